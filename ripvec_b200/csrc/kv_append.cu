// Rotary append: rotates the step's queries and keys by their positions and writes keys and values
// into their slots of the paged pools.
//
// (a, b) -> (a cos - b sin, b cos + a sin) over the first `rot` values of a head, in f32, rounded once;
// pairs are (i, i + rot / 2), or (2i, 2i + 1) when interleaved.  The rest of a head is copied.  Bound by HBM: 28.8
// thousand tokens of 32 + 8 + 8 heads of 128 (757 MB) take 125 us, 6.05 TB/s; by its launch for a few tokens (2 us).
#include "common.cuh"
#include "decode.h"

namespace rv {

namespace {

// One thread per (token, head, value pair): any alignment and any even rot.
template <typename T>
__global__ void __launch_bounds__(256) append_any_kernel(AppendArgs a) {
  const int heads = (a.q.p ? a.q_heads : 0) + 2 * a.kv_heads;
  const int half = a.head_dim / 2;
  const int64_t total = int64_t(a.n_tokens) * heads * half;
  for (int64_t w = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; w < total; w += int64_t(gridDim.x) * blockDim.x) {
    const int i = static_cast<int>(w % half);
    const int64_t th = w / half;
    int h = static_cast<int>(th % heads);
    const int t = static_cast<int>(th / heads);
    const StepToken tk = a.tokens[t];
    const T* src;
    T* dst;
    bool turn = true;
    const int nq = a.q.p ? a.q_heads : 0;
    if (h < nq) {
      src = static_cast<const T*>(a.q.p) + t * a.q.token_stride + h * a.q.head_stride;
      dst = static_cast<T*>(a.q_out) + t * a.q_out_token + h * a.q_out_head;
    } else {
      h -= nq;
      turn = h < a.kv_heads;
      if (!turn) h -= a.kv_heads;
      const Rows& r = turn ? a.k : a.v;
      src = static_cast<const T*>(r.p) + t * r.token_stride + h * r.head_stride;
      dst = static_cast<T*>(turn ? a.pool.k : a.pool.v) + tk.page * a.pool.page_stride + h * a.pool.head_stride +
            tk.slot * a.pool.slot_stride;
    }
    if (turn && 2 * i < a.rot) {
      const int i0 = a.interleaved ? 2 * i : i, i1 = a.interleaved ? 2 * i + 1 : i + a.rot / 2;
      const float c = a.cos[int64_t(tk.pos) * (a.rot / 2) + i], s = a.sin[int64_t(tk.pos) * (a.rot / 2) + i];
      const float x = Elem<T>::to_f(src[i0]), y = Elem<T>::to_f(src[i1]);
      dst[i0] = Elem<T>::from_f(x * c - y * s);
      dst[i1] = Elem<T>::from_f(y * c + x * s);
    } else {
      dst[2 * i] = src[2 * i];
      dst[2 * i + 1] = src[2 * i + 1];
    }
  }
}

// 16 values of one head: two 16-byte vectors that hold the two halves of 8 half-split pairs, 8
// neighbouring pairs, or values to copy.
struct Unit {
  uint4 a, b;
};

// One CTA per token.  Thread (slot, u) handles unit u of heads slot, slot + slots, ...: all of them turn by
// the same 8 angles, which the thread reads once, and two heads' loads are in flight before the first store.
template <typename T>
__global__ void __launch_bounds__(256) append_vec_kernel(const AppendArgs a, const int units, const int slots) {
  const int u = threadIdx.x % units, slot = threadIdx.x / units;
  const int t = blockIdx.x;
  const StepToken tk = a.tokens[t];
  const int nq = a.q.p ? a.q_heads : 0, heads = nq + 2 * a.kv_heads;
  const int ru = a.rot / 16;  // units that turn
  const bool turn = u < ru;
  // Offsets of the unit's two vectors in its head.
  const int o0 = !turn || a.interleaved ? 16 * u : 8 * u;
  const int o1 = !turn || a.interleaved ? o0 + 8 : o0 + a.rot / 2;
  float c[8], s[8];
  if (turn) {
    const float4* cp = reinterpret_cast<const float4*>(a.cos + int64_t(tk.pos) * (a.rot / 2) + 8 * u);
    const float4* sp = reinterpret_cast<const float4*>(a.sin + int64_t(tk.pos) * (a.rot / 2) + 8 * u);
    *reinterpret_cast<float4*>(c) = cp[0];
    *reinterpret_cast<float4*>(c + 4) = cp[1];
    *reinterpret_cast<float4*>(s) = sp[0];
    *reinterpret_cast<float4*>(s + 4) = sp[1];
  }
  const int64_t at = tk.page * a.pool.page_stride + tk.slot * a.pool.slot_stride;
  auto source = [&](int h) -> const T* {
    if (h < nq) return static_cast<const T*>(a.q.p) + t * a.q.token_stride + h * a.q.head_stride;
    h -= nq;
    const bool key = h < a.kv_heads;
    const Rows& r = key ? a.k : a.v;
    return static_cast<const T*>(r.p) + t * r.token_stride + (key ? h : h - a.kv_heads) * r.head_stride;
  };
  auto load = [&](int h) {
    const T* p = source(h);
    return Unit{*reinterpret_cast<const uint4*>(p + o0), *reinterpret_cast<const uint4*>(p + o1)};
  };
  auto store = [&](int h, const Unit& in) {
    Unit r = in;
    if (turn && h < nq + a.kv_heads) {
      float x[8], y[8], p[8], q[8];
      unpack8<T>(in.a, x);
      unpack8<T>(in.b, y);
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[2 * i] = x[2 * i] * c[i] - x[2 * i + 1] * s[i];
          p[2 * i + 1] = x[2 * i + 1] * c[i] + x[2 * i] * s[i];
          q[2 * i] = y[2 * i] * c[4 + i] - y[2 * i + 1] * s[4 + i];
          q[2 * i + 1] = y[2 * i + 1] * c[4 + i] + y[2 * i] * s[4 + i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = x[i] * c[i] - y[i] * s[i];
          q[i] = y[i] * c[i] + x[i] * s[i];
        }
      }
      r.a = pack8<T>(p);
      r.b = pack8<T>(q);
    }
    T* d;
    if (h < nq) {
      d = static_cast<T*>(a.q_out) + t * a.q_out_token + h * a.q_out_head;
    } else {
      h -= nq;
      const bool key = h < a.kv_heads;
      d = static_cast<T*>(key ? a.pool.k : a.pool.v) + at + (key ? h : h - a.kv_heads) * a.pool.head_stride;
    }
    *reinterpret_cast<uint4*>(d + o0) = r.a;
    *reinterpret_cast<uint4*>(d + o1) = r.b;
  };
  int h = slot;
  for (; h + slots < heads; h += 2 * slots) {
    const Unit x = load(h), y = load(h + slots);
    store(h, x);
    store(h + slots, y);
  }
  if (h < heads) store(h, load(h));
}

template <typename T>
cudaError_t launch(const AppendArgs& a, cudaStream_t st) {
  const int heads = (a.q.p ? a.q_heads : 0) + 2 * a.kv_heads;
  if (a.vec) {
    // As many threads as spread the heads evenly over the fewest passes of 256 threads.
    const int units = a.head_dim / 16, most = 256 / units;
    const int passes = (heads + most - 1) / most, slots = (heads + passes - 1) / passes;
    append_vec_kernel<T><<<a.n_tokens, units * slots, 0, st>>>(a, units, slots);
    return cudaGetLastError();
  }
  const int64_t total = int64_t(a.n_tokens) * heads * (a.head_dim / 2);
  const int64_t blocks = (total + 255) / 256;
  append_any_kernel<T><<<static_cast<int>(blocks < 65536 ? blocks : 65536), 256, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t kv_append(Act act, const AppendArgs& a, cudaStream_t st) {
  if (a.n_tokens <= 0) return cudaSuccess;
  return act == Act::kBf16 ? launch<__nv_bfloat16>(a, st) : launch<__half>(a, st);
}

}  // namespace rv
