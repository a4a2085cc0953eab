// Rotary append: rotates the step's queries and keys by their positions and writes keys and values
// into their slots of the paged pools.
//
// (a, b) -> (a cos - b sin, b cos + a sin) over the first `rot` values of a head, in f32, rounded once;
// pairs are (i, i + rot / 2), or (2i, 2i + 1) when interleaved.  The rest of a head is copied.
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

template <typename T>
cudaError_t launch(const AppendArgs& a, cudaStream_t st) {
  const int heads = (a.q.p ? a.q_heads : 0) + 2 * a.kv_heads;
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
