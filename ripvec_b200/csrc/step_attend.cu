// Attention of a decoding step over the paged cache: every query of a sequence sees its group's shared
// prefix and, of its sequence's own keys, those up to its own place.
#include "common.cuh"
#include "decode.h"

namespace rv {

namespace {

// One warp per (token, query head), the head's values spread over the lanes; one pass over the keys
// with a running maximum m and sum l.
template <typename T, int D>
__global__ void __launch_bounds__(128) attend_rows_kernel(AttendArgs a) {
  constexpr int kPer = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t w = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (w >= int64_t(a.n_tokens) * a.q_heads) return;
  const int t = static_cast<int>(w / a.q_heads), h = static_cast<int>(w % a.q_heads);
  const int kvh = h / (a.q_heads / a.kv_heads);
  const StepSeq s = a.seqs[a.tokens[t].seq];
  const int own = min(s.len_b, s.diag + (t - s.tok0) + 1);
  const T* q = static_cast<const T*>(a.q.p) + t * a.q.token_stride + h * a.q.head_stride;
  const float sl = a.scale * 1.4426950408889634f;
  float qr[kPer], o[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    qr[i] = Elem<T>::to_f(q[lane * kPer + i]) * sl;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int part = 0; part < 2; ++part) {
    const int n = part ? own : s.len_a;
    const int* pg = a.pages + (part ? s.pg_b : s.pg_a);
    for (int j = 0; j < n; ++j) {
      const int64_t off = pg[j / a.pool.page_size] * a.pool.page_stride + kvh * a.pool.head_stride +
                          (j % a.pool.page_size) * a.pool.slot_stride + lane * kPer;
      const T* kp = static_cast<const T*>(a.pool.k) + off;
      const T* vp = static_cast<const T*>(a.pool.v) + off;
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) x += qr[i] * Elem<T>::to_f(kp[i]);
#pragma unroll
      for (int e = 16; e > 0; e >>= 1) x += __shfl_xor_sync(0xffffffffu, x, e);
      const float mn = fmaxf(m, x);
      const float f = m == mn ? 1.f : exp2f(m - mn);
      const float p = exp2f(x - mn);
      l = l * f + p;
#pragma unroll
      for (int i = 0; i < kPer; ++i) o[i] = o[i] * f + p * Elem<T>::to_f(vp[i]);
      m = mn;
    }
  }
  T* out = static_cast<T*>(a.out) + t * a.out_token + h * a.out_head;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < kPer; ++i) out[lane * kPer + i] = Elem<T>::from_f(o[i] * inv);
  if (a.lse && lane == 0)
    a.lse[int64_t(t) * a.q_heads + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

template <typename T>
cudaError_t launch(const AttendArgs& a, cudaStream_t st) {
  const int64_t warps = int64_t(a.n_tokens) * a.q_heads;
  const int blocks = static_cast<int>((warps + 3) / 4);
  if (a.head_dim == 64) attend_rows_kernel<T, 64><<<blocks, 128, 0, st>>>(a);
  else attend_rows_kernel<T, 128><<<blocks, 128, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t step_attend(Act act, const AttendArgs& a, cudaStream_t st) {
  if (a.n_tokens <= 0) return cudaSuccess;
  return act == Act::kBf16 ? launch<__nv_bfloat16>(a, st) : launch<__half>(a, st);
}

}  // namespace rv
