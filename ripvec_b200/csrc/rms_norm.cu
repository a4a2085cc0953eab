// Residual RMS norm: h = x + residual (f32), y = h / sqrt(mean(h^2) + eps) * weight, written in 16 bits or
// as e4m3 codes with one f32 scale per group of values (scale = max|y| of the group / 448).
#include <cuda_fp8.h>

#include "common.cuh"
#include "decode.h"

namespace rv {

namespace {

constexpr float kE4m3Max = 448.f;
constexpr float kScaleFloor = 1e-12f;  // of a group whose values are all zero: codes 0, scale 1e-12 / 448

__device__ __forceinline__ float block_sum(float v, float* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < (blockDim.x >> 5); ++w) s += sh[w];
  return s;
}
__device__ __forceinline__ float block_max(float v, float* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < (blockDim.x >> 5); ++w) s = fmaxf(s, sh[w]);
  return s;
}

// One CTA per row, any width, stride and alignment; x and residual are read again for the second pass.
template <typename T>
__global__ void __launch_bounds__(256) rms_norm_any_kernel(NormArgs a) {
  __shared__ float sh[8];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* r = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    T* ro = a.residual_out ? static_cast<T*>(a.residual_out) + row * a.residual_out_stride : nullptr;
    auto at = [&](int i) { return Elem<T>::to_f(x[i]) + (r ? Elem<T>::to_f(r[i]) : 0.f); };
    float ss = 0.f;
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x) {
      const float h = at(i);
      ss += h * h;
    }
    const float inv = rsqrtf(block_sum(ss, sh) / a.hidden + a.eps);
    if (!a.scales) {
      T* o = static_cast<T*>(a.out) + row * a.out_stride;
      for (int i = threadIdx.x; i < a.hidden; i += blockDim.x) {
        const float h = at(i);
        o[i] = Elem<T>::from_f(h * inv * a.weight[i]);
        if (ro) ro[i] = Elem<T>::from_f(h);
      }
      continue;
    }
    uint8_t* o = static_cast<uint8_t*>(a.out) + row * a.out_stride;
    const int groups = a.hidden / a.group;
    for (int g = 0; g < groups; ++g) {
      float mx = 0.f;
      for (int i = g * a.group + threadIdx.x; i < (g + 1) * a.group; i += blockDim.x)
        mx = fmaxf(mx, fabsf(at(i) * inv * a.weight[i]));
      const float scale = fmaxf(block_max(mx, sh), kScaleFloor) / kE4m3Max;
      if (threadIdx.x == 0) a.scales[row * groups + g] = scale;
      for (int i = g * a.group + threadIdx.x; i < (g + 1) * a.group; i += blockDim.x) {
        const float h = at(i);
        o[i] = __nv_cvt_float_to_fp8(h * inv * a.weight[i] / scale, __NV_SATFINITE, __NV_E4M3);
        if (ro) ro[i] = Elem<T>::from_f(h);
      }
    }
  }
}

template <typename T>
cudaError_t launch(const NormArgs& a, cudaStream_t st) {
  const int64_t blocks = a.rows < 65536 ? a.rows : 65536;
  rms_norm_any_kernel<T><<<static_cast<int>(blocks), 256, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t rms_norm(Act act, const NormArgs& a, cudaStream_t st) {
  if (a.rows <= 0) return cudaSuccess;
  return act == Act::kBf16 ? launch<__nv_bfloat16>(a, st) : launch<__half>(a, st);
}

}  // namespace rv
