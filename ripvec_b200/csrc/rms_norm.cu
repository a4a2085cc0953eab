// Residual RMS norm: h = x + residual (f32), y = h / sqrt(mean(h^2) + eps) * weight, written in 16 bits or
// as e4m3 codes with one f32 scale per group of values (scale = max|y| of the group / 448).
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"
#include "decode.h"
#include "tmap.h"

namespace rv {

namespace {

constexpr float kE4m3Max = 448.f;
constexpr float kScaleFloor = 1e-12f;  // of a group whose values are all zero: codes 0, scale 1e-12 / 448

// Sum and maximum over the block.  The caller alternates between two `sh` arrays, so that one barrier a call
// is enough.
__device__ __forceinline__ float block_sum(float v, float* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < (blockDim.x >> 5); ++w) s += sh[w];
  return s;
}
__device__ __forceinline__ float block_max(float v, float* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < (blockDim.x >> 5); ++w) s = fmaxf(s, sh[w]);
  return s;
}

// kVec consecutive 16-bit values, as loaded and as f32.
template <typename T, int kVec>
using Raw = std::conditional_t<kVec == 8, uint4, T>;
template <typename T, int kVec>
__device__ __forceinline__ void widen(const Raw<T, kVec>& r, float (&v)[kVec]) {
  if constexpr (kVec == 8) unpack8<T>(r, v);
  else v[0] = Elem<T>::to_f(r);
}
template <typename T, int kVec>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[kVec]) {
  if constexpr (kVec == 8) *reinterpret_cast<uint4*>(p) = pack8<T>(v);
  else *p = Elem<T>::from_f(v[0]);
}
template <int kVec>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&v)[kVec], float mul) {
  if constexpr (kVec == 8) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i] * mul, v[4 * i + 1] * mul), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2] * mul, v[4 * i + 3] * mul), __NV_SATFINITE, __NV_E4M3);
      w[i] = lo | (hi << 16);
    }
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
    *p = __nv_cvt_float_to_fp8(v[0] * mul, __NV_SATFINITE, __NV_E4M3);
  }
}

// One pass over the data: a CTA holds its row in registers (kN vectors of kVec values a thread, vector n of
// thread i at (n * threads + i) * kVec) from the load to the store, walks rows blockIdx.x, + gridDim.x, ...
// and holds the weights for all of them.  kVec 8 wants rows on 16 bytes; kVec 1 takes any alignment.
// Threads of a CTA at most, and threads that an SM holds, by the registers that the row, its weights and the
// next row take.
template <int kVec, int kN>
constexpr int kMaxThreads = kVec * kN >= 32 ? 512 : kVec * kN >= 16 ? 384 : 256;
template <int kVec, int kN>
constexpr int kResident = kVec * kN >= 32 ? 512 : kN >= 16 ? 384 : kVec * kN >= 16 ? 768 : 1024;

template <typename T, int kVec, int kN, bool kCodes>
__global__ void __launch_bounds__(kMaxThreads<kVec, kN>, kResident<kVec, kN> / kMaxThreads<kVec, kN>) rms_norm_kernel(const NormArgs a) {
  __shared__ float sh[4][16];
  float w[kN][kVec];
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    const int i = (n * blockDim.x + threadIdx.x) * kVec;
#pragma unroll
    for (int e = 0; e < kVec; ++e) w[n][e] = i < a.hidden ? a.weight[i + e] : 0.f;
  }
  using R = Raw<T, kVec>;
  R rx[kN], rr[kN];  // the next row, loaded while the present one is worked on
  auto load = [&](int64_t row) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* r = static_cast<const T*>(a.residual) + row * a.residual_stride;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int i = (n * blockDim.x + threadIdx.x) * kVec;
      if (i < a.hidden) rx[n] = *reinterpret_cast<const R*>(x + i);
    }
    if (a.residual) {
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const int i = (n * blockDim.x + threadIdx.x) * kVec;
        if (i < a.hidden) rr[n] = *reinterpret_cast<const R*>(r + i);
      }
    }
  };
  int turn = 0;
  if (blockIdx.x < a.rows) load(blockIdx.x);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    float h[kN][kVec];
    float ss = 0.f;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int i = (n * blockDim.x + threadIdx.x) * kVec;
      if (i < a.hidden) {
        widen<T, kVec>(rx[n], h[n]);
        if (a.residual) {
          float y[kVec];
          widen<T, kVec>(rr[n], y);
#pragma unroll
          for (int e = 0; e < kVec; ++e) h[n][e] += y[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) h[n][e] = 0.f;
      }
    }
    if (row + gridDim.x < a.rows) load(row + gridDim.x);
    T* ro = static_cast<T*>(a.residual_out) + row * a.residual_out_stride;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int i = (n * blockDim.x + threadIdx.x) * kVec;
      if (a.residual_out && i < a.hidden) store_vec<T, kVec>(ro + i, h[n]);
#pragma unroll
      for (int e = 0; e < kVec; ++e) ss += h[n][e] * h[n][e];
    }
    const float inv = rsqrtf(block_sum(ss, sh[turn]) / a.hidden + a.eps);
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int e = 0; e < kVec; ++e) h[n][e] = h[n][e] * inv * w[n][e];
    if constexpr (!kCodes) {
      T* o = static_cast<T*>(a.out) + row * a.out_stride;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const int i = (n * blockDim.x + threadIdx.x) * kVec;
        if (i < a.hidden) store_vec<T, kVec>(o + i, h[n]);
      }
    } else {
      uint8_t* o = static_cast<uint8_t*>(a.out) + row * a.out_stride;
      float mx[kN], all = 0.f;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        mx[n] = 0.f;
#pragma unroll
        for (int e = 0; e < kVec; ++e) mx[n] = fmaxf(mx[n], fabsf(h[n][e]));
        all = fmaxf(all, mx[n]);
      }
      if (a.group == a.hidden) {
        const float top = fmaxf(block_max(all, sh[2 + turn]), kScaleFloor);
        if (threadIdx.x == 0) a.scales[row] = top / kE4m3Max;
#pragma unroll
        for (int n = 0; n < kN; ++n) mx[n] = top;
      } else {
        // A group of 32 .. 256 values is 4 .. 32 neighbouring lanes of one vector step (kVec 8).
        const int lanes = a.group / kVec;
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          for (int off = 1; off < lanes; off <<= 1) mx[n] = fmaxf(mx[n], __shfl_xor_sync(0xffffffffu, mx[n], off));
          mx[n] = fmaxf(mx[n], kScaleFloor);
          const int i = (n * blockDim.x + threadIdx.x) * kVec;
          if (i < a.hidden && threadIdx.x % lanes == 0) a.scales[row * (a.hidden / a.group) + i / a.group] = mx[n] / kE4m3Max;
        }
      }
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const int i = (n * blockDim.x + threadIdx.x) * kVec;
        if (i < a.hidden) store_codes<kVec>(o + i, h[n], kE4m3Max / mx[n]);
      }
    }
  }
}

// The rest: wide rows, and groups in rows off 16 bytes.  One CTA per row; x and residual are read again for
// each further pass; an element's last read and its writes are one thread's, so outputs may be inputs.
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
    __syncthreads();
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
      __syncthreads();
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

template <typename T, int kVec, int kN>
cudaError_t run(const NormArgs& a, int threads, cudaStream_t st) {
  // As many CTAs as are resident at once; each then walks its share of the rows.
  const int64_t most = int64_t(device_sm_count()) * (kResident<kVec, kN> / threads);
  const int grid = static_cast<int>(a.rows < most ? a.rows : most);
  if (a.scales) rms_norm_kernel<T, kVec, kN, true><<<grid, threads, 0, st>>>(a);
  else rms_norm_kernel<T, kVec, kN, false><<<grid, threads, 0, st>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch(const NormArgs& a, cudaStream_t st) {
  const bool vec = a.vec;
  if (vec && a.hidden <= 16384) {
    const int vecs = a.hidden / 8;
    if (vecs <= 256) return run<T, 8, 1>(a, (vecs + 31) / 32 * 32, st);
    if (vecs <= 768) return run<T, 8, 2>(a, (vecs + 63) / 64 * 32, st);
    return run<T, 8, 4>(a, (vecs + 127) / 128 * 32, st);
  }
  if (!vec && a.hidden <= 6144 && a.group == a.hidden) {
    if (a.hidden <= 1024) return run<T, 1, 4>(a, (a.hidden + 127) / 128 * 32, st);
    return run<T, 1, 16>(a, (a.hidden + 511) / 512 * 32, st);
  }
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
