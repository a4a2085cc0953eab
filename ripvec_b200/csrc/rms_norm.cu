// Residual RMS norm: h = x + residual (f32), y = h / sqrt(mean(h^2) + eps) * weight, written in 16 bits or
// as e4m3 codes with one f32 scale per group of values (scale = max|y| of the group / 448).  Bound by HBM: 28800
// rows of 4096 to codes in groups of 128 (829 MB) take 126 us, 6.58 TB/s, the rate of a copy.  It takes some 20
// instructions a value to stay there: with divisions in the row loop and unpaired arithmetic (38) it was 182 us.
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"
#include "decode.h"
#include "tmap.h"

namespace rv {

namespace {

constexpr float kE4m3Max = 448.f;
constexpr float kScaleFloor = 1e-12f;  // of a group whose values are all zero: codes 0, scale 1e-12 / 448

// Sum and maximum over the block's up to 16 warps.  The caller alternates between two `sh` arrays, so that one
// barrier a call is enough.
template <class F>
__device__ __forceinline__ float block_reduce(float v, float* sh, float none, F&& f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  const int lane = threadIdx.x & 31;
  if (lane == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < (blockDim.x >> 5) ? sh[lane] : none;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return __shfl_sync(0xffffffffu, v, 0);
}
__device__ __forceinline__ float block_sum(float v, float* sh) {
  return block_reduce(v, sh, 0.f, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float block_max(float v, float* sh) {
  return block_reduce(v, sh, 0.f, [](float a, float b) { return fmaxf(a, b); });
}

// kVec consecutive 16-bit values, as loaded and as f32.
template <typename T, int kVec>
using Raw = std::conditional_t<kVec == 8, uint4, T>;
template <typename T, int kVec>
__device__ __forceinline__ void widen(const Raw<T, kVec>& r, float* v) {
  if constexpr (kVec == 8) unpack8<T>(r, v);
  else v[0] = Elem<T>::to_f(r);
}
// kWide: vectors on 16 bytes (codes on 8), moved whole; else value by value.
template <typename T, int kVec, bool kWide>
__device__ __forceinline__ Raw<T, kVec> load_vec(const T* p) {
  if constexpr (kWide || kVec == 1) {
    return *reinterpret_cast<const Raw<T, kVec>*>(p);
  } else {
    union {
      uint4 v;
      uint16_t e[8];
    } r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r.e[e] = reinterpret_cast<const uint16_t*>(p)[e];
    return r.v;
  }
}
template <typename T, int kVec, bool kWide, int kPairs>
__device__ __forceinline__ void store_vec(T* p, const uint64_t (&v)[kPairs]) {
  float f[2 * kPairs];
#pragma unroll
  for (int e = 0; e < kPairs; ++e) f2_unpack(v[e], f[2 * e], f[2 * e + 1]);
  if constexpr (kWide && kVec == 8) {
    *reinterpret_cast<uint4*>(p) = pack8<T>(f);
  } else {
#pragma unroll
    for (int e = 0; e < kVec; ++e) p[e] = Elem<T>::from_f(f[e]);
  }
}
template <int kVec, bool kWide, int kPairs>
__device__ __forceinline__ void store_codes(uint8_t* p, const uint64_t (&v)[kPairs], float mul) {
  const uint64_t mul2 = f2_pack(mul, mul);
  float f[2 * kPairs];
#pragma unroll
  for (int e = 0; e < kPairs; ++e) f2_unpack(f2_mul(v[e], mul2), f[2 * e], f[2 * e + 1]);
  if constexpr (kVec == 8) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i], f[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i + 2], f[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
      w[i] = lo | (hi << 16);
    }
    if constexpr (kWide) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = static_cast<uint8_t>(w[e / 4] >> (8 * (e % 4)));
    }
  } else {
    *p = __nv_cvt_float_to_fp8(f[0], __NV_SATFINITE, __NV_E4M3);
  }
}

// One pass over the data: a CTA holds its row in registers (kN vectors of kVec values a thread, vector n of
// thread i at (n * threads + i) * kVec) from the load to the store, walks rows blockIdx.x, + gridDim.x, ...
// and holds the weights for all of them.  kVec 8 takes rows of whole vectors, wherever they start: the order of a row's
// sum, and so every bit of its result, does not depend on the rows' alignment (28800 rows of 4096 with the residual in and
// out: 155 us to 16 bits, 126 to codes in groups of 128; off 16 bytes, moved value by value, 632 and 448).
// Threads of a CTA at most, and threads that an SM holds, by the registers that the row, its weights and the
// next row take.
template <int kVec, int kN>
constexpr int kMaxThreads = kVec == 1 || kN == 4 ? 512 : kN == 2 ? 384 : 256;
template <int kVec, int kN>
constexpr int kResident = kVec == 1 ? (kN == 16 ? 512 : 1024) : kN == 4 ? 512 : kN == 2 ? 768 : 1024;

template <typename T, int kVec, int kN, bool kCodes, bool kWide>
__global__ void __launch_bounds__(kMaxThreads<kVec, kN>, kResident<kVec, kN> / kMaxThreads<kVec, kN>)
    rms_norm_kernel(const NormArgs a) {
  __shared__ float sh[4][16];
  // Values in pairs (a lone value has a zero beside it): one instruction works on both.
  constexpr int kPairs = (kVec + 1) / 2;
  using R = Raw<T, kVec>;
  uint64_t w[kN][kPairs];
  bool in[kN];
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    const int i = (n * blockDim.x + threadIdx.x) * kVec;
    in[n] = i < a.hidden;
#pragma unroll
    for (int e = 0; e < kPairs; ++e)
      w[n][e] = f2_pack(in[n] ? a.weight[i + 2 * e] : 0.f, in[n] && kVec > 1 ? a.weight[i + 2 * e + 1] : 0.f);
  }
  const float inv_hidden = 1.f / a.hidden;
  const int64_t at = int64_t(threadIdx.x) * kVec;
  const int step = blockDim.x * kVec;  // between a thread's vectors
  const T* x = static_cast<const T*>(a.x) + blockIdx.x * a.x_stride + at;
  const T* r = static_cast<const T*>(a.residual) + blockIdx.x * a.residual_stride + at;
  T* ro = static_cast<T*>(a.residual_out) + blockIdx.x * a.residual_out_stride + at;
  R rx[kN], rr[kN];  // the next row, loaded while the present one is worked on
  auto load = [&]() {
#pragma unroll
    for (int n = 0; n < kN; ++n)
      if (in[n]) rx[n] = load_vec<T, kVec, kWide>(x + n * step);
    if (a.residual) {
#pragma unroll
      for (int n = 0; n < kN; ++n)
        if (in[n]) rr[n] = load_vec<T, kVec, kWide>(r + n * step);
    }
    x += gridDim.x * a.x_stride;
    r += gridDim.x * a.residual_stride;
  };
  int turn = 0;
  if (blockIdx.x < a.rows) load();
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    uint64_t h[kN][kPairs];
    uint64_t ss = 0;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      float v[2 * kPairs] = {};
      if (in[n]) widen<T, kVec>(rx[n], v);
#pragma unroll
      for (int e = 0; e < kPairs; ++e) h[n][e] = f2_pack(v[2 * e], v[2 * e + 1]);
      if (a.residual) {
        if (in[n]) widen<T, kVec>(rr[n], v);
#pragma unroll
        for (int e = 0; e < kPairs; ++e) h[n][e] = f2_add(h[n][e], f2_pack(v[2 * e], v[2 * e + 1]));
      }
    }
    if (row + gridDim.x < a.rows) load();
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      if (a.residual_out && in[n]) store_vec<T, kVec, kWide>(ro + n * step, h[n]);
#pragma unroll
      for (int e = 0; e < kPairs; ++e) ss = f2_fma(h[n][e], h[n][e], ss);
    }
    ro += gridDim.x * a.residual_out_stride;
    float s0, s1;
    f2_unpack(ss, s0, s1);
    const float inv = rsqrtf(block_sum(s0 + s1, sh[turn]) * inv_hidden + a.eps);
    const uint64_t inv2 = f2_pack(inv, inv);
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int e = 0; e < kPairs; ++e) h[n][e] = f2_mul(f2_mul(h[n][e], inv2), w[n][e]);
    if constexpr (!kCodes) {
      T* o = static_cast<T*>(a.out) + row * a.out_stride + at;
#pragma unroll
      for (int n = 0; n < kN; ++n)
        if (in[n]) store_vec<T, kVec, kWide>(o + n * step, h[n]);
    } else {
      uint8_t* o = static_cast<uint8_t*>(a.out) + row * a.out_stride + at;
      float mx[kN], all = 0.f;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        mx[n] = 0.f;
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
          f2_unpack(h[n][e], s0, s1);
          mx[n] = fmax3(mx[n], fabsf(s0), fabsf(s1));
        }
        all = fmaxf(all, mx[n]);
      }
      if (a.group == a.hidden) {
        const float top = fmaxf(block_max(all, sh[2 + turn]), kScaleFloor);
        if (threadIdx.x == 0) a.scales[row] = top * (1.f / kE4m3Max);
#pragma unroll
        for (int n = 0; n < kN; ++n) mx[n] = top;
      } else {
        // A group of 32, 64, 128 or 256 values is 4 to 32 neighbouring lanes of one vector step (kVec 8).
        const int lanes = a.group / kVec, shift = 31 - __clz(a.group);
        float* sc = a.scales + row * (a.hidden >> shift) + (at >> shift);
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          mx[n] = fmaxf(mx[n], __shfl_xor_sync(0xffffffffu, mx[n], 1));
          mx[n] = fmaxf(mx[n], __shfl_xor_sync(0xffffffffu, mx[n], 2));
          if (lanes > 4) mx[n] = fmaxf(mx[n], __shfl_xor_sync(0xffffffffu, mx[n], 4));
          if (lanes > 8) mx[n] = fmaxf(mx[n], __shfl_xor_sync(0xffffffffu, mx[n], 8));
          if (lanes > 16) mx[n] = fmaxf(mx[n], __shfl_xor_sync(0xffffffffu, mx[n], 16));
          mx[n] = fmaxf(mx[n], kScaleFloor);
          if (in[n] && (threadIdx.x & (lanes - 1)) == 0) sc[n * step >> shift] = mx[n] * (1.f / kE4m3Max);
        }
      }
#pragma unroll
      for (int n = 0; n < kN; ++n)
        // One approximate division a group and products, not a division by the scale a value: a code that lies within
        // some 2^-22 of a tie may fall to the other side.
        if (in[n]) store_codes<kVec, kWide>(o + n * step, h[n], __fdividef(kE4m3Max, mx[n]));
    }
  }
}

// The rest: wider rows.  One CTA per row; x and residual are read again for
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
      const float top = fmaxf(block_max(mx, sh), kScaleFloor), mul = __fdividef(kE4m3Max, top);
      if (threadIdx.x == 0) a.scales[row * groups + g] = top * (1.f / kE4m3Max);
      for (int i = g * a.group + threadIdx.x; i < (g + 1) * a.group; i += blockDim.x) {
        const float h = at(i);
        o[i] = __nv_cvt_float_to_fp8(h * inv * a.weight[i] * mul, __NV_SATFINITE, __NV_E4M3);
        if (ro) ro[i] = Elem<T>::from_f(h);
      }
    }
  }
}

template <typename T, int kVec, int kN, bool kWide>
cudaError_t run(const NormArgs& a, int threads, cudaStream_t st) {
  // As many CTAs as are resident at once; each then walks its share of the rows.
  const int64_t most = int64_t(device_sm_count()) * (kResident<kVec, kN> / threads);
  const int grid = static_cast<int>(a.rows < most ? a.rows : most);
  if (a.scales) rms_norm_kernel<T, kVec, kN, true, kWide><<<grid, threads, 0, st>>>(a);
  else rms_norm_kernel<T, kVec, kN, false, kWide><<<grid, threads, 0, st>>>(a);
  return cudaGetLastError();
}

template <typename T, bool kWide>
cudaError_t run8(const NormArgs& a, cudaStream_t st) {
  const int vecs = a.hidden / 8;
  if (vecs <= 256) return run<T, 8, 1, kWide>(a, (vecs + 31) / 32 * 32, st);
  if (vecs <= 768) return run<T, 8, 2, kWide>(a, (vecs + 63) / 64 * 32, st);
  return run<T, 8, 4, kWide>(a, (vecs + 127) / 128 * 32, st);
}

template <typename T>
cudaError_t launch(const NormArgs& a, cudaStream_t st) {
  if (a.hidden % 8 == 0) {
    if (a.hidden <= 16384) return a.vec ? run8<T, true>(a, st) : run8<T, false>(a, st);
  } else if (a.hidden <= 8192) {  // (no groups: they are multiples of 8)
    if (a.hidden <= 1024) return run<T, 1, 4, false>(a, (a.hidden + 127) / 128 * 32, st);
    if (a.hidden <= 4096) return run<T, 1, 8, false>(a, (a.hidden + 255) / 256 * 32, st);
    return run<T, 1, 16, false>(a, (a.hidden + 511) / 512 * 32, st);
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
