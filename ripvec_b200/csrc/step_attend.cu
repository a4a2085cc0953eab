// Attention of a decoding step: the two kernels that compute partial or final rows, and the join of tokens
// whose keys were split over several items.
#include <type_traits>

#include "step_attend.cuh"

namespace rv {

namespace {

// One warp per (token, query head): out = sum_i w_i o_i / sum_i w_i with w_i = l_i 2^(m_i - max), over the partials with
// any weight.  A partial without has l = 0, and o = 0 where it has no key for the row, NaN where it has (scores of -inf
// only); a partial with a NaN among its scores has l = NaN and so makes the row.  A row without any weight gets the sum
// of its o: zeros, or NaN as a softmax of -inf alone; and -inf.  (The logarithm of a weight, m + log2 l, would lose l
// beside a large m: of scores of 2^20 four bits of it are left.)
template <typename T, int D>
__global__ void __launch_bounds__(128) join_kernel(const int* __restrict__ tokens, int n, const AttendParams p) {
  constexpr int kPer = D / 32;  // values a lane
  using Vec = std::conditional_t<kPer == 4, float4, float2>;
  const int lane = threadIdx.x & 31;
  const int64_t w = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (w >= int64_t(n) * p.q_heads) return;
  const int tok = tokens[w / p.q_heads], head = static_cast<int>(w % p.q_heads);
  const StepParts pt = p.parts[tok];
  const int64_t at = int64_t(pt.first) * p.q_heads + head;
  wait_before();  // for the partials
  // Up to 32 partials at a time: one lane weighs each, all lanes add them, four loads in flight.
  float v[kPer] = {}, sum = 0.f, top = -INFINITY;
  for (int i0 = 0; i0 < pt.count; i0 += 32) {
    const float2 ml = i0 + lane < pt.count ? p.part_ml[at + int64_t(i0 + lane) * p.q_heads] : make_float2(-INFINITY, 0.f);
    float mx = ml.y == 0.f ? -INFINITY : ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const unsigned weighs = __ballot_sync(0xffffffffu, ml.y != 0.f);
    if (!weighs) continue;
    const float now = fmaxf(top, mx), ref = now == -INFINITY ? 0.f : now;
    const float old = ex2_approx(top - ref), f = ml.y * ex2_approx(ml.x - ref);
    top = now;
    sum *= old;
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] *= old;
    const int m = min(32, pt.count - i0);
    const Vec* src = reinterpret_cast<const Vec*>(p.part_o + (at + int64_t(i0) * p.q_heads) * D) + lane;
    const int64_t step = int64_t(p.q_heads) * 32;  // in Vec
    int i = 0;
    auto add = [&](const Vec& x, int k) {
      if (!(weighs >> k & 1)) return;
      const float g = __shfl_sync(0xffffffffu, f, k);
      sum += g;
      const float* y = reinterpret_cast<const float*>(&x);
#pragma unroll
      for (int e = 0; e < kPer; ++e) v[e] += g * y[e];
    };
    for (; i + 4 <= m; i += 4) {
      const Vec x0 = src[i * step], x1 = src[(i + 1) * step], x2 = src[(i + 2) * step], x3 = src[(i + 3) * step];
      add(x0, i);
      add(x1, i + 1);
      add(x2, i + 2);
      add(x3, i + 3);
    }
    for (; i < m; ++i) add(src[i * step], i);
  }
  float inv = 1.f / sum;
  if (sum == 0.f) {
    inv = 1.f;
    const Vec* src = reinterpret_cast<const Vec*>(p.part_o + at * D) + lane;
    for (int i = 0; i < pt.count; ++i, src += int64_t(p.q_heads) * 32) {
      const float* y = reinterpret_cast<const float*>(src);
#pragma unroll
      for (int e = 0; e < kPer; ++e) v[e] += y[e];
    }
  }
  T* dst = static_cast<T*>(p.out) + tok * p.out_token + head * p.out_head + lane * kPer;
  if constexpr (kPer == 4) {
    auto lo = Elem<T>::pack(v[0] * inv, v[1] * inv), hi = Elem<T>::pack(v[2] * inv, v[3] * inv);
    *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
  } else {
    auto x = Elem<T>::pack(v[0] * inv, v[1] * inv);
    *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<uint32_t*>(&x);
  }
  if (p.lse && lane == 0)
    p.lse[int64_t(tok) * p.q_heads + head] = (top + log2f(sum)) * 0.6931471805599453f;
}

template <typename T>
cudaError_t join(const AttendArgs& a, const AttendParams& p, cudaStream_t st) {
  const int blocks = static_cast<int>((int64_t(a.n_joined) * a.q_heads + 3) / 4);
  return launch_early(a.head_dim == 64 ? join_kernel<T, 64> : join_kernel<T, 128>, blocks, 128, 0, st, a.joined,
                      a.n_joined, p);
}

bool pool_map(CUtensorMap* m, const void* base, bool bf, const AttendArgs& a, int box) {
  const uint64_t dims[4] = {uint64_t(a.head_dim), uint64_t(a.pool.page_size), uint64_t(a.kv_heads), uint64_t(a.num_pages)};
  const uint64_t strides[3] = {uint64_t(a.pool.slot_stride) * 2, uint64_t(a.pool.head_stride) * 2,
                               uint64_t(a.pool.page_stride) * 2};
  const uint32_t b[4] = {64, uint32_t(box), 1, 1};
  return make_tmap_16bit(m, base, bf, 4, dims, strides, b);
}

}  // namespace

cudaError_t step_attend(Act act, const AttendArgs& a, cudaStream_t st) {
  if (a.n_tokens <= 0) return cudaSuccess;
  const bool bf = act == Act::kBf16;
  AttendParams p{};
  p.parts = a.parts;
  p.pages = a.pages;
  p.q_heads = a.q_heads;
  p.fold = a.fold;
  p.groups = a.q_heads / a.fold;
  p.per_kv = a.q_heads / a.kv_heads / a.fold;
  p.per = kTileRows / a.fold;
  p.page_size = a.pool.page_size;
  p.out = a.out;
  p.out_token = a.out_token;
  p.out_head = a.out_head;
  p.lse = a.lse;
  p.part_o = a.part_o;
  p.part_ml = a.part_ml;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.err = a.err;
  p.counter = a.counter;
  attention_get_stall(&p.stall, &p.wait_limit);
  CUtensorMap mk, mv, mq;
  cudaError_t e = cudaSuccess;
  if (a.n_tile_items > 0) {
    p.items = a.tile_items;
    p.n_items = a.n_tile_items;
    p.box = a.pool.page_size < kTileKeys ? a.pool.page_size : kTileKeys;
    const uint64_t dims[3] = {uint64_t(a.head_dim), uint64_t(a.q_heads), uint64_t(a.n_tokens)};
    const uint64_t strides[2] = {uint64_t(a.q.head_stride) * 2, uint64_t(a.q.token_stride) * 2};
    const uint32_t box[3] = {64, uint32_t(a.fold), uint32_t(kTileRows / a.fold)};
    if (!pool_map(&mk, a.pool.k, bf, a, p.box) || !pool_map(&mv, a.pool.v, bf, a, p.box) ||
        !make_tmap_16bit(&mq, a.q.p, bf, 3, dims, strides, box))
      return cudaErrorInvalidValue;
    e = attend_tiles(act, a.head_dim, mq, mk, mv, p, a.tile_sms, st);
    if (e != cudaSuccess) return e;
  }
  if (a.n_row_items > 0) {
    p.items = a.row_items;
    p.n_items = a.n_row_items;
    p.box = a.pool.page_size < kRowKeys ? a.pool.page_size : kRowKeys;
    if (!pool_map(&mk, a.pool.k, bf, a, p.box) || !pool_map(&mv, a.pool.v, bf, a, p.box)) return cudaErrorInvalidValue;
    e = attend_rows(act, a.head_dim, mk, mv, a.q, p, a.n_tile_items > 0, st);
    if (e != cudaSuccess) return e;
  }
  if (a.n_joined > 0) e = bf ? join<__nv_bfloat16>(a, p, st) : join<__half>(a, p, st);
  return e;
}

}  // namespace rv
