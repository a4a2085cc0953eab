// Attention of few query rows (decoding) over paged keys.
//
// Work = (item, group of `fold` query heads): at most 16 rows, the `fold` heads of each of the item's tokens,
// against the item's keys.  Persistent CTAs take work from a counter, so that they may come and go as another
// kernel's CTAs leave the SMs.  A producer warp copies 64-key tiles of K and V by TMA, page by page, into a ring of
// shared-memory stages and runs ahead into the next piece of work; each of four warps takes 16 keys of every tile:
// S = Q K^T and O += P V by mma.sync m16n8k16 with Q in registers, its own running maximum m and sum l, so that no
// warp waits for another until the end of the piece, where the four are joined.  Every key is read once and used
// for 2 * 16 rows of products, far below what the tensor cores need to be busy: the kernel is bound by HBM, and
// mma.sync keeps S and P in registers, which a 128-row tcgen05 tile would not for 16 rows.  8 sequences of 3 to 60
// thousand keys, 32 query and 8 key/value heads of 128 (637 MB): 119 us with the join, 5.4 TB/s; 13 % less without
// the products, which a ring of two tiles for each of two CTAs an SM does not hide entirely.
#include <algorithm>

#include "step_attend.cuh"

namespace rv {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * (kWarps + 1);

template <int D>
constexpr int kStages = D == 128 ? 2 : 3;
template <int D>
constexpr int kPerSm = D == 128 ? 2 : 3;  // CTAs an SM holds
template <int D>
constexpr int kTileBytes = kRowKeys * D * 2;
template <int D>
constexpr int kJoinBytes = (kWarps * kRowTile * (D + 4) + 2 * kWarps * kRowTile) * 4;
template <int D>
constexpr int kQBytes = kRowTile * D * 2;
// What the consumers need to know of a piece of work, beside its query rows.
struct alignas(16) Piece {
  StepItem it;
  int w, pad[3];
  StepParts parts[kRowTile];  // of its tokens
};
template <int D>
constexpr int kSmemBytes = 1024 + kStages<D> * 2 * kTileBytes<D> + kJoinBytes<D> + 2 * kQBytes<D> + 2 * sizeof(Piece) + 256;

// Barrier of the four consumer warps; true for all where one of them says so.
__device__ __forceinline__ bool consumers_or(bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.red.or.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(x))
      : "memory");
  return r != 0;
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (Elem<T>::kBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Address of the 16-byte chunk `chunk` (of 8) of row `row` in a tile of 128-byte rows that TMA wrote with
// 128-byte swizzling.
__device__ __forceinline__ uint32_t swizzled(uint32_t base, int row, int chunk) {
  return base + row * 128 + ((chunk ^ (row & 7)) << 4);
}

__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// Arrives on *bar when this thread's copies so far have landed (counted among the barrier's arrivals).
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Keeps of a register that holds keys k and k + 1 (low and high half) those below `valid`.
__device__ __forceinline__ uint32_t keep(uint32_t v, int k, int valid) {
  return v & ((k < valid ? 0xffffu : 0u) | (k + 1 < valid ? 0xffff0000u : 0u));
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, kPerSm<D>) attend_rows_kernel(const __grid_constant__ CUtensorMap mk,
                                                               const __grid_constant__ CUtensorMap mv,
                                                               const Rows q, const AttendParams p) {
  launch_next();
  constexpr int kHalves = D / 64, kSteps = D / 16, kOut = D / 8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* so = reinterpret_cast<float*>(ring + kStages<D> * 2 * kTileBytes<D>);  // [kWarps][16][D + 4]
  float* sm = so + kWarps * kRowTile * (D + 4);                                 // [kWarps][16] m, then l
  uint8_t* sq = reinterpret_cast<uint8_t*>(so) + kJoinBytes<D>;  // [2] query rows, 128-byte blocks swizzled like K
  Piece* piece = reinterpret_cast<Piece*>(sq + 2 * kQBytes<D>);  // [2]
  uint64_t* full = reinterpret_cast<uint64_t*>(piece + 2);
  uint64_t* empty = full + kStages<D>;
  uint64_t* w_full = empty + kStages<D>;  // [2] a piece and its queries are there
  uint64_t* w_empty = w_full + 2;         // [2] its place may be used again
  volatile int* abort_flag = reinterpret_cast<volatile int*>(w_empty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int total = p.n_items * p.groups;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages<D>; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kWarps);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&w_full[s], 64);  // each producer lane's writes and copies
      mbar_init(&w_empty[s], kWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();

  bool failed = false;
  int s = 0;
  uint32_t ph = 0;
  if (warp == kWarps) {
    if (lane == 0) {
      tma_prefetch_desc(&mk);
      tma_prefetch_desc(&mv);
    }
    // Lanes 0..15 copy K, lanes 16..31 V (a 64-key tile is at most 4 boxes of 2 halves).
    const int side = lane >> 4, l16 = lane & 15;
    int issued = 0;
    int w = blockIdx.x;  // then what the counter gives, from gridDim.x on
    StepItem it = p.items[w / p.groups];
    for (int turn = 0;; ++turn) {
      // Hand over the piece of work (or that there is none left), and ask for the next.
      Piece& pc = piece[turn & 1];
      if (!__all_sync(0xffffffffu, mbar_wait(&w_empty[turn & 1], ((turn >> 1) & 1) ^ 1u, abort_flag))) {
        failed = true;
        break;
      }
      // (Unsigned: no value of the counter leads past the items.)
      if (static_cast<unsigned>(w) >= static_cast<unsigned>(total)) {
        if (lane == 0) pc.w = total;
        mbar_arrive(&w_full[turn & 1]);
        copies_arrive(&w_full[turn & 1]);
        break;
      }
      const int next = lane == 0 ? gridDim.x + atomicAdd(p.counter, 1) : 0;
      const int hg = w % p.groups, rows = it.n * p.fold;
      KeyTile t = key_tile<kRowKeys>(it, 0);
      int page = TileCopy<kRowKeys, kHalves>::page_of(p, t, l16);
      {
        const uint32_t dst = smem_u32(sq + (turn & 1) * kQBytes<D>);
        for (int c = lane; c < rows * (D / 8); c += 32) {
          const int r = c / (D / 8), k = c % (D / 8);
          const T* src = static_cast<const T*>(q.p) + (it.tok0 + r / p.fold) * q.token_stride +
                         (hg * p.fold + r % p.fold) * q.head_stride + 8 * k;
          copy16_async(swizzled(dst + (k >> 3) * (kRowTile * 128), r, k & 7), src);
        }
        if (lane < it.n) pc.parts[lane] = p.parts ? p.parts[it.tok0 + lane] : StepParts{0, 1};
        if (lane == 0) {
          pc.it = it;
          pc.w = w;
        }
        // (Test hook: the first piece is never announced, and the consumers' wait for it runs out.)
        if (!(p.stall && turn == 0)) mbar_arrive(&w_full[turn & 1]);
        copies_arrive(&w_full[turn & 1]);
      }
      const int tiles = key_tiles<kRowKeys>(it);
      StepItem next_it{};
      for (int j = 0; j < tiles; ++j) {
        KeyTile nt{};
        int next_page = 0;
        if (j + 1 < tiles) {
          nt = key_tile<kRowKeys>(it, j + 1);
          next_page = TileCopy<kRowKeys, kHalves>::page_of(p, nt, l16);
        }
        if (!__all_sync(0xffffffffu, mbar_wait(&empty[s], ph ^ 1u, abort_flag))) {
          failed = true;
          break;
        }
        const int n = TileCopy<kRowKeys, kHalves>::copies(t, p.box);
        if (lane == 0) mbar_arrive_expect_tx(&full[s], 2 * n * p.box * D * 2);
        __syncwarp();
        TileCopy<kRowKeys, kHalves>::issue(p, t, page, l16, ring + (2 * s + side) * kTileBytes<D>, side ? &mv : &mk,
                                           &full[s], hg / p.per_kv);
        ++issued;
        if (++s == kStages<D>) {
          s = 0;
          ph ^= 1u;
        }
        if (j == 0) {
          // The next piece's record is on its way while this one's keys are.
          w = __shfl_sync(0xffffffffu, next, 0);
          if (static_cast<unsigned>(w) < static_cast<unsigned>(total)) next_it = p.items[w / p.groups];
        }
        t = nt;
        page = next_page;
      }
      if (failed) break;
      it = next_it;
    }
    if (failed && lane == 0) {
      *abort_flag = 1;
      atomicOr_system(p.err, kErrWaitTimeout);
    }
    // Copies in flight land before the CTA may leave, also when it gave up.
    volatile int no_abort = 0;
    for (int j = max(0, issued - kStages<D>); j < issued; ++j)
      mbar_wait(&full[j % kStages<D>], (j / kStages<D>) & 1, &no_abort);
    // The last CTA sets the counters back for the next launch.
    if (lane == 0) {
      __threadfence();
      if (atomicAdd(p.counter + 1, 1) == static_cast<int>(gridDim.x) - 1) {
        p.counter[0] = 0;
        p.counter[1] = 0;
      }
    }
    // This kernel may have started beside attend_tiles, of which it needs nothing; but what comes after it needs
    // both, and waits for this one only: it does not end before the other has.
    if (blockIdx.x == 0) wait_before();
    return;
  }
  auto give_up = [&]() {  // a wait of this warp ran out: ends the others'
    if (failed && lane == 0) {
      *abort_flag = 1;
      atomicOr_system(p.err, kErrWaitTimeout);
    }
  };
  for (int turn = 0;; ++turn) {
    failed = !__all_sync(0xffffffffu, mbar_wait_spin(&w_full[turn & 1], (turn >> 1) & 1, abort_flag, p.wait_limit));
    give_up();
    const Piece& pc = piece[turn & 1];
    const int w = failed ? total : pc.w;
    if (consumers_or(failed) || w >= total) break;
    const StepItem it = pc.it;
    const int hg = w % p.groups, rows = it.n * p.fold;
    const int tiles = key_tiles<kRowKeys>(it);
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float o[kOut][4];
    // Rows lane / 4 and lane / 4 + 8 of the 16: head row % fold of token row / fold.  (Rows past the last are what
    // an earlier piece left; nothing of theirs is written.)
    uint32_t a[kSteps][4];
    int lim[2];  // own keys that the row sees
#pragma unroll
    for (int i = 0; i < 2; ++i) lim[i] = it.diag + ((lane >> 2) + 8 * i) / p.fold + 1;
    {
      const uint32_t base = smem_u32(sq + (turn & 1) * kQBytes<D>);
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const int chunk = 2 * k + (lane >> 4);
        ldmatrix4(swizzled(base + (chunk >> 3) * (kRowTile * 128), lane & 15, chunk & 7), a[k]);
      }
    }
#pragma unroll
    for (int n = 0; n < kOut; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
    for (int j = 0; j < tiles; ++j) {
      const KeyTile t = key_tile<kRowKeys>(it, j);
      if (!__all_sync(0xffffffffu, mbar_wait_spin(&full[s], ph, abort_flag))) {
        failed = true;
        break;
      }
      const int k0 = 16 * warp;
      if (k0 < t.valid) {
        const uint32_t kb = smem_u32(ring + 2 * s * kTileBytes<D>), vb = kb + kTileBytes<D>;
        // Two chains of sums a block, over every other step of 16 values: the products of one chain wait for one
        // another.
        float x[2][4] = {}, y[2][4] = {};
#pragma unroll
        for (int k = 0; k < kSteps; k += 2) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            // Four 8 x 8 blocks of 8 keys and 32 values: the B operands of two K = 16 steps.
            uint32_t b[4];
            const int row = k0 + 8 * n + (lane & 7), chunk = 2 * k + (lane >> 3);
            ldmatrix4(swizzled(kb + (chunk >> 3) * (kRowKeys * 128), row, chunk & 7), b);
            mma16816<T>(x[n], a[k], b[0], b[1]);
            mma16816<T>(y[n], a[k + 1], b[2], b[3]);
          }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[n][e] += y[n][e];
        // Score e of block n: row lane / 4 (+ 8 for e >= 2), key k0 + 8 n + 2 (lane % 4) + (e & 1).
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int top = (t.own ? min(t.valid, lim[i] - t.base) : t.valid) - k0 - 2 * (lane & 3);
          float mx = -INFINITY;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float& v = x[n][2 * i + e];
              v = 8 * n + e < top ? __fmul_rn(v, p.scale_log2) : -INFINITY;  // (rounded, as m is)
              mx = fmaxf(mx, v);
            }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float mn = fmaxf(m[i], mx);
          const float ref = mn == -INFINITY ? 0.f : mn;  // a row without a key so far keeps weight 0
          const float f = ex2_approx(m[i] - ref);
          m[i] = mn;
          float sum = 0.f;
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float p0 = ex2_approx(x[n][2 * i] - ref), p1 = ex2_approx(x[n][2 * i + 1] - ref);
            sum += p0 + p1;
            auto pk = Elem<T>::pack(p0, p1);
            w[2 * n + i] = *reinterpret_cast<uint32_t*>(&pk);
          }
          l[i] = l[i] * f + sum;
          if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll
            for (int n = 0; n < kOut; ++n) {
              o[n][2 * i] *= f;
              o[n][2 * i + 1] *= f;
            }
          }
        }
        // What lies past the last key in its page may be anything, NaN included: weight 0 is not enough.
        const bool ragged = t.valid < k0 + 16;
#pragma unroll
        for (int n = 0; n < kOut; n += 2) {
          // Blocks (keys 0-7, keys 8-15) of 8 values n, then of 8 values n + 1.
          uint32_t b[4];
          const int row = k0 + (lane & 15), chunk = n + (lane >> 4);
          ldmatrix4_trans(swizzled(vb + (chunk >> 3) * (kRowKeys * 128), row, chunk & 7), b);
          if (ragged) {
            const int k = k0 + 2 * (lane & 3);
            b[0] = keep(b[0], k, t.valid);
            b[1] = keep(b[1], k + 8, t.valid);
            b[2] = keep(b[2], k, t.valid);
            b[3] = keep(b[3], k + 8, t.valid);
          }
          mma16816<T>(o[n], w, b[0], b[1]);
          mma16816<T>(o[n + 1], w, b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
      if (++s == kStages<D>) {
        s = 0;
        ph ^= 1u;
      }
    }
    give_up();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      const int r = (lane >> 2) + 8 * i;
      if (r < rows) {
#pragma unroll
        for (int n = 0; n < kOut; ++n)
          *reinterpret_cast<float2*>(&so[(warp * kRowTile + r) * (D + 4) + 8 * n + 2 * (lane & 3)]) =
              make_float2(o[n][2 * i], o[n][2 * i + 1]);
        if ((lane & 3) == 0) {
          sm[warp * kRowTile + r] = m[i];
          sm[(kWarps + warp) * kRowTile + r] = l[i];
        }
      }
    }
    // Join the four warps.
    if (consumers_or(failed)) break;
    for (int c = threadIdx.x; c < rows * (D / 8); c += 32 * kWarps) {
      const int r = c / (D / 8), d = c % (D / 8) * 8;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w * kRowTile + r]);
      // A warp without a key brings m = -inf, l = 0 and zeros; one whose scores are NaN m = -inf (fmaxf passes NaN over)
      // and l = NaN, which has to reach the row.  So the keys, not the maximum, tell a row that sees none.
      const bool sees = it.a1 > it.a0 || min(it.b1, it.diag + r / p.fold + 1) > it.b0;
      const float ref = top == -INFINITY ? 0.f : top;
      float sum = 0.f, v[8] = {};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2_approx(sm[w * kRowTile + r] - ref);
        sum += f * sm[(kWarps + w) * kRowTile + r];
        const float* src = &so[(w * kRowTile + r) * (D + 4) + d];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += f * src[e];
      }
      const float inv = 1.f / sum;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = sees ? v[e] * inv : 0.f;
      const int tok = it.tok0 + r / p.fold, head = hg * p.fold + r % p.fold;
      const StepParts pt = pc.parts[r / p.fold];
      if (pt.count == 1) {
        *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + tok * p.out_token + head * p.out_head + d) = pack8<T>(v);
        if (p.lse && d == 0) p.lse[int64_t(tok) * p.q_heads + head] = (top + log2f(sum)) * 0.6931471805599453f;
      } else {
        const int64_t at = int64_t(pt.first + it.part) * p.q_heads + head;
        float4* dst = reinterpret_cast<float4*>(p.part_o + at * D + d);
        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
        if (d == 0) p.part_ml[at] = make_float2(top, sum);
      }
    }
    consumers_or(false);  // read before the next piece's results are written, and this piece's place is used again
    if (lane == 0) mbar_arrive(&w_empty[turn & 1]);
  }
}

template <typename T, int D>
cudaError_t launch(const CUtensorMap& mk, const CUtensorMap& mv, const Rows& q, const AttendParams& p, bool early,
                   cudaStream_t st) {
  static PerDeviceOnce once;
  const cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(attend_rows_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes<D>);
  });
  if (e != cudaSuccess) return e;
  const int grid = std::min(p.n_items * p.groups, kPerSm<D> * device_sm_count());
  if (early) return launch_early(attend_rows_kernel<T, D>, grid, kThreads, kSmemBytes<D>, st, mk, mv, q, p);
  attend_rows_kernel<T, D><<<grid, kThreads, kSmemBytes<D>, st>>>(mk, mv, q, p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t attend_rows(Act act, int head_dim, const CUtensorMap& mk, const CUtensorMap& mv, const Rows& q,
                        const AttendParams& p, bool early, cudaStream_t st) {
  if (act == Act::kBf16)
    return head_dim == 64 ? launch<__nv_bfloat16, 64>(mk, mv, q, p, early, st)
                          : launch<__nv_bfloat16, 128>(mk, mv, q, p, early, st);
  return head_dim == 64 ? launch<__half, 64>(mk, mv, q, p, early, st) : launch<__half, 128>(mk, mv, q, p, early, st);
}

}  // namespace rv
