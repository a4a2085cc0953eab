// Attention of many query rows (prompts, rerank batches, and all sequences' rows against a shared prefix) over
// paged keys, on the 5th-generation tensor cores.
//
// Work = (item, group of `fold` query heads): up to two 128-row tiles, rows being the `fold` heads of
// consecutive tokens, against the item's key tiles of 128 keys (prefix tiles, then the sequence's own).  The
// kernel is persistent, one CTA per SM; both row tiles share every K and V tile that a CTA loads.  Warp roles:
//   warps 0..3, 4..7  softmax of row tile 0, 1: one row per thread,
//   warp 8            TMA of Q and K, warp 9 TMA of V: page by page into rings of 128-key slots,
//   warps 10, 11      issuers of row tile 0's, 1's S; warp 10 owns TMEM,
//   warps 12, 13      issuers of row tile 0's, 1's P V.
// Work goes by half tiles of 64 keys.  Per half tile and row tile i:
//   S_i = Q_i K^T     tcgen05.mma M=128 N<=64 into one of the row tile's two score buffers in TMEM,
//   softmax           scores by tcgen05.ld, masks, P = exp2(s - m) in 16 bits over the scores (tcgen05.st),
//   O_i += P V        P from TMEM, V as an MN-major operand.
// S of a buffer is issued as soon as the P V that read the buffer's last P is done (MMAs of different shapes and
// accumulators are not ordered among themselves), so a softmax warp finds its next scores ready when it has
// written a P.  An issuing warp spends some 100 cycles on each wait and 30 on each MMA, one after the other: with
// S and P V of a row tile from one warp that was 2300 cycles a half tile, and the softmax waited for it.  The
// reference maximum m moves only when a row's maximum grows by more than 2^8; then the row's O is rescaled in
// TMEM, once the P V before is done.  An item's O is read out after the next item's first P is written, before
// that item's first P V.  A causal prompt of 8192 tokens, 32 query and 8 key/value heads of 128: 492 to 507
// us, 1085 to 1115 TFLOP/s, in a short burst.
#include <algorithm>
#include <cfloat>

#include "step_attend.cuh"

namespace rv {

namespace {

constexpr int kThreads = 512;   // four warpgroups
// Registers a thread: the softmax warpgroups hold 64 scores of a row each and take some of the others'.  The
// launch must bring what the split adds up to (checked before the first launch): 2 * 160 + 2 * 96 = 4 * 128.
constexpr int kLaunchRegs = 128, kSoftmaxRegs = 160, kOtherRegs = 96;
static_assert(2 * kSoftmaxRegs + 2 * kOtherRegs <= 4 * kLaunchRegs, "register split");
constexpr int kTmemCols = 512;  // scores of row tile i at 128 i and 128 i + 64, O at 256 + 128 i
constexpr int kHalfKeys = 64;

constexpr int kStageBytes = 4096;  // of a softmax warp's output: 128 bytes of 32 rows
template <int D>
constexpr int kStages = D == 128 ? 2 : 4;  // of K and of V
template <int D>
constexpr int kQBytes = kTileRows * D * 2;
template <int D>
constexpr int kKeyBytes = kTileKeys * D * 2;
template <int D>
constexpr int kSmemBytes = 1024 + 2 * kQBytes<D> + 2 * kStages<D> * kKeyBytes<D> + 8 * kStageBytes + 512;

// MN-major operand of 64-value blocks with 128-byte swizzling: 8-row groups of 1024 bytes along K, blocks of
// 64 values `block_bytes` apart along N.
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr, uint32_t block_bytes) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(block_bytes >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x of a pair on the FMA pipe: x = n + f with n = rint(x), read off the sum x + 1.5 * 2^23, f exact in
// [-1/2, 1/2]; 2^f by a polynomial of degree 4, this project's own minimax fit of the relative error (2.7e-6;
// mean 4e-8, which is what a row's sum sees); times 2^n built in the exponent field.  Below -126.5 the result is 0
// (a masked score's weight), NaN stays NaN.  One pair in four of a tile's exponentials is computed so, beside the
// others on the MUFU unit: 507 -> 479 us on a causal prompt of 8192 tokens, 32 heads of 128, when it was made
// (changes of the compile since, and scores of any size, took back 3 to 5 %); every third or second pair was slower.
__device__ __forceinline__ uint64_t f2_exp2(uint64_t x) {
  float a, b;
  f2_unpack(x, a, b);
  const uint64_t y = f2_pack(max_nan(a, -127.f), max_nan(b, -127.f));
  const uint64_t shift = f2_pack(12582912.f, 12582912.f), back = f2_pack(-12582912.f, -12582912.f);
  const uint64_t t = f2_add(y, shift);
  const uint64_t f = f2_fma(f2_add(t, back), f2_pack(-1.f, -1.f), y);
  uint64_t p = f2_fma(f2_pack(0.009570102f, 0.009570102f), f, f2_pack(0.05591786f, 0.05591786f));
  p = f2_fma(p, f, f2_pack(0.24024744f, 0.24024744f));
  p = f2_fma(p, f, f2_pack(0.6931218f, 0.6931218f));
  p = f2_fma(p, f, f2_pack(0.9999993f, 0.9999993f));
  f2_unpack(t, a, b);
  return f2_mul(p, f2_pack(__int_as_float((__float_as_int(a) << 23) + 0x3f800000),
                           __int_as_float((__float_as_int(b) << 23) + 0x3f800000)));
}

// Completion wait that ignores the abort flag (bounded by time): lets copies and MMAs in flight finish.
__device__ __forceinline__ bool wait_done(uint64_t* bar, uint32_t parity) {
  volatile int no_abort = 0;
  return mbar_wait(bar, parity, &no_abort);
}

// The items of one CTA: rounds over all CTAs, every other one backwards, so that items ordered by their work
// spread evenly.  The next item's record is brought into L1 ahead of its use.
struct Walk {
  int w, round;
  int hg;
  StepItem it;
  int na;        // prefix key tiles; own ones follow
  int tiles;     // key tiles
  int count[2];  // of which row tile 0, 1 takes this many (0: no tokens)
  int own[2];    // own keys from b0 on that the row tile's last token sees

  __device__ __forceinline__ static int index(int round) {
    return round * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
  }
  __device__ __forceinline__ void load(const AttendParams& p, int total) {
    if (w >= total) return;
    hg = w % p.groups;
    it = p.items[w / p.groups];
    const int nw = index(round + 1);
    if (nw < total) {
      const char* nx = reinterpret_cast<const char*>(&p.items[nw / p.groups]);
      asm volatile("prefetch.global.L1 [%0];" ::"l"(nx));
      asm volatile("prefetch.global.L1 [%0];" ::"l"(nx + 32));
    }
    na = (it.a1 - it.a0 + kTileKeys - 1) / kTileKeys;
    tiles = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      own[i] = max(0, min(it.b1, it.diag + min(it.n, (i + 1) * p.per)) - it.b0);
      // A row tile that sees no key still takes one tile, all masked, which gives its rows their empty result.
      count[i] = i * p.per < it.n ? max(1, na + (own[i] + kTileKeys - 1) / kTileKeys) : 0;
      tiles = max(tiles, count[i]);
    }
  }
  __device__ __forceinline__ void init(const AttendParams& p, int total) {
    round = 0;
    w = index(0);
    load(p, total);
  }
  __device__ __forceinline__ void next(const AttendParams& p, int total) {
    ++round;
    w = index(round);
    load(p, total);
  }
  // Keys of tile j that some row of row tile i sees, at least 1 (masked then), in whole blocks of 16.
  __device__ __forceinline__ int seen16(int j, int i) const {
    const int k = j < na ? it.a1 - it.a0 - j * kTileKeys : own[i] - (j - na) * kTileKeys;
    return (max(1, min(kTileKeys, k)) + 15) & ~15;
  }
};

// The same walk by key tiles, as far as an issuer of one row tile needs it.
struct Steps {
  int w, round, j;
  int na, prefix, own, count, tiles;

  __device__ __forceinline__ void load(const AttendParams& p, int total, int i) {
    j = 0;
    w = Walk::index(round);
    if (w >= total) return;
    Walk wk;
    wk.w = w;
    wk.round = round;
    wk.load(p, total);
    na = wk.na;
    prefix = wk.it.a1 - wk.it.a0;
    own = i ? wk.own[1] : wk.own[0];
    count = i ? wk.count[1] : wk.count[0];
    tiles = wk.tiles;
  }
  __device__ __forceinline__ void init(const AttendParams& p, int total, int i) {
    round = 0;
    load(p, total, i);
  }
  __device__ __forceinline__ void next(const AttendParams& p, int total, int i) {
    if (++j < tiles) return;
    ++round;
    load(p, total, i);
  }
  // As Walk::seen16, 0 where the row tile has no part in the key tile.
  __device__ __forceinline__ int seen16() const {
    if (j >= count) return 0;
    const int k = j < na ? prefix - j * kTileKeys : own - (j - na) * kTileKeys;
    return (max(1, min(kTileKeys, k)) + 15) & ~15;
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) attend_tiles_kernel(const __grid_constant__ CUtensorMap mq,
                                                                   const __grid_constant__ CUtensorMap mk,
                                                                   const __grid_constant__ CUtensorMap mv,
                                                                   const AttendParams p) {
  launch_next();  // attend_rows may start on the SMs that this kernel leaves free
  constexpr int kHalves = D / 64;
  constexpr int kSt = kStages<D>;
  constexpr bool kBf = Elem<T>::kBf16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                            // [2]
  uint8_t* sK = sQ + 2 * kQBytes<D>;             // [kSt]
  uint8_t* sV = sK + kSt * kKeyBytes<D>;         // [kSt]
  uint8_t* sO = sV + kSt * kKeyBytes<D>;         // [8] outputs on their way out
  uint64_t* bar = reinterpret_cast<uint64_t*>(sO + 8 * kStageBytes);
  uint64_t* q_full = bar;              // [2] Q of the row tile landed
  uint64_t* q_empty = q_full + 2;      // [2] its last S is done
  uint64_t* k_full = q_empty + 2;      // [kSt]
  uint64_t* k_empty = k_full + kSt;    // [kSt] both row tiles' S are done
  uint64_t* v_full = k_empty + kSt;    // [kSt]
  uint64_t* v_empty = v_full + kSt;    // [kSt] both row tiles' P V are done
  uint64_t* v_land = v_empty + kSt;    // [kSt] a ragged V tile landed, to be cleared past its keys
  uint64_t* s_full = v_land + kSt;     // [2][2] scores of the row tile's buffer in TMEM
  uint64_t* p_full = s_full + 4;       // [2][2] P of the buffer
  uint64_t* pv_done = p_full + 4;      // [2][2] P V of the buffer's P
  uint64_t* o_full = pv_done + 4;      // [2] the item's last P V
  uint64_t* o_empty = o_full + 2;      // [2] the item's O has been read
  uint64_t* drain = o_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((2 + 2 + 5 * kSt + 4 + 4 + 4 + 2 + 2 + 2) * 8 + 8 <= 512, "barrier area");

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int total = p.n_items * p.groups;
  const int per = p.per;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      for (int k = 0; k < 2; ++k) {
        mbar_init(&s_full[2 * i + k], 1);
        mbar_init(&p_full[2 * i + k], 4);
        mbar_init(&pv_done[2 * i + k], 1);
      }
      mbar_init(&o_full[i], 1);
      mbar_init(&o_empty[i], 4);
    }
    for (int s = 0; s < kSt; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 2);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 2);
      mbar_init(&v_land[s], 1);
    }
    mbar_init(&drain[0], 2);
    mbar_init(&drain[1], 2);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&mq);
    tma_prefetch_desc(&mk);
    tma_prefetch_desc(&mv);
  }
  if (warp == 10) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  if (warp == 8 || warp == 9) {
    // ---------------------------------------------------------------- TMA producers
    const bool keys = warp == 8;
    uint8_t* ring = keys ? sK : sV;
    uint64_t* full = keys ? k_full : v_full;
    uint64_t* empty = keys ? k_empty : v_empty;
    Walk wk;
    wk.init(p, total);
    int s = 0, loaded = 0, q_loads[2] = {0, 0};
    uint32_t ph = 0;
    uint32_t on_land = 0, land_ph = 0;  // by slot: the last copy was a ragged V tile's; parity of v_land
    int ragged = 0, ragged_slot = 0;    // keys of the ragged tile that is still to be cleared
    auto clear = [&](int slot, int valid) {
      if (!__all_sync(0xffffffffu, mbar_wait(&v_land[slot], (land_ph >> slot) & 1, abort_flag))) return false;
      land_ph ^= 1u << slot;
      const int upto = (valid + 15) & ~15;
      for (int c = lane; c < (upto - valid) * kHalves * 8; c += 32) {
        const int row = valid + c / (kHalves * 8), h = c / 8 % kHalves;
        *reinterpret_cast<uint4*>(sV + slot * kKeyBytes<D> + h * (kTileKeys * 128) + row * 128 + c % 8 * 16) =
            make_uint4(0, 0, 0, 0);
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_full[slot]);
      return true;
    };
    bool ok = true;
    int page = 0;
    KeyTile t{};
    if (wk.w < total) {
      t = key_tile<kTileKeys>(wk.it, 0);
      page = TileCopy<kTileKeys, kHalves>::page_of(p, t, lane);
    }
    while (ok && wk.w < total) {
      if (keys) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (!ok || !wk.count[i]) continue;
          ok = __all_sync(0xffffffffu, mbar_wait(&q_empty[i], (q_loads[i] & 1) ^ 1u, abort_flag));
          if (!ok) continue;
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full[i], per * p.fold * D * 2);
            for (int h = 0; h < kHalves; ++h)
              tma_load_3d(sQ + i * kQBytes<D> + h * (kTileRows * 128), &mq, &q_full[i], 64 * h, wk.hg * p.fold,
                          wk.it.tok0 + i * per);
          }
          ++q_loads[i];
        }
      }
      for (int j = 0; ok && j < wk.tiles; ++j) {
        const int hg = wk.hg;
        const bool last = j + 1 == wk.tiles;
        const int n = TileCopy<kTileKeys, kHalves>::copies(t, p.box);
        if (ragged) {
          // The tile before: its copy has had the time that this slot takes to fall free.
          ok = clear(ragged_slot, ragged);
          ragged = 0;
          if (!ok) break;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], ph ^ 1u, abort_flag));
        if (!ok) break;
        // What lies past the last key of a page may be anything, NaN included, and P V would meet it with weights
        // of 0: a V tile that ends inside a block of 16 keys lands on a barrier of its own, and this warp clears
        // the rest of the block before it is announced.
        uint64_t* land = !keys && (t.valid & 15) ? &v_land[s] : &full[s];
        if (lane == 0) mbar_arrive_expect_tx(land, n * p.box * D * 2);
        __syncwarp();
        TileCopy<kTileKeys, kHalves>::issue(p, t, page, lane, ring + s * kKeyBytes<D>, keys ? &mk : &mv, land,
                                            hg / p.per_kv);
        ++loaded;
        const uint32_t bit = 1u << s;
        on_land = land == &full[s] ? on_land & ~bit : on_land | bit;
        if (on_land & bit) {
          ragged = t.valid;
          ragged_slot = s;
        }
        if (++s == kSt) {
          s = 0;
          ph ^= 1u;
        }
        // The next tile's page numbers are on their way before the wait for its slot.
        if (last) break;
        t = key_tile<kTileKeys>(wk.it, j + 1);
        page = TileCopy<kTileKeys, kHalves>::page_of(p, t, lane);
      }
      wk.next(p, total);
      if (wk.w < total) {
        t = key_tile<kTileKeys>(wk.it, 0);
        page = TileCopy<kTileKeys, kHalves>::page_of(p, t, lane);
      }
    }
    if (ok && ragged) {
      ok = clear(ragged_slot, ragged);
      ragged = 0;
    }
    if (!ok && lane == 0) {
      *abort_flag = 1;
      atomicOr_system(p.err, kErrWaitTimeout);
    }
    // Every copy lands before the CTA leaves, also when another role gave up before using it.
    for (int q = 0; q < kSt && q < loaded; ++q) {
      if (!((on_land >> q) & 1)) wait_done(&full[q], ((loaded - 1 - q) / kSt) & 1);
      else if (ragged && ragged_slot == q) wait_done(&v_land[q], (land_ph >> q) & 1);  // not cleared: gave up
    }
    if (keys)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (q_loads[i]) wait_done(&q_full[i], (q_loads[i] - 1) & 1);
  } else if (warp < 14) {
    // ---------------------------------------------------------------- MMA issuers
    // The whole warp walks the key tiles; one elected lane issues.  Every issuer waits for every K (V), also where
    // its row tile has no part in it: a slot is released once by each row tile, in the fill that it holds.
    const int i = warp & 1;
    Steps st;
    st.init(p, total, i);
    int slot = 0;
    uint32_t ph = 0, t_ph = 0;  // parity of the ring, of this row tile's key tiles
    uint32_t q_ph = 0, oe_ph = 1;
    bool ok = true;
    const uint32_t ts = tmem + i * 128, to = tmem + 256 + i * 128;
    auto wait = [&](uint64_t* b, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, mbar_wait_spin(b, parity, abort_flag));
    };
    if (warp < 12) {
      const uint64_t dq = smem_desc_sw128(smem_u32(sQ + i * kQBytes<D>)), dk = smem_desc_sw128(smem_u32(sK));
      while (st.w < total) {
        const int seen = st.seen16();
        const bool last = st.j == st.count - 1;
        ok = wait(&k_full[slot], ph);
        if (ok && seen && st.j == 0) {
          ok = wait(&q_full[i], q_ph);
          q_ph ^= 1u;
        }
        if (seen) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // The last P of the buffer has been used.
            ok = ok && wait(&pv_done[2 * i + h], t_ph ^ 1u);
            if (!ok) break;
            tc_fence_after();
            const int n = min(kHalfKeys, seen - h * kHalfKeys);
            const uint32_t id = idesc_f16(kTileRows, n, kBf);
            const uint64_t b = dk + static_cast<uint64_t>(slot * (kKeyBytes<D> >> 4) + h * (kHalfKeys * 128 >> 4));
            if (elect_one()) {
              if (n > 0) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                  const uint64_t off = (k / 4) * (kTileRows * 128 >> 4) + 2 * (k % 4);
                  tc_mma_f16(ts + h * kHalfKeys, dq + off, b + off, id, k > 0);
                }
              }
              // (Test hook: the first scores are never announced, and the softmax's wait for them runs out.)
              if (!(p.stall && st.round == 0 && st.j == 0 && h == 0)) tc_commit(&s_full[2 * i + h]);
              if (h == 1) {
                tc_commit(&k_empty[slot]);
                if (last) tc_commit(&q_empty[i]);
              }
            }
            __syncwarp();
          }
          t_ph ^= 1u;
        } else if (ok && lane == 0) {
          mbar_arrive(&k_empty[slot]);
        }
        if (!ok) break;
        if (++slot == kSt) {
          slot = 0;
          ph ^= 1u;
        }
        st.next(p, total, i);
      }
    } else {
      const uint64_t dv = desc_mn(smem_u32(sV), kTileKeys * 128);
      while (st.w < total) {
        const int seen = st.seen16();
        const bool last = st.j == st.count - 1;
        ok = wait(&v_full[slot], ph);
        if (ok && seen && st.j == 0) {
          // The previous item's O has been read out of the accumulator.
          ok = wait(&o_empty[i], oe_ph);
          oe_ph ^= 1u;
        }
        if (seen) {
          const uint32_t acc = st.j > 0;
          constexpr uint32_t id = idesc_f16(kTileRows, D, kBf) | (1u << 16);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ok = ok && wait(&p_full[2 * i + h], t_ph);
            if (!ok) break;
            tc_fence_after();
            const int n16 = (seen - h * kHalfKeys) >> 4;
            const uint64_t b = dv + static_cast<uint64_t>(slot * (kKeyBytes<D> >> 4) + h * (kHalfKeys * 128 >> 4));
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k < n16)
                  tc_mma_f16_ts(to, ts + h * kHalfKeys + 8 * k, b + 128 * k, id, h > 0 || k > 0 ? 1u : acc);
              tc_commit(&pv_done[2 * i + h]);
              if (h == 1) {
                tc_commit(&v_empty[slot]);
                if (last) tc_commit(&o_full[i]);
              }
            }
            __syncwarp();
          }
          t_ph ^= 1u;
        } else if (ok && lane == 0) {
          mbar_arrive(&v_empty[slot]);
        }
        if (!ok) break;
        if (++slot == kSt) {
          slot = 0;
          ph ^= 1u;
        }
        st.next(p, total, i);
      }
    }
    if (elect_one()) {
      if (!ok) {
        *abort_flag = 1;
        atomicOr_system(p.err, kErrWaitTimeout);
      }
      tc_commit(&drain[i]);  // every MMA is done before TMEM is released
    }
    __syncwarp();
    if (!wait_done(&drain[i], 0) && lane == 0) atomicOr_system(p.err, kErrWaitTimeout);
  }
  } else {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int i = warp >> 2;                       // row tile
    const int r = (warp & 3) * 32 + lane;          // row = TMEM lane
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t to = tmem + lanes + 256 + i * 128;
    const int my_tok = i * per + r / p.fold, my_head = r % p.fold;
    constexpr float kRescale = 8.f;  // P stays below 2^8
    constexpr float kNone = -FLT_MAX;  // no key seen yet, or scores of -inf only
    // Beyond this m, s * scale - m is taken of the rounded product, as m is one: fused it leaves at the largest score
    // what m lost in its rounding, up to 2^-12 here but beyond the range of 2^x for scores of 2^28 and more.  (Never
    // fused: the products apart are one more instruction a pair.  Packed ones would not do: the compiler joins
    // mul.rn.f32x2 and add.rn.f32x2 to a fused one.)  Rows without a key so far count as such: a test for them took 1
    // to 3 % of a prompt's time.
    constexpr float kBig = 4096.f;
    const uint64_t sl2 = f2_pack(p.scale_log2, p.scale_log2);
    Walk wk;
    wk.init(p, total);
    uint32_t t_ph = 0;   // parity of the row tile's key tiles
    uint32_t items = 0;  // items read out
    bool fail = false, fin = false, fin_live = false;
    float fin_l = 0.f, fin_m = 0.f;
    int fin_tok = 0, fin_head = 0, fin_part = 0;
    // Writes the finished item's rows: O / l from TMEM, by way of 4 KB of shared memory a warp, so that eight lanes
    // write 128 consecutive bytes of a row.
    uint8_t* stage = sO + warp * kStageBytes;
    auto write_rows = [&](uint8_t* dst, int block) {
      // dst: this lane's row, or null; row r of the staged 128 bytes at chunk c ^ (r & 7).
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int row = 4 * k + (lane >> 3), c = lane & 7;
        uint8_t* d = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), row));
        const uint4 x = *reinterpret_cast<const uint4*>(stage + row * 128 + ((c ^ (row & 7)) << 4));
        if (d) *reinterpret_cast<uint4*>(d + block * 128 + c * 16) = x;
      }
      __syncwarp();
    };
    auto read_out = [&]() {
      const bool none = fin_l < 0.f;  // the row saw no key
      const float inv = 1.f / fin_l;
      uint8_t *dst = nullptr, *part = nullptr;
      if (fin_live) {
        const StepParts pt = p.parts ? p.parts[fin_tok] : StepParts{0, 1};
        if (pt.count == 1) {
          dst = reinterpret_cast<uint8_t*>(static_cast<T*>(p.out) + fin_tok * p.out_token + fin_head * p.out_head);
          if (p.lse)
            p.lse[int64_t(fin_tok) * p.q_heads + fin_head] = none ? -INFINITY : (fin_m + log2f(fin_l)) * 0.6931471805599453f;
        } else {
          const int64_t at = int64_t(pt.first + fin_part) * p.q_heads + fin_head;
          part = reinterpret_cast<uint8_t*>(p.part_o + at * D);
          p.part_ml[at] = make_float2(fin_m, none ? 0.f : fin_l);
        }
      }
      if (__any_sync(0xffffffffu, dst != nullptr)) {
#pragma unroll
        for (int b = 0; b < D / 64; ++b) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float t[32];
            tmem_read(to + 64 * b + 32 * c, t);
#pragma unroll
            for (int e = 0; e < 32; ++e) t[e] = none ? 0.f : t[e] * inv;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((4 * c + e) ^ (lane & 7)) << 4)) = pack8<T>(t + 8 * e);
          }
          write_rows(dst, b);
        }
      }
      if (__any_sync(0xffffffffu, part != nullptr)) {
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
          float t[32];
          tmem_read(to + 32 * b, t);
#pragma unroll
          for (int e = 0; e < 32; ++e) t[e] = none ? 0.f : t[e] * inv;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<float4*>(stage + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                make_float4(t[4 * e], t[4 * e + 1], t[4 * e + 2], t[4 * e + 3]);
          write_rows(part, b);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_empty[i]);
      fin = false;
    };
    while (!fail && wk.w < total) {
      const int n = i ? wk.count[1] : wk.count[0];
      const int own = wk.it.diag + my_tok + 1 - wk.it.b0;  // own keys from b0 on that the row sees
      // A row that sees no key keeps l = -inf.  (One whose scores are all -inf gets to 0, and NaN for its result.)
      const bool sees = wk.it.a1 > wk.it.a0 || min(wk.it.b1 - wk.it.b0, own) > 0;
      float m = kNone, l = sees ? 0.f : -INFINITY;
      for (int j = 0; !fail && j < n; ++j) {
        const int seen = wk.seen16(j, i);
        const int left = j < wk.na ? wk.it.a1 - wk.it.a0 - j * kTileKeys
                                   : min(wk.it.b1 - wk.it.b0, own) - (j - wk.na) * kTileKeys;  // the row's keys
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          const int lim = left - h * kHalfKeys;  // the row sees the half's keys below
          const uint32_t ts = tmem + lanes + i * 128 + h * kHalfKeys;
          fail = !__all_sync(0xffffffffu, mbar_wait_spin(&s_full[2 * i + h], t_ph, abort_flag, p.wait_limit));
          if (fail) break;
          if (h * kHalfKeys >= seen) {  // no keys: nothing to read, nothing to multiply
            if (lane == 0) mbar_arrive(&p_full[2 * i + h]);
            continue;
          }
          tc_fence_after();
          float s[64];
          float mt;
          tmem_read(ts, s);  // where S has fewer columns the rest is something else, and masked
          if (!__all_sync(0xffffffffu, lim >= kHalfKeys)) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int k = lim - 32 * c;
              const uint32_t vis = k <= 0 ? 0u : k >= 32 ? 0xffffffffu : (1u << k) - 1u;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((vis >> e) & 1u)) s[32 * c + e] = -INFINITY;
            }
          }
          float mx[6];
#pragma unroll
          for (int e = 0; e < 6; ++e) mx[e] = fmaxf(s[2 * e], s[2 * e + 1]);
#pragma unroll
          for (int e = 12; e < 64; e += 2) mx[e / 2 % 6] = fmax3(mx[e / 2 % 6], s[e], s[e + 1]);
          mt = fmaxf(fmax3(mx[0], mx[1], mx[2]), fmax3(mx[3], mx[4], mx[5]));
          mt = __fmul_rn(mt, p.scale_log2);  // (m - mt below is not to be fused either)
          const bool need = m != kNone && mt > m + kRescale;
          if (m == kNone) m = fmaxf(m, mt);
          uint64_t mul = sl2;
          if (__any_sync(0xffffffffu, need || fabsf(m) > kBig)) {
            if (__any_sync(0xffffffffu, need)) {
              // The P V before is done, and this half's has not been issued.
              fail = !__all_sync(0xffffffffu, mbar_wait_spin(&pv_done[2 * i + (h ^ 1)], t_ph ^ (h ^ 1), abort_flag));
              if (fail) break;
              tc_fence_after();
              const float alpha = need ? ex2_approx(m - mt) : 1.f;
#pragma unroll
              for (int c = 0; c < D / 16; ++c) {
                float o[16];
                tmem_read(to + 16 * c, o);
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(o[e] * alpha);
                tmem_st16(to + 16 * c, w);
              }
              tc_wait_st();
              if (need) {
                l *= alpha;
                m = mt;
              }
            }
            if (__any_sync(0xffffffffu, fabsf(m) > kBig)) {
#pragma unroll
              for (int e = 0; e < 64; ++e) s[e] = __fmul_rn(s[e], p.scale_log2);
              mul = f2_pack(1.f, 1.f);
            }
          }
          const uint64_t nm2 = f2_pack(-m, -m);
          uint64_t ps[2] = {0ull, 0ull};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const uint64_t x = f2_fma(f2_pack(s[32 * c + 2 * e], s[32 * c + 2 * e + 1]), mul, nm2);
              float p0, p1;
              uint64_t pair;
              if ((e & 3) == 3) {
                pair = f2_exp2(x);
                f2_unpack(pair, p0, p1);
              } else {
                f2_unpack(x, p0, p1);
                p0 = ex2_approx(p0);
                p1 = ex2_approx(p1);
                pair = f2_pack(p0, p1);
              }
              ps[e & 1] = f2_add(ps[e & 1], pair);
              auto v = Elem<T>::pack(p0, p1);
              w[e] = *reinterpret_cast<uint32_t*>(&v);
            }
            tmem_st16(ts + 16 * c, w);
          }
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * i + h]);
          float p0, p1, p2, p3;
          f2_unpack(ps[0], p0, p1);
          f2_unpack(ps[1], p2, p3);
          l += (p0 + p1) + (p2 + p3);
          if (fin) {
            fail = !__all_sync(0xffffffffu, mbar_wait_spin(&o_full[i], items & 1, abort_flag));
            if (fail) break;
            ++items;
            tc_fence_after();
            read_out();
          }
        }
        t_ph ^= 1u;
      }
      if (fail) break;
      if (n) {
        fin = true;
        fin_live = my_tok < wk.it.n && r < per * p.fold;
        fin_l = l;
        fin_m = m;
        fin_tok = wk.it.tok0 + my_tok;
        fin_head = wk.hg * p.fold + my_head;
        fin_part = wk.it.part;
      }
      wk.next(p, total);
    }
    if (!fail && fin) {
      fail = !__all_sync(0xffffffffu, mbar_wait_spin(&o_full[i], items & 1, abort_flag));
      if (!fail) {
        tc_fence_after();
        read_out();
      }
    }
    if (fail && lane == 0) {
      *abort_flag = 1;
      atomicOr_system(p.err, kErrWaitTimeout);
    }
  }
  __syncthreads();
  if (warp == 10) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <typename T, int D>
cudaError_t launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const AttendParams& p,
                   int ctas, cudaStream_t st) {
  static PerDeviceOnce once;
  const cudaError_t e = once.run([] {
    cudaFuncAttributes attr;
    const cudaError_t g = cudaFuncGetAttributes(&attr, attend_tiles_kernel<T, D>);
    if (g != cudaSuccess) return g;
    if (attr.numRegs != kLaunchRegs) return cudaErrorInvalidConfiguration;  // the split would wait forever
    return cudaFuncSetAttribute(attend_tiles_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes<D>);
  });
  if (e != cudaSuccess) return e;
  const int total = p.n_items * p.groups;
  attend_tiles_kernel<T, D><<<std::min(total, ctas), kThreads, kSmemBytes<D>, st>>>(mq, mk, mv, p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t attend_tiles(Act act, int head_dim, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                         const AttendParams& p, int ctas, cudaStream_t st) {
  if (act == Act::kBf16)
    return head_dim == 64 ? launch<__nv_bfloat16, 64>(mq, mk, mv, p, ctas, st)
                          : launch<__nv_bfloat16, 128>(mq, mk, mv, p, ctas, st);
  return head_dim == 64 ? launch<__half, 64>(mq, mk, mv, p, ctas, st) : launch<__half, 128>(mq, mk, mv, p, ctas, st);
}

}  // namespace rv
