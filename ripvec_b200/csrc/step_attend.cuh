// Shared by the attention kernels of a decoding step.
#pragma once

#include <utility>

#include "common.cuh"
#include "decode.h"
#include "tmap.h"

namespace rv {

// What a launch of either kernel needs beside its tensor maps.
struct AttendParams {
  const StepItem* items;
  const StepParts* parts;  // null: one partial a token
  const int* pages;
  int n_items, q_heads, fold;
  int groups, per_kv;  // head groups of `fold` query heads: all, and to a key/value head
  int per;             // tokens of a row tile of the tensor-core kernel
  int page_size, box;                  // box: keys of one page copy
  void* out;
  int64_t out_token, out_head;
  float *lse, *part_o;
  float2* part_ml;
  float scale_log2;
  unsigned int* err;
  int* counter;  // [2] of the few-row kernel: work taken, CTAs done; 0 between launches
  long long wait_limit;  // cycles after which the wait that the test hook starves gives up (and ends the others)
  int stall;             // test hook: withhold each CTA's first signal to the consumers
};

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// True in one lane of the (converged) warp.  tcgen05 instructions take their operands from uniform registers;
// behind this election the compiler knows that one lane runs them, and issues them back to back, which behind
// `lane == 0` it does not.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 r;\n\t"
      "elect.sync r|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(p));
  return p != 0;
}

// Each thread of the warp reads 16, 32 or 64 consecutive 32-bit columns of its own TMEM lane and waits for them.
// The wait stands in the same statement: apart, nothing would keep the compiler from using the registers
// before it.
__device__ __forceinline__ void tmem_read(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=&r"(r[0]), "=&r"(r[1]), "=&r"(r[2]), "=&r"(r[3]), "=&r"(r[4]), "=&r"(r[5]), "=&r"(r[6]), "=&r"(r[7]),
        "=&r"(r[8]), "=&r"(r[9]), "=&r"(r[10]), "=&r"(r[11]), "=&r"(r[12]), "=&r"(r[13]), "=&r"(r[14]),
        "=&r"(r[15])
      : "r"(taddr + 0));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_read(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=&r"(r[0]), "=&r"(r[1]), "=&r"(r[2]), "=&r"(r[3]), "=&r"(r[4]), "=&r"(r[5]), "=&r"(r[6]), "=&r"(r[7]),
        "=&r"(r[8]), "=&r"(r[9]), "=&r"(r[10]), "=&r"(r[11]), "=&r"(r[12]), "=&r"(r[13]), "=&r"(r[14]),
        "=&r"(r[15]), "=&r"(r[16]), "=&r"(r[17]), "=&r"(r[18]), "=&r"(r[19]), "=&r"(r[20]), "=&r"(r[21]),
        "=&r"(r[22]), "=&r"(r[23]), "=&r"(r[24]), "=&r"(r[25]), "=&r"(r[26]), "=&r"(r[27]), "=&r"(r[28]),
        "=&r"(r[29]), "=&r"(r[30]), "=&r"(r[31])
      : "r"(taddr + 0));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_read(uint32_t taddr, float (&v)[64]) {
  uint32_t r[64];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=&r"(r[0]), "=&r"(r[1]), "=&r"(r[2]), "=&r"(r[3]), "=&r"(r[4]), "=&r"(r[5]), "=&r"(r[6]), "=&r"(r[7]),
        "=&r"(r[8]), "=&r"(r[9]), "=&r"(r[10]), "=&r"(r[11]), "=&r"(r[12]), "=&r"(r[13]), "=&r"(r[14]),
        "=&r"(r[15]), "=&r"(r[16]), "=&r"(r[17]), "=&r"(r[18]), "=&r"(r[19]), "=&r"(r[20]), "=&r"(r[21]),
        "=&r"(r[22]), "=&r"(r[23]), "=&r"(r[24]), "=&r"(r[25]), "=&r"(r[26]), "=&r"(r[27]), "=&r"(r[28]),
        "=&r"(r[29]), "=&r"(r[30]), "=&r"(r[31]), "=&r"(r[32]), "=&r"(r[33]), "=&r"(r[34]), "=&r"(r[35]),
        "=&r"(r[36]), "=&r"(r[37]), "=&r"(r[38]), "=&r"(r[39]), "=&r"(r[40]), "=&r"(r[41]), "=&r"(r[42]),
        "=&r"(r[43]), "=&r"(r[44]), "=&r"(r[45]), "=&r"(r[46]), "=&r"(r[47]), "=&r"(r[48]), "=&r"(r[49]),
        "=&r"(r[50]), "=&r"(r[51]), "=&r"(r[52]), "=&r"(r[53]), "=&r"(r[54]), "=&r"(r[55]), "=&r"(r[56]),
        "=&r"(r[57]), "=&r"(r[58]), "=&r"(r[59]), "=&r"(r[60]), "=&r"(r[61]), "=&r"(r[62]), "=&r"(r[63])
      : "r"(taddr + 0), "r"(taddr + 32));
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z,
                                            int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// Key tile j of an item: first key, how many there are, and the page list it is read through.
struct KeyTile {
  int base, valid, pg;
  bool own;
};
template <int kKeys>
__device__ __forceinline__ KeyTile key_tile(const StepItem& it, int j) {
  const int na = (it.a1 - it.a0 + kKeys - 1) / kKeys;
  KeyTile t;
  t.own = j >= na;
  t.base = t.own ? it.b0 + (j - na) * kKeys : it.a0 + j * kKeys;
  t.valid = min(kKeys, (t.own ? it.b1 : it.a1) - t.base);
  t.pg = t.own ? it.pg_b : it.pg_a;
  return t;
}
template <int kKeys>
__device__ __forceinline__ int key_tiles(const StepItem& it) {
  return (it.a1 - it.a0 + kKeys - 1) / kKeys + (it.b1 - it.b0 + kKeys - 1) / kKeys;
}

// One lane's share of a key tile's copies: lane (copy * kHalves + half) brings 64 values of the head from the
// box of keys `copy`.  The page number is read ahead of the copy by page_of.
template <int kKeys, int kHalves>
struct TileCopy {
  static __device__ __forceinline__ int copies(const KeyTile& t, int box) { return (t.valid + box - 1) / box; }
  static __device__ __forceinline__ int page_of(const AttendParams& p, const KeyTile& t, int lane) {
    const int c = lane / kHalves;
    if (c >= copies(t, p.box)) return 0;
    return __ldg(&p.pages[t.pg + (t.base + c * p.box) / p.page_size]);
  }
  static __device__ __forceinline__ void issue(const AttendParams& p, const KeyTile& t, int page, int lane,
                                               uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int kv_head) {
    const int c = lane / kHalves, half = lane % kHalves;
    if (c >= copies(t, p.box)) return;
    tma_load_4d(dst + half * (kKeys * 128) + c * p.box * 128, map, bar, half * 64, (t.base + c * p.box) % p.page_size,
                kv_head, page);
  }
};

// Programmatic launch: a kernel launched so may start when every CTA of the kernel before it in the stream has
// called launch_next() (or ended), and sees that kernel's results after wait_before().
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <class... P, class... A>
cudaError_t launch_early(void (*kernel)(P...), int grid, int block, int smem, cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}

// early: attend_tiles was launched just before.
cudaError_t attend_rows(Act act, int head_dim, const CUtensorMap& mk, const CUtensorMap& mv, const Rows& q,
                        const AttendParams& p, bool early, cudaStream_t st);
cudaError_t attend_tiles(Act act, int head_dim, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                         const AttendParams& p, int ctas, cudaStream_t st);

}  // namespace rv
