// Decoder-side operators over a paged key/value cache: the device records that the host plan of one
// decoding step (decode.cpp) hands to the kernels, and the kernels' launchers.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"

namespace rv {

// A new token of the step: the pool page and the slot in it that its key and value go to, its
// position (prefix length + place among its sequence's own tokens) and its sequence.
struct alignas(16) StepToken {
  int page, slot, pos, seq;
};

// A piece of attention work for each group of query heads: tokens tok0 .. tok0 + n - 1 against prefix keys
// [a0, a1) (pages from pages[pg_a]) and own keys [b0, b1) (pages from pages[pg_b]), of which token i sees
// those below diag + i + 1.  a0 and b0 are multiples of the key tile.  The result is partial number `part`
// of each of its tokens (StepParts).
struct alignas(16) StepItem {
  int tok0, n, pg_a, a0, a1, pg_b, b0, b1, diag, part, pad0, pad1;
};

// Partial results of a token: partials first .. first + count - 1 of the workspace; with count 1 its item
// writes the output itself.
struct alignas(8) StepParts {
  int first, count;
};

// Key and value pools of one layer: element (page, head, slot, d) of either at
// page * page_stride + head * head_stride + slot * slot_stride + d.
struct KvPool {
  void *k, *v;
  int64_t page_stride, head_stride, slot_stride;
  int page_size;
};

// [tokens, heads, head_dim] rows with unit stride along head_dim.
struct Rows {
  const void* p;
  int64_t token_stride, head_stride;
};

struct AppendArgs {
  const StepToken* tokens;
  int n_tokens, q_heads, kv_heads, head_dim;
  Rows q, k, v;  // q.p may be null: keys and values only
  void* q_out;
  int64_t q_out_token, q_out_head;
  KvPool pool;
  const float *cos, *sin;  // [positions, rot / 2]
  int rot;
  bool interleaved;
  bool vec;  // every address and stride a multiple of 16 bytes, rot and head_dim of 16 elements
};
cudaError_t kv_append(Act act, const AppendArgs& a, cudaStream_t st);

// Query heads that share key/value loads: a row tile holds `fold` heads of every token.
constexpr int kRowTile = 16;         // rows of an item of the few-row kernel
constexpr int kRowKeys = 64;         // keys of its tile
constexpr int kTileRows = 128;       // rows of one of the two row tiles of a tensor-core item
constexpr int kTileKeys = 128;       // keys of its tile

struct AttendArgs {
  const StepItem* row_items;   // for attend_rows: n * fold <= kRowTile
  const StepItem* tile_items;  // for attend_tiles: n <= 2 * (kTileRows / fold), most work first
  const StepParts* parts;      // by token; null where every token has one partial
  const int* joined;           // tokens with a partial count other than 1
  const int* pages;
  int n_row_items, n_tile_items, n_joined;
  int tile_sms;  // CTAs of attend_tiles at most
  int n_tokens, q_heads, kv_heads, head_dim, fold;
  Rows q;
  void* out;
  int64_t out_token, out_head;
  float* lse;     // [tokens, q_heads] or null
  float* part_o;  // [partials, q_heads, head_dim] results of items, divided by their own sums
  float2* part_ml;  // [partials, q_heads] reference exponents m and sums l of 2^(score - m) (0: no weight)
  KvPool pool;
  int64_t num_pages;
  float scale;
  unsigned int* err;  // error word that the host reads
  int* counter;       // [2] zeros, left as zeros
};
cudaError_t step_attend(Act act, const AttendArgs& a, cudaStream_t st);

struct NormArgs {
  const void *x, *residual;  // residual may be null
  const float* weight;
  int64_t rows;
  int hidden;
  int64_t x_stride, residual_stride, residual_out_stride, out_stride;
  void* residual_out;  // may be null
  void* out;           // 16-bit rows, or e4m3 codes when scales is given
  float* scales;       // [rows, hidden / group]
  int group;           // values a scale stands for (hidden: one scale a row)
  float eps;
  bool vec;  // hidden a multiple of 8, every row of x, residual and the outputs on 16 bytes (codes: 8)
};
cudaError_t rms_norm(Act act, const NormArgs& a, cudaStream_t st);

}  // namespace rv
