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

// What one sequence's queries see: keys [0, len_a) of the prefix whose pages start at pages[pg_a],
// then keys of its own, pages from pages[pg_b]: token i of the sequence (tokens tok0 .. tok0 + n - 1)
// sees own keys j < min(len_b, diag + i + 1).
struct alignas(16) StepSeq {
  int tok0, n, pg_a, len_a, pg_b, len_b, diag, pad;
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

struct AttendArgs {
  const StepToken* tokens;
  const StepSeq* seqs;
  const int* pages;
  int n_tokens, q_heads, kv_heads, head_dim;
  Rows q;
  void* out;
  int64_t out_token, out_head;
  float* lse;  // [tokens, q_heads] or null
  KvPool pool;
  float scale;
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
};
cudaError_t rms_norm(Act act, const NormArgs& a, cudaStream_t st);

}  // namespace rv
