// Internal launch interface between the 8-bit cache's C ABI (fp8_cache_abi.hip) and its gfx950 kernels
// (fp8_cache_append.hip, fp8_cache_attend.hip). Not installed; the public surface is
// include/bikv_pagecopy.h.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "host_logic/attend_plan.h"
#include "host_logic/fp8_logic.h"

namespace bikv {

// The sequences of one call: where their pages are, how long they are, which rows of the caller's
// tensors are theirs. All arrays are device memory.
struct SeqArgs {
  const int64_t* table;      // [n_seqs][max_pages], rows table_stride elements apart
  int64_t table_stride;
  const int64_t* kv_lens;    // tokens of each sequence, the call's own included
  const int64_t* q_starts;   // n_seqs + 1 row numbers, or null: sequence b owns row b
  int64_t n_seqs;
  int64_t n_rows;            // rows of the caller's tensors
  int64_t max_len;           // max_pages * page_tokens, at most 2^30: a few steps more still fit an int
};

// One layer of the cache.
struct LayerArgs {
  char* k;                   // payload planes
  char* v;
  char* ks;                  // scale planes, fp32
  char* vs;
  int64_t n_pages;
  int64_t page_stride;       // bytes
  int64_t token_stride;      // bytes
  int64_t scale_stride;      // bytes between the scales of two pages
  FastDiv page_tokens;
  int32_t heads;
};

struct AppendArgs {
  SeqArgs seq;
  LayerArgs layer;
  const uint16_t* k;         // [n_rows][heads][head_dim]
  const uint16_t* v;
  int64_t k_row, k_head, v_row, v_head;   // strides in elements
  int64_t units;             // page slots of the launch, see the kernel
  uint32_t* status;
};
// type: 0 = bf16, 1 = fp16
hipError_t launch_fp8_append(int head_dim, int type, const AppendArgs& a, hipStream_t stream);

// Few rows: what a slot says of the row tile that begins in its share and ends in a later one.
struct JoinHead {
  int64_t first_row;         // of the tile's sequence
  int32_t tile;
  int32_t rows;              // 0: there is none
  int32_t parts;
  int32_t first_index;       // of its first part; the i-th other one is 2 * (slot + i)
};

struct AttendArgs {
  SeqArgs seq;
  LayerArgs layer;
  const uint16_t* q;         // [n_rows][heads * group][head_dim]
  uint16_t* out;
  float* lse;                // [n_rows][heads * group], or null
  int64_t q_row, q_head, o_row, o_head;   // strides in elements
  FastDiv group;             // query heads to a KV head
  int32_t causal;
  float scale_log2;          // softmax scale * log2(e)
  float* part_o;             // partial results, see the kernels
  float* part_ml;
  JoinHead* part_join;       // few rows: one per slot
  int32_t slots;             // few rows: shares the work is cut into, 0 = a workgroup per tile; many rows: parts a tile's keys are cut into
  int32_t min_steps;         // few rows: key steps a share has at least
  int32_t begin_cost;        // few rows: steps' worth of room before a tile's steps
  int32_t heads_per_group;   // few rows: KV heads of a workgroup
  int64_t tiles;             // row tiles of the launch
  uint32_t* status;
};
hipError_t launch_fp8_attend(const AttendPlan& plan, int head_dim, int type, const AttendArgs& a, hipStream_t stream);

}  // namespace bikv
