// What the pool data movers of every element type share: where an append's tokens go, what a gather writes, and how
// the packed gather's grid is dealt out.
#pragma once
#include "common.h"

namespace pace_kv {
// Where the tokens go: either an explicit slot id per token, or "position
// seq_lens[b] + pos_offset + t of sequence b" resolved through the block table.
struct AppendDest {
  const int64_t* slots;
  const int32_t* table;
  const int32_t* seq_lens;
  int32_t table_stride;
  int32_t pos_offset;
  const int32_t* offset_dev;  // optional: one more offset, read on the device (a counter a captured graph advances)
};

// Two output forms: dense [B][H*n_rep][out_len][D] and packed [sum len][H*n_rep][D] (see kv_gather_kernel).
struct GatherOut {
  uint16_t* k;
  uint16_t* v;
  const int32_t* cu_seqlens;  // packed form only
  int64_t stride_b;           // dense: elements between sequences
  int64_t stride_h;           // elements between output heads
  int64_t stride_t;           // elements between token rows
  int32_t out_len;            // dense: rows per sequence; packed: unused
  int32_t zero_fill;          // dense: write zeros to rows in [len, out_len)
  int32_t batch;              // packed: sequences (cu_seqlens has batch + 1 entries)
  int32_t total_rows;         // packed: rows of the outputs
  int32_t dense_rows;         // packed grid (one workgroup per block that exists), rows written in the dense layout
};

// Packed grid: which (sequence, head, logical block) workgroup `entry` stands for.
// One grid entry per (logical block that can exist, KV head): sequence b owns the block entries
// [cu[b] / 16 + b, cu[b+1] / 16 + b + 1) -- at least ceil(len_b / 16) of them, disjoint, in order -- so a
// ragged batch launches (almost) no workgroup without rows.  Entries run sequence by sequence, head by
// head, block by block (the order of the dense grid: with the heads of a block side by side instead the
// launch measured 6 % slower).  The owner is found by bisection, uniform over the workgroup: scalar loads
// from a table that stays in the scalar cache.
__device__ __forceinline__ void packed_entry(const int32_t* __restrict__ cu, int batch, int H, unsigned entry, int& b, int& h, int& j) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((int64_t)(cu[mid] / PACE_KV_BLOCK_TOKENS + mid) * H <= (int64_t)entry) lo = mid; else hi = mid;
  }
  b = lo;
  const int first = cu[b] / PACE_KV_BLOCK_TOKENS + b;
  const int n = cu[b + 1] / PACE_KV_BLOCK_TOKENS + b + 1 - first;  // >= 1
  const int r = (int)((int64_t)entry - (int64_t)first * H);
  h = min(r / n, H - 1), j = r % n;
}

// Pools of 4-bit rows (q4_ops.hip); arguments are already checked.
int launch_q4_append(const char* who, const pace_kv_pool_t* pool, const void* k_new, const void* v_new, int64_t stride_b,
                     int64_t stride_h, int64_t stride_t, int32_t batch, int32_t n_tokens, const AppendDest& dest, bool paged,
                     hipStream_t stream);
int launch_q4_gather(const char* who, const pace_kv_pool_t* pool, const int32_t* block_table, int32_t table_stride,
                     const int32_t* seq_lens, int32_t seq_len_bias, int32_t n_rep, const GatherOut& out, int64_t n_blocks, int32_t batch,
                     bool packed, hipStream_t stream);

}  // namespace pace_kv
