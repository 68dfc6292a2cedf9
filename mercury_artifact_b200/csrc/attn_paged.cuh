// Arguments shared by the two attention kernels over pages and their host side.
#pragma once

#include "paged_common.cuh"

namespace mb {

struct PagedAttnArgs {
  PagedView c;
  const __nv_bfloat16* q;
  long long q_sb, q_st, q_sh;  // element strides: sequence (0 with offsets), token, head
  __nv_bfloat16* o;
  long long o_sb, o_st, o_sh;
  float* lse;
  long long lse_sb, lse_sh;
  int hq, group, max_queries, max_keys, causal;
  float scale_log2;  // softmax scale * log2(e): maxima are kept in units of the exponent of two
  // rows of a sequence: new tokens x heads of a group.  Sequences with at most `few` rows belong to the kernel for
  // few rows, the others to the kernel for tiles.
  int few;
  // partial results: [slot][head of a CTA][row][128] and (maximum, sum) [slot][head][row]; open: the unit that a CTA began and
  // left to the next ones (sequence, K/V head / heads of a CTA, number of CTAs, block of rows; first token, rows; CTAs 0: none)
  float* part_o;
  float2* part_ml;
  int4* open;
  int whole;  // few rows: CTA i has unit i, and nothing is joined
  // tiles: keys (in tiles of 128) of a share of a unit; partial results [CTA][32 column groups][256 rows], (maximum, sum)
  // [CTA][256]; tile_open: the split unit whose first share a CTA has (sequence, K/V head, row block, shares; 0: none).
  // All null where no unit is split.
  int share_tiles;
  // tiles: the sequences [b_begin, b_end); where their keys and values lie one after the other in bf16, [b_end - b_begin,
  // packed_rows, hkv, 128] (null: in pages)
  int b_begin, b_end;
  const __nv_bfloat16 *packed_k, *packed_v;
  int packed_rows;
  float4* tile_o;
  float2* tile_ml;
  int4* tile_open;
};

constexpr float kLn2 = 0.6931471805599453f;

// heads: neighbouring K/V heads of a CTA, 1 or 2 (e4m3 only)
int launch_paged_rows(const PagedAttnArgs& a, bool fp8, int rows, int heads, int ctas, cudaStream_t stream);
long long paged_rows_slots(int rows, int heads, int ctas);  // rows of partial results
long long paged_rows_workspace(int rows, int heads, int ctas);
int paged_rows_padded(int rows);
int paged_rows_step(bool fp8);  // keys of one head
// The first a.packed_rows keys and values of the sequences [a.b_begin, a.b_end) with at least min_new new tokens, in bf16.
int launch_read_e4m3(const PagedAttnArgs& a, int min_new, cudaStream_t stream);
int launch_paged_tiles(const PagedAttnArgs& a, int ctas, cudaStream_t stream);
int launch_paged_tiles_merge(const PagedAttnArgs& a, int ctas, cudaStream_t stream);
int launch_paged_rows_merge(const PagedAttnArgs& a, int rows, int heads, int ctas, cudaStream_t stream);
long long paged_tiles_workspace(long long ctas);

}  // namespace mb
