// Attention over keys and values in pages: checks, the choice between the two kernels, workspaces.
#include "attn_paged.cuh"

namespace mb {

// Most rows of a sequence (new tokens x heads of a group) that the kernel for few rows takes.  bf16: 17 to 32 rows are faster
// as (an eighth of) a tile, 64 sequences of 8 tokens, 32/8 heads, up to 8 192 keys: 252 us, 428 as rows; 8 of them: 61, 112.
// e4m3: a tile's sequence is first brought into bf16, which few rows do not pay for: 64 sequences as 32 rows take 330 us.  From
// there on it depends: with 10 tokens they take 562 us as tiles and 468 as 40 rows, 8 of them 89 and 113, 64 up to 1 000 keys
// 94 and 160, one of 32 768 keys 85 and 56.
constexpr int kFewRows = 16, kFewRowsE4m3 = 32;
// Steps up to which a unit of few rows is left to one CTA where there are no more units than SMs.  One token, 16 sequences of
// 2 000 keys, 8 heads: 27 us, split 32; one sequence, 2 heads: 20 and 28 (the host's time included).
constexpr int kWholeSteps = 16;
// e4m3: sequences that go to the tiles are brought into bf16 in groups that take no more than this (or one by one).  64
// sequences of 16 tokens, up to 8 192 keys: 563 us; groups of 256 MiB 706, of 4 GiB 557, which is not worth the memory.
constexpr long long kPackedBytes = 1ll << 30;

struct PagedPlan {
  int few;
  int rows, row_heads, row_ctas;    // rows of its units, K/V heads of a CTA, its grid (0: it has nothing to do)
  bool whole;            // a unit is one CTA's
  int tile_ctas;         // grid of the kernel for tiles (0: it has nothing to do)
  int share_tiles;
  bool split;
  int group;             // sequences of a launch of tiles
  long long rows_bytes, packed_bytes, split_bytes;  // workspaces
};

static long long align_up(long long n) { return (n + 255) & ~255ll; }

// Everything here goes by the bounds that the host knows; the lengths are on the device.
static int plan_paged(const mb_attn_paged_args* x, PagedPlan* p) {
  const mb_paged_kv& kv = x->kv;
  if (x->hq <= 0 || kv.hkv <= 0 || x->hq % kv.hkv != 0) return MB_E_INVALID;
  if (x->max_queries < 0 || x->max_keys < 0 || !(x->softmax_scale > 0.f) || x->softmax_scale > 2e38f /* (times log2(e)) */) return MB_E_INVALID;
  if (kv.batch < 0 || kv.tokens < 0 || kv.page_size <= 0 || kv.max_pages < 0) return MB_E_INVALID;
  // The kernels divide the work by the rows that a sequence has.  In a padded batch these are known, whatever the bound.
  const bool padded = kv.cu_seqlens == nullptr, e4m3 = kv.dtype == MB_DTYPE_E4M3;
  // (a ragged batch with a bound of no new tokens is launched all the same: the kernel reports the sequences that have some)
  const int queries = padded && kv.batch > 0 ? kv.tokens / kv.batch : max(x->max_queries, 1);
  const long long heads = x->hq / kv.hkv, rows = queries * heads;
  if (rows > 0x7fffff00ll) return MB_E_UNSUPPORTED;
  // steps of a launch are counted in 32 bits
  if ((double)kv.batch * kv.hkv * ((double)x->max_keys / 128 + 1) > 2e9) return MB_E_UNSUPPORTED;
  const int sms = sm_count();
  if (sms <= 0) return MB_E_CUDA;
  memset(p, 0, sizeof(*p));
  // Beside chunks the sequences with few rows are single tokens as a rule, which the kernels for fewer rows take faster.
  p->few = rows > kFewRows && heads <= 8 ? 8 : kFewRows;
  if (e4m3 && rows <= kFewRowsE4m3) p->few = kFewRowsE4m3;
  p->few = (int)min(rows, (long long)p->few);
  if (rows <= p->few || !padded) {
    p->rows = p->few;
    const int block = paged_rows_padded(p->rows);
    const long long units = (long long)kv.batch * kv.hkv * ((p->few + block - 1) / block);
    const int step = paged_rows_step(e4m3);
    // Few short units are not split over SMs: the launch that joins the parts would take longer than the steps it saves.
    p->whole = units <= sms && x->max_keys <= kWholeSteps * step;
    p->row_ctas = p->whole ? (int)units : sms;
    // A head's row of e4m3 is 128 bytes.  Two neighbours at once read 256 in a row, as bf16 does: 64 single tokens, 32/8 heads, up
    // to 16 384 keys 182 us, 202 one by one; 8 tokens each, up to 8 192 keys 330, 409.  Whole units stay one head's, which spreads
    // them over twice the SMs.
    p->row_heads = e4m3 && !p->whole && kv.hkv % 2 == 0 ? 2 : 1;
    p->rows_bytes = p->whole ? 0 : paged_rows_workspace(p->rows, p->row_heads, p->row_ctas);
  }
  if (rows > p->few) {
    const long long seq_bytes = (long long)x->max_keys * kv.hkv * 4 * kHeadDim;
    p->group = kv.batch;
    if (e4m3) {
      p->group = (int)max(1ll, min((long long)kv.batch, kPackedBytes / max(seq_bytes, 1ll)));
      p->packed_bytes = align_up(p->group * seq_bytes);
    }
    // units: blocks of 256 rows of a sequence and K/V head.  A ragged batch has at most one partly filled block per sequence.
    const long long most = p->group * ((rows + 255) / 256);
    const long long blocks = padded ? most : min(most, kv.tokens * heads / 256 + p->group);
    const long long units = blocks * kv.hkv, tiles = max(1, (x->max_keys + 127) / 128);
    // Costs in steps of one K/V tile against both query tiles: starting and ending a CTA, and joining the shares.
    constexpr double kCta = 2.0, kMerge = 2.0, kSlot = 0.02;
    long long best = 1;
    double t_best = ((units + sms - 1) / sms) * (tiles + kCta);
    for (long long ns = 2; ns <= 64 && ns <= tiles && units * ns <= 3ll * sms; ++ns) {
      const double t = ((units * ns + sms - 1) / sms) * ((tiles + ns - 1) / ns + kCta) + kMerge + kSlot * units * ns;
      if (t < t_best) {
        t_best = t;
        best = ns;
      }
    }
    p->share_tiles = (int)((tiles + best - 1) / best);
    const long long ctas = units * ((tiles + p->share_tiles - 1) / p->share_tiles);
    if (ctas > 0x7fffff00ll) return MB_E_UNSUPPORTED;
    p->tile_ctas = (int)ctas;
    p->split = best > 1;
    if (p->split) p->split_bytes = align_up(paged_tiles_workspace(p->tile_ctas));
  }
  return MB_SUCCESS;
}

// [bf16 copy | shares of the tiles | parts of the rows]
static long long workspace_of(const PagedPlan& p) { return p.packed_bytes + p.split_bytes + p.rows_bytes; }

long long attn_paged_workspace(const mb_attn_paged_args* x) {
  PagedPlan p;
  if (x == nullptr || plan_paged(x, &p) != MB_SUCCESS) return 0;
  return workspace_of(p);
}

int launch_attn_paged(const mb_attn_paged_args* x, void* ws, unsigned long long ws_bytes, cudaStream_t stream) {
  if (x == nullptr) return MB_E_INVALID;
  PagedAttnArgs a;
  memset(&a, 0, sizeof(a));
  int rc = paged_view(&x->kv, &a.c);
  if (rc != MB_SUCCESS) return rc;
  PagedPlan p;
  rc = plan_paged(x, &p);
  if (rc != MB_SUCCESS) return rc;
  if (x->max_keys > (long long)x->kv.max_pages * x->kv.page_size) return MB_E_INVALID;
  if (a.c.cu == nullptr && a.c.per_seq > x->max_queries) return MB_E_INVALID;
  if (a.c.batch == 0 || a.c.tokens == 0) return MB_SUCCESS;
  if (x->q == nullptr || x->o == nullptr || x->lse == nullptr) return MB_E_INVALID;
  const uintptr_t al = reinterpret_cast<uintptr_t>(x->q) | reinterpret_cast<uintptr_t>(x->o) | (uintptr_t)(x->q_stride_b * 2) |
                       (uintptr_t)(x->q_stride_t * 2) | (uintptr_t)(x->q_stride_h * 2) | (uintptr_t)(x->o_stride_b * 2) |
                       (uintptr_t)(x->o_stride_t * 2) | (uintptr_t)(x->o_stride_h * 2);
  if (al & 15u) return MB_E_INVALID;
  const long long need = workspace_of(p);
  if (need > 0 && (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 15u) || ws_bytes < (unsigned long long)need)) return MB_E_INVALID;

  a.q = static_cast<const __nv_bfloat16*>(x->q);
  a.q_sb = a.c.cu != nullptr ? 0 : x->q_stride_b;
  a.q_st = x->q_stride_t;
  a.q_sh = x->q_stride_h;
  a.o = static_cast<__nv_bfloat16*>(x->o);
  a.o_sb = a.c.cu != nullptr ? 0 : x->o_stride_b;
  a.o_st = x->o_stride_t;
  a.o_sh = x->o_stride_h;
  a.lse = x->lse;
  a.lse_sb = a.c.cu != nullptr ? 0 : x->lse_stride_b;
  a.lse_sh = x->lse_stride_h;
  a.hq = x->hq;
  a.group = x->hq / x->kv.hkv;
  a.max_queries = x->max_queries;
  a.max_keys = x->kv.pages > 0 ? x->max_keys : 0;  // (without pages there are no keys: longer sequences are errors)
  a.causal = x->causal ? 1 : 0;
  const bool e4m3 = x->kv.dtype == MB_DTYPE_E4M3;
  a.scale_log2 = x->softmax_scale * 1.4426950408889634f;
  a.few = p.few;
  a.share_tiles = max(p.share_tiles, 1);

  uint8_t* at = static_cast<uint8_t*>(ws);
  if (p.tile_ctas > 0 && e4m3 && a.max_keys > 0) {  // [keys | values]
    a.packed_rows = x->max_keys;
    a.packed_k = reinterpret_cast<const __nv_bfloat16*>(at);
    a.packed_v = a.packed_k + (long long)p.group * x->max_keys * a.c.hkv * kHeadDim;
    at += p.packed_bytes;
  }
  if (p.split) {  // [rows | (maximum, sum) | split units]
    a.tile_o = reinterpret_cast<float4*>(at);
    a.tile_ml = reinterpret_cast<float2*>(a.tile_o + (long long)p.tile_ctas * (256 * kHeadDim / 4));
    a.tile_open = reinterpret_cast<int4*>(a.tile_ml + (long long)p.tile_ctas * 256);
    at += p.split_bytes;
  }
  a.whole = p.whole;
  if (p.row_ctas > 0 && !p.whole) {  // [partial rows | (maximum, sum) | open units]
    const long long slots = paged_rows_slots(p.rows, p.row_heads, p.row_ctas);
    a.part_o = reinterpret_cast<float*>(at);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + slots * kHeadDim);
    a.open = reinterpret_cast<int4*>(a.part_ml + slots);
  }

  for (int b = 0; p.tile_ctas > 0 && b < a.c.batch; b += p.group) {
    a.b_begin = b;
    a.b_end = min(b + p.group, a.c.batch);
    if (a.packed_k != nullptr) {
      rc = launch_read_e4m3(a, p.few / a.group + 1, stream);
      if (rc != MB_SUCCESS) return rc;
    }
    rc = launch_paged_tiles(a, p.tile_ctas, stream);
    if (rc != MB_SUCCESS) return rc;
    if (p.split) {
      rc = launch_paged_tiles_merge(a, p.tile_ctas, stream);
      if (rc != MB_SUCCESS) return rc;
    }
  }
  if (p.row_ctas > 0) {
    rc = launch_paged_rows(a, e4m3, p.rows, p.row_heads, p.row_ctas, stream);
    if (rc != MB_SUCCESS) return rc;
  }
  return p.row_ctas > 0 && !p.whole ? launch_paged_rows_merge(a, p.rows, p.row_heads, p.row_ctas, stream) : MB_SUCCESS;
}

}  // namespace mb
