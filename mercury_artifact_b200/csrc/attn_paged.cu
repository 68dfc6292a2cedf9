// Attention over keys and values in pages: checks, the choice between the two kernels, workspaces.
#include "attn_paged.cuh"

namespace mb {

constexpr int kPackedRows = 512;            // e4m3: with more rows in a sequence the tiles read a bf16 copy,
constexpr long long kPackedBytes = 1ll << 30;  // if it takes no more than this
static long long align_up(long long n) { return (n + 255) & ~255ll; }
constexpr int kFewRows = 32;  // most rows that paged_rows_kernel takes

struct PagedPlan {
  int few;               // most rows of a sequence that go to the kernel for few rows
  int rows, row_ctas;    // rows of its units (0: it has nothing to do)
  int tile_ctas;         // grid of the kernel for tiles (0: it has nothing to do)
  int share_tiles;
  bool split;
  int packed_rows;  // e4m3: rows of a sequence in the bf16 copy that the tiles read (0: none)
  long long rows_bytes, tiles_bytes;  // workspaces
};

// Everything here goes by the bounds that the host knows; the lengths are on the device.
static int plan_paged(const mb_attn_paged_args* x, PagedPlan* p) {
  if (x->hq <= 0 || x->kv.hkv <= 0 || x->hq % x->kv.hkv != 0) return MB_E_INVALID;
  if (x->max_queries < 0 || x->max_keys < 0 || !(x->softmax_scale > 0.f) || x->softmax_scale > 3e38f) return MB_E_INVALID;
  if (x->kv.batch < 0 || x->kv.tokens < 0 || x->kv.page_size <= 0 || x->kv.max_pages < 0) return MB_E_INVALID;
  const long long group = x->hq / x->kv.hkv, rows = x->max_queries * group;
  if (rows > 0x7fffff00ll) return MB_E_TOO_LARGE;
  // steps of a launch are counted in 32 bits
  if ((double)x->kv.batch * x->kv.hkv * ((double)x->max_keys / 128 + 1) > 2e9) return MB_E_TOO_LARGE;
  const int sms = sm_count();
  if (sms <= 0) return MB_E_CUDA;
  memset(p, 0, sizeof(*p));
  const bool padded = x->kv.cu_seqlens == nullptr;
  // Beside chunks the sequences with few rows are single tokens as a rule, which the kernel for 16 rows takes faster than
  // that for 32 (11 of them against up to 8 192 e4m3 keys, 4 rows each: 24 us, 31 with room for 32 rows).
  p->few = rows > kFewRows && group <= 16 ? 16 : kFewRows;
  if (rows <= kFewRows || !padded) {
    p->rows = (int)min(rows, (long long)p->few);
    p->row_ctas = paged_rows_ctas();
    p->rows_bytes = paged_rows_workspace(p->rows, p->row_ctas);
  }
  if (rows > kFewRows) {
    // units: blocks of 256 rows of a sequence and K/V head.  A ragged batch has at most one partly filled block per sequence.
    const long long blocks = padded ? x->kv.batch * ((rows + 255) / 256) : min(x->kv.batch * ((rows + 255) / 256), x->kv.tokens * group / 256 + x->kv.batch);
    const long long units = blocks * x->kv.hkv, tiles = max(1, (x->max_keys + 127) / 128);
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
    if (units * best > 0x7fffff00ll) return MB_E_TOO_LARGE;
    p->share_tiles = (int)((tiles + best - 1) / best);
    p->split = best > 1;
    p->tile_ctas = (int)(units * ((tiles + p->share_tiles - 1) / p->share_tiles));
    if (p->split) p->tiles_bytes = paged_tiles_workspace(p->tile_ctas);
    // Every block of 256 rows turns the codes that it reads into f16 for itself, which takes the tiles from 1.60 to 2.65 us
    // (two tiles of 128 rows, one of keys).  From two blocks on it is faster to bring the sequence into bf16 once (776
    // bytes a key and head), as long as that copy stays small.
    const long long packed = (long long)x->kv.batch * x->max_keys * x->kv.hkv * 4 * kHeadDim;
    if (x->kv.dtype == MB_DTYPE_E4M3 && rows > kPackedRows && packed <= kPackedBytes) {
      p->packed_rows = x->max_keys;
      p->tiles_bytes += align_up(packed);
    }
  }
  return MB_SUCCESS;
}

long long attn_paged_workspace(const mb_attn_paged_args* x) {
  PagedPlan p;
  if (x == nullptr || plan_paged(x, &p) != MB_SUCCESS) return 0;
  return max(p.rows_bytes, p.tiles_bytes);
}

int launch_attn_paged(const mb_attn_paged_args* x, void* ws, unsigned long long ws_bytes, cudaStream_t stream) {
  if (x == nullptr) return MB_E_INVALID;
  PagedAttnArgs a;
  int rc = paged_view(&x->kv, &a.c);
  if (rc != MB_SUCCESS) return rc;
  PagedPlan p;
  rc = plan_paged(x, &p);
  if (rc != MB_SUCCESS) return rc;
  if (x->max_keys > (long long)x->kv.max_pages * x->kv.page_size) return MB_E_INVALID;
  if (a.c.cu == nullptr && a.c.per_seq > x->max_queries) return MB_E_INVALID;
  if (a.c.batch == 0 || a.c.tokens == 0 || x->max_queries == 0) return MB_SUCCESS;
  if (x->q == nullptr || x->o == nullptr || x->lse == nullptr) return MB_E_INVALID;
  const uintptr_t al = reinterpret_cast<uintptr_t>(x->q) | reinterpret_cast<uintptr_t>(x->o) | (uintptr_t)(x->q_stride_b * 2) |
                       (uintptr_t)(x->q_stride_t * 2) | (uintptr_t)(x->q_stride_h * 2) | (uintptr_t)(x->o_stride_b * 2) |
                       (uintptr_t)(x->o_stride_t * 2) | (uintptr_t)(x->o_stride_h * 2);
  if (al & 15u) return MB_E_INVALID;
  const long long need = max(p.rows_bytes, p.tiles_bytes);
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
  a.max_keys = x->max_keys;
  a.causal = x->causal ? 1 : 0;
  const bool fp8 = x->kv.dtype == MB_DTYPE_E4M3;
  a.scale_log2 = x->softmax_scale * 1.4426950408889634f;
  a.few = p.few;
  a.share_tiles = max(p.share_tiles, 1);
  a.head_bytes = fp8 ? 2 * kHeadDim : 4 * kHeadDim;
  a.tile_o = nullptr;
  a.tile_ml = nullptr;
  a.tile_open = nullptr;
  a.packed_k = a.packed_v = nullptr;
  a.packed_rows = p.packed_rows;
  a.part_o = nullptr;
  a.part_ml = nullptr;
  a.open = nullptr;

  // The two kernels run one after the other and use the workspace in turn.
  if (p.tile_ctas > 0) {
    uint8_t* at = static_cast<uint8_t*>(ws);
    if (p.packed_rows > 0) {  // [keys | values]
      const long long half = (long long)a.c.batch * p.packed_rows * a.c.hkv * kHeadDim;
      a.packed_k = reinterpret_cast<const __nv_bfloat16*>(at);
      a.packed_v = a.packed_k + half;
      rc = launch_read_e4m3(a.c, at, at + half * 2, p.packed_rows, p.few / a.group + 1, a.max_queries, stream);
      if (rc != MB_SUCCESS) return rc;
      at += align_up(half * 4);
    }
    if (p.split) {  // [rows | (maximum, sum) | split units]
      a.tile_o = reinterpret_cast<float4*>(at);
      a.tile_ml = reinterpret_cast<float2*>(a.tile_o + (long long)p.tile_ctas * (256 * kHeadDim / 4));
      a.tile_open = reinterpret_cast<int4*>(a.tile_ml + (long long)p.tile_ctas * 256);
    }
    rc = launch_paged_tiles(a, fp8, p.tile_ctas, stream);
    if (rc != MB_SUCCESS) return rc;
  }
  if (p.row_ctas > 0) {
    // [partial rows | (maximum, sum) | open units]
    const long long slots = 2ll * p.row_ctas * paged_rows_padded(p.rows);
    a.part_o = static_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + slots * kHeadDim);
    a.open = reinterpret_cast<int4*>(a.part_ml + slots);
    rc = launch_paged_rows(a, fp8, p.rows, p.row_ctas, stream);
  }
  return rc;
}

}  // namespace mb
