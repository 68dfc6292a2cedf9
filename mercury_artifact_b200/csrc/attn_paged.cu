// Attention over keys and values in pages: checks, the choice between the two kernels, workspaces.
#include "attn_paged.cuh"

namespace mb {

constexpr int kFewRows = 32;  // most rows that paged_rows_kernel takes

struct PagedPlan {
  int few, rows, ctas;
  long long rows_bytes;  // workspace of the kernel for few rows
};

static int plan_paged(const mb_attn_paged_args* x, PagedPlan* p) {
  if (x->hq <= 0 || x->kv.hkv <= 0 || x->hq % x->kv.hkv != 0) return MB_E_INVALID;
  if (x->max_queries < 0 || x->max_keys < 0 || !(x->softmax_scale > 0.f) || x->softmax_scale > 3e38f) return MB_E_INVALID;
  if (x->kv.batch < 0 || x->kv.page_size <= 0 || x->kv.max_pages < 0) return MB_E_INVALID;
  const int group = x->hq / x->kv.hkv;
  if ((long long)x->max_queries * group > 0x7fffff00ll) return MB_E_INVALID;
  // steps of a launch are counted in 32 bits
  if ((double)x->kv.batch * x->kv.hkv * ((double)x->max_keys / 128 + 1) > 2e9) return MB_E_TOO_LARGE;
  p->few = kFewRows;
  p->rows = min(x->max_queries * group, kFewRows);
  p->ctas = paged_rows_ctas();
  if (p->ctas <= 0) return MB_E_CUDA;
  p->rows_bytes = paged_rows_workspace(p->rows, p->ctas);
  return MB_SUCCESS;
}

long long attn_paged_workspace(const mb_attn_paged_args* x) {
  PagedPlan p;
  if (x == nullptr || plan_paged(x, &p) != MB_SUCCESS) return 0;
  return p.rows_bytes;
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
  if (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 15u) || ws_bytes < (unsigned long long)p.rows_bytes) return MB_E_INVALID;

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
  const float unbias = fp8 ? (float)(1ull << kScaleBias) : 1.f;
  a.scale = x->softmax_scale * unbias;
  a.scale_log2 = x->softmax_scale * 1.4426950408889634f * unbias;
  a.out_scale = unbias;
  a.few = p.few;
  if (x->max_queries * a.group > kFewRows) return MB_E_UNSUPPORTED;

  // [partial rows | (maximum, sum) | open units]
  const long long slots = 2ll * p.ctas * (p.rows <= 16 ? 16 : 32);
  a.part_o = static_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + slots * kHeadDim);
  a.open = reinterpret_cast<int4*>(a.part_ml + slots);
  return launch_paged_rows(a, fp8, p.rows, p.ctas, stream);
}

}  // namespace mb
