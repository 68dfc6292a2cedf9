// Writing keys and values into pages (bf16, or e4m3 with a power of two per 32 values) and reading them back.
//
// Both move every byte once: the bound is HBM, and for few tokens the latency of the chain lengths -> page number -> row.
// A group of lanes moves one row (the 128 values of a head of K or V of a token): 16 lanes of 8 values in bf16, 8 lanes
// of 16 values in e4m3, so that every access is 16 bytes a lane and whole rows at a time.  A block takes a run of
// rows, its threads look the places of its tokens up first (in shared memory), then every group moves its rows with
// all loads issued before the first store.  Four rows a group measured best for many tokens (e4m3, two prompts of 32 768, 8
// heads, one turn: 1, 2, 4 and 8 rows a group: 100, 85, 81, 99 us), one for few, which have too few blocks otherwise.
//
// Measured: that write 74-76 us, 407 MB, 5.4 TB/s of the 6.5 of a plain copy; three prompts of 1 500 to 9 001 tokens in bf16
// 18 us, 5.5 TB/s; reading 62 768 e4m3 keys of 8 heads back 66 us, 5.9 TB/s; single tokens of 32 sequences 9 us, all of it the
// host's launch.
//
// Why powers of two: a code has 4 significant bits, so code * 2^e is exact in bf16 (for every e that a write chooses).  What is
// read back, and what the attention kernels multiply, is the stored value itself with no second rounding; a factor of amax / 448 would use
// the top of the range a little better (at most one binade), but e4m3's step is relative, so that nothing is gained.
#include "attn_paged.cuh"

namespace mb {

int paged_view(const mb_paged_kv* x, PagedView* c) {
  if (x == nullptr) return MB_E_INVALID;
  if (x->head_dim != kHeadDim) return MB_E_UNSUPPORTED;
  if (x->dtype != MB_DTYPE_BF16 && x->dtype != MB_DTYPE_E4M3) return MB_E_UNSUPPORTED;
  if (x->batch < 0 || x->tokens < 0 || x->pages < 0 || x->page_size <= 0 || x->max_pages < 0 || x->hkv <= 0) return MB_E_INVALID;
  if (x->tokens > 0x7fffff00 || x->hkv > 1 << 20) return MB_E_UNSUPPORTED;  // (indices in 32 bits)
  const int size = x->dtype == MB_DTYPE_E4M3 ? 1 : 2;
  if (x->batch > 0 && (x->seq_lens == nullptr || (x->max_pages > 0 && x->page_table == nullptr))) return MB_E_INVALID;
  if (x->pages > 0) {
    if (x->k == nullptr || x->v == nullptr) return MB_E_INVALID;
    if (size == 1 && (x->k_scale == nullptr || x->v_scale == nullptr)) return MB_E_INVALID;
    const uintptr_t a = reinterpret_cast<uintptr_t>(x->k) | reinterpret_cast<uintptr_t>(x->v) |
                        (uintptr_t)(x->stride_page * size) | (uintptr_t)(x->stride_slot * size) |
                        (uintptr_t)(x->stride_h * size);
    if (a & 15u) return MB_E_INVALID;
    if ((reinterpret_cast<uintptr_t>(x->k_scale) | reinterpret_cast<uintptr_t>(x->v_scale)) & 3u) return MB_E_INVALID;
  }
  // positions are 32-bit; a sequence may use at most this many keys of its table's capacity
  if ((long long)x->max_pages * x->page_size > 0x7fffff00ll) return MB_E_INVALID;
  if (x->cu_seqlens == nullptr && x->batch > 0 && x->tokens % x->batch != 0) return MB_E_INVALID;
  memset(c, 0, sizeof(*c));
  c->k = static_cast<uint8_t*>(x->k);
  c->v = static_cast<uint8_t*>(x->v);
  c->page_sb = x->stride_page * size;
  c->slot_sb = x->stride_slot * size;
  c->head_sb = x->stride_h * size;
  // the stride of a dimension of one entry is never used; tensor maps want one that makes sense
  if (x->hkv == 1) c->head_sb = kHeadDim * size;
  if (x->page_size == 1) c->slot_sb = c->head_sb * x->hkv;
  if (x->pages == 1) c->page_sb = c->slot_sb * x->page_size;
  c->k_scale = x->k_scale;
  c->v_scale = x->v_scale;
  c->table = x->page_table;
  c->table_stride = x->page_table_stride;
  c->seq_lens = x->seq_lens;
  c->cu = x->cu_seqlens;
  c->batch = x->batch;
  c->tokens = x->tokens;
  c->per_seq = x->cu_seqlens == nullptr && x->batch > 0 ? x->tokens / x->batch : 0;
  c->pages = x->pages;
  c->page_size = x->page_size;
  c->page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (x->page_size == 1 << s) c->page_shift = s;
  c->max_pages = x->max_pages;
  c->hkv = x->hkv;
  c->status = x->status ? x->status : default_status_word();
  return c->status == nullptr ? MB_E_CUDA : MB_SUCCESS;
}

struct CacheMoveArgs {
  PagedView c;
  uint8_t* k;  // tokens' rows: source of a write, destination of a read (bf16)
  uint8_t* v;
  long long sb, st, sh;  // bytes
  int rows;              // read: rows per sequence
  int first_seq;         // read: sequences from this one on, the first one's rows at k, v
  int min_new, max_new;  // read: those with at least min_new new tokens only
  bool zeros;            // read: rows of bad pages become zeros, which the attention takes there (else they are left alone)
};

constexpr int kMoveThreads = 256;
template <bool kFp8>
struct MoveShape {
  static constexpr int kLanes = kFp8 ? 8 : 16;                 // lanes of a row
  static constexpr int kGroups = kMoveThreads / kLanes;        // rows at a time
};

// 16 bf16 values as e4m3 codes under 2^e, and the block's scale byte (the two lanes of a block agree on it).
__device__ __forceinline__ uint4 quantise16(const uint4 (&x)[2], uint32_t& byte) {
  const uint32_t w[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);  // |x| of bf16 orders like its bits
  m = max(m & 0xffffu, m >> 16);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  // amax = 1.f * 2^(E - 127) <= 448 * 2^e = 1.75 * 2^(e + 8)
  const int e = min(max((int)(m >> 7) - 135 + ((m & 0x7fu) > 0x60u ? 1 : 0), kMinScale - 127), kMaxScale - 127);
  byte = m >= 0x7f80u ? kNanScale : e + 127;
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);  // 2^-e
  uint32_t q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint16_t lo, hi;
    const float a0 = __uint_as_float(w[2 * i] << 16) * inv, a1 = __uint_as_float(w[2 * i] & 0xffff0000u) * inv;
    const float b0 = __uint_as_float(w[2 * i + 1] << 16) * inv, b1 = __uint_as_float(w[2 * i + 1] & 0xffff0000u) * inv;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(a1), "f"(a0));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(b1), "f"(b0));
    q[i] = (uint32_t)lo | ((uint32_t)hi << 16);
  }
  return make_uint4(q[0], q[1], q[2], q[3]);
}

// Rows of a block: r = (token * 2 + which) * hkv + head, `kIters` rows per group of lanes at a time.  Blocks of e4m3, which
// are bound by their instructions and barriers as much as by memory, take two turns of them for one lookup (the prompts above:
// 80.6 us with one turn, 75.8, 74.1 with four, which however leave short prompts too few blocks; bf16, two prompts of 32 768:
// 83.6, 84.8, 86.9).
template <bool kFp8, int kIters>
constexpr int kTurns = kFp8 && kIters > 1 ? 2 : 1;
// (four blocks an SM, which the compiler does not aim for by itself: the prompts in e4m3 74.0 us, 77.6 without)
template <bool kFp8, int kIters>
__global__ void __launch_bounds__(kMoveThreads, kFp8 && kIters > 1 ? 4 : 1) kv_cache_write_kernel(const __grid_constant__ CacheMoveArgs a) {
  using S = MoveShape<kFp8>;
  constexpr int kRows = S::kGroups * kIters * kTurns<kFp8, kIters>;
  __shared__ long long place[kRows / 2 + 2], source[kRows / 2 + 2];  // of a token: byte offsets (-1: not stored)
  __shared__ long long place_scale[kFp8 ? kRows / 2 + 2 : 1];
  __shared__ int bad;  // the offsets do not ascend within the tokens
  const PagedView& c = a.c;
  const int per_token = 2 * c.hkv;
  const long long total = (long long)c.tokens * per_token;
  const long long row0 = (long long)blockIdx.x * kRows;
  const int t0 = (int)(row0 / per_token), t1 = (int)min((row0 + kRows - 1) / per_token, c.tokens - 1ll);
  grid_dependents_launch();
  grid_dependency_wait();

  int first = 0;  // sequence of token t0
  if (threadIdx.x == 0) bad = 0;
  if (c.cu != nullptr) {
    for (int b = 0; b < c.batch; b += kMoveThreads) {
      const int i = b + threadIdx.x;
      const int lo = i < c.batch ? c.cu[i] : 0, hi = i < c.batch ? c.cu[i + 1] : 0;
      first += __syncthreads_count(i < c.batch && hi <= t0);
      if (lo < 0 || hi < lo || hi > c.tokens) bad = 1;
    }
  }
  for (int t = t0 + threadIdx.x; t <= t1; t += kMoveThreads) {
    int b, end;
    if (c.cu != nullptr) {
      b = first;
      while (b < c.batch && c.cu[b + 1] <= t) ++b;
      if (b < c.batch && c.cu[b] > t) b = c.batch;  // rows before the first sequence
      end = b < c.batch ? c.cu[b + 1] : 0;
    } else {
      b = t / c.per_seq;
      end = (b + 1) * c.per_seq;
    }
    long long to = -1, to_scale = 0, from = 0;
    if (b < c.batch) {
      const int len = c.seq_lens[b];
      const long long pos = (long long)len - (end - t);
      from = c.cu != nullptr ? t * a.st : b * a.sb + (t - (end - c.per_seq)) * a.st;
      if (len < 0 || len > c.max_pages * c.page_size) {
        paged_error(c);
      } else if (pos >= 0) {
        const int p = page_index(c, (int)pos), slot = (int)pos - p * c.page_size;
        const int id = c.table[b * c.table_stride + p];
        if (id < 0 || id >= c.pages) {
          paged_error(c);
        } else {
          to = paged_offset(c, id, slot, 0);
          to_scale = scale_offset(c, id, slot, 0);
        }
      }
    }
    place[t - t0] = to;
    source[t - t0] = from;
    if constexpr (kFp8) place_scale[t - t0] = to_scale;
  }
  __syncthreads();
  // Offsets that do not ascend within the tokens do not say which key a token is: every block sees them, and none stores (a
  // token at a wrong position would replace a key).
  if (bad && threadIdx.x == 0) paged_error(c);

  const int group = threadIdx.x / S::kLanes, lane = threadIdx.x % S::kLanes;
  // a group's i-th row and the end, counted from the first row of token t0 (divisions in 32 bits)
  const int row_in = (int)(row0 - (long long)t0 * per_token) + group;
  const int rows = bad ? 0 : (int)min(total - (long long)t0 * per_token, (long long)(kRows + per_token));
#pragma unroll 1
  for (int turn = 0; turn < kTurns<kFp8, kIters>; ++turn) {
    uint4 x[kIters][kFp8 ? 2 : 1];
    uint8_t* dst[kIters];
    uint8_t* dst_scale[kIters];
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      const int r = row_in + (turn * kIters + i) * S::kGroups;
      dst[i] = nullptr;
      dst_scale[i] = nullptr;
#pragma unroll
      for (int j = 0; j < (kFp8 ? 2 : 1); ++j) x[i][j] = make_uint4(0, 0, 0, 0);
      if (r < rows) {
        const int in = r / per_token, rem = r - in * per_token;
        const int which = rem >= c.hkv, h = rem - which * c.hkv;
        if (place[in] >= 0) {
          const uint4* src = reinterpret_cast<const uint4*>((which ? a.v : a.k) + source[in] + h * a.sh);
#pragma unroll
          for (int j = 0; j < (kFp8 ? 2 : 1); ++j) x[i][j] = __ldcs(src + lane * (kFp8 ? 2 : 1) + j);
          dst[i] = (which ? c.v : c.k) + place[in] + h * c.head_sb + lane * 16;
          if constexpr (kFp8)
            dst_scale[i] = (which ? c.v_scale : c.k_scale) + place_scale[in] + (long long)h * c.page_size * kScalesPerRow;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      if constexpr (kFp8) {
        uint32_t byte;
        const uint4 q = quantise16(x[i], byte);
        // the row's four bytes to its first lane
        byte |= __shfl_down_sync(0xffffffffu, byte, 2, 8) << 8;
        byte |= __shfl_down_sync(0xffffffffu, byte, 4, 8) << 16;
        if (dst[i] != nullptr) {
          __stcs(reinterpret_cast<uint4*>(dst[i]), q);
          if (lane == 0) *reinterpret_cast<uint32_t*>(dst_scale[i]) = byte;
        }
      } else {
        if (dst[i] != nullptr) __stcs(reinterpret_cast<uint4*>(dst[i]), x[i][0]);
      }
    }
  }
}

// Rows of a block: token positions [blockIdx.x * kTokens, + kTokens) of sequence blockIdx.y.
constexpr int kReadTokens = 16;
template <bool kFp8>
__global__ void __launch_bounds__(kMoveThreads) kv_cache_read_kernel(const __grid_constant__ CacheMoveArgs a) {
  using S = MoveShape<kFp8>;
  __shared__ long long place[kReadTokens], place_scale[kFp8 ? kReadTokens : 1];
  const PagedView& c = a.c;
  const int b = a.first_seq + blockIdx.y, p0 = blockIdx.x * kReadTokens;
  grid_dependents_launch();
  grid_dependency_wait();
  const PagedSeq seq = paged_seq(c, b, a.max_new, c.max_pages * c.page_size);
  const int len = seq.len;
  if (seq.n < a.min_new) return;
  const int n = min(min(len, a.rows) - p0, kReadTokens);
  if (n <= 0) return;
  if (threadIdx.x < n) {
    const int pos = p0 + threadIdx.x, p = page_index(c, pos), slot = pos - p * c.page_size;
    const int id = c.table[b * c.table_stride + p];
    const bool bad = id < 0 || id >= c.pages;
    if (bad) {
      paged_error(c);
      for (int i = 0; a.zeros && i < 2 * c.hkv * (kHeadDim / 8); ++i) {  // (here, where it costs the loop below nothing)
        const int row = i / (kHeadDim / 8), h = row >> 1;
        reinterpret_cast<uint4*>((row & 1 ? a.v : a.k) + blockIdx.y * a.sb + pos * a.st + h * a.sh)[i % (kHeadDim / 8)] = make_uint4(0, 0, 0, 0);
      }
    }
    place[threadIdx.x] = bad ? -1 : paged_offset(c, id, slot, 0);
    if constexpr (kFp8) place_scale[threadIdx.x] = bad ? 0 : scale_offset(c, id, slot, 0);
  }
  __syncthreads();
  const int group = threadIdx.x / S::kLanes, lane = threadIdx.x % S::kLanes;
  const int per_token = 2 * c.hkv;
#pragma unroll 4
  for (int r = group; r < n * per_token; r += S::kGroups) {
    const int t = r / per_token, rem = r - t * per_token;
    const int which = rem >= c.hkv, h = rem - which * c.hkv;
    if (place[t] < 0) continue;
    const uint4 x = __ldg(reinterpret_cast<const uint4*>((which ? c.v : c.k) + place[t] + h * c.head_sb) + lane);
    uint4* dst = reinterpret_cast<uint4*>((which ? a.v : a.k) + blockIdx.y * a.sb + (p0 + t) * a.st + h * a.sh) + lane * (kFp8 ? 2 : 1);
    if constexpr (kFp8) {
      const uint32_t byte = __ldg((which ? c.v_scale : c.k_scale) + place_scale[t] + (long long)h * c.page_size * kScalesPerRow + lane / 2);
      const uint32_t own = byte > (uint32_t)kMaxScale ? 0x7fc07fc0u : byte == 0 ? 0x00400040u : (byte << 7) * 0x10001u;
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
      uint32_t y[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[2 * i] = mul_bf16x2(f16_bf16(e4m3_f16(w[i])), own);
        y[2 * i + 1] = mul_bf16x2(f16_bf16(e4m3_f16_high(w[i])), own);
      }
      dst[0] = make_uint4(y[0], y[1], y[2], y[3]);
      dst[1] = make_uint4(y[4], y[5], y[6], y[7]);
    } else {
      dst[0] = x;
    }
  }
}

// Rows of 16-byte aligned bf16 tensors with strides in elements.
static bool aligned_rows(const void* p, const void* q, long long sb, long long st, long long sh) {
  return ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q) | (uintptr_t)(sb * 2) | (uintptr_t)(st * 2) |
           (uintptr_t)(sh * 2)) & 15u) == 0;
}

int launch_kv_cache_write(const mb_paged_kv* kv, const void* k_new, const void* v_new, long long sb, long long st,
                          long long sh, cudaStream_t stream) {
  CacheMoveArgs a;
  const int rc = paged_view(kv, &a.c);
  if (rc != MB_SUCCESS) return rc;
  if (a.c.batch == 0 || a.c.tokens == 0) return MB_SUCCESS;
  if (k_new == nullptr || v_new == nullptr || !aligned_rows(k_new, v_new, sb, st, sh)) return MB_E_INVALID;
  a.k = static_cast<uint8_t*>(const_cast<void*>(k_new));
  a.v = static_cast<uint8_t*>(const_cast<void*>(v_new));
  a.sb = sb * 2; a.st = st * 2; a.sh = sh * 2;
  a.rows = a.first_seq = a.min_new = a.max_new = 0;
  a.zeros = false;
  const long long rows = (long long)a.c.tokens * 2 * a.c.hkv;
  const bool fp8 = kv->dtype == MB_DTYPE_E4M3;
  const int groups = fp8 ? MoveShape<true>::kGroups : MoveShape<false>::kGroups;
  const bool many = rows >= 4ll * groups * sm_count();
  const int block = groups * (many ? 4 * (fp8 ? kTurns<true, 4> : kTurns<false, 4>) : 1);
  const long long blocks = (rows + block - 1) / block;
  if (blocks > 0x7fffffffll) return MB_E_INVALID;
  const auto kernel = fp8 ? (many ? kv_cache_write_kernel<true, 4> : kv_cache_write_kernel<true, 1>)
                          : (many ? kv_cache_write_kernel<false, 4> : kv_cache_write_kernel<false, 1>);
  return launch_overlapped("launch kv_cache_write_kernel", kernel, dim3((unsigned)blocks), kMoveThreads, 0, stream, a) ? MB_SUCCESS
                                                                                                               : MB_E_CUDA;
}

static int launch_read(CacheMoveArgs a, bool fp8, int sequences, cudaStream_t stream) {
  constexpr int kMost = 65535;  // of a grid's second dimension
  const auto kernel = fp8 ? kv_cache_read_kernel<true> : kv_cache_read_kernel<false>;
  for (int done = 0; done < sequences; done += kMost) {
    const dim3 grid((a.rows + kReadTokens - 1) / kReadTokens, min(sequences - done, kMost));
    if (!launch_overlapped("launch kv_cache_read_kernel", kernel, grid, kMoveThreads, 0, stream, a)) return MB_E_CUDA;
    a.first_seq += kMost;
    a.k += kMost * a.sb;
    a.v += kMost * a.sb;
  }
  return MB_SUCCESS;
}

int launch_read_e4m3(const PagedAttnArgs& x, int min_new, cudaStream_t stream) {
  CacheMoveArgs a;
  a.c = x.c;
  a.k = reinterpret_cast<uint8_t*>(const_cast<__nv_bfloat16*>(x.packed_k));
  a.v = reinterpret_cast<uint8_t*>(const_cast<__nv_bfloat16*>(x.packed_v));
  a.sh = kHeadDim * 2;
  a.st = a.sh * x.c.hkv;
  a.sb = a.st * x.packed_rows;
  a.rows = x.packed_rows;
  a.first_seq = x.b_begin;
  a.min_new = min_new;
  a.max_new = x.max_queries;
  a.zeros = true;
  return launch_read(a, true, x.b_end - x.b_begin, stream);
}

int launch_kv_cache_read(const mb_paged_kv* kv, void* k_out, void* v_out, long long sb, long long ss, long long sh,
                         int rows, cudaStream_t stream) {
  CacheMoveArgs a;
  const int rc = paged_view(kv, &a.c);
  if (rc != MB_SUCCESS) return rc;
  if (rows < 0 || rows > 0x7fffff00) return MB_E_INVALID;
  if (a.c.batch == 0 || rows == 0) return MB_SUCCESS;
  if (k_out == nullptr || v_out == nullptr || !aligned_rows(k_out, v_out, sb, ss, sh)) return MB_E_INVALID;
  a.k = static_cast<uint8_t*>(k_out);
  a.v = static_cast<uint8_t*>(v_out);
  a.sb = sb * 2; a.st = ss * 2; a.sh = sh * 2;
  a.rows = rows;
  a.first_seq = a.min_new = a.max_new = 0;
  a.zeros = false;
  a.c.cu = nullptr;
  return launch_read(a, kv->dtype == MB_DTYPE_E4M3, a.c.batch, stream);
}

}  // namespace mb
