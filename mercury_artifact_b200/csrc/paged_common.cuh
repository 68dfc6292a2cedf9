// Pieces shared by the kernels over keys and values in pages: the view of a cache, its lookups with their
// bounds checks, and the values that e4m3 codes and scale bytes stand for.
#pragma once

#include "mb_common.cuh"
#include "mb_host.h"

namespace mb {

constexpr int kHeadDim = 128;
constexpr int kScaleBlock = 32;                          // values that share a power of two
constexpr int kScalesPerRow = kHeadDim / kScaleBlock;    // bytes
constexpr int kMinScale = 77, kMaxScale = 191;           // scale bytes as written: 2^-50 .. 2^64
constexpr int kNanScale = 255;

// A cache as the kernels take it.  Strides in bytes.
struct PagedView {
  uint8_t* k;
  uint8_t* v;
  long long page_sb, slot_sb, head_sb;
  uint8_t* k_scale;
  uint8_t* v_scale;
  const int* table;
  long long table_stride;
  const int* seq_lens;
  const int* cu;
  int batch, tokens, per_seq;  // per_seq: new tokens of every sequence where cu is null
  int pages, page_size, page_shift /* log2 of page_size, -1 where it has none */, max_pages, hkv;
  int* status;
};

// New tokens [start, start + n) of a sequence that holds len keys.
struct PagedSeq {
  int start, n, len;
};

__device__ __forceinline__ void paged_error(const PagedView& c) { atomicCAS(c.status, 0, (int)MB_ERR_PAGED); }

// The sequence's lengths, brought into the bounds that the host gave.
__device__ __forceinline__ PagedSeq paged_seq(const PagedView& c, int b, int max_n, int max_len) {
  PagedSeq s;
  int len = c.seq_lens[b];
  if (c.cu != nullptr) {
    int lo = c.cu[b], hi = c.cu[b + 1];
    if (lo < 0 || hi < lo || hi > c.tokens || hi - lo > max_n) {
      paged_error(c);
      lo = min(max(lo, 0), c.tokens);
      hi = min(max(hi, lo), min(c.tokens, lo + max_n));
    }
    s.start = lo;
    s.n = hi - lo;
  } else {
    s.start = 0;
    s.n = c.per_seq;
  }
  if (len < 0 || len > max_len) {
    paged_error(c);
    len = min(max(len, 0), max_len);
  }
  s.len = len;
  return s;
}

// Page and slot of key `pos` (0 <= pos < max_pages * page_size).
__device__ __forceinline__ int page_index(const PagedView& c, int pos) {
  return c.page_shift >= 0 ? pos >> c.page_shift : pos / c.page_size;
}
// Byte offset of head `h` of the key in slot pos - p * page_size of page `id`, and of its scales (scale
// blocks of one head lie slot by slot).
__device__ __forceinline__ long long paged_offset(const PagedView& c, int id, int slot, int h) {
  return id * c.page_sb + slot * c.slot_sb + h * c.head_sb;
}
__device__ __forceinline__ long long scale_offset(const PagedView& c, int id, int slot, int h) {
  return (((long long)id * c.hkv + h) * c.page_size + slot) * kScalesPerRow;
}

// ---- e4m3 codes as bf16 ------------------------------------------------------------------
// The bits of a code, put into the fraction and the low exponent bits of a bf16, stand for its value times 2^-120
// (exponent biases 7 and 127; subnormal codes become subnormal bf16), so that one exact product gives code * 2^n.
// x holds the codes in the high byte of each half.
__device__ __forceinline__ uint32_t e4m3_bits(uint32_t x) { return (x & 0x80008000u) | ((x >> 4) & 0x07f007f0u); }
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// What the products work with is code * 2^(byte - 127 - kScaleBias): the bias keeps the multiplier 2^(byte - 7 -
// kScaleBias) of e4m3_bits a finite bf16 up to kMaxScale, and is taken out of the fp32 results, where it is exact.
constexpr int kScaleBias = 60;
constexpr uint32_t kScaleAdd = 120 - kScaleBias;  // of the exponent field
__device__ __forceinline__ uint32_t scale_mult(uint32_t byte) {  // the multiplier twice
  const uint32_t m = byte > (uint32_t)kMaxScale ? 0x7fc0u : (byte + kScaleAdd) << 7;
  return m | (m << 16);
}

int paged_view(const mb_paged_kv* kv, PagedView* c);

}  // namespace mb
