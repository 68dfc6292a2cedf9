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
// The table's entry for key `pos` of sequence b as it is; paged_id checks it.  (Entries are fetched ahead, and the check
// would wait for them.)
__device__ __forceinline__ int paged_entry(const PagedView& c, int b, int pos) {
  return c.table[b * c.table_stride + page_index(c, pos)];
}
// `entry` if it is a page, else `none`, and an error.
__device__ __forceinline__ int paged_id(const PagedView& c, int entry, int none) {
  if (entry >= 0 && entry < c.pages) return entry;
  paged_error(c);
  return none;
}
// Byte offset of head `h` of the key in slot pos - p * page_size of page `id`, and of its scales (scale
// blocks of one head lie slot by slot).
__device__ __forceinline__ long long paged_offset(const PagedView& c, int id, int slot, int h) {
  return id * c.page_sb + slot * c.slot_sb + h * c.head_sb;
}
__device__ __forceinline__ long long scale_offset(const PagedView& c, int id, int slot, int h) {
  return (((long long)id * c.hkv + h) * c.page_size + slot) * kScalesPerRow;
}

// ---- e4m3 codes as f16 and bf16 ------------------------------------------------------------
// Both hold every code as it is, and a code times a power of two is exact in bf16 (down to its least value, 2^-133).
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t f16_bf16(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\t.reg .f32 x, y;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.f32.f16 x, lo;\n\tcvt.f32.f16 y, hi;\n\t"
      "cvt.rn.bf16x2.f32 %0, y, x;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
// The kernel for few rows adds values in f16 where it can: code * 2^(n - U), with U the largest exponent of the first values that
// a warp sees of a unit.  With n - U in [-kBelowUnit, kAboveUnit] the products are exact (2^-9 * 2^-11 to 448 * 2^4, of f16's 2^-24 to
// 65504).  From the first step on that holds another n, for whatever row or column, the warp goes on in bf16, where a code
// times a power of two is exact for every n; U, which is the unit of the fp32 sums, then rises with the largest n.
// Keys that are multiplied in f16 have a U of their own and the same range; else scores are multiplied by 2^n in fp32.
// Probabilities go with the values.  f16: multiplied by 2^kLiftF16, so that the largest lies between 2^11 and 2^15 (a row's
// reference moves when a score is kAheadF16 above it).  They are rounded by 2^-11 down to 2^-25 of the largest, below that by no
// more than 2^-36 of it, against values whose blocks' largest are no more than 2^16 apart.  (Going back to f16 after other
// values would end that: small probabilities of large values would be measured by large probabilities of small ones.)
// bf16: rounded by 2^-8, whatever their size.
// (One conversion for two codes and one product; putting a code's bits into a bf16 instead takes four integer instructions at
// half rate: 64 tokens against up to 16 384 keys of 8 heads took 302 us with those and 238 without, all else alike.)
__device__ __forceinline__ uint32_t e4m3_f16(uint32_t two) {  // the two low bytes
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_f16_high(uint32_t two) {  // the two high bytes
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
constexpr int kBelowUnit = 11, kAboveUnit = 4;
constexpr int kLeastUnit = 17;  // 2^-110
constexpr float kAheadF16 = 4.f, kLiftF16 = 11.f;
// Whether one of four scale bytes lies outside the unit's range (or beyond the written one).
__device__ __forceinline__ bool outside_unit(uint32_t w, int unit) {
  const uint32_t even = w & 0x00ff00ffu, odd = (w >> 8) & 0x00ff00ffu;
  const uint32_t high = min(unit + kAboveUnit, kMaxScale) * 0x10001u, low = (unit - kBelowUnit) * 0x10001u;
  // (a difference below zero sets its half's top bit; what it borrows from the other half can only do the same there)
  return ((high - __vmaxu2(even, odd)) | (__vminu2(even, odd) - low)) & 0x80008000u;
}
// 2^(byte - unit) of a word's four bytes, to places 32 apart: in f16 for bytes inside the range,
__device__ __forceinline__ void store_unit_f16(uint16_t* to, uint32_t w, int unit) {
  const uint32_t bias = (uint32_t)(15 - unit) * 0x10001u;
  const uint32_t even = ((w & 0x00ff00ffu) + bias) << 10, odd = (((w >> 8) & 0x00ff00ffu) + bias) << 10;
  to[0] = (uint16_t)even;
  to[32] = (uint16_t)odd;
  to[64] = (uint16_t)(even >> 16);
  to[96] = (uint16_t)(odd >> 16);
}
// or twice each in a word of their own,
__device__ __forceinline__ uint4 unit_f16_pairs(uint32_t w, int unit) {
  const uint32_t bias = (uint32_t)(15 - unit) * 0x10001u;
  const uint32_t even = ((w & 0x00ff00ffu) + bias) << 10, odd = (((w >> 8) & 0x00ff00ffu) + bias) << 10;
  return make_uint4(__byte_perm(even, 0, 0x1010), __byte_perm(odd, 0, 0x1010), __byte_perm(even, 0, 0x3232), __byte_perm(odd, 0, 0x3232));
}
// in bf16 for any (zero below 2^-133; beyond the written range: not a number).
__device__ __forceinline__ void store_unit_bf16(uint16_t* to, uint32_t w, int unit) {
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const int byte = (w >> (8 * b)) & 0xffu, e = byte - unit + 127;
    to[32 * b] = (uint16_t)(byte > kMaxScale ? 0x7fc0 : e > 0 ? e << 7 : 0x80 >> min(1 - e, 15));
  }
}
// 2^(byte - 127); bytes beyond the written range: not a number.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return byte > (uint32_t)kMaxScale ? __int_as_float(0x7fc00000) : __int_as_float(max((int)(byte << 23), 0x00400000));
}
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
// The largest of four scale bytes, those beyond the written range left out.
__device__ __forceinline__ uint32_t scale_top(uint32_t w) {
  const uint32_t beyond = w & (w << 1) & 0x80808080u;
  w &= ~((beyond >> 7) * 0xffu);
  const uint32_t m = __vmaxu2(w & 0x00ff00ffu, (w >> 8) & 0x00ff00ffu);
  return max(m & 0xffffu, m >> 16);
}

// A row of 16 lanes' queries, eight bf16 values each, as f16 times a power of two, which is returned: the largest lies in [2^15,
// 2^16), so that f16 holds every value down to 2^-32 of it as it is.  A row with smaller ones is `uneven`: each block of 32
// has a power of its own, `block` times that of the row (else 1).
__device__ __forceinline__ float query_to_f16(uint4& x, float& block, bool& uneven) {
  uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t hi = 0, lo = 0x7fff7fffu;  // |x| of bf16 orders like its bits; the least one that is not zero
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t v = w[i] & 0x7fff7fffu;
    hi = __vmaxu2(hi, v);
    lo = __vminu2(lo, v | (__vcmpeq2(v, 0) & 0x7fff7fffu));
  }
  hi = max(hi & 0xffffu, hi >> 16);
  lo = min(lo & 0xffffu, lo >> 16);
  uint32_t both = hi << 16 | (0x7fffu - lo);  // (the two go through the lanes together)
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) {
    both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, d));
    if (d == 2) hi = both >> 16;
  }
  const uint32_t own = hi;  // of the block
  hi = both >> 16;
  lo = 0x7fffu - (both & 0xffffu);
  auto exponent = [](uint32_t most) { return min(max((int)(most >> 7) - 142, -126), 111); };
  const int row = exponent(hi);
  uneven = hi != 0 && (int)(hi >> 7) - (int)(lo >> 7) > 25;  // (7 bits less: bf16's subnormals have them)
  const int e = uneven ? max(exponent(own), row - 126) : row;
  block = exp2_int(e - row);
  const float inv = exp2_int(-e);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = pack_f16x2(__uint_as_float(w[i] << 16) * inv, __uint_as_float(w[i] & 0xffff0000u) * inv);
  x = make_uint4(w[0], w[1], w[2], w[3]);
  return exp2_int(row);
}

// ---- 16 or 4 bytes into shared memory, zeros where they are not real --------------------------
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(real ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All copies of this thread, in groups or not (a group's wait does not wait for copies that no group has).
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

int paged_view(const mb_paged_kv* kv, PagedView* c);

}  // namespace mb
