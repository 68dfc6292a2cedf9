// Attention of few rows over keys and values in pages: single new tokens, drafted tokens.
//
// The rows of a unit are the new tokens of one sequence times the query heads of one K/V head (row = token * group +
// head), in blocks of 8 or 16.  With r rows a key and its value, 512 bytes in bf16, make 512 r operations: up to 16
// rows that is below what HBM's rate asks of the matrix instructions by a factor of ten, so that the kernel is bound by the bytes
// of the cache, and everything else has to stay out of the way of the loads.
//
// One CTA per SM, eight warps, no roles: a warp loads its own keys and values with cp.async into its own three stages
// (16-byte pieces; rows behind the sequence's end are filled with zeros and never read, so that what lies in
// unwritten slots does not matter) and multiplies them with mma.sync: 16 keys (bf16) or 32 (e4m3) a step and warp.  The keys
// are the product's first operand, scores S^T = K Q^T, so that 8 rows of queries fill the instruction; P^T is turned with
// movmatrix and the values are the first operand again, O^T = V^T P^T.  tcgen05 would take scores and
// probabilities through tensor memory and a hand-over between roles for every 128 keys; here a step's operands never leave
// the warp's registers.  Only the end of a unit needs the other warps: their states are merged in shared memory.
//
// A CTA takes one K/V head, of e4m3 two neighbours with four warps each where it can, so that 256 bytes lie in a row.
//
// e4m3: codes are turned into f16, queries too.  Values are multiplied by their powers of two, and with 16 rows keys are; with 8
// the scores of 32 columns at a time are multiplied by the keys', in fp32 (half as many products).  This is exact as long as the powers
// lie close together (see paged_common.cuh).  The loop over steps leaves at the first step where they do not, and a second one goes
// on, with values by way of bf16, keys' and queries' powers in fp32, and P in bf16: 64 tokens against up to 16 384 keys take
// 181 us in the first loop and 226 in the second.  Half of a step's instructions go there.  P is rounded with the values, scores and
// sums are fp32.
//
// The work of a launch is a list of steps (128 keys of one block of rows in bf16, 256 in e4m3), sequence by
// sequence, head by head; every CTA takes an equal, contiguous part, so that lengths need not balance.  The lengths are on
// the device: every CTA finds its part itself (one look at the sequences and a scan).  A unit that lies in
// several CTAs leaves a partial state in each, and paged_merge_kernel joins them in order: results do not depend on timing.
//
// Measured among other calls, one token each of 64 sequences, 32 query and 8 K/V heads, pages of 16: bf16, 50 to 8 192 keys,
// 1.15 GB: 187-195 us, 5.9-6.1 TB/s (a plain copy: 6.5); e4m3, 100 to 16 384 keys, 1.04 GB: 185-199 us, 5.2-5.6 TB/s.  What is left
// of the difference is the start (lengths, page numbers, first rows: a chain of loads) and the merge, some 4 us each, and unequal
// ends.
#include "attn_paged.cuh"

namespace mb {

constexpr int kRowWarps = 8;
constexpr int kRowThreads = 32 * kRowWarps;
constexpr int kRowStages = 3;

template <bool kFp8>
struct RowShape {
  static constexpr int kKeys = kFp8 ? 32 : 16;                     // keys of a warp's stage
  static constexpr int kRowBytes = kFp8 ? kHeadDim : 2 * kHeadDim;
  static constexpr int kPieces = kRowBytes / 16;
  static constexpr int kHalf = kKeys * kRowBytes;                  // K or V of a stage: 4 KiB
  static constexpr int kScaleBytes = kFp8 ? kKeys * kScalesPerRow : 0;
  static constexpr int kStage = 2 * kHalf + 2 * kScaleBytes;
  static_assert(kStage % 256 == 0, "rows are aligned to their size");
};
constexpr int kPitch = 132;  // of the merge buffers' rows, in floats: what the lanes of a warp store falls into different banks

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

struct RowSmem {
  int warp_sum[kRowWarps];
  int b, step;                               // where this CTA's part starts: sequence, and step inside it
  float2 ml[kRowWarps][16];                  // of a unit: every warp's maximum and sum,
  float part_l[kRowWarps][16], row_top[32];  // its sum relative to the rows' maxima, these
  float q_scale[32];     // e4m3: power of two that a row of queries was divided by,
  float q_block[32][4];  // and what its blocks were divided by beside it
};

template <bool kFp8, int kHeads>
constexpr int row_smem_bytes() {
  // queries of 16 rows a head; merge buffers: 32 rows, of as many warps as fit
  return kRowWarps * kRowStages * RowShape<kFp8>::kStage + kHeads * 16 * 2 * kHeadDim + 32 * kPitch * 4 + (int)sizeof(RowSmem);
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// An 8 x 8 matrix of 16-bit values, a row's pairs over four lanes, the other way round.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool kF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A place in the list of steps.  A sequence's units: K/V heads (kHeads neighbours at once), and blocks of kRows rows of each.
struct RowIter {
  int b, h, block, blocks;  // heads / kHeads; block of rows, how many the sequence has
  int step, steps;          // of the unit
  PagedSeq s;
};

template <int kStep>
__device__ __forceinline__ int unit_steps(const PagedAttnArgs& a, const PagedSeq& s) {
  return s.n > 0 && s.n * a.group <= a.few ? (s.len + kStep - 1) / kStep : 0;
}
template <int kRows>
__device__ __forceinline__ int rows_blocks(const PagedAttnArgs& a, const PagedSeq& s) {
  return (s.n * a.group + kRows - 1) / kRows;
}
template <int kStep, int kRows, int kHeads>
__device__ __forceinline__ int sequence_steps(const PagedAttnArgs& a, const PagedSeq& s) {
  const int steps = unit_steps<kStep>(a, s);
  return steps == 0 ? 0 : steps * rows_blocks<kRows>(a, s) * (a.c.hkv / kHeads);
}
template <int kStep, int kRows, int kHeads>
__device__ __forceinline__ void next_unit(const PagedAttnArgs& a, RowIter& it) {
  it.step = 0;
  if (++it.block < it.blocks) return;
  it.block = 0;
  if (++it.h < a.c.hkv / kHeads) return;
  it.h = 0;
  it.steps = 0;
  while (++it.b < a.c.batch) {
    it.s = paged_seq(a.c, it.b, a.max_queries, a.max_keys);
    it.steps = unit_steps<kStep>(a, it.s);
    it.blocks = rows_blocks<kRows>(a, it.s);
    if (it.steps > 0) return;
  }
}
template <int kStep, int kRows, int kHeads>
__device__ __forceinline__ void next_step(const PagedAttnArgs& a, RowIter& it) {
  if (++it.step >= it.steps) next_unit<kStep, kRows, kHeads>(a, it);
}

// Inclusive scan over the block of one value per thread, plus `before`; `all`: the last one's.
__device__ __forceinline__ int row_scan(int mine, int before, int* warp_sum, int& all) {
  int incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, d);
    if ((int)(threadIdx.x & 31) >= d) incl += up;
  }
  if ((threadIdx.x & 31) == 31) warp_sum[threadIdx.x >> 5] = incl;
  __syncthreads();
  int add = before;
  all = before;
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) {
    if (w < (int)(threadIdx.x >> 5)) add += warp_sum[w];
    all += warp_sum[w];
  }
  __syncthreads();
  return incl + add;
}

// CTA i of n takes steps [total * i / n, total * (i + 1) / n).  Short lists use fewer CTAs: at least kMinSteps each.
constexpr int kMinSteps = 2;
__device__ __forceinline__ int row_ctas(int total, int grid) { return max(1, min(grid, total / kMinSteps)); }
__device__ __forceinline__ int row_begin(int total, int i, int n) { return (int)((long long)total * i / n); }

template <bool kFp8, int kTiles, int kHeads>
__global__ void __launch_bounds__(kRowThreads, 1) paged_rows_kernel(const __grid_constant__ PagedAttnArgs a) {
  using S = RowShape<kFp8>;
  constexpr int kWarps = kRowWarps / kHeads;  // of a head
  constexpr int kKeys = S::kKeys, kStep = kWarps * kKeys, kGroups = kKeys / 16, kRows = 8 * kTiles;
  constexpr bool kKeyUnits = kFp8 && kTiles > 1;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int wh = warp / kWarps, wi = warp % kWarps;  // head of this warp, which of its warps it is
  uint8_t* stages = smem_raw + warp * (kRowStages * S::kStage);
  uint8_t* queries = smem_raw + kRowWarps * kRowStages * S::kStage;  // rows of 256 bytes, pieces swapped like the keys'
  float* merge = reinterpret_cast<float*>(queries + kHeads * 16 * 2 * kHeadDim);
  RowSmem* sm = reinterpret_cast<RowSmem*>(merge + 32 * kPitch);
  // e4m3: a step's powers of two: [32 keys][4 blocks] for the keys, [4 blocks][32 keys] in f16 or bf16 for the values; where
  // the states are merged at a unit's end
  float* key_scale = merge + warp * 192;
  uint16_t* value_scale = reinterpret_cast<uint16_t*>(key_scale + 128);
  const uint32_t stage0 = smem_u32(stages);

  grid_dependents_launch();
  grid_dependency_wait();

  // This CTA's part of the list.  A thread looks at every 256th sequence; up to 256 of them are looked at once.
  RowIter in;  // what is loaded next
  int total = 0, ctas = 1, first = 0, last;
  bool empty = false;  // there is a sequence without keys
  if (a.whole) {
    const int most = (a.few + kRows - 1) / kRows;  // blocks of a sequence, at most
    int i = blockIdx.x;
    in.b = i / (a.c.hkv / kHeads * most);
    i -= in.b * (a.c.hkv / kHeads * most);
    in.h = i / most;
    in.block = i - in.h * most;
    in.step = 0;
    in.s = paged_seq(a.c, in.b, a.max_queries, a.max_keys);
    in.blocks = rows_blocks<kRows>(a, in.s);
    in.steps = unit_steps<kStep>(a, in.s);
    last = total = in.block < in.blocks ? in.steps : 0;
    empty = in.steps == 0 && in.h == 0 && in.block == 0;
  } else {
    int mine = 0, incl = 0;
    for (int b0 = 0; b0 < a.c.batch; b0 += kRowThreads) {
      const int b = b0 + tid;
      mine = 0;
      if (b < a.c.batch) {
        const PagedSeq s = paged_seq(a.c, b, a.max_queries, a.max_keys);
        mine = sequence_steps<kStep, kRows, kHeads>(a, s);
        empty |= s.len == 0;
      }
      incl = row_scan(mine, total, sm->warp_sum, total);
    }
    ctas = row_ctas(total, gridDim.x);
    if (tid == 0) a.open[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
    first = row_begin(total, blockIdx.x, ctas);
    last = row_begin(total, blockIdx.x + 1, ctas);
    int before = 0;
    for (int b0 = 0; b0 < a.c.batch; b0 += kRowThreads) {
      const int b = b0 + tid;
      if (a.c.batch > kRowThreads) {
        mine = b < a.c.batch ? sequence_steps<kStep, kRows, kHeads>(a, paged_seq(a.c, b, a.max_queries, a.max_keys)) : 0;
        incl = row_scan(mine, before, sm->warp_sum, before);
      }
      if (first >= incl - mine && first < incl) {
        sm->b = b;
        sm->step = first - (incl - mine);
      }
    }
    empty = __syncthreads_or(empty);
    if ((int)blockIdx.x >= ctas) total = 0;
  }
  // rows of sequences without keys see nothing
  for (int b = a.whole ? in.b : blockIdx.x; empty && b < a.c.batch; b += a.whole ? a.c.batch : gridDim.x) {
    const PagedSeq seq = paged_seq(a.c, b, a.max_queries, a.max_keys);
    if (seq.len > 0 || seq.n * a.group > a.few) continue;
    for (int i = warp; i < seq.n * a.hq; i += kRowWarps) {
      const int tok = seq.start + i / a.hq, hd = i % a.hq;
      *reinterpret_cast<uint2*>(a.o + b * a.o_sb + (long long)tok * a.o_st + (long long)hd * a.o_sh + lane * 4) = make_uint2(0, 0);
      if (lane == 0) a.lse[b * a.lse_sb + hd * a.lse_sh + tok] = -INFINITY;
    }
  }
  if (total == 0) return;
  if (!a.whole) {
    in.b = sm->b;
    in.s = paged_seq(a.c, in.b, a.max_queries, a.max_keys);
    in.steps = unit_steps<kStep>(a, in.s);
    in.blocks = rows_blocks<kRows>(a, in.s);
    const int unit = sm->step / in.steps;
    in.step = sm->step - unit * in.steps;
    in.h = unit / in.blocks;
    in.block = unit - in.h * in.blocks;
  }
  RowIter at = in;  // what is computed next

  // the page table's entry for this lane's key of the step to load, fetched one step ahead
  auto entry_of = [&](const RowIter& it) {
    const int pos = it.step * kStep + wi * kKeys + (lane & (kKeys - 1));
    return pos < it.s.len ? paged_entry(a.c, it.b, pos) : 0;
  };
  int entry = entry_of(in);

  auto load = [&](int stage) {
    const int pos = in.step * kStep + wi * kKeys + (lane & (kKeys - 1));
    const int slot = pos - page_index(a.c, pos) * a.c.page_size;
    const int page = pos < in.s.len ? paged_id(a.c, entry, -1) : -1;
    const int head = in.h * kHeads + wh;
    const long long off = page >= 0 ? paged_offset(a.c, page, slot, head) : -1;
    // Piece p of row r lies at place p ^ (r & 7) of its row.  With r = i * n + r0 (n: rows of a pass, a power of two above
    // r0) that is (p ^ r0) ^ (i * n & 7): one exclusive or with a constant, as rows are aligned to their size.
    constexpr int kPass = 32 / S::kPieces;
    const uint32_t dst = stage0 + stage * S::kStage;
    const uint32_t dst0 = dst + (lane / S::kPieces) * S::kRowBytes + (((lane % S::kPieces) ^ (lane / S::kPieces)) << 4);
    const int piece = lane % S::kPieces;
#pragma unroll
    for (int i = 0; i < kKeys / kPass; ++i) {
      const long long from = __shfl_sync(0xffffffffu, off, i * kPass + lane / S::kPieces);
      const bool real = from >= 0;
      const uint32_t to = (dst0 ^ (((i * kPass) & 7) << 4)) + i * kPass * S::kRowBytes;
      cp_async16(to, real ? a.c.k + from + piece * 16 : a.c.k, real);
      cp_async16(to + S::kHalf, real ? a.c.v + from + piece * 16 : a.c.v, real);
    }
    if constexpr (kFp8) {
      const long long so = page >= 0 ? scale_offset(a.c, page, slot, head) : 0;
      cp_async4(dst + 2 * S::kHalf + lane * 4, a.c.k_scale + so, page >= 0);
      cp_async4(dst + 2 * S::kHalf + S::kScaleBytes + lane * 4, a.c.v_scale + so, page >= 0);
    }
  };

  int to_load = last - first;
#pragma unroll
  for (int i = 0; i < kRowStages - 1; ++i) {
    if (to_load > 0) {
      load(i);
      if (--to_load > 0) {
        next_step<kStep, kRows, kHeads>(a, in);
        entry = entry_of(in);
      }
    }
    cp_async_commit();
  }

  // Queries: the next unit's are fetched into registers while this one's are in use (from shared memory).
  RowIter nx = at;  // the unit behind this one
  constexpr int kPasses = (kHeads * kTiles + 1) / 2;  // sixteen threads have a row, 16 rows at a time
  uint4 qx[kPasses];
  auto fetch_q = [&]() {
#pragma unroll
    for (int m = 0; m < kPasses; ++m) {
      const int at_row = m * 16 + (tid >> 4), h = at_row / kRows, row = nx.block * kRows + at_row % kRows;
      const int tok = row / a.group, hd = row - tok * a.group;
      qx[m] = make_uint4(0, 0, 0, 0);
      if (nx.b < a.c.batch && h < kHeads && row < nx.s.n * a.group)
        qx[m] = __ldg(reinterpret_cast<const uint4*>(a.q + nx.b * a.q_sb + (long long)(nx.s.start + tok) * a.q_st +
                                                     (long long)((nx.h * kHeads + h) * a.group + hd) * a.q_sh) + (tid & 15));
    }
  };
  // A lane of the matrix instruction takes element pairs (2 t, 2 t + 1) and (8 + 2 t, ...) of 16 along head_dim.  Of e4m3 keys
  // it gets four neighbouring values at once, so that its two pairs are 4 t .. 4 t + 3; the queries are put in that order.
  auto store_q = [&]() {
    bool uneven = false;
#pragma unroll
    for (int m = 0; m < kPasses; ++m) {
      const int r = m * 16 + (tid >> 4), piece = tid & 15;
      uint8_t* row = queries + r * 2 * kHeadDim;
      if constexpr (kFp8) {
        float block;
        bool row_uneven;
        const float scale = query_to_f16(qx[m], block, row_uneven);
        uneven |= row_uneven;
        if (piece == 0) sm->q_scale[r] = scale;
        if ((piece & 3) == 0) sm->q_block[r][piece >> 2] = block;
      }
      if constexpr (!kFp8) {
        *reinterpret_cast<uint4*>(row + ((piece ^ (r & 7)) << 4)) = qx[m];
      } else {
        *reinterpret_cast<uint2*>(row + (((piece & 14) ^ (r & 7)) << 4) + (piece & 1) * 8) = make_uint2(qx[m].x, qx[m].z);
        *reinterpret_cast<uint2*>(row + (((piece | 1) ^ (r & 7)) << 4) + (piece & 1) * 8) = make_uint2(qx[m].y, qx[m].w);
      }
    }
    return uneven;
  };
  // Queries of 8 rows as the second operand, for 32 elements along head_dim (two products)
  const uint32_t q_addr = smem_u32(queries) + (wh * kRows + (lane & 7)) * 2 * kHeadDim + (((lane >> 3) ^ (lane & 7)) << 4);
  auto queries_of = [&](uint32_t (&qf)[4], int m, int k2) { ldsm4(qf, (q_addr ^ (k2 << 6)) + m * 8 * 2 * kHeadDim); };

  fetch_q();
  int stage = 0;
  for (int s = first; s < last;) {
    // ---- a unit, or this CTA's part of it: steps [at.step, at.step + unit_end - s)
    const bool from_start = at.step == 0;  // its earlier steps are not another CTA's
    const int unit_end = min(last, s + at.steps - at.step);
    const bool done = unit_end == s + at.steps - at.step;
    bool uneven = store_q();
    next_unit<kStep, kRows, kHeads>(a, nx);
    fetch_q();
    // the queries are there, and the buffers of the unit before are free again
    if constexpr (kFp8) uneven = __syncthreads_or(uneven);
    else __syncthreads();
    float acc[kTiles][8][4], m_ref[kTiles][2], l[kTiles][2];
    int limit[kTiles][2];        // keys that the row sees; the first of the unit's rows sees the fewest
    float c[kTiles][2];          // of its scores; e4m3: with the power of two of the row's queries
    uint32_t qk[kTiles][4][4];
    int unit = 0, key_unit = 0;  // e4m3: acc is in units of 2^(unit - 127), scores of 2^(key_unit - 127) (0: no step yet)
    const int row0 = at.block * kRows, rows = min(at.s.n * a.group - row0, kRows);
    auto factor = [&](int m, int e, float keys) {  // of a row's scores, in units of the exponent of two
      // (not zero and not infinite, with which hidden or zero scores would make no number)
      return kFp8 ? fminf(fmaxf(a.scale_log2 * sm->q_scale[wh * kRows + m * 8 + 2 * t + e] * keys, 1.2e-38f), 3.4e38f) : a.scale_log2;
    };
    const int seen_by_all = a.causal ? at.s.len - at.s.n + row0 / a.group + 1 : at.s.len;
#pragma unroll
    for (int m = 0; m < kTiles; ++m) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[m][j][e] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = m * 8 + 2 * t + e;
        m_ref[m][e] = -INFINITY;
        l[m][e] = 0.f;
        limit[m][e] = a.causal ? min(at.s.len, at.s.len - at.s.n + (row0 + r) / a.group + 1) : at.s.len;
        c[m][e] = factor(m, e, 1.f);
      }
#pragma unroll
      for (int k2 = 0; k2 < 4; ++k2) queries_of(qk[m][k2], m, k2);
    }

    // ---- one step; kWide (e4m3): values by way of bf16, blocks of queries with powers of their own.  False, and nothing done, where
    // the step needs kWide.  (That is asked where the maximum is looked at: a branch of its own before the products cost 3 to 5 %.)
    uint32_t kw = 0, vw = 0;  // e4m3: the powers of two of this lane's key and value
    auto step = [&](auto wide) {
      constexpr bool kWide = decltype(wide)::value, kF16 = kFp8 && !kWide, kKeysF16 = kKeyUnits && !kWide;
      const uint32_t sk = stage0 + stage * S::kStage, sv = sk + S::kHalf;
      const int key0 = at.step * kStep + wi * kKeys;
      float sc[kTiles][kGroups][4];  // of 16 keys each
#pragma unroll
      for (int m = 0; m < kTiles; ++m)
#pragma unroll
        for (int j = 0; j < kGroups; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[m][j][e] = 0.f;
      if constexpr (!kFp8) {
        // four 8 x 8 matrices: keys 0-7 and 8-15 of one 16-byte piece, then of the next
        const uint32_t k_addr = sk + (lane & 15) * S::kRowBytes + (((lane >> 4) ^ (lane & 7)) << 4);
#pragma unroll
        for (int k2 = 0; k2 < 4; ++k2) {
          uint32_t k0[4], k1[4];
          ldsm4(k0, k_addr ^ (k2 << 6));
          ldsm4(k1, k_addr ^ (k2 << 6) ^ 32);
#pragma unroll
          for (int m = 0; m < kTiles; ++m) {
            const uint32_t(&q)[4] = qk[m][k2];
            mma16816<kFp8>(sc[m][0], k0, q[0], q[1]);
            mma16816<kFp8>(sc[m][0], k1, q[2], q[3]);
          }
        }
      } else {
        // Keys are multiplied by their powers of two in f16, or the scores of 32 columns at a time in fp32.
        if constexpr (kKeysF16)
          *reinterpret_cast<uint4*>(key_scale + lane * 4) = unit_f16_pairs(kw, key_unit);
        else
          *reinterpret_cast<float4*>(key_scale + lane * 4) =
              make_float4(scale_value(kw & 0xffu), scale_value((kw >> 8) & 0xffu), scale_value((kw >> 16) & 0xffu), scale_value(kw >> 24));
        if constexpr (kWide) store_unit_bf16(value_scale + lane, vw, unit);
        else store_unit_f16(value_scale + lane, vw, unit);
        __syncwarp();
        // four matrices: the 32 keys x one piece of 16 values, which makes two operands of 16 keys x 16 values
        const uint32_t k_addr = sk + lane * S::kRowBytes + ((lane & 7) << 4);
#pragma unroll
        for (int k2 = 0; k2 < 4; ++k2) {
          float mult[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) mult[j] = key_scale[(j * 8 + g) * 4 + k2];
          uint32_t kf[2][2][4];  // [piece][16 keys]
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t b[4];
            ldsm4(b, k_addr ^ ((2 * k2 + i) << 4));
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              kf[i][j][0] = e4m3_f16(b[2 * j]);
              kf[i][j][1] = e4m3_f16(b[2 * j + 1]);
              kf[i][j][2] = e4m3_f16_high(b[2 * j]);
              kf[i][j][3] = e4m3_f16_high(b[2 * j + 1]);
              if constexpr (kKeysF16) {
#pragma unroll
                for (int e = 0; e < 4; ++e) kf[i][j][e] = mul_f16x2(kf[i][j][e], __float_as_uint(mult[2 * j + (e & 1)]));
              }
            }
          }
#pragma unroll
          for (int m = 0; m < kTiles; ++m) {
            const uint32_t(&q)[4] = qk[m][k2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              if constexpr (kKeysF16) {
                mma16816<kFp8>(sc[m][j], kf[0][j], q[0], q[1]);
                mma16816<kFp8>(sc[m][j], kf[1][j], q[2], q[3]);
                continue;
              }
              float part[4] = {0.f, 0.f, 0.f, 0.f};
              mma16816<kFp8>(part, kf[0][j], q[0], q[1]);
              mma16816<kFp8>(part, kf[1][j], q[2], q[3]);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if constexpr (kWide) part[e] *= sm->q_block[wh * kRows + m * 8 + 2 * t + (e & 1)][k2];
                sc[m][j][e] = fmaf(part[e], mult[2 * j + (e >> 1)], sc[m][j][e]);
              }
            }
          }
        }
      }

      // ---- softmax; a lane holds keys 16 j + g and 16 j + 8 + g of rows 2 t and 2 t + 1 of a tile
      if (key0 + kKeys > seen_by_all) {
#pragma unroll
        for (int m = 0; m < kTiles; ++m)
#pragma unroll
          for (int j = 0; j < kGroups; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key0 + j * 16 + (e >> 1) * 8 + g >= limit[m][e & 1]) sc[m][j][e] = -INFINITY;
      }
      // A row's reference only moves when a score exceeds it by kAhead.  Each lane looks at its own keys, and the row's maximum is
      // only taken when one of them does.
      constexpr float kAhead = kFp8 ? kAheadF16 : 8.f;
      float top[kTiles][2];
      bool need = false;
#pragma unroll
      for (int m = 0; m < kTiles; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(sc[m][0][e], sc[m][0][2 + e]);
          if constexpr (kGroups == 2) x = max3(x, sc[m][kGroups - 1][e], sc[m][kGroups - 1][2 + e]);
          top[m][e] = x == -INFINITY ? -INFINITY : x * c[m][e];
          need |= top[m][e] - m_ref[m][e] > kAhead;
        }
      if constexpr (kF16) need |= outside_unit(vw, unit) || (kKeyUnits && outside_unit(kw, key_unit));
      if (__any_sync(0xffffffffu, need)) {
        if constexpr (kF16) {
          if (__any_sync(0xffffffffu, outside_unit(vw, unit) || (kKeyUnits && outside_unit(kw, key_unit)))) return false;
        }
#pragma unroll
        for (int m = 0; m < kTiles; ++m)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = top[m][e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
            const bool moves = x - m_ref[m][e] > kAhead;
            const float f = moves ? fast_exp2(m_ref[m][e] - x) : 1.f;
            if (moves) m_ref[m][e] = x;
            l[m][e] *= f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              acc[m][j][e] *= f;
              acc[m][j][2 + e] *= f;
            }
          }
      }
      uint32_t pf[kTiles][kGroups][2];  // probabilities as the second operand: [16 keys][rows], keys 0-7 and 8-15
#pragma unroll
      for (int m = 0; m < kTiles; ++m) {
        float lift[2], sum[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 2; ++e) lift[e] = (kFp8 ? kLiftF16 : 0.f) - (m_ref[m][e] == -INFINITY ? 0.f : m_ref[m][e]);
#pragma unroll
        for (int j = 0; j < kGroups; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float p0 = fast_exp2(fmaf(sc[m][j][2 * i], c[m][0], lift[0]));
            const float p1 = fast_exp2(fmaf(sc[m][j][2 * i + 1], c[m][1], lift[1]));
            sum[0] += p0;
            sum[1] += p1;
            pf[m][j][i] = transpose8x8(kF16 ? pack_f16x2(p0, p1) : pack_bf16x2(p0, p1));
          }
#pragma unroll
        for (int e = 0; e < 2; ++e) l[m][e] += sum[e];
      }

      // ---- values, transposed, as the first operand: 16 columns x 16 keys
      if constexpr (!kFp8) {
        // four matrices: two pieces of 8 values of keys 0-7, then of keys 8-15
        const uint32_t v_addr = sv + ((lane & 7) + ((lane >> 4) << 3)) * S::kRowBytes + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t v[4];
          ldsm4_t(v, v_addr ^ (j << 5));
#pragma unroll
          for (int m = 0; m < kTiles; ++m) mma16816<kFp8>(acc[m][j], v, pf[m][0][0], pf[m][0][1]);
        }
      } else {
        // Transposed 16-bit units are pairs of neighbouring values: a lane gets values (2 g, 2 g + 1) of keys (2 t, 2 t + 1) of
        // each 8; the even ones are the product's rows 0-7, the odd ones rows 8-15.
        const uint32_t v_addr = sv + lane * S::kRowBytes + ((lane & 7) << 4);
#pragma unroll
        for (int j2 = 0; j2 < 4; ++j2) {
          uint32_t mult[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) mult[i] = *reinterpret_cast<const uint32_t*>(value_scale + j2 * kKeys + i * 8 + 2 * t);
#pragma unroll
          for (int j = 2 * j2; j < 2 * j2 + 2; ++j) {
            uint32_t b[4];
            ldsm4_t(b, v_addr ^ (j << 4));
            uint32_t v[2][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t x = __byte_perm(b[i], 0, 0x3120);  // the even ones of both keys, then the odd ones
              const uint32_t even = e4m3_f16(x), odd = e4m3_f16_high(x);
              v[i >> 1][(i & 1) * 2] = kF16 ? mul_f16x2(even, mult[i]) : mul_bf16x2(f16_bf16(even), mult[i]);
              v[i >> 1][(i & 1) * 2 + 1] = kF16 ? mul_f16x2(odd, mult[i]) : mul_bf16x2(f16_bf16(odd), mult[i]);
            }
#pragma unroll
            for (int m = 0; m < kTiles; ++m) {
              mma16816<kF16>(acc[m][j], v[0], pf[m][0][0], pf[m][0][1]);
              mma16816<kF16>(acc[m][j], v[1], pf[m][kGroups - 1][0], pf[m][kGroups - 1][1]);
            }
          }
        }
      }
      __syncwarp();
      stage = stage + 1 == kRowStages ? 0 : stage + 1;
      return true;
    };
    auto fetch = [&]() {  // keeps the loads going, and waits for the step's own
      if (to_load > 0) {
        load(stage == 0 ? kRowStages - 1 : stage - 1);
        if (--to_load > 0) {
          next_step<kStep, kRows, kHeads>(a, in);
          entry = entry_of(in);
        }
      }
      cp_async_commit();
      cp_async_wait<kRowStages - 1>();
      __syncwarp();
      if constexpr (kFp8) {  // (behind the sequence's end: of no effect on the unit, and a number)
        const uint32_t* words = reinterpret_cast<const uint32_t*>(stages + stage * S::kStage + 2 * S::kHalf);
        const bool real = at.step * kStep + wi * kKeys + lane < at.s.len;
        kw = real ? words[lane] : key_unit * 0x01010101u;
        vw = real ? words[kKeys + lane] : unit * 0x01010101u;
      }
    };
    fetch();
    if constexpr (kFp8) {  // the units, by the first step
      const bool real = at.step * kStep + wi * kKeys + lane < at.s.len;
      unit = max((int)__reduce_max_sync(0xffffffffu, scale_top(vw)), kLeastUnit);
      if (!real) vw = unit * 0x01010101u;
      if constexpr (kKeyUnits) {
        key_unit = max((int)__reduce_max_sync(0xffffffffu, scale_top(kw)), kMinScale);
        if (!real) kw = key_unit * 0x01010101u;
#pragma unroll
        for (int m = 0; m < kTiles; ++m)
#pragma unroll
          for (int e = 0; e < 2; ++e) c[m][e] = factor(m, e, exp2_int(key_unit - 127));
      }
    }
    bool more = true;
    if (!kFp8 || !uneven) {
#pragma unroll 1
      while (step(No{})) {
        ++s;
        ++at.step;
        more = s < unit_end;
        if (!more) break;
        fetch();
      }
    }
    if (kFp8 && more) {
      if constexpr (kKeyUnits) {
#pragma unroll
        for (int m = 0; m < kTiles; ++m)
#pragma unroll
          for (int e = 0; e < 2; ++e) c[m][e] = factor(m, e, 1.f);
      }
#pragma unroll 1
      while (true) {
        const int most = (int)__reduce_max_sync(0xffffffffu, scale_top(vw));
        if (most > unit + kAboveUnit) {
          const float f = unit - most < -126 ? 0.f : exp2_int(unit - most);
#pragma unroll
          for (int m = 0; m < kTiles; ++m)
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[m][j][e] *= f;
          unit = most;
        }
        step(Yes{});
        ++s;
        ++at.step;
        if (s == unit_end) break;
        fetch();
      }
    }

    // ---- the warps' states become one: through as many buffers as fit, in turns where these are fewer than warps
#pragma unroll
    for (int m = 0; m < kTiles; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if constexpr (kFp8) m_ref[m][e] -= kLiftF16;
        float x = l[m][e];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
        if (g == 0) sm->ml[warp][m * 8 + 2 * t + e] = make_float2(m_ref[m][e], x);
      }
    __syncthreads();
    float f[kTiles][2];
#pragma unroll
    for (int m = 0; m < kTiles; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = m * 8 + 2 * t + e;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm->ml[wh * kWarps + w][r].x);
        f[m][e] = m_ref[m][e] == -INFINITY ? 0.f : fast_exp2(m_ref[m][e] - top);
        // a warp without a visible key has nothing, whatever its masked products gave
        const float mine = sm->ml[warp][r].y;
        if (m_ref[m][e] == -INFINITY && mine == mine) {
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[m][j][e] = acc[m][j][2 + e] = 0.f;
        }
        // (from here on: the row's maximum, and the warp's sum relative to it)
        if (g == 0) sm->part_l[warp][r] = m_ref[m][e] == -INFINITY ? mine : mine * f[m][e];
        if (g == 0 && wi == 0) sm->row_top[wh * kRows + r] = top;
        if constexpr (kFp8) f[m][e] *= exp2_int(unit - 127);
      }
    const int buffers = (rows <= 4 ? 8 : 4 / kTiles) / kHeads;  // of a head
    const int pitch = rows <= 4 ? 4 * kPitch : kRows * kPitch;
#pragma unroll 1
    for (int round = 0; round < kWarps; round += buffers) {
      if (wi >= round && wi < round + buffers) {
        float* buf = merge + (wh * buffers + wi - round) * pitch;
#pragma unroll
        for (int m = 0; m < kTiles; ++m)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = m * 8 + 2 * t + e;
            if (r < rows) {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                // columns 16 j + g and 16 j + 8 + g; e4m3: 16 j + 2 g and the next
                float* p = buf + r * kPitch + j * 16 + (kFp8 ? 2 * g : g);
                float x0 = acc[m][j][e] * f[m][e], x1 = acc[m][j][2 + e] * f[m][e];
                if (round > 0) {
                  x0 += p[0];
                  x1 += p[kFp8 ? 1 : 8];
                }
                p[0] = x0;
                p[kFp8 ? 1 : 8] = x1;
              }
            }
          }
      }
      __syncthreads();
    }
    const bool whole = from_start && done;
    const int slot = 2 * blockIdx.x + (from_start ? 1 : 0);
    for (int i = warp; i < kHeads * rows; i += kRowWarps) {
      const int h = kHeads == 1 ? 0 : i / rows, r = i - h * rows;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += sm->part_l[h * kWarps + w][r];
      const float top = sm->row_top[h * kRows + r];
      const float* buf = merge + h * buffers * pitch + r * kPitch + lane * 4;
      float4 x = *reinterpret_cast<const float4*>(buf);
      for (int b = 1; b < buffers; ++b) {
        const float4 y = *reinterpret_cast<const float4*>(buf + b * pitch);
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
      }
      if (whole) {
        const int tok = (row0 + r) / a.group, hd = (at.h * kHeads + h) * a.group + row0 + r - tok * a.group;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const uint2 w = make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
        *reinterpret_cast<uint2*>(a.o + at.b * a.o_sb + (long long)(at.s.start + tok) * a.o_st + (long long)hd * a.o_sh + lane * 4) = w;
        if (lane == 0)
          a.lse[at.b * a.lse_sb + hd * a.lse_sh + at.s.start + tok] = sum == 0.f ? -INFINITY : top * kLn2 + __logf(sum);
      } else {
        const long long to = ((long long)slot * kHeads + h) * kRows + r;
        *reinterpret_cast<float4*>(a.part_o + to * kHeadDim + lane * 4) = x;
        if (lane == 0) a.part_ml[to] = make_float2(top, sum);
      }
    }
    if (from_start && !done && tid == 0) {
      // the unit goes on in the next CTAs: how many of them it takes
      const int end = s + at.steps - at.step;  // behind its last step
      int n = 1;
      while (row_begin(total, blockIdx.x + n, ctas) < end) ++n;
      a.open[2 * blockIdx.x] = make_int4(at.b, at.h, n, at.block);
      a.open[2 * blockIdx.x + 1] = make_int4(at.s.start, rows, 0, 0);
    }
    at = nx;
  }
}

// Joins the partial states of the unit that CTA blockIdx.x of the launch before began and did not finish (if there is one):
// four rows of a head a block, two warps a row, each every other part; a lane has four columns.  The parts are added in order.
// Bound by latency: the first parts are fetched before the maximum is known.
constexpr int kMergeRows = 4, kMergeAhead = 4;
template <int kRows, int kHeads>
__global__ void __launch_bounds__(64 * kMergeRows) paged_merge_kernel(const __grid_constant__ PagedAttnArgs a) {
  __shared__ float4 part[kMergeRows][32];
  __shared__ float part_l[kMergeRows];
  const int row = threadIdx.x >> 6, odd = (threadIdx.x >> 5) & 1, lane = threadIdx.x & 31;
  grid_dependents_launch();
  grid_dependency_wait();
  const int4 unit = a.open[2 * blockIdx.x], more = a.open[2 * blockIdx.x + 1];
  const int n = unit.z, rows = more.y;
  if (n == 0) return;
  const int groups = gridDim.y / kHeads, h = blockIdx.y / groups, r = (blockIdx.y - h * groups) * kMergeRows + row;
  const bool real = r < rows;
  float sum = 0.f, top = -INFINITY;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (real) {
    // row of the unit's p-th CTA: it ends the list of the first one and starts those of the others
    auto slot = [&](int p) { return ((long long)(2 * (blockIdx.x + p) + (p == 0 ? 1 : 0)) * kHeads + h) * kRows + r; };
    auto state = [&](int p) { return a.part_ml[slot(p)]; };
    auto values = [&](int p) { return *reinterpret_cast<const float4*>(a.part_o + slot(p) * kHeadDim + lane * 4); };
    auto add = [&](const float2& ml, const float4& y) {
      // (a part without visible keys holds zeros, or what is not a number)
      const float w = ml.x == -INFINITY ? 1.f : fast_exp2(ml.x - top);
      sum = fmaf(w, ml.y, sum);
      x.x = fmaf(w, y.x, x.x);
      x.y = fmaf(w, y.y, x.y);
      x.z = fmaf(w, y.z, x.z);
      x.w = fmaf(w, y.w, x.w);
    };
    float2 ml[kMergeAhead];
    float4 y[kMergeAhead];
#pragma unroll
    for (int i = 0; i < kMergeAhead; ++i) {
      const int p = min(odd + 2 * i, n - 1);
      ml[i] = state(p);
      y[i] = values(p);
    }
    for (int p = lane; p < n; p += 32) top = fmaxf(top, state(p).x);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
#pragma unroll
    for (int i = 0; i < kMergeAhead; ++i)
      if (odd + 2 * i < n) add(ml[i], y[i]);
#pragma unroll 4
    for (int p = odd + 2 * kMergeAhead; p < n; p += 2) add(state(p), values(p));
    if (odd) {
      part[row][lane] = x;
      if (lane == 0) part_l[row] = sum;
    }
  }
  __syncthreads();
  if (!real || odd) return;
  const float4 y = part[row][lane];
  sum += part_l[row];
  const int first = unit.w * kRows + r, tok = first / a.group, hd = (unit.y * kHeads + h) * a.group + first - tok * a.group;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const uint2 w = make_uint2(pack_bf16x2((x.x + y.x) * inv, (x.y + y.y) * inv), pack_bf16x2((x.z + y.z) * inv, (x.w + y.w) * inv));
  *reinterpret_cast<uint2*>(a.o + unit.x * a.o_sb + (long long)(more.x + tok) * a.o_st + (long long)hd * a.o_sh + lane * 4) = w;
  if (lane == 0) a.lse[unit.x * a.lse_sb + hd * a.lse_sh + more.x + tok] = sum == 0.f ? -INFINITY : top * kLn2 + __logf(sum);
}

int paged_rows_step(bool fp8) { return kRowWarps * (fp8 ? RowShape<true>::kKeys : RowShape<false>::kKeys); }

// Rows of a block, for which the kernel is compiled
int paged_rows_padded(int rows) { return rows <= 8 ? 8 : 16; }

long long paged_rows_slots(int rows, int heads, int ctas) { return 2ll * ctas * heads * paged_rows_padded(rows); }
long long paged_rows_workspace(int rows, int heads, int ctas) {
  return paged_rows_slots(rows, heads, ctas) * (kHeadDim * (long long)sizeof(float) + (long long)sizeof(float2)) +
         2ll * ctas * (long long)sizeof(int4);
}

template <bool kFp8, int kTiles, int kHeads>
static int launch_rows(const PagedAttnArgs& a, int ctas, cudaStream_t stream) {
  static bool attr_set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return MB_E_CUDA;
  constexpr int bytes = row_smem_bytes<kFp8, kHeads>();
  static_assert(bytes <= 232448, "shared memory budget of one CTA");
  const auto kernel = paged_rows_kernel<kFp8, kTiles, kHeads>;
  if (!attr_set[dev]) {
    if (!cuda_ok(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "paged_rows_kernel shared memory"))
      return MB_E_CUDA;
    attr_set[dev] = true;
  }
  return launch_overlapped("launch paged_rows_kernel", kernel, dim3(ctas), kRowThreads, bytes, stream, a) ? MB_SUCCESS : MB_E_CUDA;
}

int launch_paged_rows(const PagedAttnArgs& a, bool fp8, int rows, int heads, int ctas, cudaStream_t stream) {
  const bool one = paged_rows_padded(rows) == 8;
  if (!fp8) return one ? launch_rows<false, 1, 1>(a, ctas, stream) : launch_rows<false, 2, 1>(a, ctas, stream);
  if (heads == 1) return one ? launch_rows<true, 1, 1>(a, ctas, stream) : launch_rows<true, 2, 1>(a, ctas, stream);
  return one ? launch_rows<true, 1, 2>(a, ctas, stream) : launch_rows<true, 2, 2>(a, ctas, stream);
}

int launch_paged_rows_merge(const PagedAttnArgs& a, int rows, int heads, int ctas, cudaStream_t stream) {
  const int block = paged_rows_padded(rows);
  const auto kernel = block == 8 ? (heads == 1 ? paged_merge_kernel<8, 1> : paged_merge_kernel<8, 2>)
                                 : (heads == 1 ? paged_merge_kernel<16, 1> : paged_merge_kernel<16, 2>);
  const dim3 grid(ctas, heads * ((min(rows, block) + kMergeRows - 1) / kMergeRows));
  return launch_overlapped("launch paged_merge_kernel", kernel, grid, 64 * kMergeRows, 0, stream, a) ? MB_SUCCESS : MB_E_CUDA;
}

}  // namespace mb
