// Attention of many rows over keys and values in pages: chunks of a prompt, cross attention.
//
// The rows of a unit are the new tokens of one sequence times the query heads of one K/V head (row = token * group +
// head): the heads of a group share every key and value that is loaded.  One CTA owns two tiles of 128 rows and
// streams tiles of 128 keys through them, like attn_fwd_kernel, whose tensor-memory layout and hand-overs it has: scores
// S = Q K^T by tcgen05 into one score region that the two query tiles use in turn, online softmax with one thread
// per row, probabilities in bf16 as the tensor-memory operand of O += P V.
//
// What differs is how keys and values arrive.  A page may end anywhere inside a tile, pages lie anywhere, and
// the slots behind a sequence's end hold anything (values that are not numbers among it).  Two ways:
//   kBoxes   bf16, pages of a multiple of 8 slots: TMA boxes of the largest power of two of slots that divides a page; boxes
//            behind the end are fetched from behind the last page, which fills in zeros, and the rows of the
//            last box that lie behind the end are cleared before the values are used (hidden scores are replaced anyway).
//            Lanes issue one after the other, some 55 cycles a box, so that two warps share them, and four where boxes
//            have fewer than 64 slots (kSmallBoxes; 512 threads, whose softmax warps have fewer registers).
//            2 048 tokens against 32 768 keys, 32/8 heads, with two warps and with four, in a short burst (attn_fwd over
//            contiguous keys: 808; under the power limit 947, pages of 64): pages of 64 840 and 858 us, of 32 960 and 844, of
//            16 1 120 and 965, of 8 1 347 and 1 110.
//   kRows    bf16, other pages: four more warps gather row by row with cp.async, 16 bytes a piece, straight into the
//            swizzled layout that tcgen05 reads: the same with pages of 17 takes 1 094 us.
// Codes (e4m3) are brought into bf16 before, into a buffer where every sequence is one page (launch_read_e4m3): 820 us for the
// same tokens.  Turning them on their way into shared memory instead, by four more warps, took 1 354 us, because the tiles
// then stall on the conversion's instructions; with 128 tokens against 8 192 keys 141 us where the copy and the tiles take 115.
// (Only one block of rows per sequence gained: 64 tokens 89 us, 99 by the copy.)
//
//   warps 0-3   softmax + epilogue of query tile 0 (one thread per row)
//   warps 4-7   softmax + epilogue of query tile 1; warps 0-7 also gather the queries
//   warp  8     issues Q K^T, owns tensor memory;  warp 10 issues P V;  warps 9 and 11 issue TMA (kSmallBoxes: 12 and 13 too)
//   warps 12-15 gather keys and values (kRows)
//
// A launch has one CTA per (sequence, 256 rows, K/V head, share of the keys), found on the device from the lengths that
// are there; CTAs beyond the last of them return.  Shares leave their unnormalised rows, maxima and sums in
// the workspace and paged_tiles_merge_kernel joins them in order.
//
// Bound by the tensor cores and, as in attn_fwd, by the exponentials beside them: a step of 128 keys takes an SM some 1.9 us.
// Unequal sequences cost more than that: 16 e4m3 sequences, 5 of them chunks of up to 512 tokens, up to 8 192 keys, take
// 172 us, of which the longest unit's 64 steps are 118.  Choosing the shares on the device by the lengths that are there was
// built: 187 us where this took 170, as smaller shares only bring the tiles to 105-110 us and cost a launch.
#include "attn_paged.cuh"
#include "attn_fwd_common.cuh"

namespace mb {

enum TileMode { kBoxes, kSmallBoxes, kRows };

// Threads; registers at launch, of the softmax warps and of the others (an increase beyond what the CTA was launched with
// would block forever, hence the check).
template <int kMode>
struct TileShape {
  static constexpr int kThreads = kMode == kBoxes ? 384 : 512;
  static constexpr int kLaunch = kMode == kBoxes ? 160 : 128;
  static constexpr int kSoftmax = kMode == kBoxes ? 216 : 208, kOthers = 48;
  static_assert(256 * kSoftmax + (kThreads - 256) * kOthers <= kThreads * kLaunch, "more registers than the CTA is launched with");
};
constexpr int kTileStages = 4;  // of 32 KiB: a tile of keys or values
template <int kRegs>
__device__ __forceinline__ void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}

struct TileMaps {
  CUtensorMap k, v;
  int box;     // slots of a box
  int pages;   // behind the last one
  int packed;  // a page is all of a sequence
};

struct TileSmem {
  uint64_t q_full, kv_full[4], kv_empty[4], s_full[2], s_free, p_full[2][2], o_full[2], drain, tail;
  uint32_t tmem_base;
  int abort_word;
  int valid;                // this CTA has an item
  int b, h, block, part, parts;
  PagedSeq seq;
  int first, last[2];       // tiles of 128 keys: [first, last[i]) of query tile i
  alignas(16) long long off[3][kBN];       // byte offsets of a tile's rows in k and v (-1: zeros)
};

constexpr int tile_smem_bytes() {
  return (2 + kTileStages) * kTileBytes + 1024 /* alignment */ + (int)sizeof(TileSmem);
}
static_assert(tile_smem_bytes() <= 232448, "shared memory budget of one CTA");

__device__ __forceinline__ int tiles_of(int keys) { return (keys + kBN - 1) / kBN; }

// Tiles that rows up to `row` (inclusive) of a sequence see.
__device__ __forceinline__ int visible_keys(const PagedAttnArgs& a, const PagedSeq& s, int row) {
  return a.causal ? min(s.len, max(0, s.len - s.n + row / a.group + 1)) : s.len;
}
// Blocks of 256 rows of a sequence, and shares of the keys of each of its units.
__device__ __forceinline__ int row_blocks(const PagedAttnArgs& a, const PagedSeq& s) {
  const int rows = s.n * a.group;
  return rows > a.few ? (rows + 2 * kBM - 1) / (2 * kBM) : 0;
}
__device__ __forceinline__ int key_shares(const PagedAttnArgs& a, const PagedSeq& s) {
  return max(1, (tiles_of(s.len) + a.share_tiles - 1) / a.share_tiles);
}

// The item of this CTA: sequences one after the other, up to 32 of them the longest first (then short units fill the end: 8
// sequences of 100 to 448 tokens, 200 to 1 500 keys, 16 heads: 36.3 us, 38.8 in their own order); inside one, blocks of heads
// whose keys and values fit a part of L2, in such a block the row blocks from the last (longest) to the first, then
// heads, then shares.  (One warp.)
__device__ __forceinline__ void find_item(const PagedAttnArgs& a, TileSmem* ctl, int lane) {
  int before = 0, found = 0;
  const int want = blockIdx.x, sequences = a.b_end - a.b_begin;
  for (int b0 = a.b_begin; b0 < a.b_end && !found; b0 += 32) {
    const int b = b0 + lane;
    PagedSeq s{0, 0, 0};
    int items = 0;
    if (b < a.b_end) {
      s = paged_seq(a.c, b, a.max_queries, a.max_keys);
      items = row_blocks(a, s) * a.c.hkv * key_shares(a, s);
    }
    int incl = items;
    if (sequences <= 32) {
      incl = 0;
      for (int i = 0; i < sequences; ++i) {
        const int theirs = __shfl_sync(0xffffffffu, items, i), len = __shfl_sync(0xffffffffu, s.len, i);
        if (len > s.len || (len == s.len && i <= lane)) incl += theirs;
      }
    } else {
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += up;
      }
      incl += before;
    }
    const bool mine = want < incl && want >= incl - items;
    if (mine) {
      const int shares = key_shares(a, s), blocks = row_blocks(a, s);
      int i = want - (incl - items);
      ctl->part = i % shares;
      i /= shares;
      const long long head_bytes = max(1ll, (long long)s.len * (4 * kHeadDim));
      const int fit = (int)min((long long)a.c.hkv, max(1ll, (48ll << 20) / head_bytes));
      const int hb = (a.c.hkv + (a.c.hkv + fit - 1) / fit - 1) / ((a.c.hkv + fit - 1) / fit);  // equal blocks
      const int group = i / (hb * blocks), rem = i - group * hb * blocks;
      const int n = min(hb, a.c.hkv - group * hb);
      ctl->b = b;
      ctl->h = group * hb + rem % n;
      ctl->block = blocks - 1 - rem / n;
      ctl->parts = shares;
      ctl->seq = s;
    }
    found = __any_sync(0xffffffffu, mine);
    before = __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) ctl->valid = found;
}

template <int kMode>
__global__ void __maxnreg__(TileShape<kMode>::kLaunch)
paged_tiles_kernel(const __grid_constant__ TileMaps maps, const __grid_constant__ PagedAttnArgs a) {
  using Shape = TileShape<kMode>;
  constexpr int kStages = kTileStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + 2 * kTileBytes;
  TileSmem* ctl = reinterpret_cast<TileSmem*>(sKV + kStages * kTileBytes);
  volatile int* abort_word = &ctl->abort_word;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  grid_dependency_wait();
  grid_dependents_launch();
  if (warp == 0) {
    find_item(a, ctl, lane);
    __syncwarp();
    if (lane == 0) {
      if (ctl->valid) {
        const PagedSeq s = ctl->seq;
        const int rows = s.n * a.group, row0 = ctl->block * 2 * kBM;
        int n[2];
        for (int i = 0; i < 2; ++i)
          n[i] = row0 + i * kBM < rows ? tiles_of(visible_keys(a, s, min(row0 + (i + 1) * kBM, rows) - 1)) : 0;
        const long long all = max(n[0], n[1]);
        ctl->first = (int)(all * ctl->part / ctl->parts);
        const int end = (int)(all * (ctl->part + 1) / ctl->parts);
        ctl->last[0] = min(n[0], end);
        ctl->last[1] = min(n[1], end);
      }
      // the merge finds a split unit at the CTA of its first share (offsets that do not ascend may ask for more CTAs than
      // there are: what the last of them begin is left out)
      if (a.tile_open != nullptr)
        a.tile_open[blockIdx.x] = ctl->valid && ctl->part == 0 && ctl->parts > 1 && blockIdx.x + ctl->parts <= gridDim.x
                                      ? make_int4(ctl->b, ctl->h, ctl->block, ctl->parts) : make_int4(0, 0, 0, 0);
    }
  } else if (warp == 1 && lane == 0) {
    mbar_init(&ctl->q_full, 256);
    mbar_init(&ctl->tail, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&ctl->kv_full[s], kMode == kRows ? 128 : 1);
      mbar_init(&ctl->kv_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->s_full[i], 1);
      mbar_init(&ctl->p_full[i][0], 128);
      mbar_init(&ctl->p_full[i][1], 128);
      mbar_init(&ctl->o_full[i], 1);
    }
    mbar_init(&ctl->s_free, 4);
    mbar_init(&ctl->drain, 2);
    ctl->abort_word = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  __syncthreads();
  if (!ctl->valid) return;
  if (warp == 8) {
    tmem_alloc(&ctl->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem_base;  // columns: S [0,128) P0 [128,192) P1 [192,256) O0 [256,384) O1 [384,512)
  const int first = ctl->first, n0 = ctl->last[0], n1 = ctl->last[1], total = max(max(n0, n1) - first, 0);

  if (warp < 8 && total > 0) {
    // queries: sixteen lanes have a row
    const int rows = ctl->seq.n * a.group, row0 = ctl->block * 2 * kBM, piece = tid & 15;
    const __nv_bfloat16* q = a.q + ctl->b * a.q_sb + ctl->seq.start * a.q_st + (long long)(ctl->h * a.group) * a.q_sh;
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
      const int x = (tid >> 4) + 16 * i, row = row0 + x, tok = row / a.group, hd = row - tok * a.group;
      const bool real = row < rows;
      cp_async16(smem_u32(sQ) + (x >> 7) * kTileBytes + (piece >> 3) * kHalfBytes + (x & 127) * 128 + (((piece & 7) ^ (x & 7)) << 4),
                 real ? q + tok * a.q_st + hd * a.q_sh + piece * 8 : a.q, real);
    }
    cp_async_wait_all();
    fence_proxy_async_smem();
    mbar_arrive(&ctl->q_full);
  }

  // Positions in the ring of K and V tiles: K0 K1 V0 K2 V1 ...; the tile at position n, and whether it is V's
  const int positions = 2 * total;
  auto tile_of = [&](int n, int& which) {
    which = n == positions - 1 || (n > 0 && (n & 1) == 0);
    return n == positions - 1 ? total - 1 : which ? n / 2 - 1 : (n + 1) / 2;
  };

  if (warp >= (kMode == kSmallBoxes ? 14 : 12)) {
    // ------------------------------------------------------------------ gather
    give_registers<Shape::kOthers>();
    const int r = tid - 12 * 32;
    bool ok = true;  // (every thread goes through the same barriers, also after a wait ran out)
    const int len = ctl->seq.len;
    if constexpr (kMode == kRows) {
      // the page table's entry for this thread's key of tile j
      auto entry_of = [&](int j) {
        const int pos = (first + j) * kBN + r;
        return j < total && pos < len ? paged_entry(a.c, ctl->b, pos) : 0;
      };
      int entry = entry_of(0);
      const int piece = r & 15, row0 = r >> 4;
      const uint32_t col = (piece >> 3) * kHalfBytes;
      for (int n = 0; n < positions; ++n) {
        int which;
        const int j = tile_of(n, which);
        if (!which) {  // where the tile's rows lie (three buffers: the values of the tile before are still to be fetched)
          const int pos = (first + j) * kBN + r, slot = pos - page_index(a.c, pos) * a.c.page_size;
          const int page = pos < len ? paged_id(a.c, entry, -1) : -1;
          ctl->off[j % 3][r] = page >= 0 ? paged_offset(a.c, page, slot, ctl->h) : -1;
          entry = entry_of(j + 1);
          asm volatile("bar.sync 2, 128;" ::: "memory");
        }
        const int stage = n % kStages, round = n / kStages;
        if (ok && round > 0) ok = mbar_wait(&ctl->kv_empty[stage], (round - 1) & 1, abort_word, MB_ERR_TIMEOUT_KV_EMPTY);
        if (ok) {
          const uint8_t* base = which ? a.c.v : a.c.k;
          const uint32_t dst = smem_u32(sKV) + stage * kTileBytes + col;
          const long long* off = ctl->off[j % 3];
#pragma unroll
          for (int i = 0; i < 16; i += 8) {
            long long from[8];  // (read before the first copy is issued: the compiler keeps their order)
#pragma unroll
            for (int e = 0; e < 8; ++e) from[e] = off[row0 + 8 * (i + e)];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int row = row0 + 8 * (i + e);
              cp_async16(dst + row * 128 + (((piece & 7) ^ (row & 7)) << 4),
                         from[e] >= 0 ? base + from[e] + piece * 16 : base, from[e] >= 0);
            }
          }
        }
        cp_async_commit();
        if (n >= 2) {
          cp_async_wait<2>();
          fence_proxy_async_smem();
          mbar_arrive(&ctl->kv_full[(n - 2) % kStages]);
        }
      }
      cp_async_wait_all();
      fence_proxy_async_smem();
      for (int n = max(positions - 2, 0); n < positions; ++n) mbar_arrive(&ctl->kv_full[n % kStages]);
    }
  } else if (warp == 9 || warp == 11 || warp >= 12) {
    give_registers<Shape::kOthers>();
    if constexpr (kMode != kRows) {
      // ---------------------------------------------------------------- TMA: a lane has a box of a tile, a warp half of
      // its columns (kSmallBoxes: of half of the boxes)
      const int half = warp == 11 || warp == 13, second = warp >= 12;
      const int len = ctl->seq.len, boxes = kBN / maps.box / (kMode == kSmallBoxes ? 2 : 1), box0 = second ? boxes : 0;
      bool ok = true;
      auto page_of = [&](int j) {
        const int pos = (first + j) * kBN + (box0 + lane) * maps.box;
        if (j >= total || lane >= boxes || pos >= len) return -1;
        return maps.packed ? ctl->b - a.b_begin : paged_entry(a.c, ctl->b, pos);
      };
      if (lane == 0) tma_prefetch_desc(half ? &maps.v : &maps.k);
      int page = page_of(0), page1 = page, page2 = page, n = 0;  // of the next keys, the last ones and those before
      for (; n < positions && ok; ++n) {
        int which;
        const int j = tile_of(n, which);
        const int stage = n % kStages, round = n / kStages;
        const int entry = !which ? page : n == positions - 1 ? page1 : page2;
        const int pos = (first + j) * kBN + (box0 + lane) * maps.box;
        const bool real = lane < boxes && pos < len;  // else zeros: a page behind the last one
        const int id = !real ? maps.pages : maps.packed ? entry : paged_id(a.c, entry, maps.pages);
        const int slot = !real ? 0 : maps.packed ? pos : pos - page_index(a.c, pos) * a.c.page_size;
        if (round > 0) ok = mbar_wait_warp(&ctl->kv_empty[stage], (round - 1) & 1, abort_word, MB_ERR_TIMEOUT_KV_EMPTY);
        if (!ok) break;
        const int k0 = (first + j) * kBN;
        const bool tail = which && k0 + kBN > len && len % maps.box != 0;  // a box holds rows behind the end
        uint64_t* full = tail ? &ctl->tail : &ctl->kv_full[stage];
        uint8_t* dst = sKV + stage * kTileBytes + (box0 + lane) * maps.box * 128;
        if (lane == 0 && warp == 9) mbar_expect_tx(full, kTileBytes);  // (of all warps)
        __syncwarp();
        if (lane < boxes) tma_load_4d(dst + half * kHalfBytes, which ? &maps.v : &maps.k, full, half * 64, ctl->h, slot, id);
        if (tail && warp == 9) {  // (the last position: no other tile reaches the end)
          ok = mbar_wait_warp(&ctl->tail, 0, abort_word, MB_ERR_TIMEOUT_KV_FULL);
          const int from = len - k0, to = (from + maps.box - 1) / maps.box * maps.box;
          for (int i = from * 16 + lane; i < to * 16; i += 32)
            *reinterpret_cast<uint4*>(sKV + stage * kTileBytes + ((i >> 3) & 1) * kHalfBytes + (i >> 4) * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctl->kv_full[stage]);
        }
        if (!which) {
          page2 = page1;
          page1 = page;
          page = page_of(j + 1);
        }
      }
      if (!ok) {
        // give copies already in flight a bounded chance to land before the CTA exits
        for (int m = max(n - kStages, 0); m < n; ++m) {
          const long long t0 = clock64();
          while (!mbar_try_wait(&ctl->kv_full[m % kStages], (m / kStages) & 1) && clock64() - t0 < kWaitCycleLimit / 16) {
          }
        }
      }
    }
  } else if (warp == 8 || warp == 10) {
    // ------------------------------------------------------------------ tcgen05 issuers (see attn_fwd.cu)
    give_registers<Shape::kOthers>();
    if (total > 0) {
      constexpr uint32_t kStageUnits = kTileBytes / 16;
      bool ok = true;
      if (warp == 8) {
        constexpr uint32_t idesc_qk = umma_idesc_bf16(kBM, kBN, false, false);
        const uint64_t q_desc = umma_smem_desc(smem_u32(sQ), 16, 1024);
        const uint64_t k_desc0 = umma_smem_desc(smem_u32(sKV), 16, 1024);
        int use = 0;
        ok = mbar_wait_warp(&ctl->q_full, 0, abort_word, MB_ERR_TIMEOUT_Q);
        for (int g = 0; g < total && ok; ++g) {
          const int pos = g == 0 ? 0 : 2 * g - 1, stage = pos % kStages;
          ok = mbar_wait_warp(&ctl->kv_full[stage], (pos / kStages) & 1, abort_word, MB_ERR_TIMEOUT_KV_FULL);
          if (!ok) break;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (first + g < (i ? n1 : n0)) {
              if (use > 0) {
                ok = mbar_wait_warp(&ctl->s_free, (use - 1) & 1, abort_word, MB_ERR_TIMEOUT_S);
                if (!ok) break;
              }
              tc_fence_after();
              issue_qk(tmem, q_desc + i * kStageUnits, k_desc0 + stage * kStageUnits, idesc_qk);
              umma_commit_elect(&ctl->s_full[i]);
              ++use;
            }
          }
          if (!ok) break;
          umma_commit_elect(&ctl->kv_empty[stage]);
        }
      } else {
        constexpr uint32_t idesc_pv = umma_idesc_bf16(kBM, kD, false, true);
        const uint64_t v_desc0 = umma_smem_desc(smem_u32(sKV), kHalfBytes, 1024);
        int cnt[2] = {0, 0};
        for (int g = 0; g < total && ok; ++g) {
          const int pos = g == total - 1 ? 2 * total - 1 : 2 * g + 2, stage = pos % kStages;
          ok = mbar_wait_warp(&ctl->kv_full[stage], (pos / kStages) & 1, abort_word, MB_ERR_TIMEOUT_KV_FULL);
          if (!ok) break;
          const uint64_t v_desc = v_desc0 + stage * kStageUnits;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (first + g < (i ? n1 : n0)) {
              const uint32_t tPi = tmem + 128 + i * 64, tOi = tmem + 256 + i * 128;
              ok = mbar_wait_warp(&ctl->p_full[i][0], cnt[i] & 1, abort_word, MB_ERR_TIMEOUT_P);
              if (!ok) break;
              tc_fence_after();
              issue_pv_half(tOi, tPi, v_desc, idesc_pv, cnt[i] == 0 ? 0u : 1u);
              ok = mbar_wait_warp(&ctl->p_full[i][1], cnt[i] & 1, abort_word, MB_ERR_TIMEOUT_P);
              if (!ok) break;
              tc_fence_after();
              issue_pv_half(tOi, tPi + 32, v_desc + 4 * 128, idesc_pv, 1u);
              umma_commit_elect(&ctl->o_full[i]);
              ++cnt[i];
            }
          }
          if (!ok) break;
          umma_commit_elect(&ctl->kv_empty[stage]);
        }
      }
      if (!ok) {
        // let tensor-core work already issued finish (bounded) before tensor memory is released
        umma_commit_elect(&ctl->drain);
        const long long t0 = clock64();
        while (!mbar_try_wait(&ctl->drain, 0) && clock64() - t0 < kWaitCycleLimit / 16) {
        }
        __syncwarp();
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax + epilogue
    take_registers<Shape::kSoftmax>();
    const int i = warp >> 2;                   // query tile
    const int row = ((warp & 3) << 5) | lane;  // row inside the tile == tensor-memory lane
    const uint32_t lane_field = static_cast<uint32_t>((warp & 3) << 5) << 16;
    const uint32_t tS = tmem + lane_field;
    const uint32_t tPi = tmem + 128 + i * 64 + lane_field;
    const uint32_t tOi = tmem + 256 + i * 128 + lane_field;
    const int tile_row = ctl->block * 2 * kBM + i * kBM;  // the tile's first row of the sequence
    const int visible = visible_keys(a, ctl->seq, tile_row + row), visible_first = visible_keys(a, ctl->seq, tile_row);
    const int last = i ? n1 : n0;

    float m_ref = -INFINITY, l = 0.f;
    int cnt = 0;
    bool ok = true;
    for (int jt = first; jt < last; ++jt) {
      ok = mbar_wait_warp(&ctl->s_full[i], cnt & 1, abort_word, MB_ERR_TIMEOUT_S);
      if (!ok) break;
      tc_fence_after();
      uint32_t sr[4][32];
      tmem_ld32(tS + 0, sr[0]);
      tmem_ld32(tS + 32, sr[1]);
      tmem_ld32(tS + 64, sr[2]);
      tmem_ld32(tS + 96, sr[3]);
      tmem_wait_ld();
      tc_fence_before();
      mbar_arrive_elect(&ctl->s_free);  // the scores are in registers: the score region has its next user

      const int k0 = jt * kBN;
      if (k0 + kBN > visible_first) {  // some row of the tile does not see all of these keys
        const int limit = visible - k0;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (c * 32 + e >= limit) sr[c][e] = 0xff800000u;  // -inf
      }
      float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        mx0 = max3(mx0, __uint_as_float(sr[0][e]), __uint_as_float(sr[0][e + 1]));
        mx1 = max3(mx1, __uint_as_float(sr[1][e]), __uint_as_float(sr[1][e + 1]));
        mx2 = max3(mx2, __uint_as_float(sr[2][e]), __uint_as_float(sr[2][e + 1]));
        mx3 = max3(mx3, __uint_as_float(sr[3][e]), __uint_as_float(sr[3][e + 1]));
      }
      float m_tile = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3));
      m_tile *= a.scale_log2;
      if (cnt == 0) {
        m_ref = m_tile;
      } else {
        // the previous P V of this query tile must be complete before its probabilities are overwritten or O is rescaled
        ok = mbar_wait_warp(&ctl->o_full[i], (cnt - 1) & 1, abort_word, MB_ERR_TIMEOUT_O);
        if (!ok) break;
        tc_fence_after();
        const float m_new = fmaxf(m_ref, m_tile);
        const bool need = m_new - m_ref > kRescaleThreshold;
        if (__any_sync(0xffffffffu, need)) {
          const float f = need ? fast_exp2(m_ref - m_new) : 1.f;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t orow[32];
            tmem_ld32(tOi + c * 32, orow);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) orow[e] = __float_as_uint(__uint_as_float(orow[e]) * f);
            tmem_st32(tOi + c * 32, orow);
          }
          tmem_wait_st();
          if (need) {
            l *= f;
            m_ref = m_new;
          }
        }
      }
      const float lift = m_ref == -INFINITY ? 0.f : -m_ref;
      const uint64_t c2 = pack2(a.scale_log2, a.scale_log2);
      const uint64_t nm2 = pack2(lift, lift);
      uint64_t sum_a = pack2(0.f, 0.f), sum_b = pack2(0.f, 0.f);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t pk[32];
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          const int c = half * 2 + cc;
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const uint64_t x2 = fma2(pack2(__uint_as_float(sr[c][e]), __uint_as_float(sr[c][e + 1])), c2, nm2);
            float x0, x1;
            unpack2(x2, x0, x1);
            const uint64_t p2 = pack2(fast_exp2(x0), fast_exp2(x1));
            if ((e >> 1) & 1) sum_b = add2(sum_b, p2);
            else sum_a = add2(sum_a, p2);
            float p0, p1;
            unpack2(p2, p0, p1);
            pk[cc * 16 + (e >> 1)] = pack_bf16x2(p0, p1);
          }
        }
        tmem_st32(tPi + half * 32, pk);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&ctl->p_full[i][half]);
      }
      float s0, s1;
      unpack2(add2(sum_a, sum_b), s0, s1);
      l += s0 + s1;
      ++cnt;
    }

    // epilogue; tiles whose rows all lie behind the sequence's skip it
    const int rows = ctl->seq.n * a.group;
    if (ok && tile_row < rows) {
      if (cnt > 0) ok = mbar_wait_warp(&ctl->o_full[i], (cnt - 1) & 1, abort_word, MB_ERR_TIMEOUT_O);
      if (ok) {
        if (cnt > 0) tc_fence_after();
        const bool store = tile_row + row < rows;
        if (ctl->parts > 1) {
          // a share: rows as they are, column group by column group (contiguous over a warp)
          const int r = i * kBM + row;
          if (cnt > 0) {
            float4* dst = a.tile_o + (long long)blockIdx.x * (32 * 2 * kBM) + r;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t orow[32];
              tmem_ld32(tOi + c * 32, orow);
              tmem_wait_ld();
#pragma unroll
              for (int v = 0; v < 8; ++v)
                dst[(c * 8 + v) * (2 * kBM)] =
                    make_float4(__uint_as_float(orow[v * 4 + 0]), __uint_as_float(orow[v * 4 + 1]),
                                __uint_as_float(orow[v * 4 + 2]), __uint_as_float(orow[v * 4 + 3]));
            }
          }
          a.tile_ml[(long long)blockIdx.x * (2 * kBM) + r] = make_float2(m_ref, l);
        } else {
          const float inv = l == 0.f ? 0.f : 1.f / l;
          const int tok = (tile_row + row) / a.group, hd = ctl->h * a.group + (tile_row + row) - tok * a.group;
          __nv_bfloat16* optr = a.o + ctl->b * a.o_sb + (long long)(ctl->seq.start + tok) * a.o_st + (long long)hd * a.o_sh;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t orow[32];
            if (cnt > 0) {
              tmem_ld32(tOi + c * 32, orow);
              tmem_wait_ld();
            }
            // a row that sees no key is zero, whatever its masked products gave
            if (cnt == 0 || l == 0.f) {
#pragma unroll
              for (int e = 0; e < 32; ++e) orow[e] = 0u;
            }
            if (store) {
              uint4* dst = reinterpret_cast<uint4*>(optr + c * 32);
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                uint4 w;
                w.x = pack_bf16x2(__uint_as_float(orow[v * 8 + 0]) * inv, __uint_as_float(orow[v * 8 + 1]) * inv);
                w.y = pack_bf16x2(__uint_as_float(orow[v * 8 + 2]) * inv, __uint_as_float(orow[v * 8 + 3]) * inv);
                w.z = pack_bf16x2(__uint_as_float(orow[v * 8 + 4]) * inv, __uint_as_float(orow[v * 8 + 5]) * inv);
                w.w = pack_bf16x2(__uint_as_float(orow[v * 8 + 6]) * inv, __uint_as_float(orow[v * 8 + 7]) * inv);
                dst[v] = w;
              }
            }
          }
          if (store)
            a.lse[ctl->b * a.lse_sb + hd * a.lse_sh + ctl->seq.start + tok] = l == 0.f ? -INFINITY : m_ref * kLn2 + __logf(l);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (tid == 0 && ctl->abort_word != 0) atomicCAS(a.c.status, 0, ctl->abort_word);
}

// Joins the shares of the unit whose first share CTA blockIdx.x had (if there is one): 8 rows a block; warp w has columns
// [16 w, 16 w + 16), a lane 4 of them of one row, so that the lanes of a column group read 128 contiguous bytes.
constexpr int kTileMergeRows = 8;
__global__ void __launch_bounds__(256) paged_tiles_merge_kernel(const __grid_constant__ PagedAttnArgs a) {
  const int lane = threadIdx.x & 31, chunk = (threadIdx.x >> 5) * 4 + (lane >> 3);
  const int r = blockIdx.y * kTileMergeRows + (lane & 7);
  grid_dependents_launch();
  grid_dependency_wait();
  const int4 unit = a.tile_open[blockIdx.x];
  if (unit.w == 0) return;
  const PagedSeq seq = paged_seq(a.c, unit.x, a.max_queries, a.max_keys);
  const int row = unit.z * 2 * kBM + r;
  if (row >= seq.n * a.group) return;
  const float2* ml = a.tile_ml + (long long)blockIdx.x * (2 * kBM) + r;
  const float4* src = a.tile_o + ((long long)blockIdx.x * 32 + chunk) * (2 * kBM) + r;
  float m = -INFINITY;
#pragma unroll 4
  for (int p = 0; p < unit.w; ++p) m = fmaxf(m, ml[p * 2 * kBM].x);
  float l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = 0; p < unit.w; ++p) {
    const float2 s = ml[p * 2 * kBM];
    if (s.y == 0.f) continue;  // a share without visible keys has stored no rows, or products of hidden keys
    const float4 x = src[(long long)p * 32 * 2 * kBM];
    const float w = s.x == -INFINITY ? 1.f : fast_exp2(s.x - m);
    l = fmaf(w, s.y, l);
    acc[0] = fmaf(w, x.x, acc[0]);
    acc[1] = fmaf(w, x.y, acc[1]);
    acc[2] = fmaf(w, x.z, acc[2]);
    acc[3] = fmaf(w, x.w, acc[3]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int tok = row / a.group, hd = unit.y * a.group + row - tok * a.group;
  const uint2 o = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  *reinterpret_cast<uint2*>(a.o + unit.x * a.o_sb + (long long)(seq.start + tok) * a.o_st + (long long)hd * a.o_sh + chunk * 4) = o;
  if (chunk == 0) a.lse[unit.x * a.lse_sb + hd * a.lse_sh + seq.start + tok] = l == 0.f ? -INFINITY : m * kLn2 + __logf(l);
}

long long paged_tiles_workspace(long long ctas) {
  return ctas * (2ll * kBM * (kHeadDim * (long long)sizeof(float) + (long long)sizeof(float2)) + (long long)sizeof(int4));
}

template <int kMode>
static int launch_tiles(const TileMaps& maps, const PagedAttnArgs& a, int ctas, cudaStream_t stream) {
  static bool attr_set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return MB_E_CUDA;
  constexpr int bytes = tile_smem_bytes();
  if (!attr_set[dev]) {
    if (!cuda_ok(cudaFuncSetAttribute(paged_tiles_kernel<kMode>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
                 "paged_tiles_kernel shared memory"))
      return MB_E_CUDA;
    attr_set[dev] = true;
  }
  if (!launch_overlapped("launch paged_tiles_kernel", paged_tiles_kernel<kMode>, dim3(ctas), TileShape<kMode>::kThreads, bytes,
                         stream, maps, a))
    return MB_E_CUDA;
  return MB_SUCCESS;
}

int launch_paged_tiles_merge(const PagedAttnArgs& a, int ctas, cudaStream_t stream) {
  return launch_overlapped("launch paged_tiles_merge_kernel", paged_tiles_merge_kernel, dim3(ctas, (2 * kBM) / kTileMergeRows),
                           256, 0, stream, a)
             ? MB_SUCCESS
             : MB_E_CUDA;
}

// Boxes of `box` slots of 64 columns of a head, out of [pages, slots, heads, 128] with strides in bytes.
static bool page_map(CUtensorMap* map, const void* ptr, int hkv, int slots, int pages, long long head_sb, long long slot_sb,
                     long long page_sb, int box) {
  const cuuint64_t dims[4] = {(cuuint64_t)kHeadDim, (cuuint64_t)hkv, (cuuint64_t)slots, (cuuint64_t)pages};
  const cuuint64_t strides[3] = {(cuuint64_t)head_sb, (cuuint64_t)slot_sb, (cuuint64_t)page_sb};
  const cuuint32_t boxes[4] = {64, 1, (cuuint32_t)box, 1}, ones[4] = {1, 1, 1, 1};
  return encode_tiled_bf16(map, const_cast<void*>(ptr), 4, dims, strides, boxes, ones) == 0;
}

int launch_paged_tiles(const PagedAttnArgs& a, int ctas, cudaStream_t stream) {
  TileMaps maps;
  memset(&maps, 0, sizeof(maps));
  const PagedView& c = a.c;
  if (a.packed_k != nullptr) {
    const long long row = (long long)c.hkv * kHeadDim * 2;
    maps.box = kBN;
    maps.pages = a.b_end - a.b_begin;
    maps.packed = 1;
    if (!page_map(&maps.k, a.packed_k, c.hkv, a.packed_rows, maps.pages, kHeadDim * 2, row, row * a.packed_rows, kBN) ||
        !page_map(&maps.v, a.packed_v, c.hkv, a.packed_rows, maps.pages, kHeadDim * 2, row, row * a.packed_rows, kBN))
      return MB_E_TENSORMAP;
    return launch_tiles<kBoxes>(maps, a, ctas, stream);
  }
  maps.box = 1;
  maps.pages = c.pages;
  while (maps.box < kBN && c.page_size % (2 * maps.box) == 0) maps.box *= 2;
  // (rows of the swizzled layout go in groups of 8; without a page or a key there is nothing to map, and nothing to fetch; a map
  // has no dimension whose entries are one, like heads that a view repeats)
  const bool repeats = c.head_sb == 0 || c.slot_sb == 0 || c.page_sb == 0;
  if (maps.box < 8 || a.max_keys == 0 || repeats) return launch_tiles<kRows>(maps, a, ctas, stream);
  if (!page_map(&maps.k, c.k, c.hkv, c.page_size, c.pages, c.head_sb, c.slot_sb, c.page_sb, maps.box) ||
      !page_map(&maps.v, c.v, c.hkv, c.page_size, c.pages, c.head_sb, c.slot_sb, c.page_sb, maps.box))
    return MB_E_TENSORMAP;
  return maps.box < 64 ? launch_tiles<kSmallBoxes>(maps, a, ctas, stream) : launch_tiles<kBoxes>(maps, a, ctas, stream);
}

}  // namespace mb
