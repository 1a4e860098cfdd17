// Attention over a key/value cache in pages for gfx950 (MI355X): each sequence's new tokens, packed one sequence after the
// other, against its own pages.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(log2(e) scale q_i . k_j - m_i)   over the keys j that row i sees:
//   j below its sequence's length; causal: j no further than the row's own position len - fresh + i; a window: within it.
//
// The key loop is the attention kernel's (attention_step.h): 64 keys a step through an LDS ring, both products transposed
// on v_mfma_f32_32x32x16 so that a query is a lane, scores, maximum and sum in 32 bits, p rounded to 16 bits for the
// second product.  What is this file's own is how work is found and how keys come into the ring.
//
// A tile is the rows of one KV head: whole tokens with all query heads of the head's group beside each other, so that K and
// V are read once a group, and a row's position is that of its token: ranges a row, ascending along the tile.  Two forms: a
// tile of 32 rows in a workgroup of one wave for calls of few rows a sequence (a generated token, a few drafted ones), one of
// 128 rows in four waves for chunks.  The first is bound by the bytes of K and V in flight: a compute unit holds two such
// workgroups at D 128, each with a ring of 64 KiB that is refilled a step ahead.
//
// How many tokens each sequence has is device data.  Every wave works the launch's deal out for itself, a lane a sequence: the
// tiles and key blocks of all sequences give the blocks an item may have for the launch to fill the chip once, a tile of
// more blocks is split, items are numbered sequence by sequence, a tile's splits next to each other, and a workgroup finds
// its item from two sums over the lanes.  The host knows bounds only: a launch has a workgroup for each item there may
// be, and those past the last leave at once.  A split leaves its accumulator, maximum and sum in f32; merge_kernel adds them
// up in the order of the splits, so a call's result depends on nothing but its inputs.
#include <hip/hip_runtime.h>

#include "kernels.h"
#include "launch.h"

#if !defined(__HIP_DEVICE_COMPILE__)  // the kernels' bodies are compiled for the device only: their helpers have no caller here
#pragma clang diagnostic ignored "-Wunused-function"
#pragma clang diagnostic ignored "-Wunused-variable"
#pragma clang diagnostic ignored "-Wunused-const-variable"
#pragma clang diagnostic ignored "-Wunneeded-internal-declaration"
#pragma clang diagnostic ignored "-Wunused-template"
#pragma clang diagnostic ignored "-Wundefined-internal"
#endif
#include "attention_step.h"
#include "pages.h"

namespace svodk {
namespace {

// A value that every lane of a wave has, in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

struct PagedParams {
  PagesArgs pages;
  const uint16_t *q;
  uint16_t *o;
  float *parts;
  int32_t *told;  // behind them: the blocks an item had
  int32_t heads, group;
  uint32_t group_rcp;
  int32_t tokens;  // of a tile: as many as have their group's rows in it
  uint32_t tokens_rcp;
  int32_t causal, win_left, win_right;
  float scale;
  int32_t splits;       // as in PagedArgs
  int32_t places;       // workgroups that the chip holds at a time
  float crowd, states;  // of blocks_an_item(): company's cost, and that of a state of every row, in steps
  int32_t slots;        // partial states there is room for
};

// ---- the deal.  What a lane's sequence asks for: tiles of query rows, and the key blocks of one of its tiles at most.
struct Demand {
  Sequence s;
  int tiles, blocks;
};
__device__ __forceinline__ Demand demand_of(const PagedParams &p, int b) {
  Demand d{};
  if (b >= p.pages.batch) return d;
  d.s = sequence_at(p.pages, b);
  d.tiles = d.s.fresh > 0 ? (int)div_by((uint32_t)d.s.fresh - 1, (uint32_t)p.tokens, p.tokens_rcp) + 1 : 0;
  d.blocks = (d.s.len + kBkv - 1) / kBkv;
  if (p.win_left >= 0) d.blocks = (int)min((int64_t)d.blocks, ((int64_t)p.win_left + p.win_right + p.tokens) / kBkv + 2);
  return d;
}
__device__ __forceinline__ int last_lane(int x) { return __builtin_amdgcn_readlane(x, 63); }

// The greatest of all lanes' values, none below 0.
__device__ __forceinline__ int most_of_lanes(int x) {
#if defined(__HIP_DEVICE_COMPILE__)
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true));  // row_shr:1
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));  // row_bcast:15 into rows 1 and 3
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));  // row_bcast:31 into rows 2 and 3
#endif
  return last_lane(x);
}
constexpr int kNoSplits = 0x7fffffff;  // an item's blocks where none is split
// A tile's splits where an item has `most` blocks.
__device__ __forceinline__ int splits_of(const PagedParams &p, int blocks, int most) {
  if (p.splits != 0) return max(1, min(p.splits, blocks));
  return blocks <= most ? 1 : (blocks + most - 1) / most;
}
// The key blocks an item may have: of those that would fill the chip once and up to twice as many, and of the longest tile's,
// what ends first by this reckoning, in steps of a block.  Items run a round of the chip's places at a time, a step of four waves
// with company on its compute unit takes `crowd` times one's alone; an item starts in kStart steps (the deal, the pages,
// the first blocks: trips to memory); a call that splits writes its rows' states, reads them and has its merge behind it.
// (By the blocks of all items over the places alone 16 sequences over 210 to 2100 keys were 528 items on 512 places, 22.9 us for 19.4;
// without the states two chunks of 1001 rows in a window of 1024 split in two, 46 us for 32.)
constexpr int kLeastBlocks = 2, kStart = 3, kMerge = 3;
__device__ __forceinline__ int blocks_an_item(const PagedParams &p, const Demand &first) {
  if (p.splits != 0) return kNoSplits;
  constexpr int kTries = 4, kQuarters[kTries] = {4, 5, 6, 8};
  int high = 0, low = 0, longest = 0, tiles = 0;
  const int lane = (int)__builtin_amdgcn_workitem_id_x() & 63;
  for (int base = 0; base < p.pages.batch; base += 64) {
    const Demand d = base == 0 ? first : demand_of(p, base + lane);
    const int64_t work = (int64_t)d.tiles * d.blocks;
    high += (int)(work >> 12), low += (int)(work & 4095);
    longest = max(longest, d.tiles > 0 ? d.blocks : 0);
    tiles += d.tiles;
  }
  const float heads = (float)p.pages.kv_heads, places = (float)p.places, all_tiles = (float)last_lane(sum_to_lane(tiles));
  const float blocks = ((float)last_lane(sum_to_lane(high)) * 4096.0f + (float)last_lane(sum_to_lane(low))) * heads;
  longest = most_of_lanes(longest);
  const float a_place = __builtin_amdgcn_rcpf(places), a_tile = __builtin_amdgcn_rcpf(all_tiles);
  const int once = max(kLeastBlocks, (int)__builtin_ceilf(blocks / places));
  int sums[kTries] = {};
  for (int base = 0; base < p.pages.batch; base += 64) {
    const Demand d = base == 0 ? first : demand_of(p, base + lane);
#pragma unroll
    for (int i = 0; i < kTries; i++) sums[i] += d.tiles * splits_of(p, d.blocks, (once * kQuarters[i] + 3) / 4);
  }
  auto time_of = [&](float items, int most) {
    const float alone = (float)most * (2.0f * items > places ? p.crowd : 1.0f) + (float)kStart;
    if (items <= places) return alone;
    return __builtin_fmaxf(alone, __builtin_ceilf(items * a_place) * (blocks * __builtin_amdgcn_rcpf(items) * p.crowd + (float)kStart));
  };
  int best = kNoSplits;
  float best_time = time_of(all_tiles * heads, longest);
#pragma unroll
  for (int i = kTries - 1; i >= 0; i--) {
    const int most = (once * kQuarters[i] + 3) / 4;
    const float items = (float)last_lane(sum_to_lane(sums[i]));
    const float time = time_of(items * heads, most) + (float)kMerge + p.states * items * a_tile;
    if (most < longest && time < best_time) best = most, best_time = time;
  }
  return best;
}

// Where an item, or a row, is in the deal.
struct Place {
  int b, tile, split, splits;
  int slot;  // of the tile's first split, in KV heads' states
  Sequence s;
  bool found;
};
// The item-th item; or, with BY_ROW, the tile of packed row `item`.
template <bool BY_ROW>
__device__ __forceinline__ Place place_of(const PagedParams &p, int item, const Demand &first, int most) {
  const int lane = (int)__builtin_amdgcn_workitem_id_x() & 63;
  Place at{};
  int items_before = 0, slots_before = 0;
  for (int base = 0; base < p.pages.batch; base += 64) {
    const Demand d = base == 0 ? first : demand_of(p, base + lane);
    const int splits = splits_of(p, d.blocks, most), items = d.tiles * splits, slots = splits > 1 ? items : 0;
    const int items_to = sum_to_lane(items), slots_to = sum_to_lane(slots);
    const uint64_t here = BY_ROW ? __builtin_amdgcn_ballot_w64(d.s.start <= item && item - d.s.start < d.s.fresh)
                                 : __builtin_amdgcn_ballot_w64(items_to > item - items_before);
    if (here != 0) {
      const int at_lane = __builtin_ctzll(here);
      at.b = base + at_lane;
      at.splits = __builtin_amdgcn_readlane(splits, at_lane);
      at.s.start = __builtin_amdgcn_readlane(d.s.start, at_lane);
      at.s.fresh = __builtin_amdgcn_readlane(d.s.fresh, at_lane);
      at.s.len = __builtin_amdgcn_readlane(d.s.len, at_lane);
      const int tiles = __builtin_amdgcn_readlane(d.tiles, at_lane);
      int order;  // the last tile, which sees the most keys, comes first
      if (BY_ROW) {
        at.tile = (int)div_by((uint32_t)(item - at.s.start), (uint32_t)p.tokens, p.tokens_rcp);
        order = tiles - 1 - at.tile;
      } else {
        const int within = item - items_before - __builtin_amdgcn_readlane(items_to - items, at_lane);
        order = within / at.splits;
        at.split = within - order * at.splits;
        at.tile = tiles - 1 - order;
      }
      at.slot = slots_before + __builtin_amdgcn_readlane(slots_to - slots, at_lane) + order * at.splits;
      at.found = true;
      return at;
    }
    items_before += last_lane(items_to);
    slots_before += last_lane(slots_to);
  }
  return at;
}

// ---- keys in pages.  A fill instruction moves 1 KiB, 16 bytes a lane: whole rows of one KV head, 16 of which never lie in two
// pages.  So a wave's fills of a block go by runs of 16 rows, with a page looked up and a descriptor made for each.
template <int D, int NW, unsigned FLAGS>
struct PagesOf {
  static constexpr bool kCodes = (FLAGS & kCoded) != 0, kStages = (FLAGS & kStaged) != 0;
  static constexpr int kRowBytes = kCodes ? D : 2 * D;
  static constexpr int kLanes = kRowBytes / 16;          // lanes a row
  static constexpr int kRows = 64 / kLanes;              // rows a fill
  static constexpr int kFills = kBkv / kRows / NW;       // a wave's fills of a tile, kStride rows apart
  static constexpr int kStride = NW * kRows;
  static constexpr int kPer = kStride >= 16 ? 1 : 16 / kStride;  // its fills of a run of 16 rows
  static constexpr int kRuns = kFills / kPer;
  static_assert(kFills * kRows * NW == kBkv && kRuns * kPer == kFills && kRows <= 16, "whole fills");
  const uint8_t *k_scale, *v_scale;  // the KV head's rows of page 0 (w.k_base and w.v_base: of the pools)
  const int32_t *table;              // the sequence's
  int columns, count;                // of the table, and pages there are
  int page_log2;
  uint32_t page_rows;                // rows of a page, all KV heads'
  int first_key;                     // the frame's
  // The pages of 128 columns from `column` on, a lane each: asked for 64 columns ahead of their use.
  int column, ids, ids_next;
  int64_t run[kRuns];                // the pool's row that each of this wave's runs of the block filled last starts at
  int run_row;                       // the first run's row of the block
  int k_src[kPer], v_src[kPer];      // a lane's offset in a run's descriptor (straight into LDS: swizzled)
  int k_dst[kPer], v_dst[kPer];      // where its 16 bytes go in a slot; of codes, widened, the second 16 go to ^ 16
  struct Stage {
    u32x4 rows[kStages ? kFills : 1];
    uint32_t scale[kCodes ? kFills : 1];
  };
  Stage k_stage, v_stage;

  __device__ int ask(int from) const {
    const int lane = (int)__builtin_amdgcn_workitem_id_x() & 63;
    return table[min(from + lane, columns - 1)];
  }
  __device__ int id_of(int at) const {  // of column `at`
    const int rel = at - column;
    const int id = rel < 64 ? __builtin_amdgcn_readlane(ids, rel) : __builtin_amdgcn_readlane(ids_next, rel & 63);
    return min(max(id, 0), count - 1);
  }
  __device__ int row_of(int r) const { return run_row + r * kStride * kPer; }
  // The runs of block `n` of the frame.
  __device__ void find(int n) {
    const int key0 = first_key + n * kBkv;
    if ((key0 >> page_log2) - column >= 64) {
      column += 64;
      ids = ids_next;
      ids_next = ask(column + 64);
    }
#pragma unroll
    for (int r = 0; r < kRuns; r++) {
      const int key = key0 + row_of(r);
      const int id = id_of(key >> page_log2);
      run[r] = (int64_t)((uint64_t)(uint32_t)id * page_rows) + (key & ((1 << page_log2) - 1));
    }
  }
};
template <int D, int NW>
struct Pages<D, NW, kPaged> : PagesOf<D, NW, kPaged> {};
template <int D, int NW>
struct Pages<D, NW, kPaged | kStaged> : PagesOf<D, NW, kPaged | kStaged> {};
template <int D, int NW>
struct Pages<D, NW, kPaged | kStaged | kCoded> : PagesOf<D, NW, kPaged | kStaged | kCoded> {};

// A descriptor over `rows` rows of `row_bytes` at `base`: rows from there on read as zeros.
[[maybe_unused]] __device__ __forceinline__ i32x4 rows_rsrc(const uint8_t *base, int rows, int row_bytes) {
  const uint64_t at = (uint64_t)(uintptr_t)base;
  // The same in every lane, and told so: a 64-bit sum that the compiler has on the VALU is no scalar to it.
  return i32x4{uniform((int)(uint32_t)at), uniform((int)(uint32_t)(at >> 32)), uniform(rows * row_bytes), 0x00020000};
}

// This wave's share of block `n` from the pool at `base`, whose runs find() has named, straight into LDS: keys past the length
// land as zeros (a page's last rows hold anything, and 0 times that is not 0).
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ void fill_pages(const Wave<D, NW, F16, FLAGS> &w, const uint8_t *base, int n, int lds_at,
                                           const int *src) {
  using P = decltype(w.pages);
#pragma unroll
  for (int r = 0; r < P::kRuns; r++) {
    const int left = min(max(w.len - n * kBkv - w.pages.row_of(r), 0), 16);
    const i32x4 rsrc = rows_rsrc(base + w.pages.run[r] * P::kRowBytes, left, P::kRowBytes);
#pragma unroll
    for (int j = 0; j < P::kPer; j++)
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                   :
                   : "s"(lds_at + (w.wave + NW * (r * P::kPer + j)) * 1024), "v"(src[j]), "s"(rsrc)
                   : "memory");
  }
}
// The same into registers, codes with their rows' scales.
template <int D, int NW, bool F16, unsigned FLAGS, typename S>
__device__ __forceinline__ void stage_pages(const Wave<D, NW, F16, FLAGS> &w, const uint8_t *base, const uint8_t *scales, int n,
                                            const int *src, S &stage) {
#if defined(__HIP_DEVICE_COMPILE__)
  using P = decltype(w.pages);
#pragma unroll
  for (int r = 0; r < P::kRuns; r++) {
    const int left = min(max(w.len - n * kBkv - w.pages.row_of(r), 0), 16);
    const auto rows = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base + w.pages.run[r] * P::kRowBytes), 0,
                                                        left * P::kRowBytes, 0x00020000);
#pragma unroll
    for (int j = 0; j < P::kPer; j++) stage.rows[r * P::kPer + j] = __builtin_amdgcn_raw_buffer_load_b128(rows, src[j], 0, 0);
    if constexpr (P::kCodes) {
      const auto scale = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(scales + w.pages.run[r]), 0, left, 0x00020000);
#pragma unroll
      for (int j = 0; j < P::kPer; j++)
        stage.scale[r * P::kPer + j] = __builtin_amdgcn_raw_buffer_load_b8(scale, src[j] / P::kRowBytes, 0, 0);
    }
  }
#endif
}
// And from there into a slot.
template <int D, int NW, bool F16, unsigned FLAGS, typename S>
__device__ __forceinline__ void land_stage(const Wave<D, NW, F16, FLAGS> &w, uint8_t *slot, const int *dst, const S &stage) {
  using P = decltype(w.pages);
#pragma unroll
  for (int i = 0; i < P::kFills; i++) {
    const u32x4 c = stage.rows[i];
    uint8_t *at = slot + (i - i % P::kPer) * P::kStride * Tile<D>::kRowBytes;
    if constexpr (P::kCodes) {
      const float scale = scale_of(stage.scale[i]);
      const u32x4 lo = {widen_codes<F16, false>(c[0], scale), widen_codes<F16, true>(c[0], scale),
                        widen_codes<F16, false>(c[1], scale), widen_codes<F16, true>(c[1], scale)};
      const u32x4 hi = {widen_codes<F16, false>(c[2], scale), widen_codes<F16, true>(c[2], scale),
                        widen_codes<F16, false>(c[3], scale), widen_codes<F16, true>(c[3], scale)};
      *reinterpret_cast<u32x4 *>(at + dst[i % P::kPer]) = lo;
      *reinterpret_cast<u32x4 *>(at + (dst[i % P::kPer] ^ 16)) = hi;
    } else {
      *reinterpret_cast<u32x4 *>(at + dst[i % P::kPer]) = c;
    }
  }
}
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ void fill_k_pages(Wave<D, NW, F16, FLAGS> &w, int n, int slot) {
  if (n >= w.end) return;
  w.pages.find(n);
  if constexpr ((FLAGS & kStaged) != 0)
    stage_pages<D, NW>(w, w.k_base, w.pages.k_scale, n, w.pages.k_src, w.pages.k_stage);
  else
    fill_pages<D, NW>(w, w.k_base, n, w.lds0 + slot * Tile<D>::kBytes, w.pages.k_src);
}
// A block's values come a step behind its keys, which have named its runs.
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ void fill_v_pages(Wave<D, NW, F16, FLAGS> &w, int n, int slot) {
  if (n >= w.end) return;
  if constexpr ((FLAGS & kStaged) != 0)
    stage_pages<D, NW>(w, w.v_base, w.pages.v_scale, n, w.pages.v_src, w.pages.v_stage);
  else
    fill_pages<D, NW>(w, w.v_base, n, w.lds0 + (2 + slot) * Tile<D>::kBytes, w.pages.v_src);
}
// The end of step `blk`: what its fills asked for goes into the ring, V(blk + 1) and K(blk + 2).
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ void land_pages(Wave<D, NW, F16, FLAGS> &w, uint8_t *smem, int blk, int par) {
  if (blk + 1 < w.end) land_stage<D, NW>(w, smem + w.v_slot(par ^ 1) * Tile<D>::kBytes, w.pages.v_dst, w.pages.v_stage);
  if (blk + 2 < w.end) land_stage<D, NW>(w, smem + w.k_slot(par) * Tile<D>::kBytes, w.pages.k_dst, w.pages.k_stage);
}

// Whether a form's tiles come through registers: codes, which are widened there; and the keys of a wave by itself, which then
// needs one slot for them and one for values, half the LDS, so that a compute unit holds twice the waves (at D 256 the
// registers do not hold a tile).
template <int D, int NW, bool CODED>
constexpr bool kStages = CODED || (NW == 1 && D <= 128);

template <int D, int NW, bool F16, bool CODED>
__device__ __forceinline__ void paged_body(uint8_t *smem, const PagedParams &p) {
  using TL = Tile<D>;
  constexpr bool kThroughRegisters = kStages<D, NW, CODED>;
  using W = Wave<D, NW, F16, kRanged | kPaged | (kThroughRegisters ? kStaged : 0u) | (CODED ? kCoded : 0u)>;
  using P = decltype(W::pages);
  constexpr int BQ = NW * kWaveRows, KS = W::KS, DB = W::DB;
  const int tid = (int)__builtin_amdgcn_workitem_id_x();
  W w;
  w.lane = tid & 63;
  w.wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
  w.g = w.lane >> 5;
  const int ln = w.lane & 31;

  // ---- the item.  The KV heads of an item are neighbours in the launch: their pages are neighbours in memory.
  const uint32_t wg = __builtin_amdgcn_workgroup_id_x();
  const int item = (int)(wg / (uint32_t)p.pages.kv_heads);
  const int kvh = (int)(wg - (uint32_t)item * (uint32_t)p.pages.kv_heads);
  const Demand first_demand = demand_of(p, w.lane);
  const int most = blocks_an_item(p, first_demand);
  const Place at = place_of<false>(p, item, first_demand, most);
  // The merge goes by the same deal: it is told what this launch went by, behind the states.
  if (wg == 0 && tid == 0 && p.slots > 0) *p.told = most;
  if (!at.found) return;
  const int slot = (at.slot + at.split) * p.pages.kv_heads + kvh;
  if (at.splits > 1 && slot >= p.slots) return;  // lengths that are none: more rows than there are

  // ---- this lane's row: query head `row % group` of the KV head's, of the tile's token row / group.
  const int tile_first = at.tile * p.tokens, base = at.s.base();
  const int row = w.wave * kWaveRows + ln;
  const int in_tile = (int)div_by((uint32_t)row, (uint32_t)p.group, p.group_rcp);
  const int token = tile_first + in_tile, last_token = min(tile_first + p.tokens, at.s.fresh) - 1;
  const bool row_ok = in_tile < p.tokens && token <= last_token;
  const int head = kvh * p.group + (row - in_tile * p.group);
  const int64_t q_row = ((int64_t)at.s.start + min(token, last_token)) * p.heads + min(head, p.heads - 1);

  // ---- the keys [lo, hi] it sees, ascending with the row; rows past the last token stand in for it.
  const int64_t pos = (int64_t)base + min(token, last_token);
  int64_t lo = 0, hi = (int64_t)at.s.len - 1;
  int first = 0, end = at.s.len;  // of the tile, in keys
  if (p.causal) {
    hi = min(hi, pos);
    end = max(0, min(end, base + last_token + 1));
  }
  if (p.win_left >= 0) {
    lo = max(lo, pos - p.win_left);
    hi = min(hi, pos + p.win_right);
    first = (int)max((int64_t)0, (int64_t)base + tile_first - p.win_left);
    end = (int)max((int64_t)0, min((int64_t)end, (int64_t)base + last_token + p.win_right + 1));
  }
  first = min(first / kBkv, (end + kBkv - 1) / kBkv);
  end = (end + kBkv - 1) / kBkv;
  if (at.splits > 1) {
    // An even share of the tile's blocks, the first splits' one more where they do not go up.
    const int n = end - first, each = n / at.splits, over = n - each * at.splits;
    first += at.split * each + min(at.split, over);
    end = first + each + (at.split < over ? 1 : 0);
  }
  // From here on in the item's own frame: keys count from its first.
  const int first_key = uniform(first * kBkv);
  end = uniform(end - first);
  w.end = end;
  w.len = max(at.s.len - first_key, 0);
  w.tk = w.len;
  w.key_mask = nullptr;
  w.mask_row = 0;
  w.mask_bytes = 1;
  w.scanned = false;
  w.mask_next = 0;
  w.row_lo = (int)(lo - first_key);
  w.row_hi = (int)(max(hi, (int64_t)-1) - first_key);
  w.lo_last = __builtin_amdgcn_readlane(w.row_lo, kWaveRows - 1);
  w.lo_first = __builtin_amdgcn_readlane(w.row_lo, 0);
  w.hi_first = __builtin_amdgcn_readlane(w.row_hi, 0);
  w.hi_last = __builtin_amdgcn_readlane(w.row_hi, kWaveRows - 1);
  w.wave_first_row = w.my_row = 0;
  w.my_row_ok = row_ok;

  // ---- the pages.
  const int64_t head_row = (int64_t)kvh << p.pages.page_log2;
  w.k_base = (const uint8_t *)p.pages.k + head_row * P::kRowBytes;
  w.v_base = (const uint8_t *)p.pages.v + head_row * P::kRowBytes;
  w.kv_bytes = 0;
  w.kv_row_bytes = P::kRowBytes;
  w.lds0 = (int)(uintptr_t)(LDS_PTR(uint8_t))(smem);
  w.nxt_end = w.end_even = 0;
  w.pages.k_scale = (const uint8_t *)p.pages.k_scale + (CODED ? head_row : 0);
  w.pages.v_scale = (const uint8_t *)p.pages.v_scale + (CODED ? head_row : 0);
  w.pages.table = p.pages.table + (int64_t)at.b * p.pages.columns;
  w.pages.columns = p.pages.columns;
  w.pages.count = p.pages.pages;
  w.pages.page_log2 = p.pages.page_log2;
  w.pages.page_rows = (uint32_t)p.pages.kv_heads << p.pages.page_log2;
  w.pages.first_key = first_key;
  w.pages.column = first_key >> p.pages.page_log2;
  w.pages.run_row = (w.wave * P::kRows) & ~15;
  w.pages.ids = w.pages.ask(w.pages.column);
  w.pages.ids_next = w.pages.ask(w.pages.column + 64);
#pragma unroll
  for (int j = 0; j < P::kPer; j++) {
    const int in_run = ((w.wave * P::kRows) & 15) + j * P::kStride + w.lane / P::kLanes, pc = w.lane % P::kLanes;
    if constexpr (kThroughRegisters) {
      w.pages.k_src[j] = w.pages.v_src[j] = in_run * P::kRowBytes + pc * 16;
      const int r = w.wave * P::kRows + j * P::kStride + w.lane / P::kLanes, chunk = CODED ? 2 * pc : pc;
      w.pages.k_dst[j] = r * TL::kRowBytes + ((chunk ^ TL::swz_k(r)) << 4);
      w.pages.v_dst[j] = r * TL::kRowBytes + ((chunk ^ (TL::swz_v(r) << 2)) << 4);
    } else {
      w.pages.k_src[j] = in_run * P::kRowBytes + ((pc ^ TL::swz_k(in_run)) << 4);
      w.pages.v_src[j] = in_run * P::kRowBytes + ((pc ^ (TL::swz_v(in_run) << 2)) << 4);
    }
  }

  // ---- Q, then K(0), V(0), K(1).
  const uint16_t *q_ptr = p.q + q_row * D + w.g * 8;
#pragma unroll
  for (int ks = 0; ks < KS; ks++) {
    u32x4 x = {0, 0, 0, 0};
    if (row_ok) x = *reinterpret_cast<const u32x4 *>(q_ptr + ks * 16);
    w.qf[ks] = x;
  }
  typename P::Stage ahead;
  if constexpr (kThroughRegisters) {
    fill_k<D, NW>(w, 0, 0);
    fill_v<D, NW>(w, 0, 0);
    if (end > 1) {
      w.pages.find(1);
      stage_pages<D, NW>(w, w.k_base, w.pages.k_scale, 1, w.pages.k_src, ahead);
    }
    if (end > 0) {
      land_stage<D, NW>(w, smem, w.pages.k_dst, w.pages.k_stage);
      land_stage<D, NW>(w, smem + W::v_slot(0) * TL::kBytes, w.pages.v_dst, w.pages.v_stage);
    }
    if (!W::kOneSlot && end > 1) land_stage<D, NW>(w, smem + TL::kBytes, w.pages.k_dst, ahead);
  } else {
    fill_k<D, NW>(w, 0, 0);
    fill_v<D, NW>(w, 0, 0);
    fill_k<D, NW>(w, 1, 1);
  }

  // ---- per-lane LDS offsets of the operand reads (as the attention kernel lays its tiles out).
#pragma unroll
  for (int ks = 0; ks < KS; ks++) w.k_read[ks] = ln * TL::kRowBytes + (((2 * ks + w.g) ^ TL::swz_k(ln)) << 4);
  const int vq = (w.lane & 15) >> 2, vc = 2 * ((w.lane >> 4) & 1) + ((w.lane & 3) >> 1);
#pragma unroll
  for (int db = 0; db < DB; db++)
    w.v_read[db] = (4 * w.g + vq) * TL::kRowBytes + ((db ^ TL::swz_v(vq)) << 6) + (vc << 4) + ((w.lane & 1) << 3);

  w.positive = p.scale > 0.0f;
  w.c_exp = p.scale * kLog2e;
  w.unit = w.positive ? w.c_exp : 1.0f;
  w.limit = kRescaleAbove / w.unit;
  w.m_run = -1e30f;
  w.l_run = 0.0f;
  const f32x16 zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int db = 0; db < DB; db++) w.acc[db] = zero;

  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  __syncthreads();

  // ---- the key loop: blocks [0, my_end) are this wave's, [0, full) of them crossed by no edge of its rows.
  const int wave_token = tile_first + (int)div_by((uint32_t)(w.wave * kWaveRows), (uint32_t)p.group, p.group_rcp);
  const bool has_rows = wave_token <= last_token && wave_token - tile_first < p.tokens;
  const int my_end = has_rows ? min(end, w.hi_last < 0 ? 0 : w.hi_last / kBkv + 1) : 0;
  float sv[32], nv[32];
  float bm = -INFINITY;
  int seen = 0;
#pragma unroll
  for (int i = 0; i < 32; i++) sv[i] = nv[i] = 0.0f;
  if (my_end > 0) {
    scores<D, NW>(w, smem, 0, sv);
    if (!w.positive) {
#pragma unroll
      for (int i = 0; i < 32; i++) sv[i] *= w.c_exp;
    }
    const uint64_t kbits0 = uniform_bits<D, NW>(w, 0, 0);
    seen = halves_seen<D, NW, false>(w, 0, kbits0);
    if (on_edge<D, NW, false>(w, 0, kbits0)) mask_scores<D, NW, false>(w, 0, kbits0, sv);
    bm = row_max(sv);
  }
  if constexpr (W::kOneSlot) {
    if (end > 1) land_stage<D, NW>(w, smem, w.pages.k_dst, ahead);
  }
  __syncthreads();  // step 0 refills the K slot those scores were read from
  int full = 0;
  if (w.positive) full = min(min(my_end, w.len / kBkv), w.hi_first < 0 ? 0 : (w.hi_first + 1) / kBkv);
  int blk = 0;
  const int lead = min(my_end, w.lo_last <= 0 ? 0 : ((w.lo_last + kBkv - 1) / kBkv + 1) & ~1);
  for (; blk < lead; blk++) edge_step<D, NW, false>(w, smem, blk, my_end, sv, bm, seen);
  for (; blk + 2 < full; blk += 2) {
    hot_step<D, NW, 0>(w, smem, blk, sv, nv, bm);
    hot_step<D, NW, 1>(w, smem, blk + 1, nv, sv, bm);
  }
  for (; blk < my_end; blk++) edge_step<D, NW, false>(w, smem, blk, my_end, sv, bm, seen);
  for (; blk < end; blk++) idle_step<D, NW>(w, smem, blk);

  const Pair lp = both_halves(w.l_run);
  const float l_tot = lp.a + lp.b;
  if (at.splits > 1) {
    // ---- the split's partial state: the accumulator as it stands, the maximum in the exponent's units and the sum.
    if (row_ok) {
      float *part = p.parts + (int64_t)slot * (BQ * (D + 2));
      if (w.g == 0) {
        part[BQ * D + row] = w.positive ? w.m_run * w.c_exp : w.m_run;
        part[BQ * D + BQ + row] = l_tot;
      }
      float *o_ptr = part + row * D + 4 * w.g;
#pragma unroll
      for (int db = 0; db < DB; db++)
#pragma unroll
        for (int c = 0; c < 4; c++)
          *reinterpret_cast<f32x4 *>(o_ptr + 32 * db + 8 * c) =
              f32x4{w.acc[db][4 * c], w.acc[db][4 * c + 1], w.acc[db][4 * c + 2], w.acc[db][4 * c + 3]};
    }
    return;
  }
  // ---- o = acc / l, zeros where no key was seen; the half-waves trade quads so that a lane stores 16 bytes.
  const float inv = 1.0f / (l_tot == 0.0f ? 1.0f : l_tot);
  uint16_t *o_ptr = p.o + q_row * D + 8 * w.g;
#pragma unroll
  for (int db = 0; db < DB; db++) {
#pragma unroll
    for (int c = 0; c < 4; c += 2) {
      uint32_t x[2], y[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        x[e] = pack2<F16>(w.acc[db][4 * c + 2 * e] * inv, w.acc[db][4 * c + 2 * e + 1] * inv);
        y[e] = pack2<F16>(w.acc[db][4 * c + 4 + 2 * e] * inv, w.acc[db][4 * c + 5 + 2 * e] * inv);
      }
      const auto lower = __builtin_amdgcn_permlane32_swap(x[0], y[0], false, false);
      const auto upper = __builtin_amdgcn_permlane32_swap(x[1], y[1], false, false);
      const u32x4 out = {lower[0], upper[0], lower[1], upper[1]};
      if (row_ok) *reinterpret_cast<u32x4 *>(o_ptr + 32 * db + 8 * c) = out;
    }
  }
}

template <int D, int NW, bool F16, bool CODED>
__global__ __launch_bounds__(NW * 64, NW == 1 ? 1 : (D <= 128 ? 2 : 1)) void paged_kernel(PagedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  paged_body<D, NW, F16, CODED>(smem, p);
#endif
}

// The rows of split tiles: each the sum of its splits' states under their common maximum.  A workgroup takes `run` pieces of a
// packed row one after the other, a piece as many heads as a wave has lanes for at eight columns each; its waves take the
// splits in turn, eight states asked for at a time with their maxima (one trip to memory for 32 splits), and the first wave adds up what they
// have, in their order.  A launch that split nothing leaves at once.
template <int D>
constexpr int kMergeHeads = 512 / D;
template <int D, int BQ, bool F16>
__global__ __launch_bounds__(256) void merge_kernel(PagedParams p, int run) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kLanes = D / 8, kAhead = 8;
  __shared__ __attribute__((aligned(16))) f32x4 of_waves[3][64][3];
  const int most = uniform(*p.told);
  if (most == kNoSplits && p.splits == 0) return;
  const int lane = (int)__builtin_amdgcn_workitem_id_x() & 63;
  const int wave = uniform((int)__builtin_amdgcn_workitem_id_x() >> 6);
  const Demand first_demand = demand_of(p, lane);
  const uint32_t pieces = (uint32_t)(p.heads + kMergeHeads<D> - 1) / kMergeHeads<D>;
  const uint32_t from = (uint32_t)__builtin_amdgcn_workgroup_id_x() * (uint32_t)run;
  int row = (int)(from / pieces), piece = (int)(from - (uint32_t)row * pieces), known = -1;
  Place at{};
  for (int i = 0; i < run && row < p.pages.rows; i++) {
    if (row != known) at = place_of<true>(p, row, first_demand, most);
    known = row;
    const int head = piece * kMergeHeads<D> + lane / kLanes, here = min(head, p.heads - 1);
    const int kvh = (int)div_by((uint32_t)here, (uint32_t)p.group, p.group_rcp);
    const int last = at.splits - 1;
    // (Slots past the workspace's: as paged_body.  The branch is the same in all waves.)
    if (at.found && last > 0 && (int64_t)(at.slot + last + 1) * p.pages.kv_heads <= p.slots) {
      const int in_tile = (row - at.s.start - at.tile * p.tokens) * p.group + here - kvh * p.group;
      const int64_t step = (int64_t)p.pages.kv_heads * (BQ * (D + 2));
      const float *part = p.parts + ((int64_t)at.slot * p.pages.kv_heads + kvh) * (BQ * (D + 2));
      const int column = lane % kLanes * 8;
      float m = -1e30f, l = 0.0f, acc[8] = {};
      for (int base = wave * kAhead; base <= last; base += 4 * kAhead) {
        f32x4 x[kAhead][2];
        float ms[kAhead], ls[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {  // one past the last asks for the last again, and weighs nothing
          const float *state = part + min(base + j, last) * step;
          ms[j] = state[BQ * D + in_tile];
          ls[j] = state[BQ * D + BQ + in_tile];
          x[j][0] = *reinterpret_cast<const f32x4 *>(state + in_tile * D + column);
          x[j][1] = *reinterpret_cast<const f32x4 *>(state + in_tile * D + column + 4);
        }
        float top = m;
#pragma unroll
        for (int j = 0; j < kAhead; j++) top = __builtin_fmaxf(top, ms[j]);
        const float keep = fast_exp2(m - top);
        m = top;
        l *= keep;
#pragma unroll
        for (int e = 0; e < 8; e++) acc[e] *= keep;
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
          const float weight = base + j <= last ? fast_exp2(ms[j] - top) : 0.0f;
          l = __builtin_fmaf(ls[j], weight, l);
#pragma unroll
          for (int e = 0; e < 8; e++) acc[e] = __builtin_fmaf(x[j][e / 4][e % 4], weight, acc[e]);
        }
      }
      const int waves = min(4, last / kAhead + 1);  // that had splits
      if (waves > 1) {
        __syncthreads();  // the piece before has been read
        if (wave > 0) {
          of_waves[wave - 1][lane][0] = f32x4{m, l, 0.0f, 0.0f};
          of_waves[wave - 1][lane][1] = f32x4{acc[0], acc[1], acc[2], acc[3]};
          of_waves[wave - 1][lane][2] = f32x4{acc[4], acc[5], acc[6], acc[7]};
        }
        __syncthreads();
        for (int o = 1; o < waves; o++) {
          const f32x4 ml = of_waves[o - 1][lane][0], x0 = of_waves[o - 1][lane][1], x1 = of_waves[o - 1][lane][2];
          const float top = __builtin_fmaxf(m, ml[0]), keep = fast_exp2(m - top), weight = fast_exp2(ml[0] - top);
          m = top;
          l = l * keep + ml[1] * weight;
#pragma unroll
          for (int e = 0; e < 8; e++) acc[e] = acc[e] * keep + (e < 4 ? x0[e % 4] : x1[e % 4]) * weight;
        }
      }
      const float inv = 1.0f / (l == 0.0f ? 1.0f : l);
      u32x4 out;
#pragma unroll
      for (int e = 0; e < 4; e++) out[e] = pack2<F16>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
      if (wave == 0 && head < p.heads) *reinterpret_cast<u32x4 *>(p.o + ((int64_t)row * p.heads + head) * D + column) = out;
    }
    piece++;
    if (piece == (int)pieces) piece = 0, row++;
  }
#endif
}

// ---- the launch.
constexpr int kUnits = 256;  // compute units of an MI355X
// Workgroups of a form that a compute unit holds: by their rings' LDS, of 160 KiB, and for four waves by their registers.
template <int D, int NW, bool CODED>
constexpr int kRing = NW == 1 && kStages<D, NW, CODED> ? 2 * Tile<D>::kBytes : Tile<D>::kLds;
constexpr int least(int a, int b) { return a < b ? a : b; }
template <int D, int NW, bool CODED>
constexpr int kResident = NW == 1 ? least(160 * 1024 / kRing<D, NW, CODED>, D == 64 ? 8 : 4) : (D <= 128 ? 2 : 1);

[[maybe_unused]] uint32_t rcp_of(uint32_t d) { return d <= 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / d); }

// Tiles there may be, of one KV head: every sequence's last may be short, and none is empty.
[[maybe_unused]] int64_t tiles_at_most(const PagedArgs &a) {
  const int64_t tokens = paged_tile_rows(a) / (a.heads / a.pages.kv_heads), rows = a.pages.rows;
  return rows < rows / tokens + a.pages.batch ? rows : rows / tokens + a.pages.batch;
}

template <int D, int NW, bool F16, bool CODED>
hipError_t launch(const PagedArgs &a, hipStream_t stream) {
  constexpr int BQ = NW * kWaveRows;
  PagedParams p{};
  p.pages = a.pages;
  p.q = (const uint16_t *)a.q;
  p.o = (uint16_t *)a.o;
  p.parts = a.workspace;
  p.heads = a.heads;
  p.group = a.heads / a.pages.kv_heads;
  p.group_rcp = rcp_of(p.group);
  p.tokens = BQ / p.group;
  p.tokens_rcp = rcp_of(p.tokens);
  p.causal = a.causal;
  p.win_left = a.win_left;
  p.win_right = a.win_right;
  p.scale = a.scale;
  p.splits = a.splits;
  p.places = kUnits * kResident<D, NW, CODED>;
  p.crowd = NW == 1 ? 1.0f : 1.25f;
  p.states = (float)((double)a.pages.rows * a.heads * (D + 2) * 8 / 7e6);  // written and read at 5 MB a us, 1.4 us a step
  const int64_t slots = paged_slots(a);
  p.slots = (int32_t)slots;
  p.told = reinterpret_cast<int32_t *>(p.parts + slots * paged_slot_floats(a));
  const int64_t grid = paged_workgroups(a);
  hipError_t e = Launch<paged_kernel<D, NW, F16, CODED>>::run(grid, NW * 64, kRing<D, NW, CODED>, kRing<D, NW, CODED>, stream, p);
  if (e != hipSuccess || slots == 0) return e;
  const int64_t pieces = (int64_t)a.pages.rows * ((a.heads + kMergeHeads<D> - 1) / kMergeHeads<D>), at_once = (int64_t)kUnits * 8;
  const int run = (int)((pieces + at_once - 1) / at_once);
  return Launch<merge_kernel<D, BQ, F16>>::run((pieces + run - 1) / run, 256, 0, 0, stream, p, run);
}

template <int D>
hipError_t launch_head(const PagedArgs &a, hipStream_t stream) {
  const bool coded = a.pages.k_scale != nullptr;
  if (paged_tile_rows(a) == 32) {
    if (a.pages.f16) return coded ? launch<D, 1, true, true>(a, stream) : launch<D, 1, true, false>(a, stream);
    return coded ? launch<D, 1, false, true>(a, stream) : launch<D, 1, false, false>(a, stream);
  }
  if (a.pages.f16) return coded ? launch<D, 4, true, true>(a, stream) : launch<D, 4, true, false>(a, stream);
  return coded ? launch<D, 4, false, true>(a, stream) : launch<D, 4, false, false>(a, stream);
}

}  // namespace

// The library's build compiles this file once per head size (SVODK_HEAD), side by side, and once for the rest (0).
#if SVODK_HEAD == 64
hipError_t launch_paged_d64(const PagedArgs &a, hipStream_t stream) { return launch_head<64>(a, stream); }
#elif SVODK_HEAD == 128
hipError_t launch_paged_d128(const PagedArgs &a, hipStream_t stream) { return launch_head<128>(a, stream); }
#elif SVODK_HEAD == 256
hipError_t launch_paged_d256(const PagedArgs &a, hipStream_t stream) { return launch_head<256>(a, stream); }
#else
int paged_tile_rows(const PagedArgs &a) {
  const int64_t group = a.heads / a.pages.kv_heads;
  return group <= 32 && a.pages.rows * group <= 32ll * a.pages.batch ? 32 : 128;
}

// An item of its own for each tile, and for each split there may be (paged_slots counts those of split tiles).
int64_t paged_workgroups(const PagedArgs &a) {
  const int64_t tiles = tiles_at_most(a) * a.pages.kv_heads;
  return a.splits > 1 ? tiles * a.splits : tiles + paged_slots(a);
}

int64_t paged_workspace(const PagedArgs &a) {
  const int64_t slots = paged_slots(a);
  return slots == 0 ? 0 : slots * paged_slot_floats(a) * 4 + 16;
}

int64_t paged_slot_floats(const PagedArgs &a) { return (int64_t)paged_tile_rows(a) * (a.pages.d + 2); }

int64_t paged_slots(const PagedArgs &a) {
  if (a.splits == 1) return 0;
  const int64_t blocks = (((int64_t)a.pages.columns << a.pages.page_log2) + kBkv - 1) / kBkv;
  if (a.splits > 1) return blocks > 1 ? tiles_at_most(a) * a.pages.kv_heads * a.splits : 0;
  // A tile of b blocks is split where b > n, the blocks an item may have, into fewer than 2 b / n: over all tiles fewer than
  // twice what fills the chip.  (And 2 for n's rounding.)
  if (blocks <= kLeastBlocks) return 0;
  const bool coded = a.pages.k_scale != nullptr;
  const int resident = paged_tile_rows(a) != 32 ? (a.pages.d <= 128 ? 2 : 1)
                       : a.pages.d == 64        ? (coded ? kResident<64, 1, true> : kResident<64, 1, false>)
                       : a.pages.d == 128       ? (coded ? kResident<128, 1, true> : kResident<128, 1, false>)
                                                : (coded ? kResident<256, 1, true> : kResident<256, 1, false>);
  return 2ll * kUnits * resident + 2;
}

hipError_t launch_paged(const PagedArgs &a, hipStream_t stream) {
  switch (a.pages.d) {
    case 64: return launch_paged_d64(a, stream);
    case 128: return launch_paged_d128(a, stream);
    case 256: return launch_paged_d256(a, stream);
    default: return hipErrorInvalidValue;
  }
}

const char *paged_config(const PagedArgs &a) {
  if (paged_tile_rows(a) == 32) return a.pages.k_scale ? "PagedCfg { rows: 32, keys: 64, e4m3 }" : "PagedCfg { rows: 32, keys: 64 }";
  return a.pages.k_scale ? "PagedCfg { rows: 128, keys: 64, e4m3 }" : "PagedCfg { rows: 128, keys: 64 }";
}
#endif

}  // namespace svodk
