// What the kernels of attention over pages share: a launch's parameters, the deal of its work, and the pages of a wave's keys.
//
// How many tokens each sequence has is device data.  Every wave works the launch's deal out for itself, a lane a sequence: the
// tiles and key blocks of all sequences give the blocks an item may have, a tile of more blocks is split, items are numbered
// sequence by sequence, a tile's splits next to each other, and a workgroup finds its item from sums over the lanes.  The host
// knows bounds only (paged_workgroups), and workgroups past the last item leave at once.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "kernels.h"
#include "pages.h"

namespace svodk {

// What the deal goes by.  A launch has these as arguments of their own, which arrive in registers with the wave.
struct Deal {
  const void *lens, *starts;
  int batch, wide;        // wide: bit 0 lens, bit 1 starts are 64-bit
  int limit, rows;        // the most tokens a table holds, the packed rows
  int tokens;             // of a tile: as many as have their group's rows in it
  uint32_t tokens_rcp;
  int window_blocks;      // the most key blocks a window leaves a tile
  int kv_heads;
  uint32_t kvh_rcp;
};
#define SVODK_DEAL_PARAMS                                                                                                   \
  uint64_t deal_lens, uint64_t deal_starts, uint32_t deal_batch, uint32_t deal_wide, uint32_t deal_limit,                   \
      uint32_t deal_rows, uint32_t deal_tokens, uint32_t deal_tokens_rcp, uint32_t deal_window_blocks,                      \
      uint32_t deal_kv_heads, uint32_t deal_kvh_rcp
#define SVODK_DEAL                                                                                                          \
  Deal {                                                                                                                    \
    (const void *)deal_lens, (const void *)deal_starts, (int)deal_batch, (int)deal_wide, (int)deal_limit, (int)deal_rows,   \
        (int)deal_tokens, deal_tokens_rcp, (int)deal_window_blocks, (int)deal_kv_heads, deal_kvh_rcp                        \
  }
#define SVODK_DEAL_ARGS(d)                                                                                                  \
  (uint64_t)(uintptr_t)(d).lens, (uint64_t)(uintptr_t)(d).starts, (uint32_t)(d).batch, (uint32_t)(d).wide,                  \
      (uint32_t)(d).limit, (uint32_t)(d).rows, (uint32_t)(d).tokens, (d).tokens_rcp, (uint32_t)(d).window_blocks,           \
      (uint32_t)(d).kv_heads, (d).kvh_rcp

struct PagedParams {
  const uint16_t *q;
  uint16_t *o;
  const void *k, *v, *k_scale, *v_scale;
  const int32_t *table;
  float *parts;
  int32_t *told;  // behind them: the blocks an item had
  int32_t columns, pages, page_log2;
  int32_t heads, group;
  uint32_t group_rcp;
  int32_t causal, win_left, win_right;
  float scale;
  int32_t splits;        // as in PagedArgs
  int32_t slots;         // partial states there is room for
  // Of blocks_an_item(): the fewest blocks of an item, the workgroups that the chip holds at a time; and in us a block of a
  // workgroup by itself and with company on its compute unit, a state of every row, and a block's bytes at the rate that memory gives.
  float least;
  int32_t places;
  float step, crowded, states, stream;
};

namespace {

constexpr int kKeys = 64;  // of a key block

// A value that every lane of a wave has, in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// n / d for n < 2^32 with rcp = floor(2^32 / d) (2^32 - 1 for d = 1): the estimate is the quotient or one less.
__device__ __forceinline__ uint32_t over(uint32_t n, uint32_t d, uint32_t rcp) {
  const uint32_t q = __umulhi(n, rcp);
  return n - q * d >= d ? q + 1 : q;
}
__device__ __forceinline__ int last_lane(int x) { return __builtin_amdgcn_readlane(x, 63); }
__device__ __forceinline__ int lane_id() { return (int)__builtin_amdgcn_workitem_id_x() & 63; }

// x folded over the lanes up to and with this one, with `op` of a lane's value and the one before it; op(0, x) is x.
template <typename T, typename Op>
__device__ __forceinline__ T fold_to_lane(T x, Op op) {
#if defined(__HIP_DEVICE_COMPILE__)
#define SVODK_MOVED(CTRL, ROWS, ZERO) __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, ZERO))
  x = op(x, SVODK_MOVED(0x111, 0xf, true));  // row_shr:1
  x = op(x, SVODK_MOVED(0x112, 0xf, true));
  x = op(x, SVODK_MOVED(0x114, 0xf, true));
  x = op(x, SVODK_MOVED(0x118, 0xf, true));
  x = op(x, SVODK_MOVED(0x142, 0xa, false));  // row_bcast:15 into rows 1 and 3
  x = op(x, SVODK_MOVED(0x143, 0xc, false));  // row_bcast:31 into rows 2 and 3
#undef SVODK_MOVED
#endif
  return x;
}
__device__ __forceinline__ int sum_to(int x) {
  return fold_to_lane(x, [](int a, int b) { return a + b; });
}

constexpr float kMerge = 5.0f;  // us, the merge's launch
// What a lane's sequence asks for: tiles of query rows, and the key blocks of one of its tiles at most.
struct Demand {
  int start, fresh, len;  // as in Sequence
  int tiles, blocks;
};
// A 32- or 64-bit integer's halves held in [0, most].
__device__ __forceinline__ int held(int lo, int hi, bool wide, int most) {
  const int n = wide ? (hi < 0 ? 0 : (hi > 0 || lo < 0 ? 0x7fffffff : lo)) : lo;
  return min(max(n, 0), most);
}
__device__ __forceinline__ Demand demand_of(const Deal &d, int b) {
  // Everything is asked for at once: no load stands under a branch.
  const int at = min(b, d.batch - 1);
  const bool lw = (d.wide & 1) != 0, sw = (d.wide & 2) != 0;
  const int *l = (const int *)d.lens + (int64_t)at * (lw ? 2 : 1), *s = (const int *)d.starts + (int64_t)at * (sw ? 2 : 1);
  const int l0 = l[0], l1 = l[lw ? 1 : 0], s0 = s[0], s1 = s[sw ? 1 : 0], e0 = s[sw ? 2 : 1], e1 = s[sw ? 3 : 1];
  Demand x;
  x.len = held(l0, l1, lw, d.limit);
  x.start = held(s0, s1, sw, d.rows);
  x.fresh = b < d.batch ? max(held(e0, e1, sw, d.rows) - x.start, 0) : 0;
  x.tiles = x.fresh > 0 ? (int)over((uint32_t)x.fresh - 1, (uint32_t)d.tokens, d.tokens_rcp) + 1 : 0;
  x.blocks = min((x.len + kKeys - 1) / kKeys, d.window_blocks);
  return x;
}

constexpr int kNoSplits = 0x7fffffff;  // an item's blocks where none is split
// A tile's splits where an item has `most` blocks.  (The estimate is off by one at most: there are no more splits than places.)
__device__ __forceinline__ int splits_of(const PagedParams &p, int blocks, int most) {
  if (p.splits != 0) return max(1, min(p.splits, blocks));
  if (most == kNoSplits) return 1;
  const int up = blocks + most - 1;
  int n = (int)((float)up * __builtin_amdgcn_rcpf((float)most));
  n -= n * most > up ? 1 : 0;
  n += up - n * most >= most ? 1 : 0;
  return max(n, 1);
}
// The key blocks an item may have.  W blocks of all tiles in items of n are W / n + tiles items at most.  With a tile for half
// of the chip's places or fewer, n is what keeps all items on places at once (a few more than there are places would wait for a
// whole round); with more, n makes two items a place, which then even out.  Splitting has to win back its merge and
// the states that it writes and reads: it does not for tiles that are short, nor for ones that are alike and many.
// This stands in front of a workgroup's first load, and what it costs is its length: a launch's instructions come from memory the
// first time.  (Five counts of items weighed against each other, by sums over the lanes each, were 1.3 us where this is XX.)
__device__ __forceinline__ int blocks_an_item(const Deal &deal, const PagedParams &p, const Demand &first) {
  if (p.splits != 0) return kNoSplits;
  const int lane = lane_id();
  float work = 0.0f;
  int longest = 0, tiles = 0;
  for (int base = 0; base < deal.batch; base += 64) {
    const Demand d = base == 0 ? first : demand_of(deal, base + lane);
    work += (float)d.tiles * (float)d.blocks;
    longest = max(longest, d.tiles > 0 ? d.blocks : 0);
    tiles += d.tiles;
  }
  const float heads = (float)deal.kv_heads, places = (float)p.places;
  const float blocks = heads * __uint_as_float((uint32_t)last_lane((int)__float_as_uint(fold_to_lane(work, [](float a, float b) { return a + b; }))));
  const float units = heads * (float)last_lane(sum_to(tiles)), most = (float)last_lane(fold_to_lane(longest, [](int a, int b) { return max(a, b); }));
  const bool sparse = units * 2.0f <= places;
  const float n = __builtin_fmaxf(p.least, __builtin_ceilf(blocks * __builtin_amdgcn_rcpf(sparse ? places - units : 2.0f * places) * (1.0f + 1e-6f)));
  // In us: a tile whole, or its items one after the other, as many rounds as there are; and what memory takes.
  const float stream = blocks * p.stream;
  const float whole = __builtin_fmaxf(most * (sparse ? p.step : p.crowded), stream);
  const float split = __builtin_fmaxf(sparse ? n * p.crowded : blocks * __builtin_amdgcn_rcpf(places) * p.crowded + 0.5f * n * p.crowded, stream) +
                      kMerge + p.states * (blocks * __builtin_amdgcn_rcpf(n * units) + 1.0f);
  return n < most && split < whole ? (int)n : kNoSplits;
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
__device__ __forceinline__ Place place_of(const Deal &deal, const PagedParams &p, int item, const Demand &first, int most) {
  const int lane = lane_id();
  const bool splitting = p.splits > 1 || most != kNoSplits;
  Place at{};
  int items_before = 0, slots_before = 0;
  for (int base = 0; base < deal.batch; base += 64) {
    const Demand d = base == 0 ? first : demand_of(deal, base + lane);
    const int splits = splitting ? splits_of(p, d.blocks, most) : 1, items = d.tiles * splits;
    const int items_to = BY_ROW ? 0 : sum_to(items);
    const uint64_t here = BY_ROW ? __builtin_amdgcn_ballot_w64(d.start <= item && item - d.start < d.fresh)
                                 : __builtin_amdgcn_ballot_w64(items_to > item - items_before);
    const int slots = splits > 1 ? items : 0, slots_to = splitting ? sum_to(slots) : 0;
    if (here != 0) {
      const int at_lane = __builtin_ctzll(here);
      at.b = base + at_lane;
      at.splits = __builtin_amdgcn_readlane(splits, at_lane);
      at.s.start = __builtin_amdgcn_readlane(d.start, at_lane);
      at.s.fresh = __builtin_amdgcn_readlane(d.fresh, at_lane);
      at.s.len = __builtin_amdgcn_readlane(d.len, at_lane);
      const int tiles = __builtin_amdgcn_readlane(d.tiles, at_lane);
      int order;  // the last tile, which sees the most keys, comes first
      if (BY_ROW) {
        at.tile = (int)over((uint32_t)(item - at.s.start), (uint32_t)deal.tokens, deal.tokens_rcp);
        order = tiles - 1 - at.tile;
      } else {
        const int within = item - items_before - __builtin_amdgcn_readlane(items_to - items, at_lane);
        order = at.splits == 1 ? within : within / at.splits;
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

// A workgroup's item: the KV heads of one are neighbours in the launch, their pages are neighbours in memory.
struct Work {
  Place at;
  int kvh;
  int slot;  // where its partial state goes, of a split tile
  int first, end;            // its key blocks
  int tile_first, last;      // the tile's first token, and its last, of the sequence's new ones
  bool some;
};
__device__ __forceinline__ Work work_of(const Deal &deal, const PagedParams &p) {
  const uint32_t wg = __builtin_amdgcn_workgroup_id_x();
  Work w{};
  const int item = (int)over(wg, (uint32_t)deal.kv_heads, deal.kvh_rcp);
  w.kvh = (int)(wg - (uint32_t)item * (uint32_t)deal.kv_heads);
  const Demand first_demand = demand_of(deal, lane_id());
  const int most = blocks_an_item(deal, p, first_demand);
  w.at = place_of<false>(deal, p, item, first_demand, most);
  // The merge goes by the same deal: it is told what this launch went by, behind the states.
  if (wg == 0 && __builtin_amdgcn_workitem_id_x() == 0 && p.slots > 0) *p.told = most;
  w.slot = (w.at.slot + w.at.split) * deal.kv_heads + w.kvh;
  // (Slots there is no room for: starts that descend give more rows than there are.)
  w.some = w.at.found && (w.at.splits == 1 || w.slot < p.slots);
  if (!w.some) return w;
  const Sequence &s = w.at.s;
  w.tile_first = w.at.tile * deal.tokens;
  w.last = min(w.tile_first + deal.tokens, s.fresh) - 1;
  int first = 0, end = s.len;  // in keys
  if (p.causal) end = max(0, min(end, s.base() + w.last + 1));
  if (p.win_left >= 0) {
    first = max(0, s.base() + w.tile_first - p.win_left);
    end = max(0, min(end, s.base() + w.last + p.win_right + 1));
  }
  first = min(first / kKeys, (end + kKeys - 1) / kKeys);
  end = (end + kKeys - 1) / kKeys;
  if (w.at.splits > 1) {
    // An even share of the tile's blocks, the first splits' one more where they do not go up.
    const int n = end - first, each = n / w.at.splits, more = n - each * w.at.splits;
    first += w.at.split * each + min(w.at.split, more);
    end = first + each + (w.at.split < more ? 1 : 0);
  }
  w.first = uniform(first);
  w.end = uniform(end);
  return w;
}

// A lane's query row of a tile: query head row % group of the KV head's, of the tile's token row / group.  The keys [lo, hi] it
// sees ascend with the row; rows past the last token stand in for it.
struct Row {
  bool there;
  int64_t at;  // of (packed row, head), in heads
  int lo, hi;
};
__device__ __forceinline__ Row row_of_tile(const Deal &deal, const PagedParams &p, const Work &w, int row) {
  Row r;
  const int in_tile = (int)over((uint32_t)row, (uint32_t)p.group, p.group_rcp), token = w.tile_first + in_tile;
  r.there = in_tile < deal.tokens && token <= w.last;
  const int held_token = min(token, w.last), head = w.kvh * p.group + (row - in_tile * p.group);
  r.at = ((int64_t)w.at.s.start + held_token) * p.heads + min(head, p.heads - 1);
  // Positions and reaches are below 2^30: the sums stay in 32 bits.
  const int pos = w.at.s.base() + held_token;
  int lo = 0, hi = w.at.s.len - 1;
  if (p.causal) hi = min(hi, pos);
  if (p.win_left >= 0) lo = max(lo, pos - p.win_left), hi = min(hi, pos + p.win_right);
  r.lo = lo;
  r.hi = max(hi, -1);
  return r;
}

// The pages of 128 columns of a sequence's table from `column` on, a lane each: asked for 64 columns ahead of their use.
struct PageIds {
  const int32_t *table;
  int columns, count;
  int column, ids, ids_next;
  __device__ __forceinline__ int ask(int from) const { return table[min(from + lane_id(), columns - 1)]; }
  __device__ __forceinline__ void begin(const PagedParams &p, int b, int at) {
    table = p.table + (int64_t)b * p.columns, columns = p.columns, count = p.pages;
    column = at;
    ids = ask(at), ids_next = ask(at + 64);
  }
  // To column `at`, less than 64 on from the last.
  __device__ __forceinline__ void go(int at) {
    if (at - column >= 64) {
      column += 64;
      ids = ids_next;
      ids_next = ask(column + 64);
    }
  }
  __device__ __forceinline__ int of(int at) const {
    const int rel = at - column;
    const int id = rel < 64 ? __builtin_amdgcn_readlane(ids, rel) : __builtin_amdgcn_readlane(ids_next, rel & 63);
    return min(max(id, 0), count - 1);
  }
};

}  // namespace

// What a call's launches go by, worked out once.
struct PagedLaunch {
  Deal deal;
  PagedParams p;
  int64_t grid;
};
PagedLaunch paged_launch(const PagedArgs &a);
constexpr int kPagedUnits = 256;  // compute units of an MI355X
// The form of few rows (paged_few_kernel.hip), and its workgroups that a compute unit holds at a time.
hipError_t launch_paged_few(const PagedArgs &a, const PagedLaunch &l, hipStream_t stream);
int paged_few_resident(int d, int rows);

}  // namespace svodk
