// What the kernels of attention over pages share: a launch's parameters, the deal of its work, and the pages of a wave's keys.
//
// How many tokens each sequence has is device data.  Every wave works the launch's deal out for itself, a lane a sequence.  A
// tile of query rows has parts: one, or as many as make its parts short enough to keep the chip busy, or one a key block.  The
// parts of a KV head are numbered sequence by sequence, a tile's next to each other, and a workgroup takes a run of them: one part, or, of
// parts of a block, an even share of all.  So it finds its own from sums over the lanes.  The host knows bounds only
// (paged_workgroups), and workgroups past the last part leave at once.
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
  int32_t *told;        // behind them: the deal, for the merge of tiles of 128 rows
  uint64_t *arrivals;   // or a word a workgroup, for those of few rows, of any content
  uint64_t tag;         // the launch's
  int32_t columns, pages, page_log2;
  int32_t heads, group;
  uint32_t group_rcp;
  int32_t causal, win_left, win_right;
  float scale;
  int32_t splits;        // as in PagedArgs
  int32_t slots;         // partial states there is room for
  int32_t shares;        // whether workgroups may take shares of all blocks: few rows, and tiles for more than half of the chip's places
  // Of parts_of_all(): the fewest blocks of a part, the workgroups that the chip holds at a time, and how many times as many parts there may
  // be; and in us a block of a workgroup by itself and with company on its compute unit, a state of every row, a block's bytes at
  // the rate that memory gives, and a block of a workgroup among as many as there are places, when it is the last and when all are busy.
  float least, turn;  // turn: 1 over the blocks that a workgroup takes at a time
  int32_t places, spread, rounds;  // spread: of the places, those that parts go to where there are tiles for a quarter of them or fewer
  float step, crowded, states, stream, tail, even;
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
// The same, of which the compiler knows nothing: what a turn works out from it is not kept in registers from one to the next.
__device__ __forceinline__ int lane_of_turn() {
  int lane = lane_id();
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+v"(lane));
#endif
  return lane;
}

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

constexpr float kStart = 5.0f, kMerge = 5.0f;  // us: from a part's place to its first block, and the merge
// A share of all blocks: how much of the time of uneven tiles its blocks take, its own start and its two merges in us, and a tile's start in it.
// (Fitted, with PagedParams' tail and even, on 98 calls of a token each of 30 to 128 sequences of 500 to 8000 keys, whole and in shares.  Over 48 that
// it was not fitted on, of 40 to 200 sequences of 100 to 9000 keys, head sizes 64, 128 and 256, both kinds of pools, tiles of 16 and 32 rows
// and a window, what is chosen is 0.7 % over the better of whole and chosen on average and 7.6 % at most, 200 sequences of 500 to 2500 keys, 8
// KV heads of 128 in codes, 143 us where whole is 133; whole throughout would be 11 % over.  Shares win where lengths differ and are long: 40
// sequences of 1600 to 8000 keys whole 197 us, 148 in shares; of 110 to 1100 keys 28.6 and 35.  It knows nothing of a chunk, whose many
// tiles read the same keys: one of 2048 beside 255 tokens over 600 keys, 16 query heads over 8 of 128, takes 480 in shares and 296 whole.)
constexpr float kShareOf = 0.8f, kShare = 14.0f, kShareTile = 9.0f;
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

constexpr int kNoSplits = 0x7fffffff;  // a part's blocks where no tile is split
// The blocks that a part of a split tile has at most, and the parts that a workgroup takes: more than one are of a block each.
struct Parts {
  int most, run;
};
// A tile's parts.  (The estimate is off by one at most: there are no more parts than places.)
__device__ __forceinline__ int parts_of(const PagedParams &p, int blocks, const Parts &parts) {
  if (p.splits != 0) return max(1, min(p.splits, blocks));
  if (parts.run > 1) return max(blocks, 1);
  if (parts.most == kNoSplits) return 1;
  const int up = blocks + parts.most - 1;
  int n = (int)((float)up * __builtin_amdgcn_rcpf((float)parts.most));
  n -= n * parts.most > up ? 1 : 0;
  n += up - n * parts.most >= parts.most ? 1 : 0;
  return max(n, 1);
}
// W blocks of all tiles in parts of n are W / n + tiles parts at most.  With a tile for half of the chip's places or fewer, n is what
// keeps all parts on places at once (a few more than there are places would wait for a whole round; and as many fewer leave compute units
// with one where others have two: 2 sequences of 4700 keys, 8 KV heads of 128, in 192 parts 16.6 us, 320 18.2, 512 16.9), or, of tiles of 128 rows, what
// fills two rounds where that comes out ahead: parts of a tile for a third of the places or more fit one round badly (chunks of 591 and 340
// over 17526 and 10077 keys, 32 heads over 8, 290 us in one round, 243 in two).  With more tiles
// they are whole, but: where rows are few and the lengths differ so much or leave a last round so empty that it pays, every place
// takes an even share of all blocks, in which a few tiles begin and end; of tiles of 128 rows, which want their sequence's
// others beside them in the same L2 (4 chunks of 2048 over 16384 keys 964 us, 1072 in shares), only those are split that are more than
// twice what a place has of all blocks.  Splitting has to win back its merge and the states that it writes and reads, a
// share the start of every tile in it.
// This stands in front of a workgroup's first load, and what it costs is its length: a launch's instructions come from memory the
// first time.  (Five counts of parts weighed against each other, by sums over the lanes each, were 1.3 us where this is 0.5.)
template <bool SHARES>
__device__ __forceinline__ Parts parts_of_all(const Deal &deal, const PagedParams &p, const Demand &first) {
  Parts parts = {kNoSplits, 1};
  if (p.splits != 0) return parts;
  const int lane = lane_id();
  int work = 0, longest = 0, tiles = 0;
  for (int base = 0; base < deal.batch; base += 64) {
    const Demand d = base == 0 ? first : demand_of(deal, base + lane);
    work += d.tiles * max(d.blocks, 1);
    longest = max(longest, d.tiles > 0 ? d.blocks : 0);
    tiles += d.tiles;
  }
  const int blocks = last_lane(sum_to(work));  // of a KV head's tiles
  const float heads = (float)deal.kv_heads, places = (float)p.places, a_place = __builtin_amdgcn_rcpf(places);
  const float all = heads * (float)blocks, units = heads * (float)last_lane(sum_to(tiles));
  const float most = (float)last_lane(fold_to_lane(longest, [](int a, int b) { return max(a, b); }));
  const float stream = all * p.stream;
  if (units * 2.0f <= places) {
    const float spread = units * 4.0f <= (float)p.spread ? (float)p.spread : places;
    float best = __builtin_fmaxf(most * p.step, stream);
    for (int round = 1; round <= p.rounds; round++) {
      // What keeps the parts to the places whatever the lengths: a part a tile too many; fewer where the lengths go up, or where with half a part
      // a tile too many the longest take fewer turns.
      const float all_places = spread * (float)round;
      auto fewest = [&](float slack) {
        return __builtin_fmaxf(p.least, __builtin_ceilf(all * __builtin_amdgcn_rcpf(all_places - slack * units) * (1.0f + 1e-6f)));
      };
      auto fit = [&](float n) {
        const Parts tried = {(int)n, 1};
        int count = 0;
        for (int base = 0; base < deal.batch; base += 64) {
          const Demand d = base == 0 ? first : demand_of(deal, base + lane);
          count += d.tiles * parts_of(p, d.blocks, tried);
        }
        return heads * (float)last_lane(sum_to(count)) <= all_places;
      };
      float n = fewest(1.0f);
      const float tight = fewest(0.0f), half = fewest(0.5f);
      if (fit(tight))
        n = tight;
      else if (__builtin_ceilf(half * p.turn) < __builtin_ceilf(n * p.turn) && fit(half))
        n = half;
      const float split = __builtin_fmaxf(n * (float)round * p.crowded, stream) + kMerge + p.states * (all * __builtin_amdgcn_rcpf(n * units) + 1.0f);
      if (n < most && split < best) best = split, parts.most = (int)n;
    }
  } else if (!SHARES) {
    const float n = __builtin_fmaxf(p.least, __builtin_ceilf(2.0f * all * a_place * (1.0f + 1e-6f)));
    const float rest = all * a_place * p.crowded;
    if (p.slots > 0 && n < most && rest + 0.5f * n * p.crowded + kMerge + p.states * (all * __builtin_amdgcn_rcpf(n * units) + 1.0f) < most * p.step)
      parts.most = (int)n;
  } else if constexpr (SHARES) {
    const int share = p.places / deal.kv_heads > 0 ? (blocks + p.places / deal.kv_heads - 1) / (p.places / deal.kv_heads) : blocks;
    const float even = all * a_place * p.even;
    const float whole = kStart * __builtin_ceilf(units * a_place) + __builtin_fmaxf(most * p.tail, even);
    const float shared = kShareOf * even + kShare + kShareTile * units * a_place;
    if (p.slots > 0 && share > 1 && shared < whole) parts.run = share;
  }
  return parts;
}

// Where a part of a KV head, or a packed row, is in the deal.
struct Place {
  int b, tile;
  int part, parts;   // of the tile's
  int tile_at;       // the number of its first part
  Sequence s;
  bool found;
};
// Rows up to which a tile is a stream of keys (paged_few.h), whatever the call's form.
constexpr int kFewRows = 16;
// The part of number `at`; or, with BY_ROW, the tile of packed row `at`.  CHUNKS: the parts of sequences of more than kFewRows
// rows come first.  They are what holds such a launch, and at its front they get compute units of their own, and those of
// few rows the places beside them.
template <bool BY_ROW, bool CHUNKS>
__device__ __forceinline__ Place place_of(const Deal &deal, const PagedParams &p, int at, const Demand &first, const Parts &all) {
  const int lane = lane_id();
  Place x{};
  const int few = CHUNKS ? (int)over(kFewRows, (uint32_t)p.group, p.group_rcp) : 0;  // tokens
  auto in_front = [&](const Demand &d) { return CHUNKS && d.fresh > few; };
  int chunks = 0;  // the parts in front
  if (CHUNKS)
    for (int base = 0; base < deal.batch; base += 64) {
      const Demand d = base == 0 ? first : demand_of(deal, base + lane);
      chunks += last_lane(sum_to(in_front(d) ? d.tiles * parts_of(p, d.blocks, all) : 0));
    }
  int before_front = 0, before = chunks;
  for (int base = 0; base < deal.batch; base += 64) {
    const Demand d = base == 0 ? first : demand_of(deal, base + lane);
    const int parts = parts_of(p, d.blocks, all), sum = d.tiles * parts;
    const bool front = in_front(d);
    const int to = before + sum_to(front ? 0 : sum), to_front = CHUNKS ? before_front + sum_to(front ? sum : 0) : 0;
    const int end = front ? to_front : to;  // of the lane's own parts
    const uint64_t here = BY_ROW ? __builtin_amdgcn_ballot_w64(d.start <= at && at - d.start < d.fresh)
                                 : __builtin_amdgcn_ballot_w64(end > at && end - sum <= at);
    if (here != 0) {
      const int at_lane = __builtin_ctzll(here);
      x.b = base + at_lane;
      x.parts = __builtin_amdgcn_readlane(parts, at_lane);
      x.s.start = __builtin_amdgcn_readlane(d.start, at_lane);
      x.s.fresh = __builtin_amdgcn_readlane(d.fresh, at_lane);
      x.s.len = __builtin_amdgcn_readlane(d.len, at_lane);
      const int tiles = __builtin_amdgcn_readlane(d.tiles, at_lane), start = __builtin_amdgcn_readlane(end - sum, at_lane);
      int order;  // the last tile, which sees the most keys, comes first
      if (BY_ROW) {
        x.tile = (int)over((uint32_t)(at - x.s.start), (uint32_t)deal.tokens, deal.tokens_rcp);
        order = tiles - 1 - x.tile;
      } else {
        const int within = at - start;
        order = x.parts == 1 ? within : (int)((uint32_t)within / (uint32_t)x.parts);
        x.part = within - order * x.parts;
        x.tile = tiles - 1 - order;
      }
      x.tile_at = start + order * x.parts;
      x.found = true;
      return x;
    }
    before = last_lane(to);
    if (CHUNKS) before_front = last_lane(to_front);
  }
  return x;
}

// What a workgroup does: parts [at, to) of a KV head.  The KV heads of a part are neighbours in the launch, their pages are
// neighbours in memory.
struct Turn {
  int kvh, mine, at;
  Parts parts;
  Demand first;
  __device__ __forceinline__ void whose(const Deal &deal) {
    const uint32_t wg = __builtin_amdgcn_workgroup_id_x();
    mine = (int)over(wg, (uint32_t)deal.kv_heads, deal.kvh_rcp);
    kvh = (int)(wg - (uint32_t)mine * (uint32_t)deal.kv_heads);
  }
  __device__ __forceinline__ int to() const { return mine * parts.run + parts.run; }
};
template <bool SHARES>
__device__ __forceinline__ Turn turn_of(const Deal &deal, const PagedParams &p) {
  Turn t;
  t.whose(deal);
  t.first = demand_of(deal, lane_id());
  t.parts = parts_of_all<SHARES>(deal, p, t.first);
  t.at = t.mine * t.parts.run;
  // The merge's kernel goes by the same deal: it is told what this launch went by.
  if (p.told != nullptr && __builtin_amdgcn_workgroup_id_x() == 0 && __builtin_amdgcn_workitem_id_x() == 0) p.told[0] = t.parts.most, p.told[1] = t.parts.run;
  return t;
}
// The workgroups that have a tile of several parts: one a part, or those in whose shares it lies; and the slots of their partial
// states, one a workgroup, or two where they take shares, of the tile that a share begins in and of the one that it ends in.
struct Sharers {
  int first, last;    // workgroups of the KV head
  int64_t slot, next; // the first one's, and the second one's
  int step;           // from there on
  // Whether all of them are in the launch, with slots.  (Starts that descend give more tiles than there are rows, whose last have none.  A tile
  // that some could count themselves in for and others not would leave its word between two counts for the next replay.)
  __device__ bool fit(int slots) const {
    return first >= 0 && last >= first && (last == first ? slot : next + (int64_t)(last - first - 1) * step) < slots;
  }
};
__device__ __forceinline__ Sharers sharers_of(const Deal &deal, const Place &at, int kvh, const Parts &parts) {
  Sharers x;
  x.first = parts.run > 1 ? at.tile_at / parts.run : at.tile_at;
  x.last = parts.run > 1 ? (at.tile_at + at.parts - 1) / parts.run : at.tile_at + at.parts - 1;
  const int each = parts.run > 1 ? 2 : 1;
  x.slot = ((int64_t)x.first * deal.kv_heads + kvh) * each + (at.tile_at != x.first * parts.run ? 1 : 0);
  x.next = ((int64_t)(x.first + 1) * deal.kv_heads + kvh) * each;
  x.step = deal.kv_heads * each;
  return x;
}
// A tile's parts from the first of a turn's on, as many as the turn has left of them.
struct Work {
  Place at;
  int kvh;
  int taken;             // of the tile's parts
  bool whole;
  Sharers sharers;       // of a tile that is not whole
  int64_t slot;          // and where its partial state goes
  bool some;
  int first, end;        // its key blocks
  int tile_first, last;  // the tile's first token, and its last, of the sequence's new ones
};
template <bool SHARES, bool CHUNKS>
__device__ __forceinline__ Work work_of(const Deal &deal, const PagedParams &p, const Turn &t) {
  Work w{};
  w.kvh = t.kvh;
  w.at = place_of<false, CHUNKS>(deal, p, t.at, t.first, t.parts);
  if (!w.at.found) return w;
  w.taken = SHARES ? min(w.at.parts - w.at.part, t.to() - t.at) : 1;
  w.whole = w.taken == w.at.parts;
  w.some = true;
  if (!w.whole) {
    w.sharers = sharers_of(deal, w.at, t.kvh, t.parts);
    const int which = t.mine - w.sharers.first;
    w.slot = which == 0 ? w.sharers.slot : w.sharers.next + (int64_t)(which - 1) * w.sharers.step;
    w.some = w.sharers.fit(p.slots);
  }
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
  if (!w.whole) {
    const int n = end - first;
    if (SHARES && t.parts.run > 1) {
      // A part a block, of as many as the sequence's longest tile has.
      end = first + min(n, w.at.part + w.taken);
      first += min(n, w.at.part);
    } else {
      // An even share of the tile's blocks, the first parts' one more where they do not go up.
      const int each = n / w.at.parts, more = n - each * w.at.parts;
      first += w.at.part * each + min(w.at.part, more);
      end = first + each + (w.at.part < more ? 1 : 0);
    }
  }
  w.first = uniform(first);
  w.end = uniform(end);
  return w;
}

// The first key that a row of the tile sees.
__device__ __forceinline__ int lowest_key(const PagedParams &p, const Work &w) {
  return p.win_left >= 0 ? max(0, w.at.s.base() + w.tile_first - p.win_left) : 0;
}

// A lane's query row of a tile: query head row % group of the KV head's, of the tile's token row / group.  The keys [lo, hi] it
// sees ascend with the row; rows past the last token stand in for it.  A token in front of its sequence's first (a length short of
// its new rows) sees none, whatever the mask.
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
  r.hi = pos < 0 ? -1 : max(hi, -1);
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
// A word of arrivals: its low bits count, the others are the launch's tag.  Words are on lines of their own.
constexpr int kPagedCountBits = 20, kPagedWord = 16;
constexpr uint64_t kPagedEnded = (1 << kPagedCountBits) - 1, kPagedTags = (uint64_t)-1 >> kPagedCountBits;
// The form of few rows (paged_few_kernel.hip), and its workgroups that a compute unit holds at a time.
hipError_t launch_paged_few(const PagedArgs &a, const PagedLaunch &l, hipStream_t stream);
int paged_few_resident(int d, int rows);

}  // namespace svodk
