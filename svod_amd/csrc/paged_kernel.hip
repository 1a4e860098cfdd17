// Attention over a key/value cache in pages for gfx950 (MI355X): each sequence's new tokens, packed one sequence after the
// other, against its own pages.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(log2(e) scale q_i . k_j - m_i)   over the keys j that row i sees:
//   j below its sequence's length; causal: j no further than the row's own position len - fresh + i; a window: within it.
//
// A tile is the rows of one KV head: whole tokens with all query heads of the head's group beside each other, so that K and
// V are read once a group, and a row's position is that of its token: ranges a row, ascending along the tile.  Two forms:
// this file's, tiles of 128 rows for chunks of tokens, bound by the matrix pipes; and paged_few_kernel.hip's, tiles of 16 or 32
// rows for calls of few rows a sequence (a generated token, a few drafted ones), bound by the stream of K and V.
//
// The key loop here is the attention kernel's (attention_step.h): 64 keys a step through an LDS ring, both products transposed
// on v_mfma_f32_32x32x16 so that a query is a lane, scores, maximum and sum in 32 bits, p rounded to 16 bits for the
// second product.  What is this file's own is how keys come into the ring.  A split leaves its accumulator, maximum and sum
// in f32; merge_kernel adds them up, so a call's result depends on nothing but its inputs.  (4 chunks of 2048 over 12288 to 16384 keys, 16 heads
// over 8 of 128: 960 us, 994 TFLOP/s, over codes 1060; two chunks of 1001 beside 30 tokens, in codes, in a window of 1024: 41 us.)
#include <hip/hip_runtime.h>

#include <algorithm>

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
#include "paged.h"
#include "paged_few.h"

namespace svodk {
namespace {

// ---- keys in pages.  A fill instruction moves 1 KiB, 16 bytes a lane: whole rows of one KV head, 16 of which never lie in two
// pages.  So a wave's fills of a block go by runs of 16 rows, with a page looked up and a descriptor made for each.
template <int D, int NW, unsigned FLAGS>
struct PagesOf {
  static constexpr bool kCodes = (FLAGS & kCoded) != 0;
  static constexpr int kRowBytes = kCodes ? D : 2 * D;
  static constexpr int kLanes = kRowBytes / 16;          // lanes a row
  static constexpr int kRows = 64 / kLanes;              // rows a fill
  static constexpr int kFills = kBkv / kRows / NW;       // a wave's fills of a tile, kStride rows apart
  static constexpr int kStride = NW * kRows;
  static constexpr int kPer = kStride >= 16 ? 1 : 16 / kStride;  // its fills of a run of 16 rows
  static constexpr int kRuns = kFills / kPer;
  static_assert(kFills * kRows * NW == kBkv && kRuns * kPer == kFills && kRows <= 16, "whole fills");
  const uint8_t *k_scale, *v_scale;  // the KV head's rows of page 0 (w.k_base and w.v_base: of the pools)
  PageIds ids;
  int page_log2;
  uint32_t page_rows;                // rows of a page, all KV heads'
  int first_key;                     // the frame's
  int lowest;                        // the first key that a row of the tile sees
  int64_t run[kRuns];                // the pool's row that each of this wave's runs of the block filled last starts at
  int run_row;                       // the first run's row of the block
  int k_src[kPer], v_src[kPer];      // a lane's offset in a run's descriptor (straight into LDS: swizzled)
  int k_dst[kPer], v_dst[kPer];      // where its 16 codes go in a slot, widened: 16 bytes there, 16 at ^ 16
  struct Stage {
    u32x4 rows[kCodes ? kFills : 1];
    uint32_t scale[kCodes ? kFills : 1];
  };
  Stage k_stage, v_stage;
  uint8_t *ring;

  __device__ int row_of(int r) const { return run_row + r * kStride * kPer; }
  // The rows that run r of block n has for the tile, whose keys end at `len`.  None of 16 in front of a window, which are the first
  // block's: a sequence may have given pages away that its window has left.
  template <bool FIRST>
  __device__ int rows_of(int n, int r, int len) const {
    const int key = n * kBkv + row_of(r);
    return !FIRST || key + 16 > lowest ? min(max(len - key, 0), 16) : 0;
  }
  // The runs of block `n` of the frame.
  __device__ void find(int n) {
    const int key0 = first_key + n * kBkv;
    ids.go(key0 >> page_log2);
#pragma unroll
    for (int r = 0; r < kRuns; r++) {
      const int key = key0 + row_of(r);
      run[r] = (int64_t)((uint64_t)(uint32_t)ids.of(key >> page_log2) * page_rows) + (key & ((1 << page_log2) - 1));
    }
  }
};
template <int D, int NW>
struct Pages<D, NW, kPaged> : PagesOf<D, NW, kPaged> {};
template <int D, int NW>
struct Pages<D, NW, kPaged | kCoded> : PagesOf<D, NW, kPaged | kCoded> {};

// A descriptor over `rows` rows of `row_bytes` at `base`: rows from there on read as zeros.
[[maybe_unused]] __device__ __forceinline__ i32x4 rows_rsrc(const uint8_t *base, int rows, int row_bytes) {
  const uint64_t at = (uint64_t)(uintptr_t)base;
  // The same in every lane, and told so: a 64-bit sum that the compiler has on the VALU is no scalar to it.
  return i32x4{uniform((int)(uint32_t)at), uniform((int)(uint32_t)(at >> 32)), uniform(rows * row_bytes), 0x00020000};
}

// This wave's share of block `n` from the pool at `base`, whose runs find() has named, straight into LDS: keys past the length
// land as zeros (a page's last rows hold anything, and 0 times that is not 0).
template <int D, int NW, bool FIRST, bool F16, unsigned FLAGS>
__device__ __forceinline__ void fill_pages(const Wave<D, NW, F16, FLAGS> &w, const uint8_t *base, int n, int lds_at,
                                           const int *src) {
  using P = decltype(w.pages);
#pragma unroll
  for (int r = 0; r < P::kRuns; r++) {
    const int left = w.pages.template rows_of<FIRST>(n, r, w.len);
    const i32x4 rsrc = rows_rsrc(base + w.pages.run[r] * P::kRowBytes, left, P::kRowBytes);
#pragma unroll
    for (int j = 0; j < P::kPer; j++)
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                   :
                   : "s"(lds_at + (w.wave + NW * (r * P::kPer + j)) * 1024), "v"(src[j]), "s"(rsrc)
                   : "memory");
  }
}
// The same of codes: into registers, with their rows' scales.
template <int D, int NW, bool FIRST, bool F16, unsigned FLAGS, typename S>
__device__ __forceinline__ void stage_pages(const Wave<D, NW, F16, FLAGS> &w, const uint8_t *base, const uint8_t *scales, int n,
                                            const int *src, S &stage) {
#if defined(__HIP_DEVICE_COMPILE__)
  using P = decltype(w.pages);
#pragma unroll
  for (int r = 0; r < P::kRuns; r++) {
    const int left = w.pages.template rows_of<FIRST>(n, r, w.len);
    const auto rows = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base + w.pages.run[r] * P::kRowBytes), 0,
                                                        left * P::kRowBytes, 0x00020000);
#pragma unroll
    for (int j = 0; j < P::kPer; j++) stage.rows[r * P::kPer + j] = __builtin_amdgcn_raw_buffer_load_b128(rows, src[j], 0, 0);
    const auto scale = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(scales + w.pages.run[r]), 0, left, 0x00020000);
#pragma unroll
    for (int j = 0; j < P::kPer; j++)
      stage.scale[r * P::kPer + j] = __builtin_amdgcn_raw_buffer_load_b8(scale, src[j] / P::kRowBytes, 0, 0);
  }
#endif
}
// And from there, widened, into a slot.
template <int D, int NW, bool F16, unsigned FLAGS, typename S>
__device__ __forceinline__ void land_stage(const Wave<D, NW, F16, FLAGS> &w, uint8_t *slot, const int *dst, const S &stage) {
  using P = decltype(w.pages);
#pragma unroll
  for (int i = 0; i < P::kFills; i++) {
    const u32x4 c = stage.rows[i];
    uint8_t *at = slot + (i - i % P::kPer) * P::kStride * Tile<D>::kRowBytes;
    const float scale = scale_of(stage.scale[i]);
    const u32x4 lo = {widen_codes<F16, false>(c[0], scale), widen_codes<F16, true>(c[0], scale),
                      widen_codes<F16, false>(c[1], scale), widen_codes<F16, true>(c[1], scale)};
    const u32x4 hi = {widen_codes<F16, false>(c[2], scale), widen_codes<F16, true>(c[2], scale),
                      widen_codes<F16, false>(c[3], scale), widen_codes<F16, true>(c[3], scale)};
    *reinterpret_cast<u32x4 *>(at + dst[i % P::kPer]) = lo;
    *reinterpret_cast<u32x4 *>(at + (dst[i % P::kPer] ^ 16)) = hi;
  }
}
// Codes are asked for a step ahead of their place in the ring: a step writes what the one before asked for, and asks for the next block's.
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ void fill_k_pages(Wave<D, NW, F16, FLAGS> &w, int n, int slot) {
  if (n >= w.end) return;
  if constexpr ((FLAGS & kCoded) != 0) {
    land_stage<D, NW>(w, w.pages.ring + slot * Tile<D>::kBytes, w.pages.k_dst, w.pages.k_stage);
    if (n + 1 >= w.end) return;
    w.pages.find(n + 1);
    stage_pages<D, NW, false>(w, w.k_base, w.pages.k_scale, n + 1, w.pages.k_src, w.pages.k_stage);
  } else {
    w.pages.find(n);
    fill_pages<D, NW, false>(w, w.k_base, n, w.lds0 + slot * Tile<D>::kBytes, w.pages.k_src);
  }
}
// A block's values come a step behind its keys, which have named its runs.
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ void fill_v_pages(Wave<D, NW, F16, FLAGS> &w, int n, int slot) {
  if (n >= w.end) return;
  if constexpr ((FLAGS & kCoded) != 0) {
    land_stage<D, NW>(w, w.pages.ring + (2 + slot) * Tile<D>::kBytes, w.pages.v_dst, w.pages.v_stage);
    if (n + 1 < w.end) stage_pages<D, NW, false>(w, w.v_base, w.pages.v_scale, n + 1, w.pages.v_src, w.pages.v_stage);
  } else {
    fill_pages<D, NW, false>(w, w.v_base, n, w.lds0 + (2 + slot) * Tile<D>::kBytes, w.pages.v_src);
  }
}

template <int D, int NW, bool F16, bool CODED>
__device__ __forceinline__ void paged_item(uint8_t *smem, const Deal &deal, const PagedParams &p, const Work &work) {
  using TL = Tile<D>;
  using W = Wave<D, NW, F16, kRanged | kPaged | (CODED ? kCoded : 0u)>;
  using P = decltype(W::pages);
  constexpr int BQ = NW * kWaveRows, KS = W::KS, DB = W::DB;
  W w;
  w.lane = lane_of_turn();
  w.wave = uniform((int)__builtin_amdgcn_workitem_id_x() >> 6);
  w.g = w.lane >> 5;
  const int ln = w.lane & 31;

  const int row = w.wave * kWaveRows + ln;
  const Row mine = row_of_tile(deal, p, work, row);
  // From here on in the item's own frame: keys count from its first.
  const int first_key = work.first * kBkv, end = work.end - work.first;
  w.end = end;
  w.len = max(work.at.s.len - first_key, 0);
  w.tk = w.len;
  w.key_mask = nullptr;
  w.mask_row = 0;
  w.mask_bytes = 1;
  w.scanned = false;
  w.mask_next = 0;
  w.row_lo = mine.lo - first_key;
  w.row_hi = mine.hi - first_key;
  w.lo_last = __builtin_amdgcn_readlane(w.row_lo, kWaveRows - 1);
  w.lo_first = __builtin_amdgcn_readlane(w.row_lo, 0);
  w.hi_first = __builtin_amdgcn_readlane(w.row_hi, 0);
  w.hi_last = __builtin_amdgcn_readlane(w.row_hi, kWaveRows - 1);
  w.wave_first_row = w.my_row = 0;
  w.my_row_ok = mine.there;

  // ---- the pages.
  const int64_t head_row = (int64_t)work.kvh << p.page_log2;
  w.k_base = (const uint8_t *)p.k + head_row * P::kRowBytes;
  w.v_base = (const uint8_t *)p.v + head_row * P::kRowBytes;
  w.kv_bytes = 0;
  w.kv_row_bytes = P::kRowBytes;
  w.lds0 = (int)(uintptr_t)(LDS_PTR(uint8_t))(smem);
  w.nxt_end = w.end_even = 0;
  w.pages.k_scale = (const uint8_t *)p.k_scale + (CODED ? head_row : 0);
  w.pages.v_scale = (const uint8_t *)p.v_scale + (CODED ? head_row : 0);
  w.pages.page_log2 = p.page_log2;
  w.pages.page_rows = (uint32_t)deal.kv_heads << p.page_log2;
  w.pages.first_key = first_key;
  w.pages.lowest = lowest_key(p, work) - first_key;
  w.pages.run_row = (w.wave * P::kRows) & ~15;
  w.pages.ids.begin(p, work.at.b, first_key >> p.page_log2);
#pragma unroll
  for (int j = 0; j < P::kPer; j++) {
    const int in_run = ((w.wave * P::kRows) & 15) + j * P::kStride + w.lane / P::kLanes, pc = w.lane % P::kLanes;
    if constexpr (CODED) {
      w.pages.k_src[j] = w.pages.v_src[j] = in_run * P::kRowBytes + pc * 16;
      const int r = w.wave * P::kRows + j * P::kStride + w.lane / P::kLanes, chunk = 2 * pc;
      w.pages.k_dst[j] = r * TL::kRowBytes + ((chunk ^ TL::swz_k(r)) << 4);
      w.pages.v_dst[j] = r * TL::kRowBytes + ((chunk ^ (TL::swz_v(r) << 2)) << 4);
    } else {
      w.pages.k_src[j] = in_run * P::kRowBytes + ((pc ^ TL::swz_k(in_run)) << 4);
      w.pages.v_src[j] = in_run * P::kRowBytes + ((pc ^ (TL::swz_v(in_run) << 2)) << 4);
    }
  }

  // ---- Q, then K(0), V(0), K(1).
  const uint16_t *q_ptr = p.q + mine.at * D + w.g * 8;
#pragma unroll
  for (int ks = 0; ks < KS; ks++) {
    u32x4 x = {0, 0, 0, 0};
    if (mine.there) x = *reinterpret_cast<const u32x4 *>(q_ptr + ks * 16);
    w.qf[ks] = x;
  }
  if constexpr (CODED) {
    w.pages.ring = smem;
    typename P::Stage ahead;
    auto k_of = [&](int n, typename P::Stage &stage) { stage_pages<D, NW, false>(w, w.k_base, w.pages.k_scale, n, w.pages.k_src, stage); };
    auto v_of = [&](int n) { stage_pages<D, NW, false>(w, w.v_base, w.pages.v_scale, n, w.pages.v_src, w.pages.v_stage); };
    if (end > 0) {
      w.pages.find(0);
      stage_pages<D, NW, true>(w, w.k_base, w.pages.k_scale, 0, w.pages.k_src, w.pages.k_stage);
      stage_pages<D, NW, true>(w, w.v_base, w.pages.v_scale, 0, w.pages.v_src, w.pages.v_stage);
    }
    if (end > 1) {
      w.pages.find(1);
      k_of(1, ahead);
    }
    if (end > 0) {
      land_stage<D, NW>(w, smem, w.pages.k_dst, w.pages.k_stage);
      land_stage<D, NW>(w, smem + 2 * TL::kBytes, w.pages.v_dst, w.pages.v_stage);
    }
    // V(1) and K(2), which the first step writes.
    if (end > 1) v_of(1);
    if (end > 2) {
      w.pages.find(2);
      k_of(2, w.pages.k_stage);
    }
    if (end > 1) land_stage<D, NW>(w, smem + TL::kBytes, w.pages.k_dst, ahead);
  } else {
    if (end > 0) {
      w.pages.find(0);
      fill_pages<D, NW, true>(w, w.k_base, 0, w.lds0, w.pages.k_src);
      fill_pages<D, NW, true>(w, w.v_base, 0, w.lds0 + 2 * TL::kBytes, w.pages.v_src);
    }
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

  if constexpr (!CODED) __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  __syncthreads();

  // ---- the key loop: blocks [0, my_end) are this wave's, [0, full) of them crossed by no edge of its rows.
  const int wave_token = (int)over((uint32_t)(w.wave * kWaveRows), (uint32_t)p.group, p.group_rcp);  // of the tile's
  const bool has_rows = wave_token <= work.last - work.tile_first && wave_token < deal.tokens;
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
  for (; blk < end; blk++) idle_step<D, NW>(w, blk);

  const Pair lp = both_halves(w.l_run);
  const float l_tot = lp.a + lp.b;
  if (!work.whole) {
    // ---- the split's partial state: the accumulator as it stands, the maximum in the exponent's units and the sum.
    if (mine.there) {
      float *part = p.parts + work.slot * (BQ * (D + 2));
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
  uint16_t *o_ptr = p.o + mine.at * D + 8 * w.g;
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
      if (mine.there) *reinterpret_cast<u32x4 *>(o_ptr + 32 * db + 8 * c) = out;
    }
  }
}

template <int D, int NW, bool F16, bool CODED>
__global__ __launch_bounds__(NW * 64, D <= 128 ? 2 : 1) void paged_kernel(SVODK_DEAL_PARAMS, PagedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  static_assert(few::Few<D, 1>::kLds <= Tile<D>::kLds, "both forms' LDS");
  const Deal deal = SVODK_DEAL;
  const Work work = work_of<false, true>(deal, p, turn_of<false>(deal, p));
  if (!work.some) return;
  // A sequence of few rows beside chunks is a stream of keys here too: one wave of four with rows would take a step a block.  (30
  // tokens beside two chunks of 1001 in a window of 1024, e4m3: 52.5 us without, 44.4 with this and the chunks in front.)
  if (work.whole && (work.last - work.tile_first + 1) * p.group <= kFewRows)
    few::item<D, 1, F16, CODED, false>(smem, deal, p, work);
  else
    paged_item<D, NW, F16, CODED>(smem, deal, p, work);
#endif
}

// The rows of split tiles: each the sum of its splits' states under their common maximum.  A workgroup takes `run` pieces of a
// packed row one after the other, a piece as many heads as a wave has lanes for at eight columns each; its waves take the
// splits in turn, eight states asked for at a time with their maxima (one trip to memory for 32 splits), and the first wave adds up what they
// have, in their order.  A launch that split nothing leaves at once.
template <int D>
constexpr int kMergeHeads = 512 / D;
template <int D, int BQ, bool F16>
__global__ __launch_bounds__(256) void merge_kernel(SVODK_DEAL_PARAMS, PagedParams p, int run) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kLanes = D / 8, kAhead = 8;
  __shared__ __attribute__((aligned(16))) f32x4 of_waves[3][64][3];
  const Deal deal = SVODK_DEAL;
  const Parts parts = {uniform(p.told[0]), uniform(p.told[1])};
  if (parts.most == kNoSplits && parts.run == 1 && p.splits == 0) return;
  const int lane = lane_id();
  const int wave = uniform((int)__builtin_amdgcn_workitem_id_x() >> 6);
  const Demand first_demand = demand_of(deal, lane);
  const uint32_t pieces = (uint32_t)(p.heads + kMergeHeads<D> - 1) / kMergeHeads<D>;
  const uint32_t from = (uint32_t)__builtin_amdgcn_workgroup_id_x() * (uint32_t)run;
  int row = (int)(from / pieces), piece = (int)(from - (uint32_t)row * pieces), known = -1;
  Place at{};
  for (int i = 0; i < run && row < deal.rows; i++) {
    if (row != known) at = place_of<true, true>(deal, p, row, first_demand, parts);
    known = row;
    const int head = piece * kMergeHeads<D> + lane / kLanes, here = min(head, p.heads - 1);
    const int kvh = (int)over((uint32_t)here, (uint32_t)p.group, p.group_rcp);
    const Sharers sharers = sharers_of(deal, at, kvh, parts);
    const int last = at.found ? sharers.last - sharers.first : 0;
    // (No slots: as work_of(), here for all of the lanes' heads.  The branch is the same in all waves.)
    if (last > 0 && sharers.first >= 0 && sharers.next + (int64_t)(last - 1) * sharers.step - kvh + deal.kv_heads <= p.slots) {
      const int in_tile = (row - at.s.start - at.tile * deal.tokens) * p.group + here - kvh * p.group;
      const int column = lane % kLanes * 8;
      float m = -1e30f, l = 0.0f, acc[8] = {};
      for (int base = wave * kAhead; base <= last; base += 4 * kAhead) {
        f32x4 x[kAhead][2];
        float ms[kAhead], ls[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {  // one past the last asks for the last again, and weighs nothing
          const int which = min(base + j, last);
          const float *state = p.parts + (which == 0 ? sharers.slot : sharers.next + (int64_t)(which - 1) * sharers.step) * (BQ * (D + 2));
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

#if SVODK_HEAD != 0
template <int D, int BQ, bool F16>
hipError_t merge(const PagedLaunch &l, hipStream_t stream) {
  const int64_t pieces = (int64_t)l.deal.rows * ((l.p.heads + kMergeHeads<D> - 1) / kMergeHeads<D>), at_once = (int64_t)kPagedUnits * 8;
  const int run = (int)((pieces + at_once - 1) / at_once);
  return Launch<merge_kernel<D, BQ, F16>>::run((pieces + run - 1) / run, 256, 0, 0, stream, SVODK_DEAL_ARGS(l.deal), l.p, run);
}

template <int D, bool F16, bool CODED>
hipError_t launch(const PagedArgs &a, hipStream_t stream) {
  const int rows = paged_tile_rows(a);
  const PagedLaunch l = paged_launch(a);
  if (rows != 128) return launch_paged_few(a, l, stream);
  const hipError_t e =
      Launch<paged_kernel<D, 4, F16, CODED>>::run(l.grid, 256, Tile<D>::kLds, Tile<D>::kLds, stream, SVODK_DEAL_ARGS(l.deal), l.p);
  return e != hipSuccess || l.p.slots == 0 ? e : merge<D, 128, F16>(l, stream);
}

template <int D>
hipError_t launch_head(const PagedArgs &a, hipStream_t stream) {
  const bool coded = a.pages.k_scale != nullptr;
  if (a.pages.f16) return coded ? launch<D, true, true>(a, stream) : launch<D, true, false>(a, stream);
  return coded ? launch<D, false, true>(a, stream) : launch<D, false, false>(a, stream);
}
#endif

}  // namespace

// The library's build compiles this file once per head size (SVODK_HEAD), side by side, and once for the rest (0).
#if SVODK_HEAD == 64
hipError_t launch_paged_d64(const PagedArgs &a, hipStream_t stream) { return launch_head<64>(a, stream); }
#elif SVODK_HEAD == 128
hipError_t launch_paged_d128(const PagedArgs &a, hipStream_t stream) { return launch_head<128>(a, stream); }
#elif SVODK_HEAD == 256
hipError_t launch_paged_d256(const PagedArgs &a, hipStream_t stream) { return launch_head<256>(a, stream); }
#else
namespace {
uint32_t rcp_of(uint32_t d) { return d <= 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / d); }

// Tiles there may be, of one KV head: every sequence's last may be short, and none is empty.
int64_t tiles_at_most(const PagedArgs &a) {
  const int64_t tokens = paged_tile_rows(a) / (a.heads / a.pages.kv_heads), rows = a.pages.rows;
  return rows < rows / tokens + a.pages.batch ? rows : rows / tokens + a.pages.batch;
}
// Workgroups that a compute unit holds at a time.
int resident(const PagedArgs &a) {
  const int rows = paged_tile_rows(a);
  return rows == 128 ? (a.pages.d <= 128 ? 2 : 1) : paged_few_resident(a.pages.d, rows);
}
int64_t places(const PagedArgs &a) { return (int64_t)kPagedUnits * resident(a); }
// Whether there may be tiles for more than half of the chip's places.
bool dense(const PagedArgs &a) { return 2 * tiles_at_most(a) * a.pages.kv_heads > places(a); }
// The places that parts go to where there are tiles for a quarter of them or fewer: of few rows over 16 bits one workgroup a compute unit,
// which take what the memory gives; codes want the second one's waves beside them.
int64_t spread(const PagedArgs &a) { return paged_tile_rows(a) != 128 && a.pages.k_scale == nullptr ? kPagedUnits : places(a); }
// Rounds of places that parts may take: two where tiles of 128 rows may be for a quarter of the places and more (parts_of_all).
int rounds(const PagedArgs &a) {
  return paged_tile_rows(a) == 128 && !dense(a) && 4 * tiles_at_most(a) * a.pages.kv_heads >= places(a) ? 2 : 1;
}
// Key blocks that a window leaves a tile.
int64_t window_blocks(const PagedArgs &a) {
  const int64_t tokens = paged_tile_rows(a) / (a.heads / a.pages.kv_heads);
  return a.win_left < 0 ? 0x7fffffff : std::min<int64_t>(((int64_t)a.win_left + a.win_right + tokens) / kBkv + 2, 0x7fffffff);
}
int64_t blocks_at_most(const PagedArgs &a) {
  return std::min((((int64_t)a.pages.columns << a.pages.page_log2) + kBkv - 1) / kBkv, window_blocks(a));
}
}  // namespace

int paged_tile_rows(const PagedArgs &a) {
  const int64_t group = a.heads / a.pages.kv_heads, rows = a.pages.rows * group;
  if (group <= 16 && rows <= 16ll * a.pages.batch) return 16;
  return group <= 32 && rows <= 32ll * a.pages.batch && a.pages.d <= 128 ? 32 : 128;
}

// A state a workgroup; two where it may take a share of all blocks, which it does on the chip's places only.
int64_t paged_slots(const PagedArgs &a) {
  const int64_t blocks = blocks_at_most(a), tiles = tiles_at_most(a) * a.pages.kv_heads;
  if (a.splits == 1 || blocks <= 1) return 0;
  if (a.splits > 1) return tiles * a.splits;
  const bool few = paged_tile_rows(a) != 128;
  // A state for each of many tiles of 128 rows would be gigabytes, where none is more than a small part of the launch.
  if (!few && tiles > 4 * places(a)) return 0;
  // Too short to be worth a merge, whatever the lengths.  (us whole, and as the device deals it out from the bound on; 16 query heads over 8
  // of 128 in 16 bits, a key block 64 keys.)
  //   few rows, 9: one sequence of 8 blocks 11.3, in four splits 10.3, 16 sequences 12.8 and 14.4; one of 9 13.4 and 14.1, of 10 13.4 and 11.8, 16
  //   of 10 15.2 and 15.8, of 16 19.2 and 19.6.
  //   few rows, dense, 32: no shares win below (40 sequences of 110 to 1100 keys 28.6 and 35.0), and from there on they may (300 to 3000 75.1 and
  //   65.1); a call that does not take any pays 1.5 for having the choice (64 of 204 to 2048 62.6 and 64.1).
  // Of 128 rows the merge is a launch, paid for split or not:
  //   8: a chunk of 128 in 7 blocks 14.6, in four splits 15.0; in 8 15.4 and 15.6 (codes 18.6 and 16.5; heads of 256 22.4 and 19.6; of
  //   64 11.2 and 12.3), in 10 17.8 and 16.2.
  //   two rounds of places, 24: two chunks of 512 in 22 blocks 33.3, in two to four splits 33.3; in 24 35.7 and 35.5, in 32 45.2 and 39.1.
  //   dense, 64: two chunks of 1001 in a window of 1024, 256 tiles, 32.1, and 34.9 with the merge's launch; what is given up is a long
  //   sequence among short ones (20 chunks of 256, one of them in 63 blocks and the others in 300 keys, 96.4; in 64 97.2 and 63.8).
  // And blocks of all tiles are counted in 31 bits.
  const int64_t least = few ? (dense(a) ? 32 : 9) : dense(a) ? 64 : rounds(a) > 1 ? 24 : 8;
  if (blocks < least || tiles / a.pages.kv_heads * blocks > 0x3fffffff) return 0;
  // Two a workgroup of the places, none for one that the launch has not: of a tile that such a one shared (where sums over starts that
  // descend have wrapped) the others would count themselves in, and leave its word between two counts for the next replay.
  const int64_t round = a.pages.kv_heads;
  return few && dense(a) ? 2 * ((places(a) + round) / round * round) : paged_workgroups(a);
}

// The workgroups of a launch: for every tile there may be, and for the chip's places where tiles may be split; for half of those more
// where long ones alone are (parts_of_all).  (With one for every partial state that there might be 16 sequences over 210 to 2100
// keys took 32.8 us: one without a part costs a place the deal.)
int64_t paged_workgroups(const PagedArgs &a) {
  const int64_t tiles = tiles_at_most(a) * a.pages.kv_heads, round = a.pages.kv_heads, p = ((4 * tiles <= spread(a) ? spread(a) : places(a)) * rounds(a) + round) / round * round;
  if (a.splits > 1) return tiles * a.splits;
  if (a.splits == 1) return tiles;
  if (dense(a) && paged_tile_rows(a) == 128) return tiles + (places(a) / 2 + round) / round * round;
  return tiles > p ? tiles : p;
}

// The states, and behind them two words that tell the merge of tiles of 128 rows of the deal, or a word a workgroup in which those
// that have a tile of few rows count themselves in.
int64_t state_bytes(const PagedArgs &a) { return paged_slots(a) * paged_tile_rows(a) * (a.pages.d + 2) * 4; }
int64_t paged_workspace(const PagedArgs &a) {
  const int64_t bytes = state_bytes(a);
  return bytes == 0 ? 0 : bytes + (paged_tile_rows(a) == 128 ? 16 : paged_workgroups(a) * kPagedWord * 8);
}

PagedLaunch paged_launch(const PagedArgs &a) {
  PagedLaunch l{};
  const PagesArgs &g = a.pages;
  const int rows = paged_tile_rows(a), group = a.heads / g.kv_heads;
  const bool few = rows != 128;
  Deal &d = l.deal;
  d.lens = g.lens, d.starts = g.starts, d.batch = g.batch, d.wide = (g.lens_i64 ? 1 : 0) | (g.starts_i64 ? 2 : 0);
  d.limit = g.columns << g.page_log2, d.rows = g.rows;
  d.tokens = rows / group, d.tokens_rcp = rcp_of(d.tokens);
  d.window_blocks = (int32_t)window_blocks(a);
  d.kv_heads = g.kv_heads, d.kvh_rcp = rcp_of(g.kv_heads);
  PagedParams &p = l.p;
  p.q = (const uint16_t *)a.q, p.o = (uint16_t *)a.o;
  p.k = g.k, p.v = g.v, p.k_scale = g.k_scale, p.v_scale = g.v_scale, p.table = g.table;
  const int64_t slots = paged_slots(a);
  p.parts = a.workspace;
  if (slots > 0) {
    uint8_t *behind = reinterpret_cast<uint8_t *>(p.parts) + state_bytes(a);
    if (few)
      p.arrivals = reinterpret_cast<uint64_t *>(behind), p.tag = launch_tag() & kPagedTags;
    else
      p.told = reinterpret_cast<int32_t *>(behind);
  }
  p.columns = g.columns, p.pages = g.pages, p.page_log2 = g.page_log2;
  p.heads = a.heads, p.group = group, p.group_rcp = rcp_of(group);
  p.causal = a.causal, p.win_left = a.win_left, p.win_right = a.win_right, p.scale = a.scale;
  p.splits = a.splits;
  p.slots = (int32_t)slots;
  p.shares = few && slots > 0 && a.splits == 0 && dense(a);
  p.least = few ? 4.0f : 2.0f, p.turn = few ? 0.25f : 1.0f, p.places = (int32_t)places(a), p.spread = (int32_t)spread(a), p.rounds = rounds(a);
  p.step = !few ? 1.4f : (g.k_scale ? 0.68f : 0.95f) * g.d / 128, p.crowded = few ? p.step : 1.75f;
  p.tail = g.k_scale ? 0.85f : 1.35f, p.even = (g.k_scale ? 1.65f : 2.3f) * (g.d == 256 ? 1.4f : 1.0f);
  // A state is written and read at 5 MB a us: of every row, or of two tiles a place.
  const double of_rows = (double)g.rows * a.heads, of_places = 2.0 * places(a) * rows;
  p.states = (float)((p.shares && of_places < of_rows ? of_places : of_rows) * (g.d + 2) * 8 / 5e6);
  p.stream = few ? (float)((g.k_scale ? 128.0 : 256.0) * g.d / 6.4e6) : 0.0f;  // at 6.4 MB a us
  l.grid = slots == 0 ? tiles_at_most(a) * g.kv_heads : paged_workgroups(a);
  if (slots == 0) p.splits = 1;
  return l;
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
  const bool coded = a.pages.k_scale != nullptr;
  switch (paged_tile_rows(a)) {
    case 16: return coded ? "PagedCfg { rows: 16, keys: 64, e4m3 }" : "PagedCfg { rows: 16, keys: 64 }";
    case 32: return coded ? "PagedCfg { rows: 32, keys: 64, e4m3 }" : "PagedCfg { rows: 32, keys: 64 }";
    default: return coded ? "PagedCfg { rows: 128, keys: 64, e4m3 }" : "PagedCfg { rows: 128, keys: 64 }";
  }
}
#endif

}  // namespace svodk
