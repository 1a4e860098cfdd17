// A part of a tile of few rows of attention over a key/value cache in pages: a sequence's generated token, a few drafted ones.  (What is
// computed, and the tiles of whole tokens: paged_kernel.hip.)
//
// Such a call is a stream of K and V past 16 or 32 rows: 2 flops a byte and row, so the matrix pipes run next to idle and
// what counts is bytes in flight and the length of the way from a launch to its last store.  So:
//   - products on v_mfma_f32_16x16x32, transposed (S^T = K Q^T, O^T += V^T P^T): 16 rows are what such a call has, and a
//     lane's scores of a block of 64 keys are 16 (on the 32 x 32 atom: 32, half of them of no row).
//   - K goes from memory straight into the registers that the matrix instruction reads: its A operand is 16 keys' rows, 16
//     bytes a lane, and the order of a product's terms is free.  Codes: a lane's 16 bytes are 16 codes of one key, two
//     operands, widened with that key's scale, one a lane.
//   - V has to be turned (its A operand is 8 keys of one column a lane), which LDS does (ds_read_b64_tr_b16): through registers
//     into a tile of the wave's own, codes widened on the way.  No wave waits for another inside the loop.
//   - the four waves of a workgroup take an item's key blocks in turn, each with its own state; K of a wave's next block is asked
//     for when its scores are done, V when the tile is written: 32 KiB in flight a wave at D 128, 8 waves a compute unit.
//   - their states meet in LDS at the end; those of the workgroups that share a tile in memory, where the one that counts itself in
//     last adds them up.
// (A token each, 16 query heads over 8 KV heads of 128: 16 sequences over 210 to 2100 keys 22.9 us, one over 65535 55 us, 4.9 TB/s with
// the launch's start and joining, 6 in the loop; 32 over 8, 64 sequences over 2048 to 8192 keys in codes 136 us, 5.0 TB/s.)
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "convert.h"
#include "paged.h"

namespace svodk {
namespace {
namespace few {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
#define SVODK_LDS(T) T __attribute__((address_space(3))) *

constexpr int kWaves = 4;
constexpr float kNone = -1e30f;         // the maximum of a row that has seen no key
constexpr float kRescaleAbove = 8.0f;   // a maximum is adopted when it grew by more, in the exponent's units (attention_step.h)
constexpr float kLog2e = 1.44269504088896340736f;

// D = A . B + C on the 16 x 16 x 32 atom of the operands' type.
template <bool F16>
__device__ __forceinline__ f32x4 mma(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
#else
  return c;
#endif
}

// LDS: a wave's tile of V, 64 keys of 2 D bytes; at the end a wave's state, RT * 16 rows of D + 4 floats (the 4 spread the rows
// over the banks), then their maxima and sums.
template <int D, int RT>
struct Few {
  static constexpr int kRows = 16 * RT;
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kTile = kKeys * kRowBytes;
  static constexpr int kStateRow = (D + 4) * 4;
  static constexpr int kState = kRows * kStateRow + kRows * 8;
  static constexpr int kWaveLds = kTile > kState ? kTile : kState;
  static constexpr int kLds = kWaves * kWaveLds;  // and behind it a word, and 16 bytes a wave
  // A state in memory: the rows' columns, then their maxima and sums.
  static constexpr int kStateBytes = kRows * (D + 2) * 4;
  // Waves a SIMD, which are workgroups a compute unit: by registers and LDS.
  static constexpr int kResident = D == 256 || (D == 128 && RT == 2) ? 1 : (D == 128 || RT == 2) ? 2 : 3;
  static_assert(kResident * (kLds + 16 * (1 + kWaves)) <= 160 * 1024, "the workgroups' LDS");
};
// A tile of V is read by 16 lanes as 4 rows of 32 bytes, 8 rows to half a wave: the 32-byte groups of a row are xor-ed with what
// tells 8 rows apart within the period of the banks (256 bytes: a row of 128 values, half of one of 256, two of 64).
template <int D>
__device__ __forceinline__ constexpr int turn_of(int row) {
  return D == 64 ? (row >> 1) & 3 : row & 7;
}

// x folded over the four lanes that share a query row (l % 16).
template <typename Op>
__device__ __forceinline__ float over_quarters(float x, Op op) {
#if defined(__HIP_DEVICE_COMPILE__)
  uint32_t u = __float_as_uint(x);
  auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  x = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  u = __float_as_uint(x);
  r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  x = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
#endif
  return x;
}

// Partial states that another workgroup reads go past the L2s, each of which serves one XCD, and are read the same way: stores and
// loads that are coherent over the device (the instructions' sc1 bit).
struct States {
#if defined(__HIP_DEVICE_COMPILE__)
  __amdgpu_buffer_rsrc_t rsrc;
  static constexpr int kDevice = 16;
  __device__ __forceinline__ States(float *p, uint32_t bytes) : rsrc(__builtin_amdgcn_make_buffer_rsrc(p, 0, (int)bytes, 0x00020000)) {}
  __device__ __forceinline__ void put4(uint32_t at, const f32x4 &x) const {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), rsrc, (int)at, 0, kDevice);
  }
  __device__ __forceinline__ void put2(uint32_t at, const f32x2 &x) const {
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, x), rsrc, (int)at, 0, kDevice);
  }
  __device__ __forceinline__ f32x4 got4(uint32_t at) const {
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)at, 0, kDevice));
  }
  __device__ __forceinline__ f32x2 got2(uint32_t at) const {
    return __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(rsrc, (int)at, 0, kDevice));
  }
#endif
};
// A row's state over some of its keys, eight columns of it, the maximum in the exponent's units; and another's joined to it.
struct State {
  float m, l, o[8];
  __device__ __forceinline__ void join(float m2, float l2, const f32x4 &a, const f32x4 &b, bool there = true) {
#if defined(__HIP_DEVICE_COMPILE__)
    const float top = __builtin_fmaxf(m, m2), mine = __builtin_amdgcn_exp2f(m - top);
    const float weight = there ? __builtin_amdgcn_exp2f(m2 - top) : 0.0f;
    m = top;
    l = l * mine + l2 * weight;
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = o[i] * mine + (i < 4 ? a[i % 4] : b[i % 4]) * weight;
#endif
  }
};

// A workgroup's part of a tile.  MERGES: the tile may be others' too.
template <int D, int RT, bool F16, bool CODED, bool MERGES>
__device__ __forceinline__ void item(uint8_t *smem, const Deal &deal, const PagedParams &p, const Work &work) {
#if defined(__HIP_DEVICE_COMPILE__)
  using L = Few<D, RT>;
  constexpr int kRowBytes = CODED ? D : 2 * D;  // of the pools
  constexpr int KS = D / 32;                    // terms of a score: matrix instructions
  constexpr int KL = kRowBytes / 64;            // loads of 16 keys' rows
  constexpr int DB = D / 16;                    // column blocks of O
  constexpr int kVLanes = kRowBytes / 16, kVRows = 64 / kVLanes, kVPer = 16 / kVRows;  // V: lanes a row, rows a load, loads a run of 16 rows
  const int lane = lane_of_turn(), wave = uniform((int)__builtin_amdgcn_workitem_id_x() >> 6);
  const int lr = lane & 15, lq = lane >> 4;

  const int first_key = work.first * kKeys, end = work.end - work.first;  // the item's own frame: keys count from its first
  const int len = max(work.at.s.len - first_key, 0);

  // ---- the pages.
  const int64_t head_row = (int64_t)work.kvh << p.page_log2;
  const uint8_t *k_base = (const uint8_t *)p.k + head_row * kRowBytes, *v_base = (const uint8_t *)p.v + head_row * kRowBytes;
  const uint8_t *k_scales = (const uint8_t *)p.k_scale + (CODED ? head_row : 0), *v_scales = (const uint8_t *)p.v_scale + (CODED ? head_row : 0);
  const uint32_t page_rows = (uint32_t)deal.kv_heads << p.page_log2;
  PageIds ids;
  ids.begin(p, work.at.b, (first_key + wave * kKeys) >> p.page_log2);

  // ---- Q: the B operand, 8 values of row l % 16 a lane; of codes in the order in which a lane's 16 give two operands.
  Row rows_of[RT];
  u32x4 qf[RT][KS];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    rows_of[t] = row_of_tile(deal, p, work, 16 * t + lr);
    const uint16_t *q = p.q + rows_of[t].at * D;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      u32x4 x = {0, 0, 0, 0};
      const int at = CODED ? ks / 2 * 64 + lq * 16 + ks % 2 * 8 : ks * 32 + lq * 8;
      if (rows_of[t].there) x = *reinterpret_cast<const u32x4 *>(q + at);
      qf[t][ks] = x;
    }
  }
  int lo[RT], hi[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) lo[t] = rows_of[t].lo - first_key, hi[t] = rows_of[t].hi - first_key;
  const int hi_least = __builtin_amdgcn_readlane(hi[0], 0), lo_most = __builtin_amdgcn_readlane(lo[RT - 1], 15);

  // ---- the loads of a block: its keys' rows by runs of 16, none of which lies in two pages.  Keys past the length read as
  // zeros (a page's last rows hold anything, and 0 times that is not 0), and so does a run in front of the window (whose page the
  // sequence may have given away) and all of a block past the item's last: no load stands under a branch, where the wait for one would be
  // a wait for all.
  int64_t run[4];
  int left[4];
  auto find = [&](int n, bool first) {  // first: the wave's, which alone may hold keys in front of the window
    const int key0 = first_key + n * kKeys;
    ids.go(key0 >> p.page_log2);
    const int lowest = first ? __builtin_amdgcn_readfirstlane(lo[0]) : 0;  // that a row of the tile sees
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int key = key0 + 16 * r;
      run[r] = (int64_t)((uint64_t)(uint32_t)ids.of(key >> p.page_log2) * page_rows) + (key & ((1 << p.page_log2) - 1));
      left[r] = n < end && (!first || n * kKeys + 16 * r + 16 > lowest) ? min(max(len - n * kKeys - 16 * r, 0), 16) : 0;
    }
  };
  u32x4 kf[4][KL], vf[4][kVPer];
  uint32_t k_scale[4], v_scale[4][kVPer];
  auto ask_k = [&]() {
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(k_base + run[r] * kRowBytes), 0, left[r] * kRowBytes, 0x00020000);
#pragma unroll
      for (int i = 0; i < KL; i++) kf[r][i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, lr * kRowBytes + lq * 16 + i * 64, 0, 0);
      if constexpr (CODED) {
        const auto scales = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(k_scales + run[r]), 0, left[r], 0x00020000);
        k_scale[r] = __builtin_amdgcn_raw_buffer_load_b8(scales, lr, 0, 0);
      }
    }
  };
  auto ask_v = [&]() {
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(v_base + run[r] * kRowBytes), 0, left[r] * kRowBytes, 0x00020000);
#pragma unroll
      for (int i = 0; i < kVPer; i++) vf[r][i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, lane * 16 + i * 1024, 0, 0);
      if constexpr (CODED) {
        const auto scales = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(v_scales + run[r]), 0, left[r], 0x00020000);
#pragma unroll
        for (int i = 0; i < kVPer; i++) v_scale[r][i] = __builtin_amdgcn_raw_buffer_load_b8(scales, lane / kVLanes + i * kVRows, 0, 0);
      }
    }
  };
  // The word in which the workgroups of a tile count themselves in is the workspace's and holds anything at first.  Every one
  // makes sure, before it counts, that it carries this launch's tag: it becomes (tag, 0) by one compare-and-swap out of whatever was
  // there, and no other write of the launch leaves that content again, so a late swap out of it fails.  Nothing else ever carries
  // the tag but the word as an earlier replay of the same captured launch left it, and that one counts kPagedEnded, which
  // no word of a launch under way does.  The content is asked for ahead of the keys, the swap goes out behind the loop: neither is
  // waited for.
  const bool whole = !MERGES || work.whole;
  uint64_t *const word = whole ? nullptr : p.arrivals + ((int64_t)work.sharers.first * deal.kv_heads + work.kvh) * kPagedWord;
  const bool counts = !whole && wave == 0 && lane == 0;
  uint64_t found = 0;
  if (counts) found = __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  find(wave, true);
  ask_k();
  ask_v();

  // ---- a lane's places in the wave's tile of V: where its 16 bytes of a row go, and what it reads of a column block.
  uint8_t *tile = smem + wave * L::kWaveLds;
  int v_put[kVPer], v_get[DB];
#pragma unroll
  for (int i = 0; i < kVPer; i++) {
    const int row = i * kVRows + lane / kVLanes, piece = lane % kVLanes;  // a piece: 8 values, or 16 codes
    const int group = CODED ? piece : piece >> 1;
    v_put[i] = row * L::kRowBytes + ((group ^ turn_of<D>(row)) << 5) + (CODED ? 0 : (piece & 1) << 4);
  }
#pragma unroll
  for (int db = 0; db < DB; db++) {
    const int row = 4 * lq + (lr >> 2);
    v_get[db] = row * L::kRowBytes + ((db ^ turn_of<D>(row)) << 5) + ((lane & 3) << 3);
  }

  const bool positive = p.scale > 0.0f;
  const float c_exp = p.scale * kLog2e, unit = positive ? c_exp : 1.0f, limit = kRescaleAbove / unit;
  f32x4 acc[RT][DB];
  float m[RT], l[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    m[t] = kNone, l[t] = 0.0f;
#pragma unroll
    for (int db = 0; db < DB; db++) acc[t][db] = f32x4{0, 0, 0, 0};
  }

  for (int n = wave; n < end; n += kWaves) {
    // ---- S^T: lane l has the scores of row l % 16 with keys 16 r + 4 (l / 16) + 0..3.
    f32x4 s[RT][4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
#pragma unroll
      for (int t = 0; t < RT; t++) s[t][r] = f32x4{0, 0, 0, 0};
      const float scale = CODED ? scale_of(k_scale[r]) : 0.0f;
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        u32x4 a;
        if constexpr (CODED) {
          const u32x4 c = kf[r][ks / 2];
          const uint32_t c0 = c[ks % 2 * 2], c1 = c[ks % 2 * 2 + 1];
          a = u32x4{widen_codes<F16, false>(c0, scale), widen_codes<F16, true>(c0, scale), widen_codes<F16, false>(c1, scale),
                    widen_codes<F16, true>(c1, scale)};
        } else {
          a = kf[r][ks];
        }
#pragma unroll
        for (int t = 0; t < RT; t++) s[t][r] = mma<F16>(a, qf[t][ks], s[t][r]);
      }
    }
    // The next block's keys are on their way from here on.
    find(n + kWaves, false);
    ask_k();

    // ---- the softmax's step, a row in four lanes.
    u32x4 pf[RT][2];
    const int k0 = n * kKeys;
#pragma unroll
    for (int t = 0; t < RT; t++) {
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; i++) x[i] = positive ? s[t][i / 4][i % 4] : s[t][i / 4][i % 4] * c_exp;
      if (k0 + kKeys - 1 > hi_least || k0 < lo_most) {
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int key = k0 + 16 * (i / 4) + 4 * lq + i % 4;
          x[i] = key >= lo[t] && key <= hi[t] ? x[i] : -INFINITY;
        }
      }
      float most = x[0];
#pragma unroll
      for (int i = 1; i < 16; i++) most = __builtin_fmaxf(most, x[i]);
      most = over_quarters(most, [](float a, float b) { return __builtin_fmaxf(a, b); });
      // A maximum is adopted when it grew by more than the limit; a wave whose rows all kept theirs has nothing to rescale.
      const float higher = __builtin_fmaxf(m[t], most);
      const float next = higher - m[t] > limit ? higher : m[t];
      if (__builtin_amdgcn_ballot_w64(next != m[t]) != 0) {
        const float keep = __builtin_amdgcn_exp2f((m[t] - next) * unit);
        l[t] *= keep;
#pragma unroll
        for (int db = 0; db < DB; db++) acc[t][db] *= keep;
      }
      m[t] = next;
      const float offset = next * unit;
      float sums[4] = {};
#pragma unroll
      for (int i = 0; i < 16; i++) {
        x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], unit, -offset));
        sums[i % 4] += x[i];
      }
      l[t] += (sums[0] + sums[1]) + (sums[2] + sums[3]);
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) pf[t][j][i] = narrow<F16>(x[8 * j + 2 * i], x[8 * j + 2 * i + 1]);
    }

    // ---- V into the tile, the next block's on their way, O^T += V^T P^T.
#pragma unroll
    for (int r = 0; r < 4; r++) {
#pragma unroll
      for (int i = 0; i < kVPer; i++) {
        uint8_t *to = tile + 16 * r * L::kRowBytes + v_put[i];
        const u32x4 c = vf[r][i];
        if constexpr (CODED) {
          const float scale = scale_of(v_scale[r][i]);
          *reinterpret_cast<u32x4 *>(to) = u32x4{widen_codes<F16, false>(c[0], scale), widen_codes<F16, true>(c[0], scale),
                                                 widen_codes<F16, false>(c[1], scale), widen_codes<F16, true>(c[1], scale)};
          *reinterpret_cast<u32x4 *>(to + 16) = u32x4{widen_codes<F16, false>(c[2], scale), widen_codes<F16, true>(c[2], scale),
                                                      widen_codes<F16, false>(c[3], scale), widen_codes<F16, true>(c[3], scale)};
        } else {
          *reinterpret_cast<u32x4 *>(to) = c;
        }
      }
    }
    ask_v();
#pragma unroll
    for (int j = 0; j < 2; j++) {
#pragma unroll
      for (int db = 0; db < DB; db++) {
        const uint8_t *from = tile + v_get[db] + 32 * j * L::kRowBytes;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SVODK_LDS(s16x4))(from));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SVODK_LDS(s16x4))(from + 16 * L::kRowBytes));
        const u32x4 v = __builtin_bit_cast(u32x4, (s16x8)__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int t = 0; t < RT; t++) acc[t][db] = mma<F16>(v, pf[t][j], acc[t][db]);
      }
    }
  }

  if (counts && (found >> kPagedCountBits != p.tag || (found & kPagedEnded) == kPagedEnded))
    __hip_atomic_compare_exchange_strong(word, &found, p.tag << kPagedCountBits, __ATOMIC_RELAXED, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // ---- the waves' states as one: maxima in the exponent's units.  A wave's state lies where its tile of V did.
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const float sum = over_quarters(l[t], [](float a, float b) { return a + b; });
    const int row = 16 * t + lr;
#pragma unroll
    for (int db = 0; db < DB; db++) *reinterpret_cast<f32x4 *>(tile + row * L::kStateRow + (16 * db + 4 * lq) * 4) = acc[t][db];
    if (lq == 0) *reinterpret_cast<f32x2 *>(tile + L::kRows * L::kStateRow + row * 8) = f32x2{positive ? m[t] * c_exp : m[t], sum};
  }
  __syncthreads();
  constexpr int kPieces = D / 8;  // of a row, 8 columns each
  const States states(p.parts, (uint32_t)p.slots * L::kStateBytes);
  for (int c = wave * 64 + lane; c < L::kRows * kPieces; c += kWaves * 64) {
    const int row = c / kPieces, column = c % kPieces * 8;
    const Row r = row_of_tile(deal, p, work, row);
    f32x2 ml[kWaves];
    f32x4 x[kWaves][2];
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      const uint8_t *state = smem + w * L::kWaveLds;
      ml[w] = *reinterpret_cast<const f32x2 *>(state + L::kRows * L::kStateRow + row * 8);
      x[w][0] = *reinterpret_cast<const f32x4 *>(state + row * L::kStateRow + column * 4);
      x[w][1] = *reinterpret_cast<const f32x4 *>(state + row * L::kStateRow + column * 4 + 16);
    }
    float top = ml[0][0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) top = __builtin_fmaxf(top, ml[w][0]);
    float sum = 0.0f, o[8] = {};
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      const float weight = __builtin_amdgcn_exp2f(ml[w][0] - top);
      sum += ml[w][1] * weight;
#pragma unroll
      for (int i = 0; i < 8; i++) o[i] += x[w][i / 4][i % 4] * weight;
    }
    if (!r.there) continue;
    if (whole) {
      const float inv = 1.0f / (sum == 0.0f ? 1.0f : sum);
      u32x4 out;
#pragma unroll
      for (int i = 0; i < 4; i++) out[i] = narrow<F16>(o[2 * i] * inv, o[2 * i + 1] * inv);
      *reinterpret_cast<u32x4 *>(p.o + r.at * D + column) = out;
    } else {
      const uint32_t at = (uint32_t)work.slot * L::kStateBytes;
      if (column == 0) states.put2(at + (L::kRows * D + 2 * row) * 4, f32x2{top, sum});
      states.put4(at + (row * D + column) * 4, f32x4{o[0], o[1], o[2], o[3]});
      states.put4(at + (row * D + column + 4) * 4, f32x4{o[4], o[5], o[6], o[7]});
    }
  }
  if (whole) return;

  // ---- the tile's other workgroups.  This one's state is where every other sees it before it counts itself in: it was stored
  // past the L2s, and vmcnt is at zero when the memory behind those has taken it.  No one waits for anyone.
  const int others = work.sharers.last - work.sharers.first;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int *const arrived = reinterpret_cast<int *>(smem + L::kLds);
  if (counts) {
    const uint64_t before = __hip_atomic_fetch_add(word, (uint64_t)1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const bool last = (int)(before & kPagedEnded) == others;
    if (last) __hip_atomic_store(word, p.tag << kPagedCountBits | kPagedEnded, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *arrived = last ? 1 : 0;
  }
  __syncthreads();
  if (uniform(*arrived) == 0) return;
  asm volatile("" ::: "memory");  // the states are read from here on
  // The last one has 256 threads for rows * kPieces pieces: where they are fewer, several take a piece's states in turn and join theirs
  // in LDS.  Who adds what follows from the sizes alone: the same bits whoever is last.
  const int rows = (work.last - work.tile_first + 1) * p.group, pieces = rows * kPieces;
  int teams_log2 = 0;
  while (pieces << (teams_log2 + 1) <= kWaves * 64 && (1 << teams_log2) <= others) teams_log2++;
  const int id = wave * 64 + lane, team = id / pieces, teams = 1 << teams_log2;
  constexpr int kAhead = 4;
  for (int c = teams > 1 ? id - team * pieces : id; c < pieces; c += teams > 1 ? pieces : kWaves * 64) {
    const int row = c / kPieces, column = c % kPieces * 8;
    State x{kNone, 0.0f, {}};
    if (team < teams || teams == 1) {
      const int from = teams > 1 ? team : 0;
      for (int i = from; i <= others; i += teams * kAhead) {
        f32x2 ml[kAhead];
        f32x4 o[kAhead][2];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {  // one past the last asks for the last again, and weighs nothing
          const int which = min(i + j * teams, others);
          const int64_t slot = which == 0 ? work.sharers.slot : work.sharers.next + (int64_t)(which - 1) * work.sharers.step;
          const uint32_t at = (uint32_t)slot * L::kStateBytes;
          ml[j] = states.got2(at + (L::kRows * D + 2 * row) * 4);
          o[j][0] = states.got4(at + (row * D + column) * 4);
          o[j][1] = states.got4(at + (row * D + column + 4) * 4);
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++) x.join(ml[j][0], ml[j][1], o[j][0], o[j][1], i + j * teams <= others);
      }
    }
    if (teams > 1) {
      float *const joined = reinterpret_cast<float *>(smem) + id * 12;
      if (team < teams) {
        *reinterpret_cast<f32x4 *>(joined) = f32x4{x.m, x.l, 0.0f, 0.0f};
        *reinterpret_cast<f32x4 *>(joined + 4) = f32x4{x.o[0], x.o[1], x.o[2], x.o[3]};
        *reinterpret_cast<f32x4 *>(joined + 8) = f32x4{x.o[4], x.o[5], x.o[6], x.o[7]};
      }
      __syncthreads();
      if (team == 0)
        for (int t = 1; t < teams; t++) {
          const float *from = reinterpret_cast<const float *>(smem) + (id + t * pieces) * 12;
          x.join(from[0], from[1], *reinterpret_cast<const f32x4 *>(from + 4), *reinterpret_cast<const f32x4 *>(from + 8));
        }
    }
    if (teams > 1 && team != 0) continue;
    const Row r = row_of_tile(deal, p, work, row);
    const float inv = 1.0f / (x.l == 0.0f ? 1.0f : x.l);
    u32x4 out;
#pragma unroll
    for (int i = 0; i < 4; i++) out[i] = narrow<F16>(x.o[2 * i] * inv, x.o[2 * i + 1] * inv);
    *reinterpret_cast<u32x4 *>(p.o + r.at * D + column) = out;
  }
#endif
}

}  // namespace few
}  // namespace
}  // namespace svodk
