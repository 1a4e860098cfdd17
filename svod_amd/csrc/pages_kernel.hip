// A key/value cache in pages, for gfx950 (MI355X): new tokens' keys and values into it, and its sequences out of it.
//
// Written as they are, or in 8 bits.  A row of 8 bits is e4m3 codes c_i and one exponent e, the row's values 2^e c_i:
//   e = the least whole number with max |x| <= 448 * 2^e (448 is e4m3's largest), from -117 on;   c_i = x_i * 2^-e to the nearest even
// over the row's finite values.  A power of two, not max / 448: x * 2^-e is exact, so that a value is rounded once and alike wherever
// it is computed, and a code times 2^e is exact in bf16 and, for rows that came from f16, in f16.  e4m3 gives up nothing for it but its range's last
// bit.  Where 256 * 2^e lies past the type's largest value (f16: rows that reach past 57344, e = 8), codes end at 240: a value in
// 63488 .. 65504 is within 2^-4 of 61440 still, and no finite value comes back infinite.  An infinity or a NaN comes back as NaN.
//
// Both directions are copies, bound by memory.  A wave's 1 KiB of 16-bit rows are neighbouring positions of one KV head: the pool's side is
// a run without gaps (a page holds a head's rows side by side), the other's are whole rows of D values.
#include <hip/hip_runtime.h>

#include "convert.h"
#include "kernels.h"
#include "launch.h"
#include "pages.h"

namespace svodk {
namespace {

typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;
typedef __attribute__((ext_vector_type(2))) short s16x2;

constexpr int kWaves = 4;

// The maximum of a value of [0, 2^31) over the LANES lanes of a row (neighbours, 8 to 32 of them).
template <int LANES>
__device__ __forceinline__ int row_most(int x) {
#if defined(__HIP_DEVICE_COMPILE__)
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0xb1, 0xf, 0xf, true));   // quad_perm: 1, 0, 3, 2
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x4e, 0xf, 0xf, true));   // quad_perm: 2, 3, 0, 1
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, true));  // row_half_mirror
  if constexpr (LANES >= 16) x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x140, 0xf, 0xf, true));  // row_mirror
  if constexpr (LANES >= 32) x = max(x, __shfl_xor(x, 16));
#endif
  return x;
}

// The largest magnitude of eight values' bits, those that are not finite left out with FINITE.
template <bool F16, bool FINITE>
__device__ __forceinline__ int most_of(const u32x4 &w) {
  constexpr uint32_t kInf = F16 ? 0x7c00u : 0x7f80u;
  u16x2 most = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    u16x2 x = __builtin_bit_cast(u16x2, (uint32_t)(w[i] & 0x7fff7fffu));
    if constexpr (FINITE) x = u16x2{x[0] < kInf ? x[0] : (uint16_t)0, x[1] < kInf ? x[1] : (uint16_t)0};
    most = __builtin_elementwise_max(most, x);
  }
  return max((int)most[0], (int)most[1]);
}
// Eight values of a row of LANES lanes as codes; `e` the row's exponent.  The hardware's conversion divides by the power of two and
// rounds once, to the nearest even; what is not finite becomes e4m3's NaN.  (Over all values of either type and exponents from -100 to
// 100 it gives the codes of x * 2^-e.)
template <bool F16, int LANES>
__device__ __forceinline__ u32x2 to_codes(const u32x4 &w, int &e) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kInf = F16 ? 0x7c00 : 0x7f80;
  constexpr int kTop = F16 ? 8 : 120;  // with it a code of 256 is past the type's largest value
  int most = row_most<LANES>(most_of<F16, false>(w));
  if (__builtin_amdgcn_ballot_w64(most >= kInf) != 0) most = row_most<LANES>(most_of<F16, true>(w));
  uint32_t bits;  // as an f32's
  if constexpr (F16)
    bits = __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)most));
  else
    bits = (uint32_t)most << 16;
  // 448 = 1.75 * 2^8: one more where the significand is past 1.75.
  e = max((int)((bits + 0x1fffffu) >> 23) - 135, -117);
  const float scale = __uint_as_float((uint32_t)(127 + e) << 23);
  u32x2 out;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    s16x2 c = {0, 0};
    const uint32_t lo = w[2 * i], hi = w[2 * i + 1];
    if constexpr (F16) {
      c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, __builtin_bit_cast(f16x2, lo), scale, false);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, __builtin_bit_cast(f16x2, hi), scale, true);
    } else {
      c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(bf16x2, lo), scale, false);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(bf16x2, hi), scale, true);
    }
    out[i] = __builtin_bit_cast(uint32_t, c);
  }
  if (__builtin_amdgcn_ballot_w64(e >= kTop) != 0) {
    // 240 (0x77) in the place of 256 and more, NaN (0x7f) apart.
#pragma unroll
    for (int i = 0; i < 2; i++) {
      uint32_t word = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t code = (out[i] >> (8 * j)) & 0xffu, size = code & 0x7fu;
        word |= (e >= kTop && size > 0x77u && size < 0x7fu ? (code & 0x80u) | 0x77u : code) << (8 * j);
      }
      out[i] = word;
    }
  }
  return out;
#else
  return u32x2{};
#endif
}

// ---- into the pages.  A wave takes 64 / LANES packed rows, keys and values, of HEADS KV heads one after the other: four where
// there are waves enough, so that a wave has eight loads on their way while it looks its rows up, and looks them up once (13312
// rows of 8 heads of 128 into codes 25.2 us a head a wave with the codes by arithmetic, 18.2 so; eight
// prompts of up to 2047 tokens in f16, 20 heads of 64, 26.4 and 25.5).
template <int D, bool F16, bool CODED, int HEADS>
__global__ __launch_bounds__(kWaves * 64) void write_pages_kernel(PagesArgs p, uint32_t strips, const uint16_t *__restrict__ k,
                                                                  const uint16_t *__restrict__ v) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kLanes = D / 8, kRows = 64 / kLanes;
  const int lane = (int)__builtin_amdgcn_workitem_id_x() & 63;
  const uint32_t wave = __builtin_amdgcn_workgroup_id_x() * kWaves + (uint32_t)__builtin_amdgcn_readfirstlane((int)__builtin_amdgcn_workitem_id_x() >> 6);
  const uint32_t group = wave / strips;
  const int head0 = (int)(wave - group * strips) * HEADS;
  const int64_t row0 = (int64_t)group * kRows;
  if (row0 >= p.rows) return;
  const int64_t row = row0 + lane / kLanes;
  const bool there = row < p.rows;
  const int column = lane % kLanes * 8;
  u32x4 xk[HEADS], xv[HEADS];
#pragma unroll
  for (int h = 0; h < HEADS; h++) {
    // A row or head past the last loads one that is there, and drops it.
    const int64_t from = ((there ? row : row0) * p.kv_heads + min(head0 + h, p.kv_heads - 1)) * D + column;
    xk[h] = *reinterpret_cast<const u32x4 *>(k + from), xv[h] = *reinterpret_cast<const u32x4 *>(v + from);
  }
  // The sequence and the position of each of the wave's rows: the sequences a lane each, 64 at a time.
  int b = -1, at = -1;
  for (int base = 0; base < p.batch; base += 64) {
    Fresh s{};
    if (base + lane < p.batch) s = fresh_at(p, base + lane);
    int found = 0;
#pragma unroll
    for (int r = 0; r < kRows; r++) {
      const int64_t in = row0 + r - s.start;
      const uint64_t here = __builtin_amdgcn_ballot_w64(in >= 0 && in < s.fresh);
      if (here != 0) {
        found++;
        const int one = __builtin_ctzll(here);
        const int position = __builtin_amdgcn_readlane(s.shift, one) + (int)(row0 + r);
        if (lane / kLanes == r && b < 0) b = base + one, at = position;
      }
    }
    if (found == kRows) break;
  }
  // A row of no sequence, of a position that the table has no column for, or of a page that the pool has not, goes nowhere; its
  // lanes go on, for their neighbours' sums.
  bool goes = there && b >= 0 && at >= 0 && at < p.columns << p.page_log2;
  const int page = goes ? p.table[(int64_t)b * p.columns + (at >> p.page_log2)] : 0, in_page = at & ((1 << p.page_log2) - 1);
  goes = goes && page >= 0 && page < p.pages;
#pragma unroll
  for (int h = 0; h < HEADS; h++) {
    const bool writes = goes && head0 + h < p.kv_heads;
    const int64_t to = page_row(p, page, head0 + h) + in_page;
    if constexpr (CODED) {
      int ek, ev;
      const u32x2 ck = to_codes<F16, kLanes>(xk[h], ek), cv = to_codes<F16, kLanes>(xv[h], ev);
      if (!writes) continue;
      *reinterpret_cast<u32x2 *>((uint8_t *)p.k + to * D + column) = ck;
      *reinterpret_cast<u32x2 *>((uint8_t *)p.v + to * D + column) = cv;
      if (column == 0) {
        ((uint8_t *)p.k_scale)[to] = (uint8_t)(ek + 127);
        ((uint8_t *)p.v_scale)[to] = (uint8_t)(ev + 127);
      }
    } else if (writes) {
      *reinterpret_cast<u32x4 *>((uint16_t *)p.k + to * D + column) = xk[h];
      *reinterpret_cast<u32x4 *>((uint16_t *)p.v + to * D + column) = xv[h];
    }
  }
#endif
}

// ---- and out of them.  A wave takes 64 / LANES neighbouring positions of one (sequence, KV head): no page ends inside.  (32768 rows of 8
// heads of 128 in codes, 202 MB: 33 us by itself, 6.1 TB/s; bound by memory.)
template <int D, bool F16, bool CODED>
__global__ __launch_bounds__(kWaves * 64) void read_pages_kernel(PagesArgs p, int tokens, uint32_t groups, uint16_t *__restrict__ k, uint16_t *__restrict__ v) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kLanes = D / 8, kRows = 64 / kLanes;
  static_assert(kRows <= kLeastPage, "a wave's rows lie in one page");
  const int lane = (int)__builtin_amdgcn_workitem_id_x() & 63;
  const uint32_t wave = __builtin_amdgcn_workgroup_id_x() * kWaves + (uint32_t)__builtin_amdgcn_readfirstlane((int)__builtin_amdgcn_workitem_id_x() >> 6);
  const uint32_t unit = wave / (uint32_t)p.kv_heads;
  const int head = (int)(wave - unit * (uint32_t)p.kv_heads);
  const uint32_t b = unit / groups;
  if (b >= (uint32_t)p.batch) return;
  const int at0 = (int)(unit - b * groups) * kRows;
  const int len = integer_at(p.lens, b, p.lens_i64, p.columns << p.page_log2);
  const int at = at0 + lane / kLanes;
  u32x4 xk{}, xv{};
  if (at < len) {
    const int64_t from = page_row(p, page_at(p, (int)b, at0 >> p.page_log2), head) + (at & ((1 << p.page_log2) - 1));
    if constexpr (CODED) {
      const u32x2 ck = *reinterpret_cast<const u32x2 *>((const uint8_t *)p.k + from * D + lane % kLanes * 8);
      const u32x2 cv = *reinterpret_cast<const u32x2 *>((const uint8_t *)p.v + from * D + lane % kLanes * 8);
      const float sk = scale_of(((const uint8_t *)p.k_scale)[from]), sv = scale_of(((const uint8_t *)p.v_scale)[from]);
      xk = u32x4{widen_codes<F16, false>(ck[0], sk), widen_codes<F16, true>(ck[0], sk), widen_codes<F16, false>(ck[1], sk),
                 widen_codes<F16, true>(ck[1], sk)};
      xv = u32x4{widen_codes<F16, false>(cv[0], sv), widen_codes<F16, true>(cv[0], sv), widen_codes<F16, false>(cv[1], sv),
                 widen_codes<F16, true>(cv[1], sv)};
    } else {
      xk = *reinterpret_cast<const u32x4 *>((const uint16_t *)p.k + from * D + lane % kLanes * 8);
      xv = *reinterpret_cast<const u32x4 *>((const uint16_t *)p.v + from * D + lane % kLanes * 8);
    }
  }
  if (at >= tokens) return;
  const int64_t to = (((int64_t)b * tokens + at) * p.kv_heads + head) * D + lane % kLanes * 8;
  *reinterpret_cast<u32x4 *>(k + to) = xk;
  *reinterpret_cast<u32x4 *>(v + to) = xv;
#endif
}

template <int D, bool F16, bool CODED, int HEADS>
hipError_t write_heads(const PagesArgs &a, const void *k, const void *v, hipStream_t stream) {
  const int64_t groups = ((int64_t)a.rows * D / 8 + 63) / 64, strips = (a.kv_heads + HEADS - 1) / HEADS;
  const int64_t grid = (groups * strips + kWaves - 1) / kWaves;
  if (grid > 0xffffffff / (kWaves * 64)) return hipErrorInvalidConfiguration;  // a launch's threads are counted in 32 bits
  return Launch<write_pages_kernel<D, F16, CODED, HEADS>>::run(grid, kWaves * 64, 0, 0, stream, a, (uint32_t)strips, (const uint16_t *)k,
                                                               (const uint16_t *)v);
}
template <int D, bool F16, bool CODED>
hipError_t write(const PagesArgs &a, const void *k, const void *v, hipStream_t stream) {
  // Four heads a wave from eight waves a compute unit on that have four.
  const bool many = ((int64_t)a.rows * D / 8 + 63) / 64 * (a.kv_heads / 4) >= 256 * 8;
  return many ? write_heads<D, F16, CODED, 4>(a, k, v, stream) : write_heads<D, F16, CODED, 1>(a, k, v, stream);
}
template <int D, bool F16, bool CODED>
hipError_t read(const PagesArgs &a, int32_t tokens, void *k, void *v, hipStream_t stream) {
  const int64_t groups = ((int64_t)tokens * D / 8 + 63) / 64, waves = groups * a.batch * a.kv_heads, grid = (waves + kWaves - 1) / kWaves;
  if (grid > 0xffffffff / (kWaves * 64)) return hipErrorInvalidConfiguration;  // a launch's threads are counted in 32 bits
  return Launch<read_pages_kernel<D, F16, CODED>>::run(grid, kWaves * 64, 0, 0, stream, a, tokens, (uint32_t)groups, (uint16_t *)k, (uint16_t *)v);
}

// f(D, F16, CODED) of a call.
template <template <int, bool, bool> class F, typename... A>
hipError_t of_kind(const PagesArgs &a, A... args) {
  const bool coded = a.k_scale != nullptr;
#define SVODK_KIND(D)                                                                                       \
  if (a.d == D) {                                                                                           \
    if (a.f16) return coded ? F<D, true, true>::run(a, args...) : F<D, true, false>::run(a, args...);       \
    return coded ? F<D, false, true>::run(a, args...) : F<D, false, false>::run(a, args...);                \
  }
  SVODK_KIND(64) SVODK_KIND(128) SVODK_KIND(256)
#undef SVODK_KIND
  return hipErrorInvalidValue;
}
template <int D, bool F16, bool CODED>
struct Write {
  static hipError_t run(const PagesArgs &a, const void *k, const void *v, hipStream_t stream) { return write<D, F16, CODED>(a, k, v, stream); }
};
template <int D, bool F16, bool CODED>
struct Read {
  static hipError_t run(const PagesArgs &a, int32_t tokens, void *k, void *v, hipStream_t stream) {
    return read<D, F16, CODED>(a, tokens, k, v, stream);
  }
};

}  // namespace

bool pages_support(int64_t d) { return d == 64 || d == 128 || d == 256; }

hipError_t launch_write_pages(const PagesArgs &a, const void *k, const void *v, hipStream_t stream) { return of_kind<Write>(a, k, v, stream); }
hipError_t launch_read_pages(const PagesArgs &a, int32_t tokens, void *k, void *v, hipStream_t stream) {
  return of_kind<Read>(a, tokens, k, v, stream);
}

}  // namespace svodk
