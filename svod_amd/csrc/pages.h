// A key/value cache in pages on the device: how the kernels that write, read and attend over one find a sequence's tokens.
//
// Sequence b has lens[b] tokens, the last starts[b + 1] - starts[b] of them this call's, which lie in rows starts[b] and on of
// the packed operands.  The token at position p is row p % page of page table[b][p / page]; a pool is
// [pages, kv_heads, page, D], so that a page holds a KV head's rows side by side: a stream of one head's keys runs in
// pieces of page * D values, whatever the number of heads (rows of [page, kv_heads, D] would be pieces of D).
//
// All three integers are device data that no host check sees.  What reads the cache holds them inside what is there: a length inside
// the table's columns, a row inside the packed operand, a page inside the pool.  A bad one gives a wrong result, never an access out
// of bounds.  What writes it may not: a place held inside is another token's.  A row goes to its own place or nowhere (Fresh).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "kernels.h"

namespace svodk {
namespace {

struct Sequence {
  int start, fresh, len;  // its first packed row, how many it has, and its tokens in the cache, those among them
  // The position of its first new token; negative where a length is short of the rows, whose first ones then have no place.
  __device__ int base() const { return len - fresh; }
};

// The b-th of an array of 32- or 64-bit integers, held in [0, most].
__device__ __forceinline__ int integer_at(const void *p, int64_t b, bool wide, int most) {
  const long long n = wide ? ((const long long *)p)[b] : (long long)((const int *)p)[b];
  return n < 0 ? 0 : (n < (long long)most ? (int)n : most);
}

// A sequence's new rows as they are written: those of [start, start + fresh) of the packed operands, row r at position shift + r,
// which may be any.  Unlike a Sequence's, the position goes by the length and the end as they are given: the rows of a length past the
// table, or of an end past the operands, would take the places of earlier tokens by the held ones.
struct Fresh {
  int start, fresh, shift;
};
__device__ __forceinline__ Fresh fresh_at(const PagesArgs &p, int b) {
  auto given = [](const void *x, int64_t i, bool wide) { return wide ? ((const long long *)x)[i] : (long long)((const int *)x)[i]; };
  Fresh f;
  f.start = integer_at(p.starts, b, p.starts_i64, p.rows);
  f.fresh = max(integer_at(p.starts, (int64_t)b + 1, p.starts_i64, p.rows) - f.start, 0);
  // Rows and positions are below 2^30: a shift as far out leaves every row without a place, and the sum in 32 bits.
  const long long far = 1ll << 30;
  long long shift;
  if (__builtin_sub_overflow(given(p.lens, b, p.lens_i64), given(p.starts, (int64_t)b + 1, p.starts_i64), &shift)) shift = far;
  f.shift = (int)(shift < -far ? -far : shift > far ? far : shift);
  return f;
}

// The page of a sequence's `column`-th run of `page` tokens, to be read.
__device__ __forceinline__ int page_at(const PagesArgs &p, int b, int column) {
  const int id = p.table[(int64_t)b * p.columns + min(column, p.columns - 1)];
  return min(max(id, 0), p.pages - 1);
}

// The first element of row 0 of (page, head), in rows.
__device__ __forceinline__ int64_t page_row(const PagesArgs &p, int page, int head) {
  return ((int64_t)page * p.kv_heads + head) << p.page_log2;
}

// 2^e for a scale's byte e + 127.  (The writer's bytes are 10 to 247: never the two that are no power of two in f32.)
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

typedef __attribute__((ext_vector_type(2))) _Float16 h16x2;
typedef __attribute__((ext_vector_type(2))) __bf16 b16x2;

// Two e4m3 codes of `word` (the upper two with HI) times a power of two, as a pair of the 16-bit type: exact in bf16, whose
// exponent holds every scale; in f16 exact for what was written from f16.
template <bool F16, bool HI>
__device__ __forceinline__ uint32_t widen_codes(uint32_t word, float scale) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (F16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, HI));
#else
  return 0;
#endif
}

}  // namespace
}  // namespace svodk
