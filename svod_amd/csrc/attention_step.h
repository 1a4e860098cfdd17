// What the attention kernels share: the key tile and its place in LDS, the matrix instruction, a wave's state and the steps it
// takes through the key blocks (hot_step, edge_step, idle_step).  attention_kernel.hip says how a tile is laid out over the waves and why,
// paged_kernel.hip takes the same steps over keys that lie in pages.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace svodk {
namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef __attribute__((ext_vector_type(4))) int i32x4;

#define LDS_PTR(T) T __attribute__((address_space(3))) *

constexpr int kBkv = 64;       // keys per ring slot
constexpr int kScannedBlocks = 256;  // key blocks (16384 keys) of a key mask row scanned up front
// LDS behind the ring of a workgroup that scans one: the blocks' words, then the elements of each wave's first two blocks.
constexpr int kRawElements = 128;
constexpr int mask_lds(int waves) { return kScannedBlocks * 8 + waves * kRawElements * 4; }
constexpr int kWaveRows = 32;  // query rows a wave owns: the N of the MFMA atom
constexpr int kXcds = 8;       // accelerator dies of an MI355X, each with its own L2
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kRescaleAbove = 8.0f;  // tk/src/kernels/attention.rs:379

// A ring slot holds a [64 keys, D] tile, rows unpadded (D*2 bytes), filled by
// buffer_load_dwordx4 ... lds: a wave instruction lands 64 consecutive 16-byte
// chunks, so the only freedom is WHICH global chunk a lane fetches.  Each row's
// chunks are therefore stored XOR-permuted, with a permutation chosen per tile
// so that its read pattern touches every bank once:
//   K is read one chunk per lane, 16 consecutive rows at the same logical chunk
//     (ds_read_b128 serves 16 lanes a cycle): chunk ^ sK(row) with sK distinct
//     over 16 rows modulo the 256-byte bank period;
//   V is read transposed, 4 consecutive rows x 64 contiguous bytes per 32 lanes
//     (ds_read_b64_tr_b16): the 64-byte group index ^ sV(row) with sV distinct
//     over 4 rows modulo the period.
// K runs one block ahead of V, so each has its own pair of slots:
// LDS = [K slot 0][K slot 1][V slot 0][V slot 1].
// A head of 48 takes the 64-wide tile: a row's last two chunks are never fetched (their lanes
// read past the descriptor's bound and land zeros), the score product stops at the third
// k-step, and the second half of O^T's second row block is dropped at the store.
template <int D>
struct Tile {
  static constexpr int kWide = D == 48 ? 64 : D;  // the head size the tile is laid out for
  static constexpr int kRowBytes = kWide * 2;
  static constexpr int kCpr = kWide / 8;   // 16-byte chunk places per row of the tile
  static constexpr int kChunks = D / 8;    // chunks a row holds in memory
  static constexpr int kBytes = kBkv * kRowBytes;
  static constexpr int kLds = 4 * kBytes;
  static constexpr int kInstrs = kBytes / 1024;  // wave-wide 1 KiB fills per tile
  // 32 wide: rows are 64 bytes, four to the bank period, so 16 rows at one logical chunk spread over
  // the period's 16 chunk places when the chunk is xor-ed with row / 4; a V row is one 64-byte
  // group and four consecutive rows are the whole period as they lie.
  // 256 wide: rows are two bank periods, every row starts on a period, and row & 15 spreads 16 rows
  // over the 16 chunk places of a half row as it does for 128.
  __device__ static constexpr int swz_k(int row) {
    return kWide == 32 ? ((row >> 2) & 3) : kWide == 64 ? ((row >> 1) & 7) : (row & 15);
  }
  // In units of 64-byte groups (4 chunks).
  __device__ static constexpr int swz_v(int row) {
    return kWide == 32 ? 0 : kWide == 64 ? ((row >> 1) & 1) : (row & 3);
  }
  // The byte offset, from a fill instruction's first row, of what the lane at chunk place `pc` of
  // tile row `row` fetches: logical chunk pc ^ swizzle of that row of memory, or an offset past any
  // descriptor's bound where the row has no such chunk.
  // `ahead` rows lie between the fill instruction's first row and the tile row the swizzle is the one of
  // (a wave's later fills of a tile, where they do not share the first's swizzle).
  __device__ static int source(int row, int pc, int row_bytes, bool v, int ahead = 0) {
    const int chunk = pc ^ (v ? swz_v(row + ahead) << 2 : swz_k(row + ahead));
    return chunk < kChunks ? row * row_bytes + (chunk << 4) : (int)0xfffffff0u;
  }
  // A wave's fills of a tile are NW instructions apart; where that is not a whole period of the swizzle
  // (16 rows) its even and odd fills have a swizzle each.
  __device__ static constexpr int sources(int nw) { return (nw * (64 / kCpr)) % 16 == 0 ? 1 : 2; }
};

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  return __builtin_fmaxf(__builtin_fmaxf(a, b), c);
}

// Two f32 values as a pair of the operands' 16-bit type, rounded to nearest even
// (tk/src/interp.rs:37-50).
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  f32x2 f = {lo, hi};
  if constexpr (F16) {
    f16x2 h = __builtin_convertvector(f, f16x2);
    return __builtin_bit_cast(uint32_t, h);
  } else {
    bf16x2 b = __builtin_convertvector(f, bf16x2);
    return __builtin_bit_cast(uint32_t, b);
  }
}

// D = A . B + C on the 32x32x16 atom of the operands' type: A 32 rows x 16, B 16 x 32 columns,
// eight 16-bit values a lane each.
template <bool F16>
__device__ __forceinline__ f32x16 mma(const u32x4 &a, const u32x4 &b, const f32x16 &c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// `x` of this lane and of its partner in the other half-wave (lane l <-> l^32),
// in an order that differs between the halves: v_permlane32_swap hands lanes
// < 32 (own, partner) and lanes >= 32 (partner, own).  Callers fold the pair
// with a commutative op.
struct Pair {
  float a, b;
};
__device__ __forceinline__ Pair both_halves(float x) {
  const uint32_t u = __float_as_uint(x);
  auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return {__uint_as_float(r[0]), __uint_as_float(r[1])};
}

// A raw buffer descriptor over `bytes` bytes at `base` (stride 0, 32-bit raw format): loads
// past the end return zero, which is how rows at and past a batch's key length read (the
// bounded views of tk/src/kernels/attention.rs:551-560).
// Both arguments are the same in every lane (a descriptor lives in scalar registers).  The bound is `bytes`
// clamped to [0, 2^32 - 1] on the scalar unit: written as comparisons of the 64-bit value the compiler does it on
// the VALU (v_cmp_*_i64 on broadcast operands), six vector instructions a descriptor in a loop whose VALU port is
// what bounds it.
__device__ __forceinline__ i32x4 make_rsrc(const void *base, int64_t bytes) {
  const uint64_t addr = (uint64_t)(uintptr_t)base;
  const int lo = (int)(uint32_t)(uint64_t)bytes, hi = (int)(bytes >> 32);
  int bound;
  asm("s_cmp_lt_i32 %1, 0\n\ts_cselect_b32 %0, 0, %2\n\ts_cmp_gt_i32 %1, 0\n\ts_cselect_b32 %0, -1, %0"
      : "=&s"(bound)
      : "s"(hi), "s"(lo)
      : "scc");
  i32x4 r;
  r[0] = (int)(uint32_t)addr;
  r[1] = (int)(uint32_t)((addr >> 32) & 0xffffu);
  r[2] = bound;
  r[3] = 0x00020000;
  return r;
}

// What a kernel's wave state is compiled for.
constexpr unsigned kStream = 1;  // a workgroup walks several query tiles
constexpr unsigned kRanged = 2;  // per-row key ranges: window, chunk mask, segment starts
constexpr unsigned kBiased = 4;  // an additive bias joins the scaled scores
constexpr unsigned kSided = 8;   // one of a tile's two sides: every other key block is this wave's
constexpr unsigned kPaged = 16;  // the keys lie in pages
constexpr unsigned kCoded = 32;  // as e4m3 codes, which come into the ring through registers and are widened there

// What a wave knows of its keys' pages: nothing where they lie in rows.
template <int D, int NW, unsigned FLAGS>
struct Pages {};

// Everything a wave carries through the key loop.
template <int D, int NW, bool F16, unsigned FLAGS>
struct Wave {
  static constexpr int KS = D / 16;               // k-steps of the score product
  static constexpr int DB = Tile<D>::kWide / 32;  // 32-row blocks of O^T
  static constexpr int CH = Tile<D>::kInstrs / NW;  // fills per wave per tile
  static constexpr int kStep = (FLAGS & kSided) ? 2 * kBkv : kBkv;  // keys from one of its blocks to the next
  // block constants
  const uint8_t *k_base, *v_base;
  int64_t kv_bytes;  // bytes of this (batch, kv head)'s rows below the length
  int kv_row_bytes;
  int end;           // key blocks the query tile sees
  int len, tk;
  const void *key_mask;
  int64_t mask_row;  // b * tk
  int mask_bytes;
  int lds0;          // LDS byte address of the ring
  int wave, lane, g;
  int wave_first_row, my_row;
  bool positive;  // the maximum is kept in raw score units: a positive scale and no bias (L368-370)
  // An additive bias (Attn::bias): this lane's row of it, at the tile's first key, and the keys
  // (from there) the row holds.  Unused unless `biased`.
  const uint16_t *bias_row;
  int bias_keys;
  bool my_row_ok;  // this lane's query row exists (rows past t read no bias)
  float c_exp, unit, limit;
  // Per-row key ranges (a window, a chunk mask, segment starts: tk/src/ops/attention.rs:64-71):
  // this lane's query sees keys [row_lo, row_hi] only, a causal mask already folded into row_hi.
  // Both are non-decreasing in the row, so the wave's first and last rows bound every row's:
  // lo_last, hi_first and hi_last are theirs.  No row sees a key below lo_first, the first row's left edge by the window and
  // the chunks alone (segment starts are the caller's).  All unused unless `ranged`.
  static constexpr bool ranged = (FLAGS & kRanged) != 0;
  static constexpr bool biased = (FLAGS & kBiased) != 0;
  int row_lo, row_hi;
  int lo_first, lo_last, hi_first, hi_last;
  // per-lane addressing
  // global byte offsets of this lane's chunk in this wave's fills of a tile (one per swizzle phase)
  static constexpr int NS = (FLAGS & kPaged) ? 1 : Tile<D>::sources(NW);
  int k_src[NS], v_src[NS];
  int k_read[KS], v_read[DB];
  // state
  u32x4 qf[KS];
  f32x16 acc[DB];
  float m_run, l_run;
  int mask_next;
  // A key mask whose row was scanned at the start (rows of up to kScannedBlocks blocks): the
  // blocks' 64-bit words, in LDS after the ring.  Otherwise the words are read a
  // lane a key, two blocks ahead of their use (mask_next).
  bool scanned;
  LDS_PTR(uint64_t) mask_words;
  // A streaming workgroup's next item (STREAM; nxt_end = 0: none): this item's
  // last steps request its first blocks.  The next item's blocks follow this item's at an even
  // position of the ring (end_even = end rounded up), so every item starts in slot 0.
  const uint8_t *nxt_k, *nxt_v;
  int64_t nxt_bytes;
  int nxt_end, end_even;
  // Keys in pages (paged_kernel.hip's fills).
  Pages<D, NW, FLAGS & (kPaged | kCoded)> pages;
};

// A tile's fills where its keys lie in pages: defined beside Pages.
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ void fill_k_pages(Wave<D, NW, F16, FLAGS> &w, int n, int slot);
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ void fill_v_pages(Wave<D, NW, F16, FLAGS> &w, int n, int slot);

// The fills are issued as raw instructions: the compiler's wait-count pass treats an LDS fill
// it knows about as aliasing every later LDS read and would park the wave on the NEXT tile's
// fills in the middle of the current tile.  The kernel waits for them itself (vmcnt(0) before
// the barrier that ends a step).  m0 carries the LDS address of a wave instruction's 1 KiB.
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ void fill_tile(const Wave<D, NW, F16, FLAGS> &w, const uint8_t *base, int64_t bytes, int blk,
                                          int lds_at, const int (&src)[Tile<D>::sources(NW)], int row_bytes) {
  // This wave's fills of a tile are NW instructions apart; the swizzle repeats with that period (or
  // with twice it), so they share the lanes' offsets and differ in the descriptor's base.
  constexpr int kRowsPer = 64 / Tile<D>::kCpr;  // rows a wave instruction covers
  constexpr int NS = Tile<D>::sources(NW);
  static_assert((NS * NW * kRowsPer) % 16 == 0, "the swizzle repeats over a wave's fills");
  const int64_t off = (int64_t)blk * Wave<D, NW, F16, FLAGS>::kStep * row_bytes;
  const i32x4 r = make_rsrc(base + off, bytes - off);
#pragma unroll
  for (int i = 0; i < Wave<D, NW, F16, FLAGS>::CH; i++) {
    int voff = src[i % NS] + (NW * i * kRowsPer) * row_bytes;
    if constexpr (D == 48) voff = src[i % NS] == (int)0xfffffff0u ? src[i % NS] : voff;  // a chunk the row does not have
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(lds_at + (w.wave + NW * i) * 1024), "v"(voff), "s"(r)
                 : "memory");
  }
}
// Block `n` of the stream of blocks that starts with this item's: the item's own while n < end,
// then (past the padding to an even count) the next item's.  Nothing past either.
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ void fill_k(Wave<D, NW, F16, FLAGS> &w, int n, int slot) {
  if constexpr ((FLAGS & kPaged) != 0) {
    fill_k_pages<D, NW>(w, n, slot);
  } else {
    const int at = w.lds0 + slot * Tile<D>::kBytes;
    if (n < w.end)
      fill_tile<D, NW>(w, w.k_base, w.kv_bytes, n, at, w.k_src, w.kv_row_bytes);
    else if ((FLAGS & kStream) && n >= w.end_even && n - w.end_even < w.nxt_end)
      fill_tile<D, NW>(w, w.nxt_k, w.nxt_bytes, n - w.end_even, at, w.k_src, w.kv_row_bytes);
  }
}
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ void fill_v(Wave<D, NW, F16, FLAGS> &w, int n, int slot) {
  if constexpr ((FLAGS & kPaged) != 0) {
    fill_v_pages<D, NW>(w, n, slot);
  } else {
    const int at = w.lds0 + (2 + slot) * Tile<D>::kBytes;
    if (n < w.end)
      fill_tile<D, NW>(w, w.v_base, w.kv_bytes, n, at, w.v_src, w.kv_row_bytes);
    else if ((FLAGS & kStream) && n >= w.end_even && n - w.end_even < w.nxt_end)
      fill_tile<D, NW>(w, w.nxt_v, w.nxt_bytes, n - w.end_even, at, w.v_src, w.kv_row_bytes);
  }
}

// A key mask row is read 64 keys (one per lane) a block, one block ahead: the load is issued
// before that block's fills and is long back when the block's step needs it.
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ int mask_lane(const Wave<D, NW, F16, FLAGS> &w, int blk) {
  const int key = blk * w.kStep + w.lane;
  if (w.key_mask == nullptr || key >= w.tk) return 0;
  const int64_t at = w.mask_row + key;
  return w.mask_bytes == 1 ? (int)((const uint8_t *)w.key_mask)[at] : ((const int *)w.key_mask)[at];
}

// S^T = K . Q^T of the key block in K slot `slot`, as 32 scalars: sv[16kb + i] is the score of
// key 32kb + 8(i/4) + 4g + i%4 (sub-registers of the two accumulators: no moves).
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ void scores(const Wave<D, NW, F16, FLAGS> &w, const uint8_t *smem, int slot, float (&sv)[32]) {
  using TL = Tile<D>;
  const uint8_t *ks_ = smem + slot * TL::kBytes;
  const f32x16 zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  f32x16 s0 = zero, s1 = zero;
#pragma unroll
  for (int ks = 0; ks < Wave<D, NW, F16, FLAGS>::KS; ks++) {
    const u32x4 a0 = *reinterpret_cast<const u32x4 *>(ks_ + w.k_read[ks]);
    const u32x4 a1 = *reinterpret_cast<const u32x4 *>(ks_ + w.k_read[ks] + 32 * TL::kRowBytes);
    s0 = mma<F16>(a0, w.qf[ks], s0);
    s1 = mma<F16>(a1, w.qf[ks], s1);
  }
#pragma unroll
  for (int i = 0; i < 16; i++) {
    sv[i] = s0[i];
    sv[16 + i] = s1[i];
  }
}

// The wave-uniform part of block `blk`'s mask: bit j = the block's key j is below the length and
// kept by the key mask (`word` is this lane's key-mask element of the block).
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ uint64_t uniform_bits(const Wave<D, NW, F16, FLAGS> &w, int blk, int word) {
  const int k0 = blk * w.kStep;
  uint64_t kbits = ~0ull;
  if (w.key_mask != nullptr) {
    if (w.scanned) {
      const uint64_t x = w.mask_words[blk];  // the same address in every lane
      kbits = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)x) |
              (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(x >> 32)) << 32;
    } else {
      kbits = __builtin_amdgcn_ballot_w64(word != 0);
    }
  }
  if (k0 + kBkv > w.len) kbits &= (w.len > k0) ? (~0ull >> (64 - (w.len - k0))) : 0ull;
  return kbits;
}

// The 32 bias elements this lane's scores of the 64 keys from `first` on take, as 16 packed
// pairs: keys first + 32 kb + 8 c + 4 g + {0..3}.  Keys past the row read as zero (their scores are hidden anyway).
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ void load_bias(const Wave<D, NW, F16, FLAGS> &w, int first, bool row_ok, uint32_t (&bw)[16]) {
  const int k0 = first + 4 * w.g;
  const bool aligned = ((uintptr_t)w.bias_row & 7u) == 0;  // wave-uniform when every row is: checked per lane
#pragma unroll
  for (int c = 0; c < 8; c++) {
    const int key = k0 + 32 * (c / 4) + 8 * (c % 4);
    uint32_t lo = 0, hi = 0;
    if (row_ok && aligned && key + 3 < w.bias_keys) {
      const u32x2 x = *reinterpret_cast<const u32x2 *>(w.bias_row + key);
      lo = x[0];
      hi = x[1];
    } else if (row_ok) {
      const uint32_t e0 = key + 0 < w.bias_keys ? w.bias_row[key + 0] : 0u;
      const uint32_t e1 = key + 1 < w.bias_keys ? w.bias_row[key + 1] : 0u;
      const uint32_t e2 = key + 2 < w.bias_keys ? w.bias_row[key + 2] : 0u;
      const uint32_t e3 = key + 3 < w.bias_keys ? w.bias_row[key + 3] : 0u;
      lo = e0 | e1 << 16;
      hi = e2 | e3 << 16;
    }
    bw[2 * c] = lo;
    bw[2 * c + 1] = hi;
  }
}

// biased() of L358-362: s = fma(bias, log2(e), s) on the scaled scores, before the masks.
template <bool F16>
__device__ __forceinline__ void add_bias(const uint32_t (&bw)[16], float (&sv)[32]) {
#pragma unroll
  for (int i = 0; i < 32; i++) {
    const uint32_t pair = bw[i / 2];
    const uint16_t e = (uint16_t)((i & 1) ? pair >> 16 : pair & 0xffffu);
    float x;
    if (F16) {
      x = (float)__builtin_bit_cast(_Float16, e);
    } else {
      const uint32_t wide = (uint32_t)e << 16;
      x = __builtin_bit_cast(float, wide);
    }
    sv[i] = __builtin_fmaf(x, kLog2e, sv[i]);
  }
}

// Whether a mask edge crosses block `blk` for this wave (L698-733).
template <int D, int NW, bool CAUSAL, bool F16, unsigned FLAGS>
__device__ __forceinline__ bool on_edge(const Wave<D, NW, F16, FLAGS> &w, int blk, uint64_t kbits) {
  const int k0 = blk * w.kStep;
  if (kbits != ~0ull) return true;
  // L715-731: a range's right edge for the wave's first row, its left edge for the last.
  if (w.ranged) return k0 + kBkv - 1 > w.hi_first || k0 < w.lo_last;
  return CAUSAL && (k0 + kBkv - 1 > w.wave_first_row);
}

// What the wave's rows may see of block `blk`, by halves of 32 keys: bit h when some row may see a key of half h.  An edge
// step spends exponentials and P V on those halves only (the vector unit is what short calls wait for): 32 sequences of up to
// 140 keys 14.65 -> 14.25 us, 64 of up to 40 8.7 -> 8.55, 12 of 200 with a window of 16 keys a side 9.8 -> 9.5; and a
// range's wave skips the blocks below its left edge (4 of 4096 with a window of 64 a side 30.4 -> 28.3).  The scores, masks
// and maximum stay a block's: by halves too they cost registers the kernel does not have.  Above d 64 it is not worth the
// branches: a step in pieces leaves the scheduler nothing to put beside the products (4 causal sequences of up to 1030 at d 128
// 30.1 -> 30.6, 8 of up to 300 at d 256 19.4 -> 20.7).
template <int D, int NW, bool CAUSAL, bool F16, unsigned FLAGS>
__device__ __forceinline__ int halves_seen(const Wave<D, NW, F16, FLAGS> &w, int blk, uint64_t kbits) {
  if (D > 64) return 3;
  const int k0 = blk * w.kStep;
  const int last = w.ranged ? w.hi_last : CAUSAL ? w.wave_first_row + kWaveRows - 1 : 0x7fffffff;
  int seen = ((uint32_t)kbits != 0 && k0 <= last ? 1 : 0) | ((uint32_t)(kbits >> 32) != 0 && k0 + 32 <= last ? 2 : 0);
  if (w.ranged && k0 + 31 < w.lo_first) seen &= k0 + 63 < w.lo_first ? 0 : 2;
  return seen;
}

// Scores whose bit of `mine` is clear become -inf; bit 8 (i / 4) + i % 4 (+ 32 for the second
// half) is this lane's score i: the key that many places past the lane's first.
__device__ __forceinline__ void hide_scores(uint64_t mine, float (&sv)[32]) {
  const int lo = (int)(uint32_t)mine, hi = (int)(uint32_t)(mine >> 32);
  // Two instructions a score, its bit over a whole word and a choice by bits (an and, a compare and a select were three):
  // 32 sequences of at most 140 keys 15.1 -> 14.65 us, 4 of 4096 with a window of 64 a side 28.3 -> 27.7, 4 of at most 1030,
  // causal, d 128, 30.7 -> 30.1.
  auto hidden_unless = [](float x, int bit_word) {
    const uint32_t keep = (uint32_t)bit_word, u = __float_as_uint(x);
    return __uint_as_float((u & keep) | (0xff800000u & ~keep));
  };
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const int rel = 8 * (i / 4) + (i % 4);  // key k0 + 32kb + 4g + rel
    sv[i] = hidden_unless(sv[i], __builtin_amdgcn_sbfe(lo, rel, 1));
    sv[16 + i] = hidden_unless(sv[16 + i], __builtin_amdgcn_sbfe(hi, rel, 1));
  }
}

// Scales (a non-positive scale only) and masks (L641-697) the scores of block `blk`: hidden
// scores become -inf.  `kbits` is the uniform word; causality adds a per-lane one.
template <int D, int NW, bool CAUSAL, bool F16, unsigned FLAGS>
__device__ __forceinline__ void mask_scores(const Wave<D, NW, F16, FLAGS> &w, int blk, uint64_t kbits, float (&sv)[32]) {
  const int k0 = blk * w.kStep;
  uint64_t mine = kbits;
  if (w.ranged) {
    // Keys k0 .. row_hi are seen from above and those from row_lo on from below (L659-695).
    const int seen = w.row_hi - k0 + 1;
    mine &= seen >= 64 ? ~0ull : (seen <= 0 ? 0ull : (~0ull >> (64 - seen)));
    const int below = w.row_lo - k0;
    mine &= below <= 0 ? ~0ull : (below >= 64 ? 0ull : (~0ull << below));
  } else if (CAUSAL && (k0 + kBkv - 1 > w.wave_first_row)) {
    const int seen = w.my_row - k0 + 1;  // keys k0 .. my_row are seen
    mine &= seen >= 64 ? ~0ull : (seen <= 0 ? 0ull : (~0ull >> (64 - seen)));
  }
  hide_scores(mine >> (4 * w.g), sv);
}

// The row maximum of a block's scores: in-lane tree of three-way folds, then the other
// half-wave's.
__device__ __forceinline__ float row_max(const float (&sv)[32]) {
  float t[11];
#pragma unroll
  for (int i = 0; i < 10; i++) t[i] = max3(sv[3 * i], sv[3 * i + 1], sv[3 * i + 2]);
  t[10] = __builtin_fmaxf(sv[30], sv[31]);
  const float u0 = max3(t[0], t[1], t[2]), u1 = max3(t[3], t[4], t[5]), u2 = max3(t[6], t[7], t[8]);
  const float bm = max3(max3(u0, u1, u2), t[9], t[10]);
  const Pair p = both_halves(bm);
  return __builtin_fmaxf(p.a, p.b);
}

// Half a block's probabilities: p = 2^(s*unit - m*unit) for 16 scores, summed unrounded in
// four chains, then held as bf16 (L432-444).
template <bool F16>
__device__ __forceinline__ void probabilities(const float *sv, float unit, float m_exp, float (&bs)[4],
                                              uint32_t *pk) {
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    const float p0 = fast_exp2(__builtin_fmaf(sv[i], unit, -m_exp));
    const float p1 = fast_exp2(__builtin_fmaf(sv[i + 1], unit, -m_exp));
    const float p2 = fast_exp2(__builtin_fmaf(sv[i + 2], unit, -m_exp));
    const float p3 = fast_exp2(__builtin_fmaf(sv[i + 3], unit, -m_exp));
    bs[0] += p0;
    bs[1] += p1;
    bs[2] += p2;
    bs[3] += p3;
    pk[i / 2] = pack2<F16>(p0, p1);
    pk[i / 2 + 1] = pack2<F16>(p2, p3);
  }
}

// O^T += V^T . P^T over 32 keys (half a block): chunks c of 16 keys, fragment registers 4c..4c+3.
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ void accumulate(Wave<D, NW, F16, FLAGS> &w, const uint8_t *vs_, int half, const uint32_t *pk) {
  using TL = Tile<D>;
#pragma unroll
  for (int c = 0; c < 2; c++) {
    const u32x4 pw = {pk[4 * c], pk[4 * c + 1], pk[4 * c + 2], pk[4 * c + 3]};

#pragma unroll
    for (int db = 0; db < Wave<D, NW, F16, FLAGS>::DB; db++) {
      const uint8_t *at = vs_ + w.v_read[db] + (32 * half + 16 * c) * TL::kRowBytes;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(at));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(at + 8 * TL::kRowBytes));
      const s16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      w.acc[db] = mma<F16>(__builtin_bit_cast(u32x4, both), pw, w.acc[db]);
    }
  }
}

// The running maximum's update for a block whose row maximum is `bm`: the lazy rescale of
// L418-431, and the O^T rescale that a wave skips when all its rows kept their maximum
// (L56-59).  Returns the exponent's offset m*unit; `corr` is the correction of l.
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ float adopt_maximum(Wave<D, NW, F16, FLAGS> &w, float bm, float &corr) {
  const float m_max = __builtin_fmaxf(w.m_run, bm);
  const bool grows = w.limit < (m_max - w.m_run);
  const float m_new = grows ? m_max : w.m_run;
  corr = fast_exp2((w.m_run - m_new) * w.unit);
  w.m_run = m_new;
  if (__builtin_amdgcn_ballot_w64(corr != 1.0f) != 0) {
#pragma unroll
    for (int db = 0; db < Wave<D, NW, F16, FLAGS>::DB; db++) w.acc[db] *= corr;
  }
  return m_new * w.unit;
}

// Keeps the computation of `x` where the source has it: instruction selection is otherwise free
// to let arithmetic without side effects drift past the fences between slots.
__device__ __forceinline__ void pin(float &x) { asm volatile("" : "+v"(x)); }

// One unit of the exponentials: two scores to two probabilities (p = 2^(s*unit - m*unit)),
// each added unrounded to a row-sum chain, the pair held as bf16 (L432-444).
template <bool F16>
__device__ __forceinline__ uint32_t p_unit(float s_a, float s_b, float unit, float m_exp, float &sum_a, float &sum_b) {
  const float pa = fast_exp2(__builtin_fmaf(s_a, unit, -m_exp));
  const float pb = fast_exp2(__builtin_fmaf(s_b, unit, -m_exp));
  sum_a += pa;
  sum_b += pb;
  return pack2<F16>(pa, pb);
}

// The hot step: block `blk` (parity PAR = blk & 1: V(blk) in V slot PAR, K(blk+1) in K slot
// PAR^1) when block blk+1 is this wave's too, no mask edge crosses it and the scale is
// positive.  `sv` holds S(blk) and `bm` its row maximum; S(blk+1) goes to `nv`, its maximum to
// `bm`.
//
// The step is written as a sequence of slots, one matrix instruction each, fenced so that the
// compiler keeps their order: the LDS fragment a matrix instruction reads was requested four
// slots earlier, and each slot carries its share of the VALU work, so that the matrix pipe
// never waits for the VALU's whole job.  2 KS slots compute S(blk+1) beside the exponentials
// of keys 0..31; 2 DB slots add P V of keys 0..31 beside the exponentials of keys 32..63;
// 2 DB slots add P V of keys 32..63 beside the row maximum of S(blk+1).
template <int D, int NW, int PAR, bool F16, unsigned FLAGS>
__device__ __forceinline__ void hot_step(Wave<D, NW, F16, FLAGS> &w, const uint8_t *smem, int blk, const float (&sv)[32],
                                         float (&nv)[32], float &bm) {
  using TL = Tile<D>;
  constexpr int KS = Wave<D, NW, F16, FLAGS>::KS, DB = Wave<D, NW, F16, FLAGS>::DB;
  constexpr int NQK = 2 * KS;  // score slots
  constexpr int NPV = 4 * DB;  // P V slots, half of them per 32 keys
  const uint8_t *ks_ = smem + (PAR ^ 1) * TL::kBytes;
  const uint8_t *vs_ = smem + (2 + PAR) * TL::kBytes;
  // Score fragment f: key half kb = f & 1, k-step ks = f >> 1.
  auto k_frag = [&](int f) -> u32x4 {
    return *reinterpret_cast<const u32x4 *>(ks_ + w.k_read[f >> 1] + (f & 1) * 32 * TL::kRowBytes);
  };
  // P V fragment j: 16-key chunk c = j / DB (0..3), d-block db = j % DB.
  auto v_frag = [&](int j) -> s16x8 {
    const uint8_t *at = vs_ + w.v_read[j % DB] + 16 * (j / DB) * TL::kRowBytes;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(at));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(at + 8 * TL::kRowBytes));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };

  u32x4 kf[4];
#pragma unroll
  for (int f = 0; f < 4; f++) kf[f] = k_frag(f);
  fill_v<D, NW>(w, blk + 1, PAR ^ 1);
  fill_k<D, NW>(w, blk + 2, PAR);
  w.mask_next = 0;  // hot steps run without a key mask only
  float corr;
  const float m_exp = adopt_maximum<D, NW>(w, bm, corr);
  __builtin_amdgcn_sched_barrier(0);

  float bs[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  uint32_t pk[16];
  s16x8 vf[4];
  const f32x16 zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  f32x16 s0 = zero, s1 = zero;
  // ---- S(blk+1) beside the probabilities of keys 0..31 (8 units over NQK slots).
#pragma unroll
  for (int i = 0; i < NQK; i++) {
    if (i & 1)
      s1 = mma<F16>(kf[i & 3], w.qf[i >> 1], s1);
    else
      s0 = mma<F16>(kf[i & 3], w.qf[i >> 1], s0);
    if (i + 4 < NQK)
      kf[i & 3] = k_frag(i + 4);
    else
      vf[(i + 4 - NQK) & 3] = v_frag(i + 4 - NQK);
#pragma unroll
    for (int u = 8 * i / NQK; u < 8 * (i + 1) / NQK; u++)
      pk[u] = p_unit<F16>(sv[2 * u], sv[2 * u + 1], w.unit, m_exp, bs[(2 * u) & 3], bs[(2 * u + 1) & 3]);
    if (8 * i / NQK < 8 * (i + 1) / NQK) {
#pragma unroll
      for (int x = 0; x < 4; x++) pin(bs[x]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int i = 0; i < 16; i++) {
    nv[i] = s0[i];
    nv[16 + i] = s1[i];
  }
  // ---- O += P V of keys 0..31 beside the probabilities of keys 32..63, then O += P V of keys
  // 32..63 beside the row maximum of S(blk+1).
  float t[11];
#pragma unroll
  for (int j = 0; j < NPV; j++) {
    const int c = j / DB;
    const u32x4 pw = {pk[4 * c], pk[4 * c + 1], pk[4 * c + 2], pk[4 * c + 3]};
    w.acc[j % DB] = mma<F16>(__builtin_bit_cast(u32x4, vf[j & 3]), pw, w.acc[j % DB]);
    if (j + 4 < NPV) vf[j & 3] = v_frag(j + 4);
    if (j < NPV / 2) {
#pragma unroll
      for (int u = 8 + 16 * j / NPV; u < 8 + 16 * (j + 1) / NPV; u++)
        pk[u] = p_unit<F16>(sv[2 * u], sv[2 * u + 1], w.unit, m_exp, bs[(2 * u) & 3], bs[(2 * u + 1) & 3]);
#pragma unroll
      for (int x = 0; x < 4; x++) pin(bs[x]);
    } else {
      // The row maximum's first level, ten three-way folds and one two-way, over these slots.
      const int jj = j - NPV / 2;
#pragma unroll
      for (int x = 11 * jj / (NPV / 2); x < 11 * (jj + 1) / (NPV / 2); x++)
      {
        t[x] = x < 10 ? max3(nv[3 * x], nv[3 * x + 1], nv[3 * x + 2]) : __builtin_fmaxf(nv[30], nv[31]);
        pin(t[x]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  {
    const float u0 = max3(t[0], t[1], t[2]), u1 = max3(t[3], t[4], t[5]), u2 = max3(t[6], t[7], t[8]);
    const Pair p = both_halves(max3(max3(u0, u1, u2), t[9], t[10]));
    bm = __builtin_fmaxf(p.a, p.b);
  }
  w.l_run = w.l_run * corr + ((bs[0] + bs[1]) + (bs[2] + bs[3]));
  // vmcnt(0): the fills issued this step have landed.  (Codes are in registers, for the next step to write.)
  if constexpr ((FLAGS & kCoded) == 0) __builtin_amdgcn_s_waitcnt(0x0f70);
  __syncthreads();
}

// The general step, for the blocks at the edges: any block, a next block or none, masks, any
// scale.  Slots are picked at run time.  `sv` holds the masked S(blk), `bm` its row maximum and `seen` its halves that
// any row sees; on exit they hold block blk+1's (when this wave has one).
template <int D, int NW, bool CAUSAL, bool F16, unsigned FLAGS>
__device__ __forceinline__ void edge_step(Wave<D, NW, F16, FLAGS> &w, const uint8_t *smem, int blk, int my_end, float (&sv)[32],
                                          float &bm, int &seen) {
  using TL = Tile<D>;
  const int par = blk & 1;
  const bool more = blk + 1 < my_end;
  const uint64_t kbits_next = uniform_bits<D, NW>(w, blk + 1, w.mask_next);
  // The next block's bias is asked for first: it has this block's P.V to arrive under.
  uint32_t bw[16];
  if (w.biased && more) load_bias<D, NW>(w, (blk + 1) * kBkv, w.my_row_ok, bw);
  fill_v<D, NW>(w, blk + 1, par ^ 1);
  if (!w.scanned && blk + 2 < w.end) w.mask_next = mask_lane<D, NW>(w, blk + 2);
  fill_k<D, NW>(w, blk + 2, par);
  float corr;
  const float m_exp = adopt_maximum<D, NW>(w, bm, corr);

  const uint8_t *vs_ = smem + (2 + par) * TL::kBytes;
  float bs[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  uint32_t pk[16];
  if constexpr (D > 64) {  // both halves always, in one piece for the scheduler
    probabilities<F16>(sv, w.unit, m_exp, bs, pk);
    probabilities<F16>(sv + 16, w.unit, m_exp, bs, pk + 8);
    accumulate<D, NW>(w, vs_, 0, pk);
    accumulate<D, NW>(w, vs_, 1, pk + 8);
  } else {
    if (seen & 1) {
      probabilities<F16>(sv, w.unit, m_exp, bs, pk);
      accumulate<D, NW>(w, vs_, 0, pk);
    }
    if (seen & 2) {
      probabilities<F16>(sv + 16, w.unit, m_exp, bs, pk + 8);
      accumulate<D, NW>(w, vs_, 1, pk + 8);
    }
  }
  w.l_run = w.l_run * corr + ((bs[0] + bs[1]) + (bs[2] + bs[3]));
  if (more) {
    seen = halves_seen<D, NW, CAUSAL>(w, blk + 1, kbits_next);
    bm = -INFINITY;
    if (D > 64 || !w.ranged || seen != 0) {
      scores<D, NW>(w, smem, par ^ 1, sv);
      if (!w.positive) {
#pragma unroll
        for (int i = 0; i < 32; i++) sv[i] *= w.c_exp;
      }
      if (w.biased) add_bias<F16>(bw, sv);
      if (on_edge<D, NW, CAUSAL>(w, blk + 1, kbits_next)) mask_scores<D, NW, CAUSAL>(w, blk + 1, kbits_next, sv);
      bm = row_max(sv);
    }
  }
  // vmcnt(0): the fills issued this step have landed.  (Codes are in registers, for the next step to write.)
  if constexpr ((FLAGS & kCoded) == 0) __builtin_amdgcn_s_waitcnt(0x0f70);
  __syncthreads();
}

// A step of a wave with nothing to compute: fills and the barrier only.
template <int D, int NW, bool F16, unsigned FLAGS>
__device__ __forceinline__ void idle_step(Wave<D, NW, F16, FLAGS> &w, int blk) {
  const int par = blk & 1;
  fill_v<D, NW>(w, blk + 1, par ^ 1);
  fill_k<D, NW>(w, blk + 2, par);
  if constexpr ((FLAGS & kCoded) == 0) __builtin_amdgcn_s_waitcnt(0x0f70);
  __syncthreads();
}

// n / d for n < 2^32 with rcp = floor(2^32 / d) (2^32 - 1 for d = 1) from the host: the
// estimate is the quotient or one less.
__device__ __forceinline__ uint32_t div_by(uint32_t n, uint32_t d, uint32_t rcp) {
  const uint32_t q = __umulhi(n, rcp);
  return n - q * d >= d ? q + 1 : q;
}

}  // namespace
}  // namespace svodk
