// What the attention kernels over the 4-bit key/value cache share.
//
// Operands are f16 for both types of T.  A nibble left in bits 0..3 (4..7) of
// a 16-bit half reads as the f16 subnormal q * 2^-24 (q * 2^-20), so one AND
// extracts two of them and one v_pk_fma_f16 makes two values
//   (s * 2^(24 - E)) * (q * 2^-24) + b * 2^-E = (s q + b) * 2^-E
// with a single rounding.  E, the same for the keys (the values) of one product, is
// chosen by the largest constant among them, max(|b|, 16 |s|) within 2^(E - 5): then
// s * 2^(24 - E) <= 2^15 fits f16, whatever T's range.  A value is off by at most
// 2^-11 of itself or, where it lies among f16's subnormals, by its bias's rounding
// and its own, 2^-19 each of 2^(E - 5).
//
// Tokens whose constants are far apart do not share a product, or the largest would
// take the others' bits, also from rows that do not see it.  E stays from tile to tile
// while it holds every token (their largest constants within (2^(E - 12), 2^(E - 5)]),
// so any of them is off by 2^-11 of its largest at most; else the tile's tokens are taken in
// passes, the largest first (a softmax takes its keys in any portions).  A row's sums change their unit where a product that it sees has another.
//
// fp32 operands would run the matrix instructions at a sixteenth of the rate.  What
// one rounding each of keys, values and weights costs at T = bf16: for few rows
// nothing (2-norm 0.0017 against 64 bits either way, the output's own rounding), for
// prompts 0.0018 where a form in 32 bits has 0.0016.  At T = f16, where the output's
// rounding alone is 0.0002, outputs would be off by 0.0004 to 0.0013, most of it the
// keys': keys and weights are kept whole there and the values' one rounding is left
// (0.0003; kv_decode.hip and kv_attention.hip say how).
#pragma once

#include <cfloat>

#include "../cpq_internal.hpp"
#include "common.hpp"

namespace cpq {
namespace dev {

constexpr int kKvTop = 5;    // constants stay below 2^(E - kKvTop)
constexpr int kKvBand = 6;   // exponents of tokens are E - kKvBand .. E
constexpr int kKvKeep = 2;   // E stays while it is at most this much more than a tile needs
constexpr int kKvNone = -1000;  // the exponent of a token whose constants are zero: fits all
constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ f16x2 as_f16x2(uint32_t v) { return __builtin_bit_cast(f16x2, v); }
__device__ __forceinline__ uint32_t pk_fma(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(as_f16x2(a), as_f16x2(b), as_f16x2(c)));
}
__device__ __forceinline__ uint32_t sixteenth(uint32_t a) {
  return __builtin_bit_cast(uint32_t, as_f16x2(a) * f16x2{(_Float16)0.0625f, (_Float16)0.0625f});
}
// x * 2^e, also where 2^e is no float.
__device__ __forceinline__ float scaled(float x, int e) { return __builtin_amdgcn_ldexpf(x, e); }
// The exponent e with |x| < 2^e, from x's bits (x finite).
__device__ __forceinline__ int exponent_above(float x) { return (int)(__float_as_uint(x) >> 23 & 255) - 126; }
__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= FLT_MAX; }

// The largest |scale| and |bias| of constants as T patterns in one word (both
// types order like integers; Inf and NaN come last).
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ uint32_t pk_min(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ uint32_t sizes(uint32_t m, uint32_t sb) { return pk_max(m, sb & 0x7fff7fffu); }
__device__ __forceinline__ uint32_t smallest(uint32_t m, uint32_t sb) { return pk_min(m, sb & 0x7fff7fffu); }
// What `sizes` may reach at exponent E: scales 2^(E - 9), biases 2^(E - 5), finite.
template <typename TT>
__device__ __forceinline__ uint32_t size_limits(int e) {
  const uint32_t top = Sig16<TT>::bf16 ? 0x7f7fu : 0x7bffu;
  const uint32_t s = TT::from_f32(scaled(1.f, e - kKvTop - 4)), b = TT::from_f32(scaled(1.f, e - kKvTop));
  return min(s, top) | min(b, top) << 16;
}
// Whether `sizes` of constants has none that is not finite.
template <typename TT>
__device__ __forceinline__ bool all_finite(uint32_t m) {
  return finite(TT::lo(m)) && finite(TT::hi(m));
}
// max(|b|, 16 |s|) of a constant, 0 where it is not finite.
template <typename TT>
__device__ __forceinline__ float finite_size(uint32_t sb) {
  const float s = fabsf(TT::lo(sb)), b = fabsf(TT::hi(sb));
  return s <= FLT_MAX && b <= FLT_MAX ? fminf(fmaxf(b, 16.f * s), FLT_MAX) : 0.f;
}
// The exponent for constants up to m; none for zeros.
__device__ __forceinline__ int size_exponent(float m) {
  return m > 0.f ? max(exponent_above(m), -110) + kKvTop : kKvNone;
}
// An exponent E with what goes with it: the limits of sizes that it holds, and sizes
// at or below which a token may be too small for it.
struct KvRange {
  int e = 0;
  uint32_t high = 0, low = 0;
  // m, l: `sizes` and `smallest` of constants.  False where one may not fit (a small
  // bias of one and a small scale of another look like a small token).
  __device__ __forceinline__ bool holds(uint32_t m, uint32_t l) const {
    return (pk_max(m, high) == high) & (pk_max(l, low) != low);
  }
  template <typename TT>
  __device__ __forceinline__ void set(int to) {
    e = to;
    high = size_limits<TT>(to);
    low = size_limits<TT>(to - kKvBand - 1);
  }
  // For tokens whose largest exponent is `need`; takes(x): those it holds.
  template <typename TT>
  __device__ __forceinline__ void fit(int need) {
    if (need != kKvNone && (high == 0 || need > e || need < e - kKvKeep)) set<TT>(need);
  }
  __device__ __forceinline__ bool takes(int x) const { return x == kKvNone || (x <= e && x >= e - kKvBand); }
};

// Until the wave's LDS reads and writes are done.
__device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14)); }

// Bits [lo, hi) of 32 keys.
__device__ __forceinline__ uint32_t range_bits(int lo, int hi) {
  lo = min(max(lo, 0), 32);
  hi = min(max(hi, 0), 32);
  return (uint32_t)((1ull << hi) - 1) & ~(uint32_t)((1ull << lo) - 1);
}

// Over the lanes that differ in bits 4 and 5 (16 columns are left).
template <typename F>
__device__ __forceinline__ float over_rows(float v, F f) {
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const float w = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const uint32_t x = __float_as_uint(w);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float sum_of(float a, float b) { return a + b; }
// The exponent of the unit that a row's sums take, of which `largest_sum` in units of 2^was
// is the largest, where a product comes in units of 2^to below that: not beyond what
// fp32 holds.
__device__ __forceinline__ int lower_unit(int was, int to, float largest_sum) {
  return largest_sum > 0.f ? min(max(to, was + exponent_above(largest_sum) - 120), was) : to;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

// The largest of 16 columns' values that the wave's rows share, in a scalar register.
__device__ __forceinline__ int max_of_columns(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x128, 0xf, 0xf, false));  // row_ror 8, 4, 2, 1
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x124, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x122, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x121, 0xf, 0xf, false));
  return __builtin_amdgcn_readfirstlane(v);
}

__device__ __forceinline__ int max_of_wave(int v) {
  const auto a = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  v = max((int)a[0], (int)a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
  return max_of_columns(max((int)b[0], (int)b[1]));
}

// Inclusive sum over the wave: within rows of 16 lanes, then from row to row.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15 into rows 1, 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast 31 into rows 2, 3
  return v;
}
// 16 bytes of a partial result that a workgroup on another XCD reads or wrote in
// this launch: through to the memory side and from it.  `base` is the same for
// the whole wave.
constexpr int kSc1 = 16;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t park_rsrc(const void* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7fffffff, 0x00020000);
}
__device__ __forceinline__ void park_store(const void* base, int off, f32x4 v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), park_rsrc(base), off, 0, kSc1);
}
__device__ __forceinline__ f32x4 park_load(const void* base, int off) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(park_rsrc(base), off, 0, kSc1));
}

// One sequence of a call as a workgroup sees it.
struct KvSeq {
  int rows0;  // first query row in q and out
  int n_q;
  int n;    // keys, bounded by what the table's row holds
  int pos;  // position of its first query (n_q queries stand at the end; may be negative)
  int lo;   // first key that any query sees
};

// Sequence s, or n_q = 0 where its rows are not within the call's.  `report`:
// this thread counts what is wrong with it.
__device__ __forceinline__ KvSeq kv_seq(const cpq_kv_attention_args& a, int s, int bs_shift, bool report,
                                        unsigned int* bad) {
  const uint32_t s0 = a.query_starts[s], s1 = a.query_starts[s + 1], len = a.kv_lens[s];
  KvSeq q{};
  if (s1 <= s0) {
    if (s1 < s0 && report) atomicAdd(bad, 1u);
    return q;
  }
  if (s1 > a.n_tokens || s1 - s0 > a.max_q) {
    if (report) atomicAdd(bad, 1u);
    return q;
  }
  const uint64_t room = (uint64_t)a.max_blocks << bs_shift, most = room < 0x7fff0000ull ? room : 0x7fff0000ull;
  if (len > most && report) atomicAdd(bad, 1u);
  q.rows0 = (int)s0;
  q.n_q = (int)(s1 - s0);
  q.n = (int)(len < most ? len : most);
  q.pos = q.n - q.n_q;
  q.lo = a.window && (uint64_t)(q.pos + 1 > 0 ? q.pos + 1 : 0) > a.window ? q.pos + 1 - (int)a.window : 0;
  return q;
}

// A block table's row, read through the scalar cache: nothing writes it while
// the kernel runs.
typedef const __attribute__((address_space(4))) uint32_t* KvBlocks;
__device__ __forceinline__ KvBlocks kv_blocks(const cpq_kv_attention_args& a, int s) {
  return (KvBlocks)(a.block_table + (size_t)s * a.max_blocks);
}
// The table index of 16 keys from t (a multiple of 16); past the end of the last
// keys' block (their loads are in bounds, their results masked).
__device__ __forceinline__ int kv_index(int t, int n, int bs_shift) { return min(t, (n - 1) & ~15) >> bs_shift; }
// Where 16 keys lie: the row of the first in the cache's [block][head][offset]
// order, and whether the block is one of the cache's.
struct KvPlace {
  size_t row;
  bool ok;
};
__device__ __forceinline__ KvPlace kv_place(const cpq_kv_cache& c, uint32_t id, int at, int head, int bs_shift) {
  const bool ok = id < c.n_blocks;
  return KvPlace{(((size_t)(ok ? id : 0) * c.n_kv_heads + head) << bs_shift) + (at & ((1 << bs_shift) - 1)), ok};
}
// Of 32 keys.
struct KvPlaces {
  KvPlace a, b;
};
__device__ __forceinline__ KvPlaces kv_places(const cpq_kv_cache& c, uint32_t id0, uint32_t id1, int t, int n, int head,
                                              int bs_shift) {
  return KvPlaces{kv_place(c, id0, t, head, bs_shift), kv_place(c, id1, min(t + 16, (n - 1) & ~15), head, bs_shift)};
}

// A value constant that is not finite is taken as zero and makes its group's
// dimensions NaN in the rows that see the key (a masked row would meet 0 * NaN
// otherwise): the groups of such keys among 16 from `key` in [from, to).  Only
// where a tile holds any, so a loop over memory does.
template <typename TT>
__device__ __forceinline__ uint32_t poisoned_groups(const cpq_kv_cache& c, const KvPlace& p, int key, int G, int from,
                                                    int to) {
  uint32_t groups = 0;
  if (!p.ok) return groups;
#pragma clang loop unroll(disable)
  for (int e = 0; e < 16 * G; ++e) {
    const uint32_t sb = c.v_sb[p.row * G + e];
    if (finite(TT::lo(sb)) && finite(TT::hi(sb))) continue;
    const int k = key + e / (4 * G) * 4 + (e & 3);
    groups |= (uint32_t)(k >= from && k < to) << (e / 4 % G);
  }
  return groups;
}

// Rows of q as f16 operands: 8 values of T times 2^-e, in the order of a key
// word's nibbles once extracted: (0, 4) (1, 5) (2, 6) (3, 7).
template <typename TT>
__device__ __forceinline__ u32x4 query_slice(u32x4 raw, int e) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = scaled(TT::lo(raw[i]), -e);
    x[2 * i + 1] = scaled(TT::hi(raw[i]), -e);
  }
  return u32x4{F16::pack2(x[0], x[4]), F16::pack2(x[1], x[5]), F16::pack2(x[2], x[6]), F16::pack2(x[3], x[7])};
}
template <typename TT>
__device__ __forceinline__ float largest(u32x4 raw, float m) {
#pragma unroll
  for (int i = 0; i < 4; ++i) m = fmaxf(m, fmaxf(fabsf(TT::lo(raw[i])), fabsf(TT::hi(raw[i]))));
  return m;
}
// The exponent that brings a row's largest value into [2^14, 2^15): every
// value of T down to 2^-28 of it stays exact in f16.
__device__ __forceinline__ int query_exponent(float m) { return m > 0.f ? max(exponent_above(m), -100) - 15 : 0; }

// A word of keys as an operand of 8 dimensions.
__device__ __forceinline__ u32x4 key_slice(uint32_t w, uint32_t s, uint32_t s16, uint32_t b) {
  const uint32_t w8 = w >> 8;
  return u32x4{pk_fma(w & 0x000f000fu, s, b), pk_fma(w & 0x00f000f0u, s16, b), pk_fma(w8 & 0x000f000fu, s, b),
               pk_fma(w8 & 0x00f000f0u, s16, b)};
}

}  // namespace dev
}  // namespace cpq
