// Attention of a step's queries over the 4-bit key/value cache (semantics:
// cpq_kv_attention and, scored, cpq_kv_attention_scored in cpq.h): the kernel for many
// query rows per sequence, and the choice between it and kv_decode.hpp.
//
// A workgroup takes 32 query rows a wave of one key/value head (rows run over the
// queries, then the heads of the group, so a group of any size shares the keys)
// and walks tiles of 64 keys:
//   S^T = K Q^T     v_mfma_f32_32x32x16_f16, A = 32 keys, B = 32 query rows
//   O^T += V^T P^T  A = 32 dimensions over 16 keys, B = the weights, which
//                   S^T's result layout holds as B takes them: lane (row n, h)
//                   has keys 8 x + 4 h + 0 .. 3, so a k step's 16 keys are
//                   {4 h .. 4 h + 3, 8 + 4 h ..} of either operand.
// Keys and values become f16 operands in LDS once per workgroup (kv_common.hpp).  Of
// four waves two dequantize a tile's keys and two its values.  At head_dim 128 a
// workgroup has two such teams: each stages every second tile, one team before and
// one between the products of two tiles, into the other half of four tiles of LDS,
// so that on each SIMD one wave's dequantization meets the other's matrix
// instructions; one barrier every two tiles.  At head_dim 256 (the rows take twice
// the registers), at 64 (three workgroups share a CU) and where eight waves a
// workgroup would leave CUs without one, it has one team, two tiles of LDS and a
// barrier every tile.  The packed words of a team's next tile are in
// flight meanwhile.  (4096 queries of 32 heads over 8192 keys of 8, back to back until
// the clock has settled: head_dim 128 442 us, 64 370, 256 1434; when each was chosen:
// a barrier every tile 470 us for 429, four waves a workgroup 607; head_dim 64 with
// eight waves 429 us for 344.)
//   LDS image: 16-byte units, a key's word (8 dimensions) or a dimension's 8
//   keys of a k step, XORed so that neighbouring lanes' b128 reads and writes meet
//   in different banks (measured: 8 lanes are served at a time, 8 cycles a read;
//   a key that repeats among them doubles it).
// No maximum is taken on the way: weights are 2^(score - reference), and only
// where their sums show that one leaves f16's range (the first tile's do) is the
// maximum of the half tile found, the reference raised to 2^-10 of it and its weights
// made again.  The weights of a tile's first 32 keys are made between the matrix
// instructions of the other 32 keys' scores, theirs between those of the first
// keys' values (when that came in: head_dim 64 350 -> 337 us).
//
// Bound by its instructions: 4096 queries over 8192 keys at head_dim 128 run at 933
// TFLOP/s (a large f16 product of the library: 1322), with the vector pipes busy for
// 55% of the cycles, the matrix pipes for 42%, both at once for 17%.  The first twenty
// calls after a pause take 520 us, not 442: the clock.
//
// A tile whose tokens are too far apart for one exponent is staged and multiplied again
// for each set of them that goes together (kv_common.hpp), its words loaded once more
// each time; that, like all that is rare, lies outside the loop's straight line (with it
// inside the line 7 % were lost).
//
// Where there are few row tiles their keys are split, evenly over the resident
// workgroups by the lengths on the device, and joined, in part order, by the last
// to arrive.
#pragma once

#include <algorithm>

#include "kv_common.hpp"

namespace cpq {
namespace {

using namespace dev;

constexpr int kKeys = 64;        // of a tile
constexpr int kMinTiles = 4;     // of a part
// log2 of the largest weight when the reference is set: with it one of 2^-24 of the
// largest keeps 11 bits (beside a key that draws nearly all weight and holds zeros the
// others make the output).  At 2^6 the reference is set less often: 1 % of the time.
constexpr float kRaise = 10.f;
constexpr float kMost = 65504.f;  // of 16 weights' sum, so that each fits f16
// What a wave publishes of its half of a tile: the exponent (0: all constants so
// far are zeros), which 16 keys have their block, whether a value constant is not
// finite, whether its tokens are too far apart for one exponent.
constexpr int kExpBias = 1 << 12, kOkShift = 16, kPoison = 1 << 20, kApart = 1 << 21;
// Halves of values whose exponents differ by no more than this are joined by smaller
// weights; others are too far apart.
constexpr int kMostApart = 4;

// At T = f16 queries' sums over a group enter a product as 2^-kSumShift of them.
constexpr int kSumShift = 7;

struct TileArgs {
  cpq_kv_cache c;
  cpq_kv_attention_args a;
  int few_rows;    // sequences of up to this many rows are another kernel's
  int target;      // parts to divide the tiles into, 0: no splits
  unsigned int* counters;  // per workgroup that is a first part
  float* partial;          // [workgroup][wave][D / 8 + 1][lane] f32x4: rows, then (maximum, sum)
  int report;  // this launch counts what is wrong with the sequences
  unsigned int* bad;
  KvScore score;
};

__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Unit of a key's word.
template <int W>
__device__ __forceinline__ int key_unit(int key, int w) {
  return key * W + (w ^ (key & (W < 16 ? 7 : 15)));
}
// Unit of a dimension's keys of half k step ts (2 * step + h): read at
// neighbouring dimensions, written at dimensions 8 apart (two of eight lanes
// meet there: the bank conflicts that are left, 16 cycles a wave's tile, 2.6% of the
// busy ones).  Dimensions 32 apart have the same place in their rows.
__device__ __forceinline__ int value_unit(int d, int ts) { return d * 8 + (ts ^ ((d ^ (d >> 3 & 3)) & 7)); }

// The packed words of one wave's 32 keys: as keys, lane (key, half of the
// words); as values, lane (word, half k step) -- twice at head_dim 256.
template <int D>
struct Packed {
  static constexpr int NK = D / 64;            // 16-byte loads of a key's half, and its constants
  static constexpr int VS = D == 256 ? 2 : 1;  // value words per lane
  static constexpr int N = NK > 2 * VS ? NK : 2 * VS;
  u32x4 q[N];
  u32x4 sb[2 * VS];  // values: constants of q's four keys each; keys: sb[0], one per 16-byte load
};

template <int D>
__device__ __forceinline__ void load_keys(Packed<D>& t, const cpq_kv_cache& c, size_t row_a, size_t row_b, int lane,
                                          int gw_shift) {
  constexpr int W = D / 8, NK = Packed<D>::NK;
  const int G = W >> gw_shift, half = lane >> 5;
  const size_t row = (lane & 16 ? row_b : row_a) + (lane & 15);
  const u32x4* q = reinterpret_cast<const u32x4*>(c.k_q + row * W + half * (W / 2));
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    t.q[i] = q[i];
    t.sb[0][i] = c.k_sb[row * G + ((half * (W / 2) + 4 * i) >> gw_shift)];
  }
}
template <int D>
__device__ __forceinline__ void load_values(Packed<D>& t, const cpq_kv_cache& c, size_t row_a, size_t row_b, int lane,
                                            int gw_shift) {
  constexpr int W = D / 8, L = W < 16 ? 8 : 16;  // lanes over words
  const int G = W >> gw_shift, ts = lane / L & 3;
  const size_t quad = ((ts & 2 ? row_b : row_a) >> 2) + (ts & 1);
#pragma unroll
  for (int v = 0; v < Packed<D>::VS; ++v) {
    const int w = 16 * v + lane % L;
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // keys 4 h .., 8 + 4 h ..
      t.q[2 * v + e] = *reinterpret_cast<const u32x4*>(c.v_q + ((quad + 2 * e) * W + w) * 4);
      t.sb[2 * v + e] = *reinterpret_cast<const u32x4*>(c.v_sb + ((quad + 2 * e) * G + (w >> gw_shift)) * 4);
    }
  }
}

// Exponents of constants as `Packed` has them: of a lane's key (a lane each, both halves the
// same), of the eight keys that a lane's values are of.
template <typename TT, int NK>
__device__ __forceinline__ int key_exponent(const uint32_t* sb) {
  float f = 0.f;
#pragma unroll
  for (int i = 0; i < NK; ++i) f = fmaxf(f, finite_size<TT>(sb[i]));
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(f), __float_as_uint(f), false, false);
  return size_exponent(fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])));
}
template <typename TT, int D>
__device__ __forceinline__ int value_exponent(const u32x4* sb, int e) {
  float f = 0.f;
#pragma unroll
  for (int v = 0; v < Packed<D>::VS; ++v) f = fmaxf(f, finite_size<TT>(sb[2 * v + (e >> 2)][e & 3]));
  int x = size_exponent(f);  // the largest over the words: 8 or 16 neighbouring lanes
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0xB1, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x4E, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x141, 0xf, 0xf, false));
  if (D > 64) x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x140, 0xf, 0xf, false));
  return x;
}

// 32 keys (key0 .. in the tile) as operands.  FIT: the exponent is moved to what they
// need; returns whether some are too small for it.
template <typename TT, int D, bool FIT>
__device__ __forceinline__ bool store_keys(const Packed<D>& t, u32x4* lds, int key0, int lane, KvRange& range, bool live) {
  constexpr int W = D / 8, NK = Packed<D>::NK;
  bool apart = false;
  uint32_t sb[NK];
#pragma unroll
  for (int i = 0; i < NK; ++i) sb[i] = live ? t.sb[0][i] : 0u;
  if (FIT) {
    uint32_t m = 0u, l = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      m = sizes(m, sb[i]);
      l = smallest(l, sb[i]);
    }
    if (!live) l = 0xffffffffu;
    if (__builtin_expect(!__all(range.holds(m, l)), 0)) {
      if (__all(all_finite<TT>(m))) range.template fit<TT>(max_of_wave(size_exponent(finite_size<TT>(m))));
      if (!__all(range.holds(m, l))) {
        const int x = key_exponent<TT, NK>(sb);
        range.template fit<TT>(max_of_wave(x));
        apart = __any(!range.takes(x));
      }
    }
  }
  const int key = key0 + (lane & 31), half = lane >> 5;
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const float s = scaled(TT::lo(sb[i]), 24 - range.e), b = scaled(TT::hi(sb[i]), -range.e);
    const uint32_t s0 = F16::pack2(s, s), b0 = F16::pack2(b, b), s1 = sixteenth(s0);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      lds[key_unit<W>(key, half * (W / 2) + 4 * i + e)] = key_slice(t.q[i][e], s0, s1, b0);
  }
  return apart;
}

// 32 keys for T = f16: their words as integers (a nibble's f16 subnormals, q * 2^-24 and
// q * 2^-20 in turn), scales and biases beside them.
template <int D>
__device__ __forceinline__ void store_whole_keys(const Packed<D>& t, u32x4* lds, float* scales, uint32_t* biases,
                                                 int key0, int lane, int gw_shift) {
  constexpr int W = D / 8, NK = Packed<D>::NK;
  const int key = key0 + (lane & 31), half = lane >> 5;
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const uint32_t sb = t.sb[0][i];
    const int g = (half * (W / 2) + 4 * i) >> gw_shift;
    scales[g * kKeys + key] = scaled(F16::lo(sb), 24 - kSumShift);
    biases[key * 8 + g] = __builtin_amdgcn_perm(sb, sb, 0x03020302u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t w = t.q[i][e], w8 = w >> 8;
      lds[key_unit<W>(key, half * (W / 2) + 4 * i + e)] =
          u32x4{w & 0x000f000fu, w & 0x00f000f0u, w8 & 0x000f000fu, w8 & 0x00f000f0u};
    }
  }
}

// 32 keys' values (half k steps ts0 ..) as operands, likewise; `poison`: a constant was
// not finite (those count as zeros).
template <typename TT, int D, bool FIT>
__device__ __forceinline__ bool store_values(const Packed<D>& t, u32x4* lds, int ts0, int lane, KvRange& range,
                                             uint32_t live, bool& poison) {
  constexpr int W = D / 8, L = W < 16 ? 8 : 16, VS = Packed<D>::VS;
  bool apart = false;
  u32x4 sb[2 * VS];
#pragma unroll
  for (int i = 0; i < 2 * VS; ++i) sb[i] = t.sb[i];
  uint32_t out0 = 0u, out1 = 0u;  // of the lane's own two keys: not live
  if (live != 0xffu) {
#pragma unroll
    for (int i = 0; i < 2 * VS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) sb[i][e] = live >> (4 * (i & 1) + e) & 1 ? sb[i][e] : 0u;
    out0 = live >> (lane & 3) & 1 ? 0u : 0xffffffffu;
    out1 = live >> (4 + (lane & 3)) & 1 ? 0u : 0xffffffffu;
  }
  // The lanes of a group's words have the same constants: four neighbours look at a
  // quarter of them each.
  uint32_t m = 0u, l = 0xffffffffu;
  if (FIT) {
#pragma unroll
    for (int i = 0; i < 2 * VS; ++i) {
      const uint32_t a = lane & 1 ? sb[i][1] : sb[i][0], b = lane & 1 ? sb[i][3] : sb[i][2], mine = lane & 2 ? b : a;
      m = sizes(m, mine);
      l = smallest(l, mine | (i & 1 ? out1 : out0));
    }
  }
  bool fits = FIT && __all(range.holds(m, l));
  if (FIT && __builtin_expect(!fits, 0) && __all(all_finite<TT>(m))) {
    range.template fit<TT>(max_of_wave(size_exponent(finite_size<TT>(m))));
    fits = __all(range.holds(m, l));
  }
  if (!FIT || __builtin_expect(!fits, 0)) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 2 * VS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool ok = finite(TT::lo(sb[i][e])) && finite(TT::hi(sb[i][e]));
        bad |= !ok;
        sb[i][e] = ok ? sb[i][e] : 0u;
      }
    poison = __any(bad);
    if (FIT) {
      int x[8], top = kKvNone;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = value_exponent<TT, D>(sb, e);
        top = max(top, x[e]);
      }
      range.template fit<TT>(max_of_wave(top));
      bool out = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) out |= !range.takes(x[e]);
      apart = __any(out);
    }
  }
  const int ts = ts0 + (lane / L & 3);
#pragma unroll
  for (int v = 0; v < VS; ++v) {
    uint32_t s0[4], s1[4], b0[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const uint32_t c0 = sb[2 * v + (x >> 1)][2 * (x & 1)], c1 = sb[2 * v + (x >> 1)][2 * (x & 1) + 1];
      s0[x] = F16::pack2(scaled(TT::lo(c0), 24 - range.e), scaled(TT::lo(c1), 24 - range.e));
      b0[x] = F16::pack2(scaled(TT::hi(c0), -range.e), scaled(TT::hi(c1), -range.e));
      s1[x] = sixteenth(s0[x]);
    }
    const int w = 16 * v + lane % L;
    // At head_dim 64 the wave's halves take half of a word's dimensions each.
    constexpr int NY = D == 64 ? 2 : 4;
    const int y0 = D == 64 ? 2 * (lane >> 5) : 0;
#pragma unroll
    for (int y = 0; y < NY; ++y) {
      const uint32_t sel = 0x0c040c00u + (uint32_t)(y + y0) * 0x00010001u;
      u32x4 lo, hi;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const u32x4& q4 = t.q[2 * v + (x >> 1)];
        const uint32_t b2 = __builtin_amdgcn_perm(q4[2 * (x & 1) + 1], q4[2 * (x & 1)], sel);
        lo[x] = pk_fma(b2 & 0x000f000fu, s0[x], b0[x]);
        hi[x] = pk_fma(b2 & 0x00f000f0u, s1[x], b0[x]);
      }
      lds[value_unit(8 * w + 2 * (y + y0), ts)] = lo;
      lds[value_unit(8 * w + 2 * (y + y0) + 1, ts)] = hi;
    }
  }
  return apart;
}

// What a workgroup does: rows tile `qt` of a sequence, a head, a part of the keys.
struct Item {
  int s, qt, head, part, parts;
  KvSeq q;
};
// Workgroup b's item among the sequences that this kernel takes, if any: every
// wave goes over them, 64 at a time, first for all their tiles (rows by keys)
// and from that the size of a part.
__device__ __forceinline__ bool find_item(const TileArgs& p, int b, int group, int bs_shift, int rows_per, Item& it) {
  const int n_seqs = (int)p.a.n_seqs, heads = (int)p.c.n_kv_heads, lane = threadIdx.x & 63;
  KvSeq q{};
  int row_tiles = 0, key_tiles = 0;
  auto work = [&](int s, bool report) {
    row_tiles = key_tiles = 0;
    if (s >= n_seqs) return;
    q = kv_seq(p.a, s, bs_shift, report, p.bad);
    const int rows = q.n_q * group;
    if (rows <= p.few_rows) return;
    row_tiles = (rows + rows_per - 1) / rows_per;
    // Of the last rows; a window leaves about its own length beside the rows'.
    const int reach = p.a.window ? (int)min((uint64_t)q.n, (uint64_t)p.a.window + rows_per / group) : q.n;
    key_tiles = (reach + kKeys - 1) / kKeys;
  };
  long total = 0, items = 0;
  if (p.target || p.report) {
    for (int base = 0; base < n_seqs; base += 64) {
      work(base + lane, p.report && b == 0 && threadIdx.x < 64);
      long sum = (long)row_tiles * key_tiles;
      items += __builtin_amdgcn_readlane(wave_scan(min(row_tiles * heads, 1 << 24)), 63);
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
      total += sum;
    }
  }
  // (Each row tile rounds its parts up, by half a part on average.  At least 1: where
  // the scratch leaves room for a few parts only, these come to nothing.)
  const long target = max(max(p.target - items / 2, (long)p.target / 4), 1l);
  // Query starts that are not ascending (reported) can name more row tiles than the
  // grid was made for: no splits then, or parts without a workgroup would leave their
  // arrival counters behind.
  const bool split = p.target && items <= (long)gridDim.x - p.target;
  const long per = split ? max((total * heads + target - 1) / target, (long)kMinTiles) : 1l << 40;
  int before = 0;
  for (int base = 0; base < n_seqs; base += 64) {
    work(base + lane, false);
    const int parts = max((int)min((key_tiles + per - 1) / per, (long)64), 1), items = row_tiles * parts * heads;
    const int sum = wave_scan(items), at = before + sum - items;
    before += __builtin_amdgcn_readlane(sum, 63);
    if (b < before) {
      const int l = __builtin_ctzll(__ballot(b >= at && b < at + items));
      const int k = b - __builtin_amdgcn_readlane(at, l);
      it.s = base + l;
      it.parts = __builtin_amdgcn_readlane(parts, l);
      it.head = k % heads;
      it.part = k / heads % it.parts;
      it.qt = k / heads / it.parts;
      it.q.rows0 = __builtin_amdgcn_readlane(q.rows0, l);
      it.q.n_q = __builtin_amdgcn_readlane(q.n_q, l);
      it.q.n = __builtin_amdgcn_readlane(q.n, l);
      it.q.lo = __builtin_amdgcn_readlane(q.lo, l);
      it.q.pos = it.q.n - it.q.n_q;
      return true;
    }
  }
  return false;
}

// GS: the group size at T = f16, 0 (any) at bf16.
template <typename TT, int D, int kWaves, int GS, Scores SCORES>
__global__ __launch_bounds__(kWaves * 64, D == 256 ? 1 : D == 64 && !GS ? 3 : 2) void kv_tile_kernel(TileArgs p) {
  constexpr int W = D / 8, NS = D / 16, ND = D / 32, kUnits = kKeys * W;
  constexpr int kTeams = kWaves / 4, kBufs = 2 * kTeams;
  extern __shared__ u32x4 units[];  // [kBufs][keys, values][kUnits]
  __shared__ int meta[kBufs][4];         // of the halves' keys, then their values
  __shared__ unsigned int arrived;
  __shared__ int exponents[2][kKeys];    // of tokens too far apart: keys, values
  // At T = f16 one rounding of keys and weights would show (off by 0.0005 to 0.0007 from 64
  // bits, 0.0003 now): keys enter as integers, their scales by an fma after the product
  // over a group, their biases by a product with the queries' sums, a weight with what its
  // rounding took.  A step of 13 requests 51 us instead of 46, 4096 queries over 8192 keys
  // in groups of 64 668 instead of 446, in groups of 32 726.
  constexpr bool kExact = !Sig16<TT>::bf16;
  constexpr int kGroups = kExact ? D / (GS ? GS : 1) : 1;
  __shared__ __align__(16) float key_scales[kExact ? kBufs : 1][kGroups][kExact ? kKeys : 4];
  __shared__ __align__(16) uint32_t key_biases[kExact ? kBufs : 1][kExact ? kKeys : 1][8];  // of group g, twice
  constexpr int kRows = 32 * kWaves;
  const cpq_kv_cache& c = p.c;
  const cpq_kv_attention_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, h = lane >> 5;
  const int bs_shift = 31 - __builtin_clz(c.block_size), gw_shift = 28 - __builtin_clz(GS ? GS : c.group_size);
  const int group = (int)a.n_heads / (int)c.n_kv_heads;
  Item it{};
  if (!find_item(p, blockIdx.x, group, bs_shift, kRows, it)) return;
  const KvSeq& q = it.q;
  const int head = it.head, part = it.part;
  const int rows = q.n_q * group;
  const int qt = (rows + kRows - 1) / kRows - 1 - it.qt;  // the rows that see most first
  const int row0 = qt * kRows, row1 = min(row0 + kRows, rows);

  // Keys that any of the rows sees, in tiles; this part's.
  const int pos0 = q.pos + row0 / group, pos1 = q.pos + (row1 - 1) / group;
  constexpr bool kScored = SCORES != Scores::kPlain;
  const int prefix = kScored ? kv_prefix(p.score, it.s, q.n) : 0;
  const int end = max(a.causal ? min(max(pos1 + 1, prefix), q.n) : q.n, 0);
  const int from = a.window ? (int)max((int64_t)pos0 + 1 - (int64_t)a.window, (int64_t)0) : 0;
  const int first = from / kKeys, tiles = max((end + kKeys - 1) / kKeys - first, 0);
  const int parts = max(min(it.parts, tiles / kMinTiles), 1), per = (tiles + parts - 1) / parts;
  if (part >= parts) return;
  const int begin = first + part * per, stop = min(first + tiles, begin + per);

  // This lane's query row.
  const int r = min(row0 + wave * 32 + col, rows - 1), qi = r / group, hh = head * group + r - qi * group;
  const int qpos = q.pos + qi;
  u32x4 qs[NS];
  int qe;
  {
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (size_t)(q.rows0 + qi) * a.q_token_stride +
                          (size_t)hh * a.q_head_stride + h * 8;
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      qs[i] = *reinterpret_cast<const u32x4*>(src + 16 * i);
      m = largest<TT>(qs[i], m);
    }
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    qe = query_exponent(fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])));
#pragma unroll
    for (int i = 0; i < NS; ++i) qs[i] = query_slice<TT>(qs[i], qe);
  }
  u32x4 qsum{0u, 0u, 0u, 0u};  // of groups 4 h .. 4 h + 3: high and low part
  if constexpr (kExact) {
    // (Groups that there are not; the waves that stage write the others after this.)
    for (int e = tid; e < kBufs * kKeys * 8; e += kWaves * 64) (&key_biases[0][0][0])[e] = 0u;
    __syncthreads();
    float all[kGroups];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      all[g] = 0.f;
#pragma unroll
      for (int i = g * NS / kGroups; i < (g + 1) * NS / kGroups; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) all[g] = F16::dot2(qs[i][e], 0x3c003c00u, all[g]);
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(all[g]), __float_as_uint(all[g]), false, false);
      all[g] = scaled(__uint_as_float(sw[0]) + __uint_as_float(sw[1]), -kSumShift);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float v = h ? (4 + g < kGroups ? all[(4 + g) % kGroups] : 0.f) : g < kGroups ? all[g % kGroups] : 0.f;
      const float high = F16::lo(F16::pack2(v, 0.f));
      qsum[g] = F16::pack2(high, v - high);
    }
    // The words' second and fourth pairs are in units 16 times as large.
#pragma unroll
    for (int i = 0; i < NS; ++i) qs[i] = u32x4{qs[i][0], sixteenth(qs[i][1]), qs[i][2], sixteenth(qs[i][3])};
  }
  const int see_to = a.causal ? min(max(qpos + 1, prefix), q.n) : q.n;  // keys [see_from, see_to) of this row
  const int see_from = a.window ? (int)max((int64_t)qpos + 1 - (int64_t)a.window, (int64_t)0) : 0;
  // Of the wave's rows: any sees [any_from, any_to), all see [all_from, all_to).
  const int wr0 = min(row0 + wave * 32, rows - 1), wr1 = min(row0 + wave * 32 + 31, rows - 1);
  const int wpos0 = q.pos + wr0 / group, wpos1 = q.pos + wr1 / group;
  const bool idle = row0 + wave * 32 >= rows;  // no rows of its own: it only stages
  const int any_to = idle ? 0 : a.causal ? min(max(wpos1 + 1, prefix), q.n) : q.n;
  const int all_to = a.causal ? min(max(wpos0 + 1, prefix), q.n) : q.n;
  const int any_from = a.window ? (int)max((int64_t)wpos0 + 1 - (int64_t)a.window, (int64_t)0) : 0;
  const int all_from = a.window ? (int)max((int64_t)wpos1 + 1 - (int64_t)a.window, (int64_t)0) : 0;

  KvRowScore<SCORES> score;
  if constexpr (kScored) score.head(p.score, hh, see_from, see_to);

  f32x16 o[ND];
#pragma unroll
  for (int j = 0; j < ND; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[j][e] = 0.f;
  float ref = -FLT_MAX, sum = 0.f;
  uint32_t nan_groups = 0;             // groups of dimensions that are NaN in this row
  int unit = 0;                        // o is in units of 2^unit
  float cl0 = 0.f, cl1 = 0.f;          // of the halves: log2(e) * scale * 2^(exponents of q and the keys)
  int ve = 0, d0 = 0, d1 = 0;          // the values' exponent, and the halves' less that
  int alike = 0;                       // the rows' units are ve

  // Staging: of each four waves two keys and two values of the tile's halves.
  const uint32_t* __restrict__ blocks = a.block_table + (size_t)it.s * a.max_blocks;
  const int team = wave >> 2;
  const bool is_values = ((wave >> 1) ^ team) & 1;  // on each SIMD one wave of either kind
  const int half = wave & 1;
  KvRange range;
  Packed<D> packed;
  int loaded_ok = 3;
  // The blocks of this half of 32 tiles, a lane each 16 keys (scalar loads in
  // flight would make every LDS wait a wait for all).
  uint32_t ids = 0;
  // The first key of the t-th tile of `begin` to `stop`.  With biases, which mostly fall
  // with distance, the last keys come first: forward the weights of most heads grow from tile
  // to tile, and with each the reference is raised and weights are made twice (4096 queries
  // over 8192 keys 667 us; so 485.  Slopes below 0 still have it).
  auto key_of = [&](int t) { return (biased(SCORES) ? begin + stop - 1 - t : t) * kKeys; };
  auto load = [&](int t) {
    const int lane = (int)opaque((uint32_t)(tid & 63));
    const int key = key_of(t) + half * 32;
    const int l = 2 * ((t - begin) / kTeams & 31);
    if (l == 0) {
      const int ahead = key_of(t + kTeams * (lane >> 1)) + half * 32 + 16 * (lane & 1);
      ids = blocks[min(biased(SCORES) ? max(ahead, 0) : ahead, q.n - 1) >> bs_shift];
    }
    const KvPlaces pl = kv_places(c, (uint32_t)__builtin_amdgcn_readlane((int)ids, l),
                                  (uint32_t)__builtin_amdgcn_readlane((int)ids, l + 1), min(key, (q.n - 1) & ~15), q.n,
                                  head, bs_shift);
    loaded_ok = (pl.a.ok ? 1 : 0) | (pl.b.ok ? 2 : 0);
    if (is_values) load_values<D>(packed, c, pl.a.row, pl.b.row, lane, gw_shift);
    else load_keys<D>(packed, c, pl.a.row, pl.b.row, lane, gw_shift);
  };
  // The words of a tile that `load` has taken already.
  auto load_again = [&](int t) {
    asm volatile("" : "+s"(t));  // (addresses made here, not ahead of the branch)
    const int lane = (int)opaque((uint32_t)(tid & 63));
    const int key = key_of(t) + half * 32;
    const KvPlaces pl = kv_places(c, blocks[min(key, q.n - 1) >> bs_shift], blocks[min(key + 16, q.n - 1) >> bs_shift],
                                  min(key, (q.n - 1) & ~15), q.n, head, bs_shift);
    if (is_values) load_values<D>(packed, c, pl.a.row, pl.b.row, lane, gw_shift);
    else load_keys<D>(packed, c, pl.a.row, pl.b.row, lane, gw_shift);
  };
  // The half's keys of which bit k of `seen` (from key 32 * half on) is set.
  auto live_values = [&](uint32_t seen, int lane) {
    const int ts = lane / (W < 16 ? 8 : 16) & 3;
    seen >>= 16 * (ts >> 1) + 4 * (ts & 1);
    return (seen & 15u) | (seen >> 4 & 0xf0u);
  };
  auto store = [&](int t, int buf) {
    // (The lane hidden from the optimiser: addresses made anew each time take a few
    // instructions, kept through the loop they spill registers.)
    const int lane = (int)opaque((uint32_t)(tid & 63));
    u32x4* keys = units + buf * 2 * kUnits;
    const int key = key_of(t) + half * 32;
    const bool all = key >= from && key + 32 <= end && loaded_ok == 3;
    // (Of the keys [from, end) each is seen by one of the rows.)
    if (!all && !is_values && lane == 0 &&
        ((!(loaded_ok & 1) && key < end && key + 16 > from) || (!(loaded_ok & 2) && key + 16 < end && key + 32 > from)))
      atomicAdd(p.bad, 1u);
    const uint32_t seen = all ? 0xffffffffu
                              : range_bits(from - key, end - key) &
                                    ((loaded_ok & 1 ? 0xffffu : 0u) | (loaded_ok & 2 ? 0xffff0000u : 0u));
    bool poison = false, apart;
    if (is_values)
      apart = store_values<TT, D, true>(packed, keys + kUnits, 4 * half, lane, range,
                                        all ? 0xffu : live_values(seen, lane), poison);
    else if constexpr (kExact)
      apart = false, store_whole_keys<D>(packed, keys, &key_scales[buf][0][0], &key_biases[buf][0][0], 32 * half, lane, gw_shift);
    else
      apart = store_keys<TT, D, true>(packed, keys, 32 * half, lane, range, all || (seen >> (lane & 31) & 1));
    if (lane == 0)
      meta[buf][2 * is_values + half] = (range.high ? range.e + kExpBias : 0) + (loaded_ok << kOkShift) +
                                        (poison ? kPoison : 0) + (apart ? kApart : 0);
  };

  // Byte offsets of the lane's operands in LDS; the half of LDS in turn is the
  // other value of one bit.
  constexpr uint32_t kHalf = 2 * kUnits * 16;
  const unsigned char* lds = reinterpret_cast<const unsigned char*>(units);
  uint32_t at_key[NS], at_value[kKeys / 16];
#pragma unroll
  for (int i = 0; i < NS; ++i) at_key[i] = (uint32_t)key_unit<W>(col, 2 * i + h) * 16;
#pragma unroll
  for (int k = 0; k < kKeys / 16; ++k) at_value[k] = (uint32_t)(kUnits + value_unit(col, 2 * k + h)) * 16;
  auto key_operand = [&](int u, int i) {
    return *reinterpret_cast<const u32x4*>(lds + at_key[i] + u * (32 * W * 16));
  };
  auto value_operand = [&](int j, int k) {
    return *reinterpret_cast<const u32x4*>(lds + at_value[k] + j * (32 * 8 * 16));
  };

  if (begin + team < stop) load(begin + team);
  if (begin + team < stop) {
    store(begin + team, team);
    if (begin + team + kTeams < stop) load(begin + team + kTeams);
  }
  __syncthreads();
  int known = -1;     // the published words that what follows is of
  uint64_t keep = 0;  // keys that are there
  int poison = 0, apart = 0;  // (uniform, in scalar registers)
  // The units of the rows that see some of the tile's keys `keep`.
  auto rescale = [&](int key0) {
    asm volatile("" : "+s"(key0));  // (what follows is made here, not kept)
    const int lo = see_from - key0, hi = see_to - key0;
    const uint64_t seen = (uint64_t)range_bits(lo, hi) | (uint64_t)range_bits(lo - 32, hi - 32) << 32;
    if (ref == -FLT_MAX) unit = ve;  // nothing yet
    int next = seen & keep ? ve : unit;
    if (__any(next != unit)) {
      if (__any(next < unit)) {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < ND; ++j)
#pragma unroll
          for (int x = 0; x < 16; ++x) m = fmaxf(m, fabsf(o[j][x]));
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
        m = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
        next = next < unit ? lower_unit(unit, next, m) : next;
      }
#pragma unroll
      for (int j = 0; j < ND; ++j)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[j][x] = scaled(o[j][x], unit - next);
      unit = next;
    }
    alike = __builtin_amdgcn_readfirstlane((int)!__any(unit != ve));
  };
  for (int t = begin; t < stop; ++t) {
    const int buf = (t - begin) & (kBufs - 1), key0 = key_of(t);
    const int news = meta[buf][lane & 3];
    if (__builtin_expect(__any(news != known), 0)) {
      auto word = [&](int i) { return __builtin_amdgcn_readlane(news, i); };
      auto exponent = [&](int i) { return word(i) & 0xffff ? (word(i) & 0xffff) - kExpBias : kKvNone; };
      const int k0 = exponent(0), k1 = exponent(1), v0 = exponent(2), v1 = exponent(3);
      // The keys, and the values, of all waves share the largest where it is near, so
      // that the words change seldom.
      const int own = is_values ? max(v0, v1) : max(k0, k1);
      if (range.high && own > range.e && own <= range.e + kKvKeep) range.set<TT>(own);
      const int any = word(0) | word(1) | word(2) | word(3);
      poison = any & kPoison;
      apart = any & kApart;
      if (min(v0, v1) != kKvNone && abs(v0 - v1) > kMostApart) apart = kApart;
      const uint32_t there0 = word(0) >> kOkShift & 3, there1 = word(1) >> kOkShift & 3;
      keep = (uint64_t)((there0 & 1) * 0xffffu | (there0 >> 1) * 0xffff0000u) |
             (uint64_t)((there1 & 1) * 0xffffu | (there1 >> 1) * 0xffff0000u) << 32;
      if (!apart) {
        cl0 = fmaxf(scaled(a.scale, (kExact ? kSumShift : k0 == kKvNone ? 0 : k0) + qe) * kLog2e, FLT_MIN);
        cl1 = fmaxf(scaled(a.scale, (kExact ? kSumShift : k1 == kKvNone ? 0 : k1) + qe) * kLog2e, FLT_MIN);
        if (max(v0, v1) != kKvNone) ve = max(v0, v1);
        d0 = v0 == kKvNone ? 0 : v0 - ve;
        d1 = v1 == kKvNone ? 0 : v1 - ve;
        rescale(key0);
      }
      known = alike ? news : -1;  // (else again at the next tile)
    }
    if (t + kTeams < stop && (t - begin) % kTeams == team) {
      store(t + kTeams, (t + kTeams - begin) & (kBufs - 1));
      if (t + 2 * kTeams < stop) load(t + 2 * kTeams);
    }
    uint64_t left = 0;  // keys that some row sees, of a tile whose tokens are taken in passes
    const bool mine = (t - begin) % kTeams == team;
    if (__builtin_expect(apart != 0, 0)) {
      __syncthreads();
      if (mine) {
        load_again(t);
        const int lane = (int)opaque((uint32_t)(tid & 63));
        if (is_values) {
          const int ts = lane / (W < 16 ? 8 : 16) & 3;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int x = value_exponent<TT, D>(packed.sb, e);
            if (lane % (W < 16 ? 8 : 16) == 0)
              exponents[1][32 * half + 16 * (ts >> 1) + 4 * (ts & 1) + (e & 3) + 8 * (e >> 2)] = x;
          }
        } else {
          uint32_t sb[Packed<D>::NK];
#pragma unroll
          for (int i = 0; i < Packed<D>::NK; ++i) sb[i] = packed.sb[0][i];
          const int x = key_exponent<TT, Packed<D>::NK>(sb);
          if (lane < 32) exponents[0][32 * half + lane] = x;
        }
      }
      __syncthreads();
      left = keep & __ballot(key0 + lane >= from && key0 + lane < end);
    }
    do {
      if (__builtin_expect(apart != 0, 0)) {
        const int kx = kExact ? kKvNone : exponents[0][lane], vx = exponents[1][lane];
        KvRange kr, vr;
        bool in = left >> lane & 1;
        vr.fit<TT>(max_of_wave(in ? vx : kKvNone));
        in = in && vr.takes(vx);
        kr.fit<TT>(max_of_wave(in ? kx : kKvNone));
        keep = __ballot(in && kr.takes(kx));
        left &= ~keep;
        __syncthreads();  // (the reads of the pass before)
        if (mine) {
          load_again(t);
          const int lane = (int)opaque((uint32_t)(tid & 63));
          u32x4* keys = units + buf * 2 * kUnits;
          const uint32_t seen = (uint32_t)(keep >> (32 * half));
          bool bad;
          if (is_values)
            store_values<TT, D, false>(packed, keys + kUnits, 4 * half, lane, vr, live_values(seen, lane), bad);
          else if constexpr (!kExact)
            store_keys<TT, D, false>(packed, keys, 32 * half, lane, kr, seen >> (lane & 31) & 1);
        }
        __syncthreads();
        cl0 = cl1 = fmaxf(scaled(a.scale, (kExact ? kSumShift : kr.e) + qe) * kLog2e, FLT_MIN);
        if (vr.high) ve = vr.e;
        d0 = d1 = 0;
        rescale(key0);
      }
      if (key0 >= any_to || key0 + kKeys <= any_from) continue;
      const bool whole = key0 >= all_from && key0 + kKeys <= all_to && keep == ~0ull;
      // Operands are read a step ahead of the matrix instructions that take them, and
      // the weights of one half of the keys are made between those of the other.
      f32x16 sc[2];
      constexpr int kAhead = 4;
      u32x4 op[kAhead], pw[kKeys / 16], lost[kExact ? kKeys / 16 : 1], vop[2][kExact ? 1 : ND];
      float add[2] = {0.f, 0.f};
      // Bits of half u's keys that the row sees, from the lane's first key.
      auto seen_of = [&](int u) {
        // (Kept inside the branch: hoisted, the comparisons fill the scalar registers and
        // every tile selects.)
        int at = key0 + 32 * u;
        asm volatile("" : "+s"(at));
        return (range_bits(see_from - at, see_to - at) & (uint32_t)(keep >> (32 * u))) >> (4 * h);
      };
      uint32_t seen[2];  // where not all are (scored)
      // What the scores become (apart from `sc`, whose 16 registers stay one operand).  Caps
      // bound how far they lie from the reference, which is subtracted on the way then (568
      // us instead of 578); with biases it would take their last bits where it jumps.
      constexpr bool kFolded = SCORES == Scores::kCapped;
      float rel[2];  // what `z` holds besides
      float z[kScored ? 2 : 1][16];
      auto logit = [&](int u, int x) { return kScored ? z[u][x] : sc[u][x]; };
      // Before a half's weights.
      auto mask = [&](int u) {
        if constexpr (kScored) {
          if constexpr (kFolded) rel[u] = ref == -FLT_MAX ? 0.f : (float)(u ? d1 : d0) - ref;
          // (What has no side effects is otherwise made where it is used, after the fences: the
          // operands of all sixteen scores stay in registers, 50 of them.)
          if constexpr (kExact) asm volatile("" : "+v"(sc[u]));
          score.at(p.score, key0 + 32 * u + 4 * h, u ? cl1 : cl0, kFolded ? rel[u] : 0.f);
        }
        if (__builtin_expect(whole, 1)) return;
        const uint32_t bits = seen_of(u);
        if constexpr (kScored) {
          seen[u] = bits;
          return;
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) sc[u][x] = bits >> (8 * (x >> 2) + (x & 3)) & 1 ? sc[u][x] : -INFINITY;
      };
      // Scored: two of a half's scores become what they are to be, then are masked.  In order:
      // `base` goes on to the next two keys.
      auto become = [&](int u, int i) {
        if constexpr (kScored) {
          const float next = score.step(score.base, 1.f);
          z[u][2 * i] = score.of(p.score, sc[u][2 * i], score.base);
          z[u][2 * i + 1] = score.of(p.score, sc[u][2 * i + 1], next);
          score.base = score.step(score.base, i & 1 ? 6.f : 2.f);
          asm volatile("" : "+v"(z[u][2 * i]), "+v"(z[u][2 * i + 1]), "+v"(score.base));
          if (__builtin_expect(!whole, 0)) {
            const int x = 8 * (i >> 1) + 2 * (i & 1);
            z[u][2 * i] = seen[u] >> x & 1 ? z[u][2 * i] : -INFINITY;
            z[u][2 * i + 1] = seen[u] >> (x + 1) & 1 ? z[u][2 * i + 1] : -INFINITY;
          }
        }
      };
      auto weights = [&](int u, float rel, int i) {  // two of a half's
        const float cl = u ? cl1 : cl0;
        const float w0 = __builtin_amdgcn_exp2f(kFolded   ? z[u][2 * i]
                                                : kScored ? z[u][2 * i] + rel
                                                          : fmaf(sc[u][2 * i], cl, rel));
        const float w1 = __builtin_amdgcn_exp2f(kFolded   ? z[u][2 * i + 1]
                                                : kScored ? z[u][2 * i + 1] + rel
                                                          : fmaf(sc[u][2 * i + 1], cl, rel));
        const uint32_t w = F16::pack2(w0, w1);
        pw[2 * u + (i >> 2)][i & 3] = w;
        // The sum is of the rounded weights, two at a time.
        add[u] = F16::dot2(w, 0x3c003c00u, add[u]);
        if constexpr (kExact) {
          lost[2 * u + (i >> 2)][i & 3] = F16::pack2(w0 - F16::lo(w), w1 - F16::hi(w));
          add[u] = F16::dot2(lost[2 * u + (i >> 2)][i & 3], 0x3c003c00u, add[u]);
        }
      };
      // Where a weight of half u left f16's range: a new reference, the weights again.
      auto settle = [&](int u) {
        const uint64_t redo = __ballot(!(add[u] < kMost) || (kFolded && ref == -FLT_MAX));
        if (__builtin_expect(redo != 0, 0)) {
          const float cl = kScored ? 1.f : u ? cl1 : cl0;
          float mine = logit(u, 0);
#pragma unroll
          for (int x = 1; x < 16; ++x) mine = fmaxf(mine, logit(u, x));
          mine *= cl;
          if constexpr (kFolded) mine -= rel[u];
          const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mine), __float_as_uint(mine), false, false);
          const float was = ref;
          // (Rows that need none keep theirs, and their weights: a row's result is its own.)
          if ((redo | redo >> 32) >> col & 1)
            ref = fmaxf(ref, fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) - kRaise);
          const float keep = __builtin_amdgcn_exp2f(was - ref);
          sum *= keep;
#pragma unroll
          for (int j = 0; j < ND; ++j) o[j] *= keep;
          add[u] = 0.f;
          const float to = (float)(u ? d1 : d0) - ref;
          if constexpr (kFolded) {
            const float by = to - rel[u];  // (0 where the reference stays)
#pragma unroll
            for (int x = 0; x < 16; ++x) z[u][x] += by;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) weights(u, to, i);
        }
        sum += scaled(add[u], u ? -d1 : -d0);
        // (A row whose sums are beyond these values by all that fp32 holds leaves them out.)
        if (__builtin_expect(!alike, 0)) {
          uint32_t with = unit == ve ? 0xffffffffu : 0u;
          asm volatile("" : "+v"(with));  // (a branch, not selections in every tile)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            pw[2 * u][x] &= with;
            pw[2 * u + 1][x] &= with;
            if constexpr (kExact) {
              lost[2 * u][x] &= with;
              lost[2 * u + 1][x] &= with;
            }
          }
        }
      };
      if constexpr (kExact) {
        // One half of the keys after the other: what both would hold exceeds the registers.
        constexpr int kSteps = NS / kGroups;  // of a group
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const f32x16 none{};
          sc[u] = mma(*reinterpret_cast<const u32x4*>(&key_biases[buf][32 * u + col][4 * h]), qsum, none);
#pragma unroll
          for (int i = 0; i < kAhead; ++i) op[i] = key_operand(u, i);
          fence();
          f32x16 run;  // the integers' product over a group so far
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            const bool ends = i % kSteps == kSteps - 1;
            f32x4 by[4];
            if (ends) {
#pragma unroll
              for (int x = 0; x < 4; ++x)
                by[x] = *reinterpret_cast<const f32x4*>(&key_scales[buf][i / kSteps][32 * u + 8 * x + 4 * h]);
            }
            run = mma(op[i % kAhead], qs[i], i % kSteps ? run : none);
            if (i + kAhead < NS) op[i % kAhead] = key_operand(u, i + kAhead);
            fence();
            if (!ends) continue;
#pragma unroll
            for (int x = 0; x < 16; ++x) sc[u][x] = fmaf(run[x], by[x >> 2][x & 3], sc[u][x]);
            fence();
          }
          mask(u);
          const float rel = (float)(u ? d1 : d0) - ref;
#pragma unroll
          for (int i = 0; i < kAhead; ++i) op[i] = value_operand(i % ND, 2 * u + i / ND);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            become(u, i);
            weights(u, rel, i);
            if (kScored) fence();
          }
          settle(u);
          fence();
#pragma unroll
          for (int n = 0; n < 2 * ND; ++n) {
            const int k = 2 * u + n / ND, j = n % ND;
            o[j] = mma(op[n % kAhead], pw[k], o[j]);
            o[j] = mma(op[n % kAhead], lost[k], o[j]);
            if (n + kAhead < 2 * ND) op[n % kAhead] = value_operand((n + kAhead) % ND, 2 * u + (n + kAhead) / ND);
            fence();
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) op[i] = key_operand(i / NS, i % NS);
        fence();
#pragma unroll
        for (int x = 0; x < 16; ++x) sc[0][x] = sc[1][x] = 0.f;
        auto score = [&](int i) {
          sc[i / NS] = mma(op[i % kAhead], qs[i % NS], sc[i / NS]);
          if (i + kAhead < 2 * NS) op[i % kAhead] = key_operand((i + kAhead) / NS, (i + kAhead) % NS);
        };
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          score(i);
          fence();
        }
#pragma unroll
        for (int j = 0; j < ND; ++j) vop[0][j] = value_operand(j, 0);
        fence();
        mask(0);
        const float rel0 = (float)d0 - ref;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          score(NS + i);
#pragma unroll
          for (int x = i * 8 / NS; x < (i + 1) * 8 / NS; ++x) {
            become(0, x);
            weights(0, rel0, x);
          }
          fence();
        }
        settle(0);
        mask(1);
        const float rel1 = (float)d1 - ref;
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k) {
          if (k == 2) settle(1);
#pragma unroll
          for (int j = 0; j < ND; ++j) {
            if (k + 1 < kKeys / 16) vop[(k + 1) & 1][j] = value_operand(j, k + 1);
            o[j] = mma(vop[k & 1][j], pw[k], o[j]);
            if (k < 2) {
#pragma unroll
              for (int x = (k * ND + j) * 4 / ND; x < (k * ND + j + 1) * 4 / ND; ++x) {
                become(1, x);
                weights(1, rel1, x);
              }
            }
            fence();
          }
        }
      }
    } while (__builtin_expect(left != 0, 0));
    if (__builtin_expect(poison != 0, 0) && key0 < any_to && key0 + kKeys > any_from) {
#pragma clang loop unroll(disable)
      for (int k = 0; k < kKeys && key0 + k < q.n; k += 16)
        nan_groups |= poisoned_groups<TT>(c, kv_place(c, blocks[(key0 + k) >> bs_shift], key0 + k, head, bs_shift),
                                          key0 + k, W >> gw_shift, see_from, see_to);
    }
    if (__builtin_expect(apart != 0, 0)) {
      known = -1;
      if (mine && t + 2 * kTeams < stop) load_again(t + 2 * kTeams);
    }
    const uint32_t next = kTeams > 1 && (t - begin) % kTeams ? 3 * kHalf : kHalf;
#pragma unroll
    for (int i = 0; i < NS; ++i) at_key[i] ^= next;
#pragma unroll
    for (int k = 0; k < kKeys / 16; ++k) at_value[k] ^= next;
    if ((t + 1 - begin) % kTeams == 0) __syncthreads();
  }

  {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    sum = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  }
  if (__any(nan_groups != 0)) {
#pragma unroll
    for (int j = 0; j < ND; ++j)
#pragma unroll
      for (int x = 0; x < 16; ++x)
        if (nan_groups >> ((32 * j + 8 * (x >> 2)) / 8 >> gw_shift) & 1) o[j][x] = NAN;
  }
  const bool stored = row0 + wave * 32 + col < rows;
  uint16_t* out = static_cast<uint16_t*>(a.out) + (size_t)(q.rows0 + qi) * a.out_token_stride +
                  (size_t)hh * a.out_head_stride + 4 * h;
  if (parts > 1) {
    const size_t slab = (size_t)kWaves * (D / 8 + 1) * 64;  // f32x4 of a workgroup
    const size_t first = blockIdx.x - (size_t)part * c.n_kv_heads, stride = slab * c.n_kv_heads;
    const f32x4* all = reinterpret_cast<const f32x4*>(p.partial) + first * slab + (size_t)wave * (D / 8 + 1) * 64;
    const f32x4* mine = all + part * stride;
    auto put = [&](int at, f32x4 v) { park_store(mine, (at * 64 + lane) * 16, v); };
    auto get = [&](int k, int at) { return park_load(all + k * stride, (at * 64 + lane) * 16); };
    if (!idle) {
#pragma unroll
      for (int j = 0; j < ND; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          put(4 * j + x, f32x4{scaled(o[j][4 * x], unit), scaled(o[j][4 * x + 1], unit),
                               scaled(o[j][4 * x + 2], unit), scaled(o[j][4 * x + 3], unit)});
      put(D / 8, f32x4{ref, sum, 0.f, 0.f});
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) arrived = __hip_atomic_fetch_add(&p.counters[first], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (arrived != (unsigned int)(parts - 1)) return;
    float m = -FLT_MAX;
    const int joined = idle ? 0 : parts;
    for (int k = 0; k < joined; ++k) m = fmaxf(m, get(k, D / 8)[0]);
    sum = 0.f;
    unit = 0;
#pragma unroll
    for (int j = 0; j < ND; ++j)
#pragma unroll
      for (int x = 0; x < 16; ++x) o[j][x] = 0.f;
    constexpr int U = D == 256 ? 1 : 2;  // parts whose rows are under way together
    for (int k = 0; k < joined; k += U) {
      f32x4 v[U][D / 8], ml[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        ml[u] = get(min(k + u, joined - 1), D / 8);
#pragma unroll
        for (int x = 0; x < D / 8; ++x) v[u][x] = get(min(k + u, joined - 1), x);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (k + u >= joined) break;
        const float w = __builtin_amdgcn_exp2f(ml[u][0] - m);
        sum += ml[u][1] * w;
#pragma unroll
        for (int x = 0; x < D / 8; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[x >> 2][4 * (x & 3) + e] += v[u][x][e] * w;
      }
    }
    if (tid == 0) __hip_atomic_store(&p.counters[first], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (!stored) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int j = 0; j < ND; ++j)
#pragma unroll
    for (int x = 0; x < 4; ++x)
      *reinterpret_cast<u32x2*>(out + 32 * j + 8 * x) =
          u32x2{TT::pack2(scaled(o[j][4 * x] * inv, unit), scaled(o[j][4 * x + 1] * inv, unit)),
                TT::pack2(scaled(o[j][4 * x + 2] * inv, unit), scaled(o[j][4 * x + 3] * inv, unit))};
}

template <typename TT, int D, int kWaves, int GS, Scores SCORES>
hipError_t launch_tiles(hipStream_t s, const TileArgs& p, dim3 grid) {
  const size_t lds = (size_t)(kWaves / 2) * 2 * kKeys * (D / 8) * 16;
  auto kernel = kv_tile_kernel<TT, D, kWaves, GS, SCORES>;
  static const hipError_t raised = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  if (raised != hipSuccess) return raised;
  hipLaunchKernelGGL(kernel, grid, dim3(kWaves * 64), lds, s, p);
  return hipGetLastError();
}
template <int D, int kWaves, Scores SCORES>
hipError_t launch_tiles(hipStream_t s, const TileArgs& p, dim3 grid) {
  if (p.c.dtype == CPQ_DTYPE_BF16) return launch_tiles<BF16, D, kWaves, 0, SCORES>(s, p, grid);
  switch (p.c.group_size) {
    case 32: return launch_tiles<F16, D, kWaves, 32, SCORES>(s, p, grid);
    case 64: return launch_tiles<F16, D, kWaves, 64, SCORES>(s, p, grid);
    case 128:
      if constexpr (D >= 128) return launch_tiles<F16, D, kWaves, 128, SCORES>(s, p, grid);
    default: return hipErrorInvalidValue;
  }
}

// `decode`: launch_kv_decode of the same form.
template <Scores SCORES, typename Decode>
hipError_t run_attention(const ExecCtx& ex, const cpq_kv_cache& c, const cpq_kv_attention_args& given,
                         const KvScore& score, unsigned int* bad, Decode decode) {
  // Bounds past what a sequence can have mean no more than that, and would wrap.
  constexpr size_t kLongest = 1ull << 31;
  cpq_kv_attention_args a = given;
  a.max_q = std::min(a.max_q, a.n_tokens);
  a.max_kv = std::min(a.max_kv, kLongest);
  a.window = std::min(a.window, kLongest - 1);
  const size_t group = a.n_heads / c.n_kv_heads;
  if (a.max_q * group <= kKvDecodeRows)
    return decode(a, (int)std::max<size_t>(a.max_q * group, 1), true);
  TileArgs p{};
  p.score = score;
  p.c = c;
  p.a = a;
  p.bad = bad;
  // Beside long rows a batch may hold single tokens over long keys, whose rows
  // would leave most of a tile empty and their keys to one workgroup.
  p.few_rows = a.n_seqs > 1 && group <= 16 ? 16 : 0;
  if (p.few_rows) {
    const hipError_t e = decode(a, p.few_rows, false);
    if (e != hipSuccess) return e;
  }
  p.report = 1;
  // No more row tiles than this, whatever the sequences' shares.
  auto row_tiles = [&](size_t waves) { return (a.n_tokens * group / (32 * waves) + a.n_seqs) * c.n_kv_heads; };
  // At head_dim 128 eight waves share a workgroup's dequantization; where that
  // leaves compute units without one, workgroups of four, two to a CU (a step of 13
  // requests, 590 and 115 tokens of prompts: 46.6 us, 52.6 with eight; 1024 queries
  // of 48 heads on one key/value head: 75 and 87; 4096 of 32 on 8: 502 and 432).
  // (With scores the rows that there are count, not the most row tiles that sequences may
  // round up to: a step of 13 requests, 850, 690, 270 and 115 tokens of prompts, 78 us, 103
  // with eight.)
  const size_t full = SCORES == Scores::kPlain ? row_tiles(8) : a.n_tokens * a.n_heads / 256;
  const size_t waves = c.head_dim == 128 && full >= (size_t)ex.cu_count ? 8 : 4;
  const size_t wgs = row_tiles(waves);
  // As many parts as workgroups are resident where there are fewer tiles than that,
  // as far as the scratch goes.
  const size_t slab = waves * (c.head_dim / 8 + 1) * 64 * 16;
  const size_t room = ex.scratch_bytes > kWideCounterBytes ? (ex.scratch_bytes - kWideCounterBytes) / slab : 0;
  const bool three = c.head_dim == 64 && c.dtype == CPQ_DTYPE_BF16;
  const size_t target = (size_t)(three ? 3 : c.head_dim == 64 || (c.head_dim == 128 && waves == 4) ? 2 : 1) * ex.cu_count;
  p.target = wgs < room && wgs < target ? (int)std::min(target, room - wgs) : 0;
  p.counters = static_cast<unsigned int*>(ex.scratch);
  p.partial = reinterpret_cast<float*>(static_cast<char*>(ex.scratch) + kWideCounterBytes);
  const dim3 grid((uint32_t)(wgs + p.target));
  switch (c.head_dim) {
    case 64: return launch_tiles<64, 4, SCORES>(ex.stream, p, grid);
    case 128: return waves == 4 ? launch_tiles<128, 4, SCORES>(ex.stream, p, grid) : launch_tiles<128, 8, SCORES>(ex.stream, p, grid);
    case 256: return launch_tiles<256, 4, SCORES>(ex.stream, p, grid);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace
}  // namespace cpq
