// Attention over the 4-bit key/value cache for few query rows per sequence
// (kernels/kv_attention.hpp chooses; semantics: cpq_kv_attention and, scored,
// cpq_kv_attention_scored in cpq.h).
//
// The query rows of one key/value head (n_q queries times the heads of its
// group, at most 16 NC) share its keys and values, which are read once.  A
// workgroup of four waves takes one (sequence, head, part of the keys); each
// wave walks tiles of 32 keys with a softmax of its own:
//   S^T = K Q^T     v_mfma_f32_16x16x32_f16, A = 16 keys, B = 16 query rows:
//                   lane (key i, quarter h) takes a quarter of the key's words
//   O^T += V^T P^T  A = 16 words' j-th dimension over 32 keys, B = the weights.
//                   The result layout of S^T (lane: query n, keys 4h .. 4h + 3)
//                   is B's layout of P^T as it stands, with A's keys in the same
//                   order: lane (word i, h) takes word i of keys 4h .. 4h + 3,
//                   16 bytes of the interleaved value layout.
// A dimension pair of two keys costs one v_perm, two ANDs and two v_pk_fma_f16
// (kv_common.hpp).  A tile's words and constants come into the wave's own ring
// in LDS by asynchronous copies, a tile ahead, each lane's 16 bytes as it will
// read them; no barrier until the waves' results are joined.  The constants of
// 32 keys' values are turned into f16 once per wave, not once per lane that uses
// them.  The weights' reference, 2^-12 of the largest, moves only when a tile exceeds
// that by 2^3 (weights stay below 2^15 in f16, sums are fp32).
//
// The workgroups divide the tiles of all sequences evenly, by the lengths on
// the device.  Where a sequence's keys are split, every part parks its maximum,
// sum and fp32 rows in the session's scratch, and the last to arrive joins them
// in part order, or a kernel after this one where there are many.
//
// Bound by HBM where the keys are long (64 requests of 4097 tokens, 8 heads of 128 in
// groups of 64: 63 us, 4.8 TB/s; three of 120002 in groups of 32 93 us, 5.0 TB/s), at
// T = f16 by its instructions too (the same three: 110 us, 4.2 TB/s), by fixed
// phases of 9 us where they are not: launch, search, first tile, join (48 requests of
// up to 8193 tokens: 27 us, 2.6 TB/s; one of 391 tokens, 2 heads of 64: 8.6 us).
// With a bias 17 to 32 rows at T = f16 in groups of 32 do not fit the registers (23 to 60 of
// them go to scratch memory): 3 drafts each of three requests of 60001 tokens, 64 heads of 128
// on 8, 79 us without scores, 88 capped, 108 with a bias, 115 with both; of 30001 tokens, heads
// of 256, 141, 150, 167 and 177.  In groups of 64 73, 81, 82 and 89 (256: 111, 116, 144, 152).
#pragma once

#include <algorithm>

#include "kv_common.hpp"

namespace cpq {
namespace {

using namespace dev;

constexpr int kStages = 2;  // of a wave's ring: a tile is copied while one is worked on
constexpr int kTile = 32;
constexpr int kMaxParts = 256;
// Least tiles of a part, and most that are one part all the same where parts are
// that small: a join costs 3 us, a wave's tile 1.1 us while its SIMD has no other.
// (When chosen: one request of 4001 tokens, 8 heads, 12.6 us at 8 tiles a part, 14.4 at
// 16; one of 391 tokens, 2 heads, 11.4 us as one part, 13.1 as two.)
constexpr int kPartTiles = 8, kWholeTiles = 24;
// Eight waves a workgroup instead of four halve what a wave goes over, but are
// slower to start and leave one workgroup to a CU.  They are taken where that is
// enough and a sequence is more than a tile a wave (one request of 290 tokens: 9.3 us,
// with four waves 10.6; of 250 no difference) and at most this many tiles (16
// requests of 701 tokens, 8 heads: 12.5 us, with four waves 14.8; 32 requests of 251:
// 11.7 and 10.0; one of 8001: 15.8 and 13.0).
constexpr size_t kFewTiles = 9, kEightWaves = 64;
constexpr size_t kScanSeqs = 128;
// log2 of the largest weight when the reference moves, and of how far one may pass it:
// up to 2^15 the weights take f16's whole range, so that one of 2^-26 of the largest
// still keeps 11 bits (beside a key that draws nearly all weight and holds zeros the
// others make the output).  The reference moves in the first tile and seldom after.
constexpr float kRaise = 12.f, kSlack = 3.f;

template <int D, int GS>
struct Geo {
  static constexpr int W = D / 8;               // words of a row
  static constexpr int G = D / GS;              // constants of a row
  static constexpr int GW = GS / 8;             // words of a group
  static constexpr int WL = D / 32;             // key words per lane
  static constexpr int NG = WL > GW ? WL / GW : 1;  // key constants per lane
  static constexpr int VS = D == 256 ? 2 : 1;   // sets of 16 value words
  static constexpr int NJ = D == 64 ? 4 : 8;    // result tiles per set
  static constexpr int NQ = D / 64;             // copies of 1 KiB per tile's keys (values)
  static constexpr int NL = G > 2 ? G / 2 : 1;  // copies of 256 bytes per tile's constants
  static constexpr int kLoads = 2 * NQ + 2 * NL;
  // Byte offsets in a stage: keys, values, their constants.
  static constexpr int kV = NQ * 1024, kKc = 2 * kV, kVc = kKc + NL * 256, kStage = kVc + NL * 256;
  // Waves per SIMD that the registers are to allow.
  template <int NC>
  static constexpr int kOccupancy = D == 256 ? 3 - NC : NC == 2 ? 2 : 3;
  // Behind the ring: the values' constants in f16, scales and biases [G][32].
  static constexpr int kConst = kStages * kStage, kWave = kConst + 2 * 64 * G;
};

struct DecodeArgs {
  cpq_kv_cache c;
  cpq_kv_attention_args a;
  int rows_max;    // sequences of more rows are another kernel's
  int target;      // workgroups to divide the tiles over
  int report;      // this launch counts what is wrong with the sequences
  int whole;       // sequences of up to kWholeTiles are one part whatever the others' size
  int joined;      // the parts are joined by kv_join_kernel, not by the last to arrive
  unsigned int* counters;  // per (sequence, head)
  float* partial;          // [workgroup][rows_max][D + 4]: rows, then maximum and sum
  int* starts;             // of many sequences: [n_seqs + 1] first workgroups, else null
  unsigned int* bad;
  KvScore score;
};

typedef __attribute__((address_space(3))) void* LdsPtr;
typedef const __attribute__((address_space(1))) void* GlobalPtr;
__device__ __forceinline__ void copy16(const void* src, unsigned char* lds) {
  __builtin_amdgcn_global_load_lds((GlobalPtr)src, (LdsPtr)lds, 16, 0, 0);
}
__device__ __forceinline__ void copy4(const void* src, unsigned char* lds) {
  __builtin_amdgcn_global_load_lds((GlobalPtr)src, (LdsPtr)lds, 4, 0, 0);
}

// Starts the copies of one tile into a stage: kLoads instructions.
template <int D, int GS>
__device__ __forceinline__ void start_tile(const cpq_kv_cache& c, size_t row_a, size_t row_b, int lane, unsigned char* stage) {
  using X = Geo<D, GS>;
  const int i = lane & 15, h = lane >> 4;
  const size_t mine = lane & 32 ? row_b : row_a;  // lanes 32 .. take the second 16 keys
#pragma unroll
  for (int q = 0; q < X::NQ; ++q) {
    const uint32_t *k, *v;
    if constexpr (D == 64) {  // lane: half a key; a word of four keys
      k = c.k_q + mine * 8 + (lane & 31) * 4;
      v = c.v_q + mine * 8 + (lane & 31) * 4;
    } else {
      const int u = q / (D / 128), part = q % (D / 128);
      k = c.k_q + (u ? row_b : row_a) * X::W + i * X::W + h * X::WL + 4 * part;
      v = c.v_q + (u ? row_b : row_a) * X::W + (h * X::W + 16 * part + i) * 4;
    }
    copy16(k, stage + q * 1024);
    copy16(v, stage + X::kV + q * 1024);
  }
#pragma unroll
  for (int q = 0; q < X::NL; ++q) {
    const int e = min(64 * q + lane, 32 * X::G - 1);  // constant of the tile, 16 G of each place
    const bool second = e >= 16 * X::G;
    const size_t at = (second ? row_b : row_a) * X::G + (second ? e - 16 * X::G : e);
    copy4(c.k_sb + at, stage + X::kKc + q * 256);
    copy4(c.v_sb + at, stage + X::kVc + q * 256);
  }
}

// A wave's running result, relative to 2^ref per row.
template <typename TT, int D, int GS, int NC, Scores SCORES>
struct Rows {
  using X = Geo<D, GS>;
  // At T = f16 a key's and a weight's one rounding to f16 would show in the output: a
  // scale enters in two parts whose products with a nibble are exact, the biases by
  // a product of their own with the queries' sums, a weight with what it lost.
  // (Three requests of 120002 tokens: off by 0.0003 from 64 bits instead of 0.0006 to
  // 0.0013, in 110 us instead of 93.)
  static constexpr bool kExact = !Sig16<TT>::bf16;
  u32x4 qs[NC][X::WL];
  u32x4 qsum[NC];  // sums over a lane's words of each group, in units of 2^6: high and low part
  int qe[NC];    // exponents of the query rows
  float cl[NC];  // log2(e) * scale * 2^(qe + keys.e)
  f32x4 o[X::VS][X::NJ][NC];
  float top[NC], ref[NC], sum[NC];
  int unit[NC];         // of a row's sums o: 2^unit
  KvRange keys, values;  // of the operands
  bool alike = false;   // every row's unit is the values' exponent
  static constexpr bool kScored = SCORES != Scores::kPlain;
  KvRowScore<SCORES> score[kScored ? NC : 1];

  // Chooses the keys of one pass among `left` (bit k: key k of the tile is seen by a
  // row and not yet taken) and sets the exponents to them.
  __device__ __forceinline__ uint32_t choose(const uint32_t (&ksb)[2][X::NG], const uint32_t* vc, int lane, uint32_t left) {
    const int i = lane & 15, h = lane >> 4;
    int kx[2], vx[2];  // of keys i and 16 + i
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float k = 0.f, v = 0.f;
#pragma unroll
      for (int g = 0; g < X::NG; ++g) k = fmaxf(k, finite_size<TT>(ksb[u][g]));
#pragma unroll
      for (int g = 0; g < X::G; g += 4)
        v = fmaxf(v, finite_size<TT>(vc[(4 * u + (i >> 2)) * 4 * X::G + 4 * min(g + h, X::G - 1) + (i & 3)]));
      const bool live = left >> (16 * u + i) & 1;
      kx[u] = live ? size_exponent(over_rows(k, max_of)) : kKvNone;
      vx[u] = live ? size_exponent(over_rows(v, max_of)) : kKvNone;
    }
    values.template fit<TT>(max_of_columns(max(vx[0], vx[1])));
    const bool in0 = (left >> i & 1) && values.takes(vx[0]), in1 = (left >> (16 + i) & 1) && values.takes(vx[1]);
    keys.template fit<TT>(max_of_columns(max(in0 ? kx[0] : kKvNone, in1 ? kx[1] : kKvNone)));
    const uint32_t taken = ((uint32_t)__ballot(in0 && keys.takes(kx[0])) & 0xffffu) |
                           (uint32_t)__ballot(in1 && keys.takes(kx[1])) << 16;
    return taken;
  }
  // The units of the rows that see one of the keys `taken`.
  __device__ __forceinline__ void rescale(float scale, int t, uint32_t taken, const int (&from)[NC], const int (&to)[NC]) {
    alike = true;
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
      cl[cc] = fmaxf(scaled(scale, keys.e + qe[cc]) * kLog2e, FLT_MIN);
      const bool sees = range_bits(from[cc] - t, to[cc] - t) & taken;
      if (top[cc] == -INFINITY) unit[cc] = values.e;  // nothing yet
      int next = sees ? values.e : unit[cc];
      if (__any(next != unit[cc])) {
        if (__any(next < unit[cc])) {
          float m = 0.f;
#pragma unroll
          for (int v = 0; v < X::VS; ++v)
#pragma unroll
            for (int j = 0; j < X::NJ; ++j)
#pragma unroll
              for (int x = 0; x < 4; ++x) m = fmaxf(m, fabsf(o[v][j][cc][x]));
          m = over_rows(m, max_of);
          next = next < unit[cc] ? lower_unit(unit[cc], next, m) : next;
        }
#pragma unroll
        for (int v = 0; v < X::VS; ++v)
#pragma unroll
          for (int j = 0; j < X::NJ; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[v][j][cc][x] = scaled(o[v][j][cc][x], unit[cc] - next);
        unit[cc] = next;
      }
      alike = alike && !__any(next != values.e);
    }
  }

  // One pass over the tile in `stage`, keys t on: those of `left` (bit k: key k is seen by
  // a row) that go together; `left` loses them.  Rows see keys [from, to) of theirs.
  // Returns whether a value's constants were not finite (they count as zeros).
  __device__ __forceinline__ bool add(unsigned char* wave_lds, const unsigned char* stage, int lane, bool whole,
                                      float scale, int t, uint32_t& left, const int (&from)[NC], const int (&to)[NC],
                                      const KvScore& k) {
    const int i = lane & 15, h = lane >> 4;
    const uint32_t* kc = reinterpret_cast<const uint32_t*>(stage + X::kKc);
    const uint32_t* vc = reinterpret_cast<const uint32_t*>(stage + X::kVc);
    uint16_t* cs = reinterpret_cast<uint16_t*>(wave_lds + X::kConst);  // scales, [32 G] biases

    // Constants: whether they fit the exponents (and are finite).
    uint32_t ksb[2][X::NG], vsb[X::NL];
    uint32_t ks = 0u, vs = 0u, kl = 0xffffffffu, vl = 0xffffffffu;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int g = 0; g < X::NG; ++g) {
        ksb[u][g] = kc[(16 * u + i) * X::G + h * X::WL / X::GW + g];
        ks = sizes(ks, ksb[u][g]);
        kl = smallest(kl, ksb[u][g]);
      }
#pragma unroll
    for (int q = 0; q < X::NL; ++q) {
      vsb[q] = vc[64 * q + lane];
      vs = sizes(vs, vsb[q]);
      vl = smallest(vl, vsb[q]);
    }
    uint32_t taken = left;
    bool poison = false;
    // The key of a tile's value constant e.  (One group a head: 32 constants, and the lanes
    // after them hold copies of the last.)
    auto key_of = [](int e) { return X::G > 1 ? e / (4 * X::G) * 4 + (e & 3) : min(e, 31); };
    const bool fit = __all(keys.holds(ks, kl) & values.holds(vs, vl));
    whole = whole & (left == 0xffffffffu);
    if (__builtin_expect(!(whole & alike & fit), 0)) {
      ks = vs = 0u;
      kl = vl = 0xffffffffu;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int g = 0; g < X::NG; ++g) {
          const bool live = left >> (16 * u + i) & 1;
          ks = sizes(ks, live ? ksb[u][g] : 0u);
          kl = smallest(kl, live ? ksb[u][g] : 0xffffffffu);
        }
#pragma unroll
      for (int q = 0; q < X::NL; ++q) {
        const bool live = left >> key_of(64 * q + lane) & 1;
        vs = sizes(vs, live ? vsb[q] : 0u);
        vl = smallest(vl, live ? vsb[q] : 0xffffffffu);
      }
      bool together = __all(all_finite<TT>(ks) & all_finite<TT>(vs));
      if (together) {  // nearly always: one exponent holds all
        keys.template fit<TT>(max_of_wave(size_exponent(finite_size<TT>(ks))));
        values.template fit<TT>(max_of_wave(size_exponent(finite_size<TT>(vs))));
        together = __all(keys.holds(ks, kl) & values.holds(vs, vl));
      }
      if (!together) taken = choose(ksb, vc, lane, left);
      rescale(scale, t, taken, from, to);
      whole = whole && taken == 0xffffffffu;
#pragma unroll
      for (int q = 0; q < X::NL; ++q) {  // what is not taken counts as zeros, as do values that are not finite
        const bool live = taken >> key_of(64 * q + lane) & 1;
        const bool ok = finite(TT::lo(vsb[q])) && finite(TT::hi(vsb[q]));
        poison |= live && !ok;
        vsb[q] = live && ok ? vsb[q] : 0u;
      }
      poison = __any(poison);
    }
    left &= ~taken;
    // The values' constants in f16, each once: [group][key].
    wave_lds_order();
#pragma unroll
    for (int q = 0; q < X::NL; ++q) {
      const int e = 64 * q + lane, at = e / 4 % X::G * 32 + e / (4 * X::G) * 4 + (e & 3);
      if (X::G > 1 || lane < 32) {
        cs[at] = F16::from_f32(scaled(TT::lo(vsb[q]), 24 - values.e));
        cs[32 * X::G + at] = F16::from_f32(scaled(TT::hi(vsb[q]), -values.e));
      }
    }
    wave_lds_order();

    f32x4 sc[2][NC];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t s0[X::NG], s1[X::NG], bb[X::NG], r0[X::NG], r1[X::NG];
#pragma unroll
      for (int g = 0; g < X::NG; ++g) {
        const float sv = scaled(TT::lo(ksb[u][g]), 24 - keys.e), bv = scaled(TT::hi(ksb[u][g]), (kExact ? 6 : 0) - keys.e);
        s0[g] = F16::pack2(sv, sv);
        bb[g] = F16::pack2(bv, bv);
        if constexpr (kExact) {  // 7 bits and the other 4
          const uint32_t all = s0[g];
          s0[g] = all & 0xfff0fff0u;
          r0[g] = __builtin_bit_cast(uint32_t, as_f16x2(all) - as_f16x2(s0[g]));
          r1[g] = sixteenth(r0[g]);
        }
        s1[g] = sixteenth(s0[g]);
      }
#pragma unroll
      for (int cc = 0; cc < NC; ++cc) sc[u][cc] = f32x4{0.f, 0.f, 0.f, 0.f};
      uint32_t kw[X::WL];
      if constexpr (D == 64) {
        const u32x2 v = *reinterpret_cast<const u32x2*>(stage + (16 * u + i) * 32 + h * 8);
        kw[0] = v.x;
        kw[1] = v.y;
      } else {
#pragma unroll
        for (int q = 0; q < D / 128; ++q) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(stage + (u * (D / 128) + q) * 1024 + lane * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) kw[4 * q + e] = v[e];
        }
      }
#pragma unroll
      for (int w = 0; w < X::WL; ++w) {
        const int g = w / X::GW;
        if constexpr (kExact) {
          const u32x4 high = key_slice(kw[w], s0[g], s1[g], 0u), low = key_slice(kw[w], r0[g], r1[g], 0u);
#pragma unroll
          for (int cc = 0; cc < NC; ++cc) {
            sc[u][cc] = Mfma16<F16>::run(high, qs[cc][w], sc[u][cc]);
            sc[u][cc] = Mfma16<F16>::run(low, qs[cc][w], sc[u][cc]);
          }
        } else {
          const u32x4 k = key_slice(kw[w], s0[g], s1[g], bb[g]);
#pragma unroll
          for (int cc = 0; cc < NC; ++cc) sc[u][cc] = Mfma16<F16>::run(k, qs[cc][w], sc[u][cc]);
        }
      }
      if constexpr (kExact) {
        const u32x4 b{bb[0], X::NG > 1 ? bb[X::NG - 1] : 0u, 0u, 0u};
#pragma unroll
        for (int cc = 0; cc < NC; ++cc) sc[u][cc] = Mfma16<F16>::run(b, qsum[cc], sc[u][cc]);
      }
    }

    u32x4 pw[NC], lost[NC];
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
      if constexpr (kScored) {
        score[cc].at(k, t + 4 * h, cl[cc]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float plus = score[cc].step(score[cc].base, 16.f * u);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sc[u][cc][e] = score[cc].of(k, sc[u][cc][e], plus);
            plus = score[cc].step(plus, 1.f);
          }
        }
      }
      const float cl = kScored ? 1.f : this->cl[cc];
      if (!whole) {
        const uint32_t seen = (range_bits(from[cc] - t, to[cc] - t) & taken) >> (4 * h);  // from the lane's first key
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[u][cc][e] = seen >> (16 * u + e) & 1 ? sc[u][cc][e] : -INFINITY;
      }
      float m = fmaxf(fmaxf(fmaxf(sc[0][cc][0], sc[0][cc][1]), fmaxf(sc[0][cc][2], sc[0][cc][3])),
                      fmaxf(fmaxf(sc[1][cc][0], sc[1][cc][1]), fmaxf(sc[1][cc][2], sc[1][cc][3])));
      m = over_rows(m, max_of) * cl;
      if (__builtin_expect(__any(m > top[cc] + kSlack), 0)) {
        const float was = ref[cc];
        top[cc] = fmaxf(top[cc], m);
        ref[cc] = fmaxf(top[cc] - kRaise, -FLT_MAX);
        const float keep = __builtin_amdgcn_exp2f(was - ref[cc]);
        sum[cc] *= keep;
#pragma unroll
        for (int v = 0; v < X::VS; ++v)
#pragma unroll
          for (int j = 0; j < X::NJ; ++j) o[v][j][cc] *= keep;
      }
      float w[8];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * u + e] = __builtin_amdgcn_exp2f(fmaf(sc[u][cc][e], cl, -ref[cc]));
      sum[cc] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        pw[cc][x] = F16::pack2(w[2 * x], w[2 * x + 1]);
        if constexpr (kExact)
          lost[cc][x] = F16::pack2(w[2 * x] - F16::lo(pw[cc][x]), w[2 * x + 1] - F16::hi(pw[cc][x]));
      }
      // (A row whose sums are beyond these values by all that fp32 holds leaves them out.)
      if (__builtin_expect(!alike, 0) && unit[cc] != values.e) {
#pragma unroll
        for (int x = 0; x < 4; ++x) pw[cc][x] = lost[cc][x] = 0u;
      }
    }

#pragma unroll
    for (int v = 0; v < X::VS; ++v) {
      const int word = D == 64 ? i & 7 : 16 * v + i;
      const uint16_t* mine = cs + word / X::GW * 32 + 4 * h;
      uint32_t s0[4], s1[4], bb[4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const u32x2 s = *reinterpret_cast<const u32x2*>(mine + 16 * u);
        const u32x2 b = *reinterpret_cast<const u32x2*>(mine + 32 * X::G + 16 * u);
        s0[2 * u] = s.x; s0[2 * u + 1] = s.y;
        bb[2 * u] = b.x; bb[2 * u + 1] = b.y;
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) s1[x] = sixteenth(s0[x]);
      u32x4 vq[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
        vq[u] = *reinterpret_cast<const u32x4*>(
            stage + X::kV + (D == 64 ? u * 512 + h * 128 + (i & 7) * 16 : (u * (D / 128) + v) * 1024 + lane * 16));
      const uint32_t lane_sel = D == 64 ? (uint32_t)(i >> 3) * 0x00020002u : 0u;
#pragma unroll
      for (int y = 0; y < X::NJ / 2; ++y) {
        const uint32_t sel = (0x0c040c00u + (uint32_t)y * 0x00010001u) + lane_sel;
        u32x4 lo, hi;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t b2 = __builtin_amdgcn_perm(vq[x >> 1][2 * (x & 1) + 1], vq[x >> 1][2 * (x & 1)], sel);
          lo[x] = pk_fma(b2 & 0x000f000fu, s0[x], bb[x]);
          hi[x] = pk_fma(b2 & 0x00f000f0u, s1[x], bb[x]);
        }
#pragma unroll
        for (int cc = 0; cc < NC; ++cc) {
          o[v][2 * y][cc] = Mfma16<F16>::run(lo, pw[cc], o[v][2 * y][cc]);
          o[v][2 * y + 1][cc] = Mfma16<F16>::run(hi, pw[cc], o[v][2 * y + 1][cc]);
          if constexpr (kExact) {
            o[v][2 * y][cc] = Mfma16<F16>::run(lo, lost[cc], o[v][2 * y][cc]);
            o[v][2 * y + 1][cc] = Mfma16<F16>::run(hi, lost[cc], o[v][2 * y + 1][cc]);
          }
        }
      }
    }
    return poison;
  }
};

// What a workgroup does: its sequence, head and part.
struct Item {
  int s, head, part, parts, first;  // first: workgroup of the same head's part 0
  KvSeq q;
};

__device__ __forceinline__ int tiles_of(const KvSeq& q) {
  return (max(q.n - (q.lo & ~(kTile - 1)), 0) + kTile - 1) / kTile;
}
// Sequence s and its tiles that this kernel takes.
__device__ __forceinline__ int seq_tiles(const DecodeArgs& p, int s, int group, int bs_shift, bool report, KvSeq& q) {
  if (s >= (int)p.a.n_seqs) return 0;
  q = kv_seq(p.a, s, bs_shift, report, p.bad);
  const int rows = q.n_q * group;
  return rows == 0 || rows > p.rows_max ? 0 : max(tiles_of(q), 1);  // no keys: zeros to store
}
// Tiles of a part, by those of all sequences; parts of a sequence.
__device__ __forceinline__ int part_of(const DecodeArgs& p, int total) {
  return max(kPartTiles, p.target ? (int)(((long)total * (int)p.c.n_kv_heads + p.target - 1) / p.target) : 0x3fffffff);
}
__device__ __forceinline__ int parts_of(const DecodeArgs& p, int own, int per) {
  return (per == kPartTiles || p.whole) && own <= kWholeTiles ? min(own, 1) : min((own + per - 1) / per, kMaxParts);
}
// The item of workgroup b where kv_starts_kernel has run: two steps of a search
// 64 wide (more past 4096 sequences).
__device__ __forceinline__ bool look_up(const DecodeArgs& p, int b, int group, int bs_shift, Item& it) {
  const int n_seqs = (int)p.a.n_seqs, heads = (int)p.c.n_kv_heads, lane = threadIdx.x & 63;
  if (b >= p.starts[n_seqs]) return false;
  int lo = 0, hi = n_seqs;  // starts[lo] <= b < starts[hi]
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, at = min(lo + lane * step, hi);
    const int k = (int)__builtin_popcountll(__ballot(p.starts[at] <= b)) - 1;  // lane 0's is
    lo = min(lo + k * step, hi - 1);
    hi = min(lo + step, hi);
  }
  const int first = __builtin_amdgcn_readfirstlane(p.starts[lo]), k = b - first;
  const KvSeq q = kv_seq(p.a, lo, bs_shift, false, p.bad);
  it.s = lo;
  it.parts = (__builtin_amdgcn_readfirstlane(p.starts[lo + 1]) - first) / heads;
  it.head = k % heads;
  it.part = k / heads;
  it.first = first + it.head;
  it.q.rows0 = __builtin_amdgcn_readfirstlane(q.rows0);
  it.q.n_q = __builtin_amdgcn_readfirstlane(q.n_q);
  it.q.n = __builtin_amdgcn_readfirstlane(q.n);
  it.q.lo = __builtin_amdgcn_readfirstlane(q.lo);
  it.q.pos = it.q.n - it.q.n_q;
  return true;
}
// The tiles of all sequences divided evenly: workgroup b's item, if any.  Every
// wave goes over the sequences, 64 at a time: their tiles, the size of a part
// from the sum of all, the sequence whose parts workgroup b falls among.
__device__ __forceinline__ bool find_item(const DecodeArgs& p, int b, int group, int bs_shift, Item& it) {
  const int n_seqs = (int)p.a.n_seqs, heads = (int)p.c.n_kv_heads, lane = threadIdx.x & 63;
  if (p.starts) return look_up(p, b, group, bs_shift, it);
  KvSeq q{};
  int total = 0, own = 0;
  for (int base = 0; base < n_seqs; base += 64) {
    own = seq_tiles(p, base + lane, group, bs_shift, p.report && b == 0 && threadIdx.x < 64, q);
    total += __builtin_amdgcn_readlane(wave_scan(own), 63);
  }
  const int per = part_of(p, total);
  int before = 0;
  for (int base = 0; base < n_seqs; base += 64) {
    if (n_seqs > 64) own = seq_tiles(p, base + lane, group, bs_shift, false, q);
    const int parts = parts_of(p, own, per);
    const int sum = wave_scan(parts * heads), at = before + sum - parts * heads;
    before += __builtin_amdgcn_readlane(sum, 63);
    if (b < before) {
      const int l = __builtin_ctzll(__ballot(b >= at && b < at + parts * heads));
      const int k = b - __builtin_amdgcn_readlane(at, l);
      it.s = base + l;
      it.parts = __builtin_amdgcn_readlane(parts, l);
      it.head = k % heads;
      it.part = k / heads;
      it.first = b - it.part * heads;
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

// Each sequence's first workgroup.
constexpr int kStartsThreads = 1024;
__global__ __launch_bounds__(kStartsThreads) void kv_starts_kernel(DecodeArgs p) {
  __shared__ int waves[kStartsThreads / 64];
  const int n_seqs = (int)p.a.n_seqs, heads = (int)p.c.n_kv_heads, group = (int)p.a.n_heads / heads;
  const int tid = threadIdx.x, lane = tid & 63, bs_shift = 31 - __builtin_clz(p.c.block_size);
  KvSeq q{};
  auto sum_all = [&](int v, int& before) {  // over the workgroup; before: over earlier threads
    const int sum = wave_scan(v);
    __syncthreads();
    if (lane == 63) waves[tid >> 6] = sum;
    __syncthreads();
    int all = 0;
    before = sum - v;
#pragma unroll
    for (int w = 0; w < kStartsThreads / 64; ++w) {
      if (w < tid >> 6) before += waves[w];
      all += waves[w];
    }
    return all;
  };
  int total = 0, own = 0, before = 0, at = 0;
  for (int base = 0; base < n_seqs; base += kStartsThreads) {
    own = seq_tiles(p, base + tid, group, bs_shift, p.report, q);
    total += sum_all(own, before);
  }
  const int per = part_of(p, total);
  for (int base = 0; base < n_seqs; base += kStartsThreads) {
    if (n_seqs > kStartsThreads) own = seq_tiles(p, base + tid, group, bs_shift, false, q);
    const int all = sum_all(parts_of(p, own, per) * heads, before);
    if (base + tid < n_seqs) p.starts[base + tid] = at + before;
    at += all;
  }
  if (tid == 0) p.starts[n_seqs] = at;
}

template <typename TT, int D, int GS, int NC, int kWaves, Scores SCORES>
__global__ __launch_bounds__(kWaves * 64, (Geo<D, GS>::template kOccupancy<NC>)) void kv_decode_kernel(DecodeArgs p) {
  using X = Geo<D, GS>;
  extern __shared__ __align__(16) unsigned char lds_bytes[];  // the waves' rings; then the join
  __shared__ int arrived;
  const cpq_kv_cache& c = p.c;
  const cpq_kv_attention_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, h = lane >> 4;
  const int bs_shift = 31 - __builtin_clz(c.block_size);
  const int group = (int)a.n_heads / (int)c.n_kv_heads;
  Item it{};
  if (!find_item(p, blockIdx.x, group, bs_shift, it)) return;
  const KvSeq& q = it.q;
  const int rows = q.n_q * group, head = it.head, parts = it.parts;
  const int base = q.lo & ~(kTile - 1), tiles = tiles_of(q);
  const int per = (tiles + parts - 1) / parts, last = min(tiles, (it.part + 1) * per);

  const KvBlocks blocks = kv_blocks(a, it.s);
  unsigned char* ring = lds_bytes + wave * X::kWave;
  const int t0 = it.part * per + wave;
  int ok = 0;  // two bits a stage: whether the block of either 16 keys is the cache's
  uint32_t id0 = 0, id1 = 0;  // blocks of the tile that is copied next
  auto look = [&](int ti) {
    if (ti >= last) return;
    id0 = blocks[kv_index(base + ti * kTile, q.n, bs_shift)];
    id1 = blocks[kv_index(base + ti * kTile + 16, q.n, bs_shift)];
  };
  auto start = [&](int ti) {
    const int stage = (ti - t0) / kWaves % kStages;
    const KvPlaces pl = kv_places(c, id0, id1, base + ti * kTile, q.n, head, bs_shift);
    ok = (ok & ~(3 << 2 * stage)) | (pl.a.ok ? 1 : 0) << 2 * stage | (pl.b.ok ? 2 : 0) << 2 * stage;
    start_tile<D, GS>(c, pl.a.row, pl.b.row, lane, ring + stage * X::kStage);
    look(ti + kWaves);
  };
  look(t0);
  // Query rows: column n = lane % 16 of tile cc is row r = 16 cc + n, query r / group, head r % group.
  // Their loads, the first tile's blocks and its copies are under way together.
  Rows<TT, D, GS, NC, SCORES> R;
  const int prefix = R.kScored ? kv_prefix(p.score, it.s, q.n) : 0;
  int from[NC], to[NC];  // keys that a row sees
#pragma unroll
  for (int cc = 0; cc < NC; ++cc) {
    const int r = min(16 * cc + i, rows - 1), qi = r / group, hh = head * group + r - qi * group;
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (size_t)(q.rows0 + qi) * a.q_token_stride +
                          (size_t)hh * a.q_head_stride + h * (X::WL * 8);
#pragma unroll
    for (int w = 0; w < X::WL; ++w) R.qs[cc][w] = *reinterpret_cast<const u32x4*>(src + 8 * w);
    const int pos = q.pos + qi;
    from[cc] = a.window ? (int)max((int64_t)pos + 1 - (int64_t)a.window, (int64_t)0) : 0;
    to[cc] = a.causal ? min(max(pos + 1, prefix), q.n) : q.n;
    if constexpr (R.kScored) R.score[cc].head(p.score, hh, from[cc], to[cc]);
  }
#pragma unroll
  for (int st = 0; st < kStages - 1; ++st)
    if (t0 + st * kWaves < last) start(t0 + st * kWaves);
#pragma unroll
  for (int cc = 0; cc < NC; ++cc) {
    float m = 0.f;
#pragma unroll
    for (int w = 0; w < X::WL; ++w) m = largest<TT>(R.qs[cc][w], m);
    m = over_rows(m, max_of);
    R.qe[cc] = query_exponent(m);
#pragma unroll
    for (int w = 0; w < X::WL; ++w) R.qs[cc][w] = query_slice<TT>(R.qs[cc][w], R.qe[cc]);
    if constexpr (R.kExact) {
      R.qsum[cc] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int g = 0; g < X::NG; ++g) {
        float all = 0.f;
#pragma unroll
        for (int w = g * X::WL / X::NG; w < (g + 1) * X::WL / X::NG; ++w)
#pragma unroll
          for (int e = 0; e < 4; ++e) all = F16::dot2(R.qs[cc][w][e], 0x3c003c00u, all);
        all *= 0x1p-6f;
        const float high = F16::lo(F16::pack2(all, 0.f));
        R.qsum[cc][g] = F16::pack2(high, all - high);
      }
    }
    R.cl[cc] = fmaxf(scaled(a.scale, R.qe[cc]) * kLog2e, FLT_MIN);
    R.top[cc] = -INFINITY;
    R.ref[cc] = -FLT_MAX;
    R.sum[cc] = 0.f;
    R.unit[cc] = 0;
#pragma unroll
    for (int v = 0; v < X::VS; ++v)
#pragma unroll
      for (int j = 0; j < X::NJ; ++j) R.o[v][j][cc] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Every row sees the keys [seen_from, seen_end): nothing to mask among them.
  const int seen_end = a.causal ? min(max(q.pos + 1, prefix), q.n) : q.n;
  const int seen_from = a.window ? (int)max((int64_t)q.pos + q.n_q - (int64_t)a.window, (int64_t)0) : 0;
  uint32_t nan_groups[NC] = {};  // groups of dimensions that are NaN in a row
  // The SIMD serves its oldest wave first, so of the workgroups on a CU one would
  // end long before the last.  A wave gives way as it gets ahead.
  const int quarter = (last - t0 + 3) / 4;
  __builtin_amdgcn_s_setprio(3);
  for (int ti = t0; ti < last; ti += kWaves) {
    if (ti - t0 >= quarter) {
      if (ti - t0 >= 3 * quarter) __builtin_amdgcn_s_setprio(0);
      else if (ti - t0 >= 2 * quarter) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(2);
    }
    // The stage that the wave read last is free once its reads are done.
    wave_lds_order();
    wait_lds();
    if (ti + (kStages - 1) * kWaves < last) {
      start(ti + (kStages - 1) * kWaves);
      wait_vmcnt<(kStages - 1) * X::kLoads>();
    } else {
      wait_vmcnt<0>();
    }
    wave_lds_order();
    const int stage = (ti - t0) / kWaves % kStages;
    const int t = base + ti * kTile, oks = ok >> 2 * stage & 3;
    const bool whole = t >= seen_from && t + kTile <= seen_end && oks == 3;
    // (Of the keys [q.lo, q.n) each is seen by one of the rows.)
    if (lane == 0 && ((!(oks & 1) && t < q.n && t + 16 > q.lo) || (!(oks & 2) && t + 16 < q.n))) atomicAdd(p.bad, 1u);
    uint32_t left = 0xffffffffu;  // keys that some row sees
    if (!whole)
      left = range_bits(q.lo - t, q.n - t) & ((oks & 1 ? 0xffffu : 0u) | (oks & 2 ? 0xffff0000u : 0u));
    bool poison = false;
    if (left) {
      do {
        poison |= R.add(ring, ring + stage * X::kStage, lane, whole, a.scale, t, left, from, to, p.score);
      } while (__builtin_expect(left != 0, 0));
    }
    if (__builtin_expect(poison, 0)) {
      const KvPlaces pl = kv_places(c, blocks[kv_index(t, q.n, bs_shift)], blocks[kv_index(t + 16, q.n, bs_shift)], t,
                                    q.n, head, bs_shift);
#pragma unroll
      for (int cc = 0; cc < NC; ++cc) {
        nan_groups[cc] |= poisoned_groups<TT>(c, pl.a, t, X::G, from[cc], to[cc]);
        if (t + 16 < q.n) nan_groups[cc] |= poisoned_groups<TT>(c, pl.b, t + 16, X::G, from[cc], to[cc]);
      }
    }
  }

  // The waves' results: each one's rows relative to its own maximum.
  __syncthreads();
  float* lds = reinterpret_cast<float*>(lds_bytes);  // [wave][rows][LD], then maxima and sums
  constexpr int LD = D + 4;
  float* wmax = lds + kWaves * rows * LD;  // [wave][rows]
  float* wsum = wmax + kWaves * rows;
#pragma unroll
  for (int cc = 0; cc < NC; ++cc) {
    const int r = 16 * cc + i;
    const float total = over_rows(R.sum[cc], sum_of);
    if (r < rows) {
      float* dst = lds + (wave * rows + r) * LD;
#pragma unroll
      for (int v = 0; v < X::VS; ++v)
#pragma unroll
        for (int j = 0; j < X::NJ; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int w = 4 * h + x;  // of 16: word, or word and half of its dimensions
            const int d = D == 64 ? 8 * (w & 7) + 4 * (w >> 3) + j : 8 * (16 * v + w) + j;
            dst[d] = nan_groups[cc] >> (d / GS) & 1 ? NAN : scaled(R.o[v][j][cc][x], R.unit[cc]);
          }
      if (h == 0) {
        wmax[wave * rows + r] = R.ref[cc];
        wsum[wave * rows + r] = total;
      }
    }
  }
  __syncthreads();
  const size_t slab = (size_t)p.rows_max * LD;
  auto put = [&](int r, int d, f32x4 acc, float inv) {
    const int qi = r / group, hh = head * group + r - qi * group;
    uint16_t* out = static_cast<uint16_t*>(a.out) + (size_t)(q.rows0 + qi) * a.out_token_stride +
                    (size_t)hh * a.out_head_stride + d;
    *reinterpret_cast<u32x2*>(out) = u32x2{TT::pack2(acc[0] * inv, acc[1] * inv), TT::pack2(acc[2] * inv, acc[3] * inv)};
  };
  for (int e = tid; e < rows * (D / 4); e += kWaves * 64) {
    const int r = e / (D / 4), d = e % (D / 4) * 4;
    float m = wmax[r];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, wmax[w * rows + r]);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float k = __builtin_amdgcn_exp2f(wmax[w * rows + r] - m);
      total += wsum[w * rows + r] * k;
      acc += *reinterpret_cast<const f32x4*>(lds + (w * rows + r) * LD + d) * k;
    }
    if (parts == 1) {
      put(r, d, acc, total == 0.f ? 0.f : 1.f / total);
    } else {
      const float* park = p.partial + blockIdx.x * slab;
      park_store(park, (r * LD + d) * 4, acc);
      if (d == 0) park_store(park, (r * LD + D) * 4, f32x4{m, total, 0.f, 0.f});
    }
  }
  if (parts == 1 || p.joined) return;

  // The last part to arrive joins them: the parts' weights (a lane a part) and
  // their rows, every (threads / vectors)-th part to a thread, eight loads in
  // flight, the first of them while the weights are made.
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  unsigned int* counter = p.counters + (it.s * (int)c.n_kv_heads + head);
  if (tid == 0) arrived = (int)__hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (arrived != parts - 1) return;
  const float* all = p.partial + it.first * slab;
  const int stride = (int)(slab * c.n_kv_heads);  // from part to part
  float* weight = lds;                   // [rows][parts]
  float* share = weight + rows * parts;  // [rows]: 1 / sum
  f32x4* acc_lds = reinterpret_cast<f32x4*>(lds + ((rows * parts + rows + 3) & ~3));
  const int vectors = rows * (D / 4), each = max(kWaves * 64 / vectors, 1), items = vectors * each;
  constexpr int U = 8;
  f32x4 x[U];
  auto fetch = [&](int e, int k) {
    const int v = e % vectors, r = v / (D / 4), d = v % (D / 4) * 4;
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = park_load(all, (min(k + u * each, parts - 1) * stride + r * LD + d) * 4);
  };
  fetch(min(tid, items - 1), min(tid, items - 1) / vectors);
  for (int r = wave; r < rows; r += kWaves) {
    float m = -FLT_MAX, total = 0.f;
    f32x4 ml[kMaxParts / 64];
#pragma unroll
    for (int u = 0; u < kMaxParts / 64; ++u) {
      if (64 * u >= parts) break;
      ml[u] = park_load(all, (min(64 * u + lane, parts - 1) * stride + r * LD + D) * 4);
      m = fmaxf(m, ml[u][0]);
    }
    m = wave_max(m);
#pragma unroll
    for (int u = 0; u < kMaxParts / 64; ++u) {
      if (64 * u >= parts) break;
      const float w = __builtin_amdgcn_exp2f(ml[u][0] - m);
      if (64 * u + lane < parts) {
        weight[r * parts + 64 * u + lane] = w;
        total += ml[u][1] * w;
      }
    }
    total = wave_sum(total);
    if (lane == 0) share[r] = total == 0.f ? 0.f : 1.f / total;
  }
  __syncthreads();
  for (int e = tid; e < items; e += kWaves * 64) {
    const int k0 = e / vectors, v = e - k0 * vectors, r = v / (D / 4), d = v % (D / 4) * 4;
    if (e != tid) fetch(e, k0);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int k = k0;;) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k + u * each < parts) acc += x[u] * weight[r * parts + k + u * each];
      k += U * each;
      if (k >= parts) break;
      fetch(e, k);
    }
    if (each == 1) put(r, d, acc, share[r]);
    else acc_lds[e] = acc;
  }
  if (each > 1) {
    __syncthreads();
    for (int v = tid; v < vectors; v += kWaves * 64) {
      f32x4 acc = acc_lds[v];
      for (int k = 1; k < each; ++k) acc += acc_lds[k * vectors + v];
      put(v / (D / 4), v % (D / 4) * 4, acc, share[v / (D / 4)]);
    }
  }
  if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Joins the parts of few heads' long keys.  The last workgroup to arrive takes 8 us
// to read 94 parts alone (one request of 60001 tokens, 8 heads, 4 rows of 128: 192 KB a
// head; 33 us in all), 32 workgroups together 4.5 us with their launch (24 us in all).
// At 15 parts the two come out even, at 31 it is 15 us to 13.  A workgroup joins 32
// vectors of four dimensions, a thread every eighth part.
constexpr size_t kJoinParts = 16;
constexpr int kJoinVectors = 32, kJoinSlices = 8, kJoinThreads = kJoinSlices * kJoinVectors;
template <typename TT, int D>
__global__ __launch_bounds__(kJoinThreads) void kv_join_kernel(DecodeArgs p) {
  constexpr int LD = D + 4, kRows = D < 128 ? 128 / D : 1, U = 16;  // rows of a workgroup
  static_assert(kMaxParts <= 2 * U * kJoinSlices);
  __shared__ float weight[kRows][kMaxParts];
  __shared__ float share[kRows];
  __shared__ f32x4 slices[kJoinSlices][kJoinVectors];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int heads = (int)p.c.n_kv_heads, group = (int)p.a.n_heads / heads, s = blockIdx.x / heads, head = blockIdx.x % heads;
  KvSeq q{};
  const int own = seq_tiles(p, lane, group, 31 - __builtin_clz(p.c.block_size), false, q);
  const int per = part_of(p, __builtin_amdgcn_readlane(wave_scan(own), 63));
  const int mine = parts_of(p, own, per), sum = wave_scan(mine * heads);
  const int parts = __builtin_amdgcn_readlane(mine, s), first = __builtin_amdgcn_readlane(sum - mine * heads, s) + head;
  const int rows = __builtin_amdgcn_readlane(q.n_q, s) * group, rows0 = __builtin_amdgcn_readlane(q.rows0, s);
  const int v0 = blockIdx.y * kJoinVectors, r0 = v0 / (D / 4);
  if (parts <= 1 || r0 >= rows) return;
  const size_t slab = (size_t)p.rows_max * LD;
  const float* all = p.partial + first * slab;
  const int stride = (int)(slab * heads);
  const int v = min(v0 + tid % kJoinVectors, rows * (D / 4) - 1), r = v / (D / 4), d = v % (D / 4) * 4;
  f32x4 x[U];
  auto fetch = [&](int k) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      x[u] = *reinterpret_cast<const f32x4*>(all + (size_t)min(k + u * kJoinSlices, parts - 1) * stride + r * LD + d);
  };
  fetch(tid / kJoinVectors);
  if (wave < kRows && r0 + wave < rows) {
    float m = -FLT_MAX, total = 0.f;
    f32x4 ml[kMaxParts / 64];
#pragma unroll
    for (int u = 0; u < kMaxParts / 64; ++u) {
      ml[u] = *reinterpret_cast<const f32x4*>(all + (size_t)min(64 * u + lane, parts - 1) * stride + (r0 + wave) * LD + D);
      m = fmaxf(m, ml[u][0]);
    }
    m = wave_max(m);
#pragma unroll
    for (int u = 0; u < kMaxParts / 64; ++u) {
      const float w = 64 * u + lane < parts ? __builtin_amdgcn_exp2f(ml[u][0] - m) : 0.f;
      weight[wave][64 * u + lane] = w;
      total += ml[u][1] * w;
    }
    total = wave_sum(total);
    if (lane == 0) share[wave] = total == 0.f ? 0.f : 1.f / total;
  }
  __syncthreads();
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int k = tid / kJoinVectors; k < parts; k += U * kJoinSlices) {
    if (k >= U * kJoinSlices) fetch(k);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u * kJoinSlices < parts) acc += x[u] * weight[r - r0][k + u * kJoinSlices];
  }
  slices[tid / kJoinVectors][tid % kJoinVectors] = acc;
  __syncthreads();
  if (tid >= kJoinVectors || v0 + tid >= rows * (D / 4)) return;
#pragma unroll
  for (int k = 1; k < kJoinSlices; ++k) acc += slices[k][tid];
  const int qi = r / group, hh = head * group + r - qi * group;
  uint16_t* out = static_cast<uint16_t*>(p.a.out) + (size_t)(rows0 + qi) * p.a.out_token_stride +
                  (size_t)hh * p.a.out_head_stride + d;
  acc *= share[r - r0];
  *reinterpret_cast<u32x2*>(out) = u32x2{TT::pack2(acc[0], acc[1]), TT::pack2(acc[2], acc[3])};
}

template <typename TT, int D, int GS, int NC, int kWaves, Scores SCORES>
hipError_t launch(hipStream_t s, const DecodeArgs& p, size_t grid) {
  const size_t ring = (size_t)kWaves * Geo<D, GS>::kWave;
  const size_t waves = (size_t)kWaves * p.rows_max * (D + 4 + 2) * sizeof(float);
  const size_t join = ((size_t)p.rows_max * (kMaxParts + 1) + 4 + (size_t)kWaves * 64 * 4) * sizeof(float);
  const size_t lds = std::max(ring, std::max(waves, p.target ? join : 0));
  auto kernel = kv_decode_kernel<TT, D, GS, NC, kWaves, SCORES>;
  if (lds > 60 * 1024) {
    static const hipError_t raised = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                         hipFuncAttributeMaxDynamicSharedMemorySize, 156 * 1024);
    if (raised != hipSuccess) return raised;
  }
  hipLaunchKernelGGL(kernel, dim3((uint32_t)grid), dim3(kWaves * 64), lds, s, p);
  const hipError_t launched = hipGetLastError();
  if (launched != hipSuccess || !p.joined) return launched;
  const dim3 joins((uint32_t)(p.a.n_seqs * p.c.n_kv_heads),
                   (uint32_t)((p.rows_max * (D / 4) + kJoinVectors - 1) / kJoinVectors));
  hipLaunchKernelGGL((kv_join_kernel<TT, D>), joins, dim3(kJoinThreads), 0, s, p);
  return hipGetLastError();
}

template <typename TT, int NC, int kWaves, Scores SCORES>
hipError_t launch_d(hipStream_t s, const DecodeArgs& p, size_t grid) {
  switch (p.c.head_dim * 1000 + p.c.group_size) {
    case 64032: return launch<TT, 64, 32, NC, kWaves, SCORES>(s, p, grid);
    case 64064: return launch<TT, 64, 64, NC, kWaves, SCORES>(s, p, grid);
    case 128032: return launch<TT, 128, 32, NC, kWaves, SCORES>(s, p, grid);
    case 128064: return launch<TT, 128, 64, NC, kWaves, SCORES>(s, p, grid);
    case 128128: return launch<TT, 128, 128, NC, kWaves, SCORES>(s, p, grid);
    case 256032: return launch<TT, 256, 32, NC, 4, SCORES>(s, p, grid);
    case 256064: return launch<TT, 256, 64, NC, kWaves, SCORES>(s, p, grid);
    case 256128: return launch<TT, 256, 128, NC, kWaves, SCORES>(s, p, grid);
    default: return hipErrorInvalidValue;
  }
}

template <Scores SCORES>
hipError_t run_decode(const ExecCtx& ex, const cpq_kv_cache& c, const cpq_kv_attention_args& a, const KvScore& score,
                      int rows_max, bool report, unsigned int* bad) {
  DecodeArgs p{};
  p.score = score;
  p.c = c;
  p.a = a;
  p.bad = bad;
  p.rows_max = rows_max;
  p.report = report;
  const size_t reach = a.window ? std::min<size_t>(a.max_kv, (size_t)a.window + a.max_q) : a.max_kv;
  const size_t most_tiles = (reach + kTile - 1) / kTile + 1, most_parts = most_tiles <= kWholeTiles ? 1 : most_tiles / kPartTiles;
  const bool fits = c.head_dim < 256 || c.group_size > 32;  // the rings of eight waves in LDS
  const int waves = fits && p.rows_max <= 16 && most_tiles > kFewTiles && most_tiles <= kEightWaves &&
                    a.n_seqs * c.n_kv_heads * most_parts <= (size_t)ex.cu_count
                ? 8
                : 4;
  const size_t pairs = a.n_seqs * c.n_kv_heads;
  const size_t slab = (size_t)p.rows_max * (c.head_dim + 4) * sizeof(float);
  const size_t left = ex.scratch_bytes > kWideCounterBytes ? ex.scratch_bytes - kWideCounterBytes : 0;
  // Every wave goes over the sequences, 64 at a time; over many a kernel before does
  // (up to 600 keys each: 700 sequences 67 us, 117 without; 100 sequences 18 and 16).
  const size_t starts = a.n_seqs > kScanSeqs ? (a.n_seqs + 4) / 4 * 16 : 0;
  const size_t room = left > starts ? (left - starts) / slab : 0;
  // As many parts as workgroups are resident (of eight waves one to a CU: 64 pairs of 33
  // tiles made 320 parts by the others' count, a second round: 19.3 us, now 13.4; f16 in
  // groups of 32 20.4 and 14.2); each (sequence, head) rounds its own up, by half a part
  // on average.
  p.whole = waves == 8;
  const size_t resident = (size_t)(waves == 8 ? 1 : c.head_dim == 256 || p.rows_max > 16 ? 2 : 3) * ex.cu_count;
  size_t target = std::max(resident - std::min(resident, pairs / 2), resident / 4);
  if (pairs * sizeof(unsigned int) > kWideCounterBytes || room <= pairs) target = 0;
  else target = std::min(target, room - pairs);
  p.target = (int)target;
  // Parts of a head, at most; many are joined by a kernel of its own.
  const size_t most = std::min(target / pairs + 1, (a.max_kv + kTile - 1) / kTile / kPartTiles);
  p.joined = a.n_seqs <= 64 && most >= kJoinParts;
  p.counters = static_cast<unsigned int*>(ex.scratch);
  char* rest = static_cast<char*>(ex.scratch) + kWideCounterBytes;
  if (starts && left >= starts) {
    p.starts = reinterpret_cast<int*>(rest);
    rest += starts;
    hipLaunchKernelGGL(kv_starts_kernel, dim3(1), dim3(kStartsThreads), 0, ex.stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  p.partial = reinterpret_cast<float*>(rest);
  const size_t grid = pairs + target;
  const bool bf16 = c.dtype == CPQ_DTYPE_BF16;
  if (p.rows_max > 16) return bf16 ? launch_d<BF16, 2, 4, SCORES>(ex.stream, p, grid) : launch_d<F16, 2, 4, SCORES>(ex.stream, p, grid);
  if (waves == 8) return bf16 ? launch_d<BF16, 1, 8, SCORES>(ex.stream, p, grid) : launch_d<F16, 1, 8, SCORES>(ex.stream, p, grid);
  return bf16 ? launch_d<BF16, 1, 4, SCORES>(ex.stream, p, grid) : launch_d<F16, 1, 4, SCORES>(ex.stream, p, grid);
}

}  // namespace
}  // namespace cpq
