// Attention over the 4-bit key/value cache for few query rows per sequence
// (kernels/kv_attention.hip chooses; semantics: cpq_kv_attention in cpq.h).
//
// The query rows of one key/value head (n_q queries times the heads of its
// group, at most 16 NC) share its keys and values, which are read once.  A
// workgroup of four waves takes one (sequence, head, part of the keys); each
// wave walks tiles of 32 keys with a softmax of its own:
//   S^T = K Q^T   v_mfma_f32_16x16x32_f16, A = 16 keys, B = 16 query rows:
//                 lane (key i, quarter h) holds a quarter of the key's words,
//                 16 adjacent bytes at head_dim 128, as the cache lays them out
//   O^T += V^T P^T  A = 16 words' j-th dimension over 32 keys, B = the weights.
//                 The result layout of S^T (lane: query n, keys 4h .. 4h + 3)
//                 is B's layout of P^T as it stands, with A's keys in the same
//                 order: lane (word i, h) takes word i of keys 4h .. 4h + 3, one
//                 16-byte load of the interleaved value layout.
// So nothing goes through LDS until the waves' results are joined, and a
// dimension pair of two keys costs one v_perm, two ANDs and two v_pk_fma_f16
// (kv_common.hpp).  The running maximum moves only when a tile exceeds it by
// 2^8 (weights stay below 2^8 in f16, sums are fp32).
//
// Where keys are split, every part parks its maximum, sum and fp32 rows in the
// session's scratch, and the last to arrive joins them in part order.
#include <algorithm>

#include "kv_common.hpp"

namespace cpq {
namespace {

using namespace dev;

constexpr int kWaves = 4;
constexpr int kTile = 32;
constexpr float kSlack = 8.f;  // log2 of how far a weight may pass 1

template <int D>
struct Tile {
  static constexpr int WL = D / 32;             // key words per lane
  static constexpr int NG = D == 256 ? 2 : 1;   // key constants per lane (32 dimensions each at least)
  static constexpr int VS = D == 256 ? 2 : 1;   // sets of 16 value words
  static constexpr int NJ = D == 64 ? 4 : 8;    // dimensions of a word per result tile set
  uint32_t kq[2][WL];
  uint32_t ksb[2][NG];
  u32x4 vq[2][VS];
  u32x4 vsb[2][VS];
};

struct DecodeArgs {
  cpq_kv_cache c;
  cpq_kv_attention_args a;
  int parts;       // most parts per sequence and head
  int part_tiles;  // least tiles of one part
  int rows_max;    // query rows the scratch and LDS are laid out for
  int report;      // this launch counts what is wrong with the sequences
  unsigned int* counters;
  float* partial;  // [seq * head][part][rows_max][D + 2]: rows, then maximum and sum
  unsigned int* bad;
};

template <int D>
__device__ __forceinline__ void load_tile(Tile<D>& t, const cpq_kv_cache& c, const KvPlace* p, int lane, int gw_shift) {
  using T = Tile<D>;
  constexpr int W = D / 8;
  const int G = W >> gw_shift, i = lane & 15, h = lane >> 4;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const uint32_t* kq = c.k_q + p[u].row * W + i * W + h * T::WL;
    if constexpr (T::WL == 2) {
      const u32x2 v = *reinterpret_cast<const u32x2*>(kq);
      t.kq[u][0] = v.x; t.kq[u][1] = v.y;
    } else {
#pragma unroll
      for (int q = 0; q < T::WL / 4; ++q) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(kq + 4 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) t.kq[u][4 * q + e] = v[e];
      }
    }
#pragma unroll
    for (int q = 0; q < T::NG; ++q)
      t.ksb[u][q] = c.k_sb[p[u].row * G + i * G + ((h * T::WL + 4 * q) >> gw_shift)];
#pragma unroll
    for (int q = 0; q < T::VS; ++q) {
      const int w = 16 * q + (i & (W - 1));
      t.vq[u][q] = *reinterpret_cast<const u32x4*>(c.v_q + (p[u].row >> 2) * (4 * W) + (h * W + w) * 4);
      t.vsb[u][q] =
          *reinterpret_cast<const u32x4*>(c.v_sb + (p[u].row >> 2) * (4 * G) + (h * G + (w >> gw_shift)) * 4);
    }
  }
}

template <typename TT, int D, int NC>
__global__ __launch_bounds__(kWaves * 64) void kv_decode_kernel(DecodeArgs p) {
  using T = Tile<D>;
  constexpr int W = D / 8, WL = T::WL, NJ = T::NJ, VS = T::VS;
  extern __shared__ float lds[];  // [wave][rows][D + 4], then [wave][rows] maxima and sums
  __shared__ unsigned int flag;
  const cpq_kv_cache& c = p.c;
  const cpq_kv_attention_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, h = lane >> 4;
  const int pair = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  const int head = pair % (int)c.n_kv_heads, s = pair / (int)c.n_kv_heads;
  const int bs_shift = 31 - __builtin_clz(c.block_size), gw_shift = 28 - __builtin_clz(c.group_size);
  const int group = (int)a.n_heads / (int)c.n_kv_heads;
  const KvSeq q = kv_seq(a, s, bs_shift, p.report && tid == 0 && head == 0 && part == 0, p.bad);
  const int rows = q.n_q * group;
  if (rows == 0 || rows > p.rows_max) return;  // none, not computed, or many: another kernel's

  // Tiles of this part.
  const int base = q.lo & ~(kTile - 1);
  const int tiles = (max(q.n - base, 0) + kTile - 1) / kTile;
  const int per = max(p.part_tiles, (tiles + p.parts - 1) / p.parts);
  const int parts = max((tiles + per - 1) / per, 1);
  if (part >= parts) return;
  const int last = min(tiles, (part + 1) * per);

  // Query rows: column n = lane % 16 of tile cc is row r = 16 cc + n, query r / group, head r % group.
  u32x4 qs[NC][WL];
  float cl[NC];   // log2(e) * scale * 2^(query exponent)
  int qpos[NC];   // position of the row's query
  int qe[NC];
#pragma unroll
  for (int cc = 0; cc < NC; ++cc) {
    const int r = min(16 * cc + i, rows - 1), qi = r / group, hh = head * group + r - qi * group;
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (size_t)(q.rows0 + qi) * a.q_token_stride +
                          (size_t)hh * a.q_head_stride + h * (WL * 8);
    u32x4 raw[WL];
    float m = 0.f;
#pragma unroll
    for (int w = 0; w < WL; ++w) {
      raw[w] = *reinterpret_cast<const u32x4*>(src + 8 * w);
      m = largest<TT>(raw[w], m);
    }
    m = over_rows(m, max_of);
    qe[cc] = query_exponent(m);
#pragma unroll
    for (int w = 0; w < WL; ++w) qs[cc][w] = query_slice<TT>(raw[w], qe[cc]);
    qpos[cc] = q.pos + qi;
  }

  f32x4 o[VS][NJ][NC];
  float top[NC], ref[NC], sum[NC];
#pragma unroll
  for (int cc = 0; cc < NC; ++cc) {
    top[cc] = -INFINITY;
    ref[cc] = -FLT_MAX;
    sum[cc] = 0.f;
    cl[cc] = fmaxf(scaled(a.scale * kLog2e, qe[cc]), FLT_MIN);
#pragma unroll
    for (int v = 0; v < VS; ++v)
#pragma unroll
      for (int j = 0; j < NJ; ++j) o[v][j][cc] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  int ek = 0, ev = 0;  // exponents of keys and values; zeros alone fit them so far
  uint32_t klim = 0, vlim = 0;
  const uint32_t* blocks = a.block_table + (size_t)s * a.max_blocks;

  auto places = [&](int ti, KvPlace* pl) {
    const int t = base + ti * kTile;
    pl[0] = kv_place(c, blocks, t, q.n, head, bs_shift);
    pl[1] = bs_shift > 4 && t + 16 < q.n ? KvPlace{pl[0].row + 16, pl[0].ok} : kv_place(c, blocks, t + 16, q.n, head, bs_shift);
  };
  // Every row sees all keys of [t, t + 32): nothing to mask.
  const int seen_end = a.causal ? min(q.pos + 1, q.n) : q.n;
  const int seen_from = a.window ? (int)max((int64_t)q.pos + q.n_q - (int64_t)a.window, (int64_t)0) : 0;

  Tile<D> cur, nxt;
  KvPlace now[2] = {}, then[2] = {};
  int ti = part * per + wave;
  if (ti < last) {
    places(ti, now);
    load_tile<D>(cur, c, now, lane, gw_shift);
    if (ti + kWaves < last) places(ti + kWaves, then);
  }
  for (; ti < last; ti += kWaves) {
    const bool ok0 = now[0].ok, ok1 = now[1].ok;
    if (ti + kWaves < last) {
      now[0] = then[0]; now[1] = then[1];
      load_tile<D>(nxt, c, now, lane, gw_shift);
      if (ti + 2 * kWaves < last) places(ti + 2 * kWaves, then);
    }
    const int t = base + ti * kTile;
    const bool whole = t >= seen_from && t + kTile <= seen_end && ok0 && ok1;
    if (!whole) {
      if (lane == 0 && ((!ok0 && t < q.n) || (!ok1 && t + 16 < q.n))) atomicAdd(p.bad, 1u);
      // Values that no row sees count as zeros, whatever they hold.
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = t + 16 * u + 4 * h + e;
          const bool any = key < q.n && key >= q.lo && (u ? ok1 : ok0);
#pragma unroll
          for (int v = 0; v < VS; ++v) cur.vsb[u][v][e] = any ? cur.vsb[u][v][e] : 0u;
        }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int key = t + 16 * u + i;
        const bool any = key < q.n && key >= q.lo && (u ? ok1 : ok0);
#pragma unroll
        for (int g = 0; g < T::NG; ++g) cur.ksb[u][g] = any ? cur.ksb[u][g] : 0u;
      }
    }

    // Exponents: larger constants than before (or none finite) are rare.
    uint32_t ks = klim, vs = vlim;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int g = 0; g < T::NG; ++g) ks = sizes(ks, cur.ksb[u][g]);
#pragma unroll
      for (int v = 0; v < VS; ++v)
#pragma unroll
        for (int e = 0; e < 4; ++e) vs = sizes(vs, cur.vsb[u][v][e]);
    }
    const bool careful = __any(ks != klim || vs != vlim);
    if (careful) {
      float km = 0.f, vm = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int g = 0; g < T::NG; ++g) km = fmaxf(km, finite_size<TT>(cur.ksb[u][g]));
#pragma unroll
        for (int v = 0; v < VS; ++v)
#pragma unroll
          for (int e = 0; e < 4; ++e) vm = fmaxf(vm, finite_size<TT>(cur.vsb[u][v][e]));
      }
      km = wave_max(km);
      vm = wave_max(vm);
      if (klim == 0 || size_exponent(km) > ek) {
        ek = size_exponent(km);
        klim = size_limits<TT>(ek);
#pragma unroll
        for (int cc = 0; cc < NC; ++cc) cl[cc] = fmaxf(scaled(a.scale * kLog2e, ek + qe[cc]), FLT_MIN);
      }
      if (vlim == 0 || size_exponent(vm) > ev) {
        const int e = size_exponent(vm);
#pragma unroll
        for (int v = 0; v < VS; ++v)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int cc = 0; cc < NC; ++cc)
#pragma unroll
              for (int x = 0; x < 4; ++x) o[v][j][cc][x] = scaled(o[v][j][cc][x], ev - e);
        ev = e;
        vlim = size_limits<TT>(ev);
      }
    }

    // S^T.
    f32x4 sc[2][NC];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t s0[T::NG], s1[T::NG], bb[T::NG];
#pragma unroll
      for (int g = 0; g < T::NG; ++g) {
        const float sv = scaled(TT::lo(cur.ksb[u][g]), 24 - ek), bv = scaled(TT::hi(cur.ksb[u][g]), -ek);
        s0[g] = F16::pack2(sv, sv);
        bb[g] = F16::pack2(bv, bv);
        s1[g] = sixteenth(s0[g]);
      }
#pragma unroll
      for (int cc = 0; cc < NC; ++cc) sc[u][cc] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WL; ++w) {
        const int g = T::NG == 2 ? w / 4 : 0;
        const u32x4 k = key_slice(cur.kq[u][w], s0[g], s1[g], bb[g]);
#pragma unroll
        for (int cc = 0; cc < NC; ++cc) sc[u][cc] = Mfma16<F16>::run(k, qs[cc][w], sc[u][cc]);
      }
    }

    // Weights.
    u32x4 pw[NC], seen[NC];
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
      if (!whole) {
        const int to = a.causal ? min(qpos[cc] + 1, q.n) : q.n;
        const int from = a.window ? (int)max((int64_t)qpos[cc] + 1 - (int64_t)a.window, (int64_t)0) : 0;
        uint32_t bits = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = t + 16 * u + 4 * h + e;
            const bool on = key >= from && key < to && (u ? ok1 : ok0);
            sc[u][cc][e] = on ? sc[u][cc][e] : -INFINITY;
            bits |= (uint32_t)on << (4 * u + e);
          }
#pragma unroll
        for (int x = 0; x < 4; ++x)
          seen[cc][x] = ((bits >> (2 * x) & 1) ? 0x3c00u : 0u) | ((bits >> (2 * x + 1) & 1) ? 0x3c000000u : 0u);
      } else {
        seen[cc] = u32x4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
      }
      float m = fmaxf(fmaxf(fmaxf(sc[0][cc][0], sc[0][cc][1]), fmaxf(sc[0][cc][2], sc[0][cc][3])),
                      fmaxf(fmaxf(sc[1][cc][0], sc[1][cc][1]), fmaxf(sc[1][cc][2], sc[1][cc][3])));
      m = over_rows(m, max_of) * cl[cc];
      if (__any(m > top[cc] + kSlack)) {
        const float was = ref[cc];
        top[cc] = fmaxf(top[cc], m);
        ref[cc] = fmaxf(top[cc], -FLT_MAX);
        const float keep = __builtin_amdgcn_exp2f(was - ref[cc]);
        sum[cc] *= keep;
#pragma unroll
        for (int v = 0; v < VS; ++v)
#pragma unroll
          for (int j = 0; j < NJ; ++j) o[v][j][cc] *= keep;
      }
      float w[8];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * u + e] = __builtin_amdgcn_exp2f(fmaf(sc[u][cc][e], cl[cc], -ref[cc]));
      sum[cc] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
#pragma unroll
      for (int x = 0; x < 4; ++x) pw[cc][x] = F16::pack2(w[2 * x], w[2 * x + 1]);
    }

    // O^T.
#pragma unroll
    for (int v = 0; v < VS; ++v) {
      uint32_t s0[4], s1[4], bb[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        uint32_t c0 = cur.vsb[x >> 1][v][2 * (x & 1)], c1 = cur.vsb[x >> 1][v][2 * (x & 1) + 1];
        if (careful) {  // constants that are not finite: zeros here, NaN below
          const bool f0 = finite(TT::lo(c0)) && finite(TT::hi(c0)), f1 = finite(TT::lo(c1)) && finite(TT::hi(c1));
          cur.vsb[x >> 1][v][2 * (x & 1)] = (f0 ? 0u : 0x3c00u) | (f1 ? 0u : 0x3c000000u);  // flags, as operands
          c0 = f0 ? c0 : 0u;
          c1 = f1 ? c1 : 0u;
        }
        s0[x] = F16::pack2(scaled(TT::lo(c0), 24 - ev), scaled(TT::lo(c1), 24 - ev));
        bb[x] = F16::pack2(scaled(TT::hi(c0), -ev), scaled(TT::hi(c1), -ev));
        s1[x] = sixteenth(s0[x]);
      }
      const uint32_t lane_sel = D == 64 ? (uint32_t)(i >> 3) * 0x00020002u : 0u;
#pragma unroll
      for (int y = 0; y < NJ / 2; ++y) {
        const uint32_t sel = (0x0c040c00u + (uint32_t)y * 0x00010001u) + lane_sel;
        u32x4 lo, hi;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const u32x4& q4 = cur.vq[x >> 1][v];
          const uint32_t b2 = __builtin_amdgcn_perm(q4[2 * (x & 1) + 1], q4[2 * (x & 1)], sel);
          lo[x] = pk_fma(b2 & 0x000f000fu, s0[x], bb[x]);
          hi[x] = pk_fma(b2 & 0x00f000f0u, s1[x], bb[x]);
        }
#pragma unroll
        for (int cc = 0; cc < NC; ++cc) {
          o[v][2 * y][cc] = Mfma16<F16>::run(lo, pw[cc], o[v][2 * y][cc]);
          o[v][2 * y + 1][cc] = Mfma16<F16>::run(hi, pw[cc], o[v][2 * y + 1][cc]);
        }
      }
      if (careful) {  // rows that see such a value: not a number in its group's dimensions
        const u32x4 flags{cur.vsb[0][v][0], cur.vsb[0][v][2], cur.vsb[1][v][0], cur.vsb[1][v][2]};
#pragma unroll
        for (int cc = 0; cc < NC; ++cc) {
          const f32x4 n = Mfma16<F16>::run(flags, seen[cc], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[v][j][cc][x] = n[x] > 0.f ? NAN : o[v][j][cc][x];
        }
      }
    }
    cur = nxt;
  }

  // The waves' results: each one's rows relative to its own maximum.
  constexpr int LD = D + 4;
  float* wmax = lds + kWaves * rows * LD;  // [wave][rows]
  float* wsum = wmax + kWaves * rows;
#pragma unroll
  for (int cc = 0; cc < NC; ++cc) {
    const int r = 16 * cc + i;
    const float total = over_rows(sum[cc], sum_of);
    if (r < rows) {
      float* dst = lds + (wave * rows + r) * LD;
#pragma unroll
      for (int v = 0; v < VS; ++v)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int w = 4 * h + x;  // of 16: word, or word and half of its dimensions
            const int d = D == 64 ? 8 * (w & 7) + 4 * (w >> 3) + j : 8 * (16 * v + w) + j;
            dst[d] = scaled(o[v][j][cc][x], ev);
          }
      if (h == 0) {
        wmax[wave * rows + r] = ref[cc];
        wsum[wave * rows + r] = total;
      }
    }
  }
  __syncthreads();
  const size_t slab = (size_t)p.rows_max * (D + 2);
  float* park = p.partial + ((size_t)pair * p.parts + part) * slab;
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
      const float inv = total == 0.f ? 0.f : 1.f / total;
      const int qi = r / group, hh = head * group + r - qi * group;
      uint16_t* out = static_cast<uint16_t*>(a.out) + (size_t)(q.rows0 + qi) * a.out_token_stride +
                      (size_t)hh * a.out_head_stride + d;
      *reinterpret_cast<u32x2*>(out) = u32x2{TT::pack2(acc[0] * inv, acc[1] * inv), TT::pack2(acc[2] * inv, acc[3] * inv)};
    } else {
      float* dst = park + r * (D + 2);
#pragma unroll
      for (int x = 0; x < 4; ++x) __hip_atomic_store(dst + d + x, acc[x], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (d == 0) {
        __hip_atomic_store(dst + D, m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(dst + D + 1, total, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
  if (parts == 1) return;

  // The last part to arrive joins them, in part order.
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (tid == 0) flag = __hip_atomic_fetch_add(&p.counters[pair], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (flag != (unsigned int)(parts - 1)) return;
  const float* all = p.partial + (size_t)pair * p.parts * slab;
  for (int e = tid; e < rows * D; e += kWaves * 64) {
    const int r = e / D, d = e % D;
    float m = -FLT_MAX;
    for (int k = 0; k < parts; ++k)
      m = fmaxf(m, __hip_atomic_load(all + k * slab + r * (D + 2) + D, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    float acc = 0.f, total = 0.f;
    for (int k = 0; k < parts; ++k) {
      const float* src = all + k * slab + r * (D + 2);
      const float w = __builtin_amdgcn_exp2f(
          __hip_atomic_load(src + D, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) - m);
      total += __hip_atomic_load(src + D + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) * w;
      acc += __hip_atomic_load(src + d, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) * w;
    }
    const int qi = r / group, hh = head * group + r - qi * group;
    static_cast<uint16_t*>(a.out)[(size_t)(q.rows0 + qi) * a.out_token_stride + (size_t)hh * a.out_head_stride + d] =
        TT::from_f32(total == 0.f ? 0.f : acc / total);
  }
  if (tid == 0) __hip_atomic_store(&p.counters[pair], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <typename TT, int D, int NC>
hipError_t launch(hipStream_t s, const DecodeArgs& p) {
  const size_t lds = (size_t)kWaves * p.rows_max * (D + 4 + 2) * sizeof(float);
  auto kernel = kv_decode_kernel<TT, D, NC>;
  if (lds > 60 * 1024) {
    static const hipError_t raised = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                         hipFuncAttributeMaxDynamicSharedMemorySize, 140 * 1024);
    if (raised != hipSuccess) return raised;
  }
  const dim3 grid((uint32_t)(p.a.n_seqs * p.c.n_kv_heads * p.parts));
  hipLaunchKernelGGL(kernel, grid, dim3(kWaves * 64), lds, s, p);
  return hipGetLastError();
}

template <typename TT, int NC>
hipError_t launch_d(hipStream_t s, const DecodeArgs& p) {
  switch (p.c.head_dim) {
    case 64: return launch<TT, 64, NC>(s, p);
    case 128: return launch<TT, 128, NC>(s, p);
    case 256: return launch<TT, 256, NC>(s, p);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_kv_decode(const ExecCtx& ex, const cpq_kv_cache& c, const cpq_kv_attention_args& a, int rows_max,
                            bool report, unsigned int* bad) {
  DecodeArgs p{};
  p.c = c;
  p.a = a;
  p.bad = bad;
  p.rows_max = rows_max;
  p.report = report;
  const size_t pairs = a.n_seqs * c.n_kv_heads;
  // A part is at least one tile per wave; more parts than about 4096
  // workgroups in all bring nothing but their joining.
  const size_t tiles = (std::min<size_t>(a.max_kv, a.max_blocks * c.block_size) + kTile - 1) / kTile;
  size_t parts = std::max<size_t>(std::min((tiles + kWaves - 1) / kWaves, std::max<size_t>(4096 / pairs, 1)), 1);
  const size_t slab = pairs * (size_t)p.rows_max * (c.head_dim + 2) * sizeof(float);
  const size_t room = ex.scratch_bytes > kWideCounterBytes ? ex.scratch_bytes - kWideCounterBytes : 0;
  if (pairs * sizeof(unsigned int) > kWideCounterBytes) parts = 1;
  parts = std::max<size_t>(std::min(parts, room / slab), 1);
  p.parts = (int)parts;
  p.part_tiles = kWaves;
  p.counters = static_cast<unsigned int*>(ex.scratch);
  p.partial = reinterpret_cast<float*>(static_cast<char*>(ex.scratch) + kWideCounterBytes);
  const bool bf16 = c.dtype == CPQ_DTYPE_BF16;
  if (p.rows_max <= 16) return bf16 ? launch_d<BF16, 1>(ex.stream, p) : launch_d<F16, 1>(ex.stream, p);
  return bf16 ? launch_d<BF16, 2>(ex.stream, p) : launch_d<F16, 2>(ex.stream, p);
}

}  // namespace cpq
