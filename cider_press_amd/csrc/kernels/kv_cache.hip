// The 4-bit key/value cache around its attention: blocks back to the free
// list, a step's block table and slots, the quantizing append, the
// dequantizing gather.  Layouts and semantics: cpq.h (cpq_kv_cache and after).
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "kv_common.hpp"

namespace cpq {
namespace {

using namespace dev;

constexpr int kPlanThreads = 1024;
// Heads to a thread of the gather where that leaves enough workgroups (with one head
// instead: 12000 rows of 8 heads of 128, 3000 workgroups of four heads, 13.8 us for
// 10.1; 2000 workgroups 10.5 for 9.3; up to 1500 no difference, the launch's time).
constexpr uint32_t kHeads = 4, kEnough = 1024;

// ceil(n / block) bounded by a table row's blocks.
__device__ __forceinline__ uint32_t blocks_of(uint64_t n, int bs_shift, uint32_t max_blocks) {
  const uint64_t b = (n + ((1u << bs_shift) - 1)) >> bs_shift;
  return b < max_blocks ? (uint32_t)b : max_blocks;
}

// Exclusive sum over the workgroup's threads, saturating at `top` (< 2^31, no
// addend above it: min(a + b, top) is associative over these and cannot wrap),
// on top of *carry, which becomes the sum of all.
__device__ __forceinline__ uint32_t scan(uint32_t v, uint32_t top, uint32_t* carry, uint32_t* waves) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t sum = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(sum, d, 64);
    if (lane >= d) sum = min(sum + o, top);
  }
  if (lane == 63) waves[wave] = sum;
  __syncthreads();
  uint32_t before = *carry, all = *carry;
#pragma unroll
  for (int i = 0; i < kPlanThreads / 64; ++i) {
    const uint32_t w = waves[i];
    if (i < wave) before = min(before + w, top);
    all = min(all + w, top);
  }
  __syncthreads();
  *carry = all;
  const uint32_t left = __shfl_up(sum, 1, 64);
  return lane ? min(before + left, top) : before;
}

// Every workgroup sums the released blocks of all sequences (a few KB from the
// L2) and one wave copies each finished sequence's row.
// Launch and round trips: 64 requests 2.8 us, 700 requests 3.9 us.
__global__ __launch_bounds__(kPlanThreads) void kv_release_kernel(
    const uint32_t* __restrict__ finished, const uint32_t* __restrict__ lens, const uint32_t* __restrict__ table,
    uint32_t n_seqs, uint32_t max_blocks, int bs_shift, uint32_t* __restrict__ free_list, uint32_t free_cap,
    const uint32_t* __restrict__ free_count, uint32_t* __restrict__ lens_out, uint32_t* __restrict__ free_count_out,
    unsigned int* bad) {
  __shared__ uint32_t waves[kPlanThreads / 64];
  __shared__ uint32_t first[kPlanThreads];
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  uint32_t carry = min(*free_count, free_cap);
  for (uint32_t base = 0; base < n_seqs; base += kPlanThreads) {
    const uint32_t s = base + tid;
    uint32_t n = 0;
    if (s < n_seqs) {
      const bool end = finished[s] != 0;
      const uint32_t len = lens[s];
      if (end) n = blocks_of(len, bs_shift, max_blocks);
      if (blockIdx.x == 0) lens_out[s] = end ? 0 : len;
    }
    first[tid] = scan(n, 0x7fffffffu, &carry, waves);
    __syncthreads();
    const uint32_t stop = min(n_seqs - base, (uint32_t)kPlanThreads);
    for (uint32_t i = blockIdx.x * (kPlanThreads / 64) + (tid >> 6); i < stop;
         i += gridDim.x * (kPlanThreads / 64)) {
      const uint32_t at = first[i], end = i + 1 < (uint32_t)kPlanThreads ? first[i + 1] : carry;
      for (uint32_t j = lane; at + j < min(end, free_cap); j += 64)
        free_list[at + j] = table[(size_t)(base + i) * max_blocks + j];
    }
    __syncthreads();
  }
  if (blockIdx.x == 0 && tid == 0) {
    *free_count_out = min(carry, free_cap);
    if (carry > free_cap) atomicAdd(bad, carry - free_cap);
  }
}

// One thread per slot of the step.  Every workgroup sums the new tokens and the
// new blocks of all sequences (8 bytes a sequence) into LDS: starts[s] the
// first new token of sequence s, first[s] the free block its first new one
// takes, counted from the top.  A thread then finds its token's sequence by
// bisection.  The token that opens a block enters it in the table.
// Launch and round trips: 64 requests of one token 4.4 us, 700 requests with 65536
// slots 6.6 us.
__global__ __launch_bounds__(kPlanThreads) void kv_plan_kernel(
    const uint32_t* __restrict__ lens, const uint32_t* __restrict__ new_lens, uint32_t* table, uint32_t n_seqs,
    uint32_t max_blocks, int bs_shift, const uint32_t* __restrict__ free_list, uint32_t free_cap,
    const uint32_t* __restrict__ free_count, uint32_t* __restrict__ starts_out, uint32_t* __restrict__ kv_lens,
    uint32_t* __restrict__ slots, uint32_t* __restrict__ positions, uint32_t cap,
    uint32_t* __restrict__ free_count_out, unsigned long long* bad) {
  extern __shared__ uint32_t plan_lds[];
  uint32_t* starts = plan_lds;            // [n_seqs + 1]
  uint32_t* first = plan_lds + n_seqs + 1;  // [n_seqs]
  __shared__ uint32_t waves[kPlanThreads / 64];
  const uint32_t tid = threadIdx.x, bs = 1u << bs_shift;
  const uint32_t n_free = min(*free_count, free_cap);
  uint32_t tokens = 0, blocks = 0;
  for (uint32_t base = 0; base < n_seqs; base += kPlanThreads) {
    const uint32_t s = base + tid;
    const uint32_t len = s < n_seqs ? lens[s] : 0;
    const uint32_t want = s < n_seqs ? new_lens[s] : 0;
    const uint32_t in = min(want, cap);
    const uint32_t at = scan(in, cap, &tokens, waves);
    const uint32_t n = min(at + in, cap) - at;  // new tokens that the step holds
    const uint32_t have = blocks_of(len, bs_shift, max_blocks);
    const uint32_t need = blocks_of((uint64_t)len + n, bs_shift, max_blocks) - have;
    const uint32_t top = scan(need, 0x7fffffffu, &blocks, waves);
    if (s < n_seqs) {
      starts[s] = at;
      first[s] = top;
      if (base / kPlanThreads % gridDim.x == blockIdx.x) {
        starts_out[s] = at;
        const uint32_t got = have + (top < n_free ? min(need, n_free - top) : 0u);
        const uint64_t room = (uint64_t)got << bs_shift, all = (uint64_t)len + n;
        kv_lens[s] = (uint32_t)(all < room ? all : room);
        if (want > n) atomicAdd(bad, (unsigned long long)(want - n));
      }
    }
  }
  if (tid == 0) {
    starts[n_seqs] = tokens;
    if (blockIdx.x == 0) {
      starts_out[n_seqs] = tokens;
      *free_count_out = blocks < n_free ? n_free - blocks : 0;
    }
  }
  __syncthreads();
  uint32_t lost = 0;
  for (uint32_t t = blockIdx.x * kPlanThreads + tid; t < cap; t += gridDim.x * kPlanThreads) {
    uint32_t slot = CPQ_KV_NO_SLOT, pos = 0;
    if (t < tokens) {
      uint32_t lo = 0, hi = n_seqs;  // starts[lo] <= t < starts[hi]
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (starts[mid] <= t) lo = mid;
        else hi = mid;
      }
      const uint32_t len = lens[lo];
      const uint64_t p = (uint64_t)len + (t - starts[lo]);
      const uint64_t j = p >> bs_shift;
      uint32_t block = CPQ_KV_NO_SLOT;
      if (j < max_blocks) {
        uint32_t* entry = table + (size_t)lo * max_blocks + j;
        const uint32_t have = blocks_of(len, bs_shift, max_blocks);
        if (j < have) {
          block = *entry;
        } else {
          const uint32_t i = first[lo] + ((uint32_t)j - have);
          if (i < n_free) {
            block = free_list[n_free - 1 - i];
            if ((p & (bs - 1)) == 0) *entry = block;
          }
        }
      }
      pos = (uint32_t)p;
      if (block != CPQ_KV_NO_SLOT) slot = (block << bs_shift) + ((uint32_t)p & (bs - 1));
      lost += slot == CPQ_KV_NO_SLOT;
    }
    slots[t] = slot;
    positions[t] = pos;
  }
  if (lost) atomicAdd(bad, (unsigned long long)lost);
}

// The largest exponent's bits, above which a pattern is an Inf or NaN.
template <typename TT>
constexpr uint32_t kExpBits = Sig16<TT>::bf16 ? 0x7f80u : 0x7c00u;

// Lowest (or highest) of 4, 8 or 16 adjacent lanes by DPP: lane pairs and
// quads exchanged, then halves of 8 and of 16 mirrored (either half is uniform
// by then).  All lanes of a group are active together.
template <bool MAX>
__device__ __forceinline__ float group_extreme(float v, int lanes) {
  auto step = [&](auto ctrl) {
    const float o = __uint_as_float(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), decltype(ctrl)::value,
                                                                0xf, 0xf, false));
    v = MAX ? fmaxf(v, o) : fminf(v, o);
  };
  step(std::integral_constant<int, 0xB1>{});   // quad_perm [1, 0, 3, 2]
  step(std::integral_constant<int, 0x4E>{});   // quad_perm [2, 3, 0, 1]
  if (lanes > 4) step(std::integral_constant<int, 0x141>{});  // row_half_mirror
  if (lanes > 8) step(std::integral_constant<int, 0x140>{});  // row_mirror
  return v;
}

// d / s correctly rounded, as IEEE division gives it, for d >= 0 and an s of at
// most 11 significant bits, r within a unit of 1 / s: one step of the remainder,
// which is exact in an fma.  It leaves 2^-45 of the quotient, and no quotient of 24
// bits by 11 is nearer than 2^-36 to a value halfway between two floats (nor on
// one).  In `plain` range, where no remainder falls below the normal numbers.  A
// quarter of a division's instructions, which bound the append.
__device__ __forceinline__ float quotient(float d, float s, float r) {
  const float q = d * r;
  return fmaf(fmaf(-q, s, d), r, q);
}
__device__ __forceinline__ bool plain(float v) { return v >= 0x1p-100f && v <= 0x1p100f; }

// Of three, where none is a NaN that counts (the builtins quiet each first).
__device__ __forceinline__ float min3(float a, float b, float c) {
  float o;
  asm("v_min3_f32 %0, %1, %2, %3" : "=v"(o) : "v"(a), "v"(b), "v"(c));
  return o;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float o;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(o) : "v"(a), "v"(b), "v"(c));
  return o;
}

// Eight values of T, word wi of a token's row, quantized into their place in the cache.
// The `lanes` words of a group are adjacent lanes, all of them here.
template <typename TT>
__device__ __forceinline__ void append_word(const cpq_kv_cache& c, u32x4 raw, uint32_t block, uint32_t off,
                                            uint32_t head, bool values, uint32_t wi, int w_shift, int lanes) {
  const uint32_t bs = c.block_size;
  float x[8];
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = TT::lo(raw[i]);
    x[2 * i + 1] = TT::hi(raw[i]);
    most = sizes(most, raw[i]);
  }
  const bool finite = (most & 0xffff) < kExpBits<TT> && most >> 16 < kExpBits<TT>;
  float lo = min3(min3(min3(x[0], x[1], x[2]), x[3], x[4]), min3(x[5], x[6], x[7]), x[0]);
  float hi = max3(max3(max3(x[0], x[1], x[2]), x[3], x[4]), max3(x[5], x[6], x[7]), x[0]);
  lo = group_extreme<false>(finite ? lo : 0.f, lanes);
  hi = group_extreme<true>(finite ? hi : INFINITY, lanes);  // not finite anywhere: no finite range
  const float span = hi - lo;
  const bool ok = span <= FLT_MAX;
  // (Opaque: an fma and a conversion become one instruction of one rounding, where
  // the definition rounds to float first.)
  const float step = !Sig16<TT>::bf16 || plain(span) ? quotient(span, 15.f, 1.f / 15.f) : span / 15.f;
  const uint16_t s = ok ? TT::from_f32(__uint_as_float(opaque(__float_as_uint(step)))) : 0;
  const uint16_t b = ok ? TT::from_f32(lo) : (uint16_t)(kExpBits<TT> | kExpBits<TT> >> 1);  // NaN
  const float sf = TT::to_f32(s);
  uint32_t word = 0;
  if (ok && sf != 0.f) {  // the quotient correctly rounded: ties as in the definition
    float q[8];
    if (!Sig16<TT>::bf16 || plain(sf)) {
      const float r = __builtin_amdgcn_rcpf(sf);
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = quotient(x[i] - lo, sf, r);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = (x[i] - lo) / sf;
    }
    float half[2] = {0.f, 0.f};  // four values each, exact
#pragma unroll
    for (int i = 7; i >= 0; --i) half[i >> 2] = fmaf(half[i >> 2], 16.f, rintf(fminf(q[i], 15.f)));
    word = (uint32_t)half[0] | (uint32_t)half[1] << 16;
  }
  const uint32_t w = 1u << w_shift, g = w / lanes, gi = wi / lanes;
  const size_t row = ((size_t)block * c.n_kv_heads + head) * bs;
  const uint32_t sb = s | (uint32_t)b << 16;
  if (values) {
    const size_t quad = row + (off & ~3u);
    c.v_q[quad * w + wi * 4 + (off & 3)] = word;
    if (wi % lanes == 0) c.v_sb[quad * g + gi * 4 + (off & 3)] = sb;
  } else {
    c.k_q[(row + off) * w + wi] = word;
    if (wi % lanes == 0) c.k_sb[(row + off) * g + gi] = sb;
  }
}

// A workgroup takes consecutive tokens of one head, keys or values: thread =
// one word (8 values) of one token, so a group is 4, 8 or 16 adjacent lanes
// and the words of four tokens in adjacent slots, which the value layout
// interleaves, come from one wave (head_dim 128).  Bound by its instructions, 183 a
// wave of 512 values: 8191 tokens of 8 heads of 128 in 14.5 us (3.0 TB/s; with
// IEEE divisions 17.4).  Four heads to a thread, as in the gather: no faster.
template <typename TT>
__global__ __launch_bounds__(256) void kv_append_kernel(cpq_kv_cache c, const uint16_t* __restrict__ k,
                                                        size_t k_token, size_t k_head,
                                                        const uint16_t* __restrict__ v, size_t v_token,
                                                        size_t v_head, const uint32_t* __restrict__ slots,
                                                        uint32_t n_tokens, int w_shift, int lanes, unsigned int* bad) {
  const uint32_t wi = threadIdx.x & ((1u << w_shift) - 1), t = blockIdx.x * (256u >> w_shift) + (threadIdx.x >> w_shift);
  const uint32_t head = blockIdx.y;
  const bool values = blockIdx.z;
  if (t >= n_tokens) return;
  const uint32_t slot = slots[t];
  const uint32_t bs = c.block_size, bs_shift = 31 - __builtin_clz(bs);
  const uint32_t block = slot >> bs_shift, off = slot & (bs - 1);
  if (block >= c.n_blocks) {
    if (slot != CPQ_KV_NO_SLOT && wi == 0 && head == 0 && !values) atomicAdd(bad, 1u);
    return;
  }
  const uint16_t* src = values ? v + t * v_token + head * v_head : k + t * k_token + head * k_head;
  const u32x4 raw = *reinterpret_cast<const u32x4*>(src + wi * 8);
  append_word<TT>(c, raw, block, off, head, values, wi, w_shift, lanes);
}

// Cosine and sine of an angle, off by 2^-52.  The angle less the nearest multiple of a
// quarter turn (in two parts, pi / 2 = kHigh + kLow + 2^-109: up to 2^32 quarters nothing else
// is lost), then Taylor's series about 0, whose next terms are below 2^-54 at an eighth of
// a turn.  The library's takes what is larger or not finite.
__device__ __forceinline__ void cos_sin(double angle, double& c, double& s) {
  constexpr double kQuarters = 0x1.45f306dc9c883p-1;  // 2 / pi
  constexpr double kWhole = 0x1.8p52;
  constexpr double kHigh = 0x1.921fb54442d18p+0, kLow = 0x1.1a62633145c07p-54;
  if (!(fabs(angle) < 0x1p32)) {
    sincos(angle, &s, &c);
    return;
  }
  const double whole = fma(angle, kQuarters, kWhole), k = whole - kWhole;  // rounded, its low bits at the end
  const double r = fma(-k, kLow, fma(-k, kHigh, angle)), z = r * r;
  double p = -1.0 / 1307674368000.0, q = 1.0 / 20922789888000.0;  // -1 / 15!, 1 / 16!
  p = fma(p, z, 1.0 / 6227020800.0);
  p = fma(p, z, -1.0 / 39916800.0);
  p = fma(p, z, 1.0 / 362880.0);
  p = fma(p, z, -1.0 / 5040.0);
  p = fma(p, z, 1.0 / 120.0);
  p = fma(p, z, -1.0 / 6.0);
  p = fma(p * z, r, r);
  q = fma(q, z, -1.0 / 87178291200.0);
  q = fma(q, z, 1.0 / 479001600.0);
  q = fma(q, z, -1.0 / 3628800.0);
  q = fma(q, z, 1.0 / 40320.0);
  q = fma(q, z, -1.0 / 720.0);
  q = fma(q, z, 1.0 / 24.0);
  q = fma(q, z, -0.5);
  q = fma(q, z, 1.0);
  const uint32_t quarter = (uint32_t)(unsigned long long)__double_as_longlong(whole);
  const double x = quarter & 1 ? p : q, y = quarter & 1 ? q : p;
  c = (quarter + 1) & 2 ? -x : x;
  s = quarter & 2 ? -y : y;
}

// Eight values rotated: pairs within the word, or with those of `other`.
template <typename TT, bool PAIRS, int N>
__device__ __forceinline__ u32x4 turn(u32x4 raw, u32x4 other, const double (&co)[N], const double (&si)[N]) {
  u32x4 out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double x = TT::lo(raw[i]), y = TT::hi(raw[i]);
    if constexpr (PAIRS)
      out[i] = TT::pack2((float)fma(x, co[i], -(y * si[i])), (float)fma(y, co[i], x * si[i]));
    else
      out[i] = TT::pack2((float)fma(x, co[2 * i], (double)TT::lo(other[i]) * si[2 * i]),
                         (float)fma(y, co[2 * i + 1], (double)TT::hi(other[i]) * si[2 * i + 1]));
  }
  return out;
}

// Rotation and append.  A workgroup takes 256 / W consecutive tokens (thread = one word of
// one token, as above) and `rows` of their rows: keys, values, then queries.  The cosines
// and sines of its tokens are made once, in LDS, and kept in registers over the rows; a
// rotated word takes its partner's word besides its own (from the cache: a lane nearby
// loads it too).  In fp64, whose fma runs at fp32's rate here: which of 16 steps a key's
// value falls on is a whole number, so that a rotation in fp32 would store other steps than
// an append of keys that were rotated exactly.
// Bound by HBM, and by its instructions where it is not: 8191 tokens of 32 + 8 + 8 heads of
// 128, 178 MB that no cache holds, 45.7 us, 3.9 TB/s (a copy 4.7); with the library's sine and
// rows addressed one by one 60.  1500 tokens of 16 + 4 + 4 heads of 256 9.3 us.
// Workgroups that many rows are divided over: with twice as many the cosines are made twice
// as often (50 us), half leave CUs idle towards the end (51 us).
constexpr uint32_t kRotaryEnough = 1024;
template <typename TT, bool PAIRS>
__global__ __launch_bounds__(256) void kv_append_rotary_kernel(cpq_kv_cache c, cpq_kv_append_rotary_args a, int w_shift,
                                                               int lanes, uint32_t rows, unsigned int* bad) {
  __shared__ double2 turns[1024];  // [j][token][word]: cosine and sine of its j-th
  constexpr uint32_t kTurns = PAIRS ? 4 : 8;  // of a word
  const uint32_t w = 1u << w_shift, tokens = 256u >> w_shift, t0 = blockIdx.x * tokens;
  const uint32_t wi = threadIdx.x & (w - 1), tl = threadIdx.x >> w_shift, t = t0 + tl;
  const uint32_t n_tokens = (uint32_t)a.n_tokens, kv_heads = c.n_kv_heads;
  const uint32_t all = 2 * kv_heads + (uint32_t)a.n_heads, r0 = blockIdx.y * rows, r1 = min(r0 + rows, all);
  const uint32_t half = a.rotary_dim / 2, words = half / kTurns;  // words of distinct turns
  for (uint32_t e = threadIdx.x; e < half << (8 - w_shift); e += 256) {
    const uint32_t tt = e / half, i = e - tt * half;
    if (t0 + tt >= n_tokens) break;
    double co, si;
    cos_sin((double)a.positions[t0 + tt] * (double)a.frequencies[i], co, si);
    turns[(i % kTurns * tokens + tt) * words + i / kTurns] = double2{co * a.magnitude, si * a.magnitude};
  }
  __syncthreads();
  if (t >= n_tokens) return;
  const uint32_t slot = a.slots[t];
  const uint32_t bs = c.block_size, bs_shift = 31 - __builtin_clz(bs);
  const uint32_t block = slot >> bs_shift, off = slot & (bs - 1);
  if (block >= c.n_blocks) {
    if (slot != CPQ_KV_NO_SLOT && wi == 0 && r0 == 0) atomicAdd(bad, 1u);
    return;
  }
  const bool turned = wi < a.rotary_dim / 8, second = !PAIRS && wi >= words;
  const int partner = !turned || PAIRS ? 0 : second ? -(int)words * 8 : (int)words * 8;  // from the own word
  double co[kTurns], si[kTurns];
  if (turned) {
#pragma unroll
    for (uint32_t j = 0; j < kTurns; ++j) {
      const double2 v = turns[(j * tokens + tl) * words + (second ? wi - words : wi)];
      co[j] = v.x;
      si[j] = PAIRS || second ? v.y : -v.y;
    }
  }
  auto load = [](const uint16_t* p) { return *reinterpret_cast<const u32x4*>(p); };
  uint32_t head = min(r0, kv_heads), end = min(r1, kv_heads);
  const uint16_t* src = static_cast<const uint16_t*>(a.k) + t * a.k_token_stride + head * a.k_head_stride + wi * 8;
  for (; head < end; ++head, src += a.k_head_stride) {
    u32x4 raw = load(src);
    if (turned) raw = turn<TT, PAIRS>(raw, load(src + partner), co, si);
    append_word<TT>(c, raw, block, off, head, false, wi, w_shift, lanes);
  }
  head = max(r0, kv_heads) - kv_heads;
  end = max(min(r1, 2 * kv_heads), kv_heads) - kv_heads;
  src = static_cast<const uint16_t*>(a.v) + t * a.v_token_stride + head * a.v_head_stride + wi * 8;
  for (; head < end; ++head, src += a.v_head_stride)
    append_word<TT>(c, load(src), block, off, head, true, wi, w_shift, lanes);
  // Queries, U rows' loads in flight together (four: no faster).
  constexpr uint32_t U = 2;
  head = max(r0, 2 * kv_heads) - 2 * kv_heads;
  end = max(r1, 2 * kv_heads) - 2 * kv_heads;
  src = static_cast<const uint16_t*>(a.q) + t * a.q_token_stride + head * a.q_head_stride + wi * 8;
  uint16_t* dst = static_cast<uint16_t*>(a.q_out) + t * a.q_out_token_stride + head * a.q_out_head_stride + wi * 8;
  for (; head < end; head += U) {
    u32x4 raw[U], other[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      raw[u] = load(src);
      if (!PAIRS) other[u] = load(src + partner);
      if (head + u + 1 < end) src += a.q_head_stride;  // (the last one's again)
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      if (head + u >= end) break;
      if (turned) raw[u] = turn<TT, PAIRS>(raw[u], other[u], co, si);
      *reinterpret_cast<u32x4*>(dst) = raw[u];
      dst += a.q_out_head_stride;
    }
  }
}

// The same split, U heads to a thread (their loads in flight together, and what
// neighbouring workgroups write lies together); a word in, 16 bytes out.  Bound by
// HBM: 65536 rows of 8 heads of 128 in 67 us, 5.1 TB/s read and written (99 us with
// one head to a thread, 91 with two, 69 with eight).  Few rows: one head to a
// thread, or the launch fills a part of the chip.
template <typename TT, int U>
__global__ __launch_bounds__(256) void kv_gather_kernel(cpq_kv_cache c, const uint32_t* __restrict__ slots,
                                                        uint32_t n_rows, uint16_t* __restrict__ k_out,
                                                        uint16_t* __restrict__ v_out, int w_shift, int lanes,
                                                        unsigned int* bad) {
  const uint32_t wi = threadIdx.x & ((1u << w_shift) - 1), t = blockIdx.x * (256u >> w_shift) + (threadIdx.x >> w_shift);
  const uint32_t head0 = blockIdx.y * U, heads = c.n_kv_heads;
  const bool values = k_out ? blockIdx.z : true;
  if (t >= n_rows) return;
  const uint32_t slot = slots[t];
  const uint32_t bs = c.block_size, bs_shift = 31 - __builtin_clz(bs);
  const uint32_t block = slot >> bs_shift, off = slot & (bs - 1);
  const uint32_t w = 1u << w_shift, g = w / lanes, gi = wi / lanes;
  uint16_t* out = (values ? v_out : k_out) + (((size_t)t * heads + head0) << (w_shift + 3)) + wi * 8;
  if (block >= c.n_blocks) {
    if (slot != CPQ_KV_NO_SLOT && wi == 0 && head0 == 0 && blockIdx.z == 0) atomicAdd(bad, 1u);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (head0 + u < heads) *reinterpret_cast<u32x4*>(out + ((size_t)u << (w_shift + 3))) = u32x4{0u, 0u, 0u, 0u};
    return;
  }
  uint32_t word[U], sb[U];
  const uint32_t* q = values ? c.v_q + wi * 4 + (off & 3) : c.k_q + wi;
  const uint32_t* p = values ? c.v_sb + gi * 4 + (off & 3) : c.k_sb + gi;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const size_t row = ((size_t)block * heads + min(head0 + u, heads - 1)) * bs + (values ? off & ~3u : off);
    word[u] = q[row * w];
    sb[u] = p[row * g];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float s = TT::lo(sb[u]), b = TT::hi(sb[u]);
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[i] = TT::pack2(fmaf(s, (float)(word[u] >> (8 * i) & 15u), b), fmaf(s, (float)(word[u] >> (8 * i + 4) & 15u), b));
    u32x4* dst = reinterpret_cast<u32x4*>(out + ((size_t)u << (w_shift + 3)));
    if (head0 + u < heads) {
      if (U > 1) __builtin_nontemporal_store(o, dst);  // more than the caches keep
      else *dst = o;
    }
  }
}

int log2_of(uint32_t v) { return 31 - __builtin_clz(v); }

}  // namespace

hipError_t launch_kv_release(hipStream_t s, const uint32_t* finished, const uint32_t* lens, const uint32_t* table,
                             uint32_t n_seqs, uint32_t max_blocks, uint32_t block_size, uint32_t* free_list,
                             uint32_t free_cap, const uint32_t* free_count, uint32_t* lens_out,
                             uint32_t* free_count_out, unsigned int* bad) {
  const uint32_t waves = kPlanThreads / 64;
  const uint32_t grid = std::min(std::max((std::min(n_seqs, (uint32_t)kPlanThreads) + waves - 1) / waves, 1u), 64u);
  hipLaunchKernelGGL(kv_release_kernel, dim3(grid), dim3(kPlanThreads), 0, s, finished, lens, table, n_seqs,
                     max_blocks, log2_of(block_size), free_list, free_cap, free_count, lens_out, free_count_out, bad);
  return hipGetLastError();
}

hipError_t launch_kv_plan(hipStream_t s, const uint32_t* lens, const uint32_t* new_lens, uint32_t* table,
                          uint32_t n_seqs, uint32_t max_blocks, uint32_t block_size, const uint32_t* free_list,
                          uint32_t free_cap, const uint32_t* free_count, uint32_t* starts, uint32_t* kv_lens,
                          uint32_t* slots, uint32_t* positions, uint32_t cap, uint32_t* free_count_out,
                          unsigned long long* bad) {
  const uint32_t grid = std::min(std::max((cap + kPlanThreads - 1) / kPlanThreads, 1u), 256u);
  const size_t lds = (2 * (size_t)n_seqs + 1) * 4;  // at most 64 KiB + 4
  if (lds > 64 * 1024 - 1024) {
    static const hipError_t raised = hipFuncSetAttribute(reinterpret_cast<const void*>(kv_plan_kernel),
                                                         hipFuncAttributeMaxDynamicSharedMemorySize, 80 * 1024);
    if (raised != hipSuccess) return raised;
  }
  hipLaunchKernelGGL(kv_plan_kernel, dim3(grid), dim3(kPlanThreads), lds, s, lens, new_lens, table, n_seqs, max_blocks,
                     log2_of(block_size), free_list, free_cap, free_count, starts, kv_lens, slots, positions, cap,
                     free_count_out, bad);
  return hipGetLastError();
}

hipError_t launch_kv_append(hipStream_t s, const cpq_kv_cache& c, const void* k, size_t k_token, size_t k_head,
                            const void* v, size_t v_token, size_t v_head, const uint32_t* slots, uint32_t n_tokens,
                            unsigned int* bad) {
  const int w_shift = log2_of(c.head_dim / 8), lanes = (int)c.group_size / 8;
  const dim3 grid((n_tokens + (256u >> w_shift) - 1) / (256u >> w_shift), c.n_kv_heads, 2);
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, c, static_cast<const uint16_t*>(k), k_token, k_head,
                       static_cast<const uint16_t*>(v), v_token, v_head, slots, n_tokens, w_shift, lanes, bad);
    return hipGetLastError();
  };
  return c.dtype == CPQ_DTYPE_BF16 ? run(kv_append_kernel<BF16>) : run(kv_append_kernel<F16>);
}

hipError_t launch_kv_append_rotary(hipStream_t s, const cpq_kv_cache& c, const cpq_kv_append_rotary_args& a,
                                   unsigned int* bad) {
  const int w_shift = log2_of(c.head_dim / 8), lanes = (int)c.group_size / 8;
  const uint32_t per = 256u >> w_shift, blocks = ((uint32_t)a.n_tokens + per - 1) / per;
  const uint32_t all = 2 * c.n_kv_heads + (uint32_t)a.n_heads;
  // (At most 65535 workgroups along the rows.)
  const uint32_t rows = (uint32_t)std::max<size_t>((size_t)all * blocks / kRotaryEnough, (all + 65534) / 65535);
  const dim3 grid(blocks, (all + rows - 1) / rows);
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, c, a, w_shift, lanes, rows, bad);
    return hipGetLastError();
  };
  if (a.interleaved)
    return c.dtype == CPQ_DTYPE_BF16 ? run(kv_append_rotary_kernel<BF16, true>) : run(kv_append_rotary_kernel<F16, true>);
  return c.dtype == CPQ_DTYPE_BF16 ? run(kv_append_rotary_kernel<BF16, false>) : run(kv_append_rotary_kernel<F16, false>);
}

hipError_t launch_kv_gather(hipStream_t s, const cpq_kv_cache& c, const uint32_t* slots, uint32_t n_rows, void* k_out,
                            void* v_out, unsigned int* bad) {
  const int w_shift = log2_of(c.head_dim / 8), lanes = (int)c.group_size / 8;
  const uint32_t blocks = (n_rows + (256u >> w_shift) - 1) / (256u >> w_shift), sides = k_out && v_out ? 2 : 1;
  const bool wide = (size_t)blocks * ((c.n_kv_heads + kHeads - 1) / kHeads) * sides >= kEnough;
  const dim3 grid(blocks, wide ? (c.n_kv_heads + kHeads - 1) / kHeads : c.n_kv_heads, sides);
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, c, slots, n_rows, static_cast<uint16_t*>(k_out),
                       static_cast<uint16_t*>(v_out), w_shift, lanes, bad);
    return hipGetLastError();
  };
  if (wide) return c.dtype == CPQ_DTYPE_BF16 ? run(kv_gather_kernel<BF16, kHeads>) : run(kv_gather_kernel<F16, kHeads>);
  return c.dtype == CPQ_DTYPE_BF16 ? run(kv_gather_kernel<BF16, 1>) : run(kv_gather_kernel<F16, 1>);
}

}  // namespace cpq
