// Routed-expert plumbing around gather_qmm for gfx950: the router's top-k
// selection, the sort of (token, slot) rows by expert that gather_qmm's
// sorted form consumes, and the weighted combine back to tokens.
//
// Reference: the reference names this feature but has not built it
// (docs/inference/feed-forward.md:98-107, 131-137: router scores, top-k
// experts per token, gather_qmm dispatch, loop-or-fuse).  The kernel it would
// feed is MLX's affine_gather_qmm_rhs (quantized.h:2242-2436), which expects
// rows sorted by expert.  The semantics here are the usual ones for that
// pipeline, stated exactly so they can be tested:
//   route:   p = softmax(logits[t, :]) in fp32; the k largest p (ties: lower
//            expert index first), in descending order; with `normalize`
//            they are divided by their sum.
//   sort:    rows r = t*k + j ordered by expert, stably (equal experts keep
//            row order) -- a stable argsort of the flattened expert ids.
//            lhs[p] = token of the row at sorted position p, rhs[p] = its
//            expert, inv[r] = the sorted position of row r, offsets[e] =
//            first sorted position of expert e (offsets[E] = T*k).
//   combine: out[t, :] = RNE_T(sum_j scores[t*k + j] * y[inv[t*k + j], :]),
//            fp32, j ascending.
// All three are tiny next to the expert matmuls (bytes: T*E logits;
// 16*T*k of indices; (k + 1)*T*N*sizeof(T) for the combine).
#include <algorithm>
#include <type_traits>

#include "../cpq_internal.hpp"
#include "common.hpp"

namespace cpq {
namespace {

using namespace dev;

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 16;
constexpr int kSortRows = 256;  // rows per sort block (four waves of 64)

template <int L>
__device__ __forceinline__ float logit_at(const void* p, size_t i) {
  if constexpr (L == 0) return static_cast<const float*>(p)[i];
  else if constexpr (L == 1) return F16::to_f32(static_cast<const uint16_t*>(p)[i]);
  else return BF16::to_f32(static_cast<const uint16_t*>(p)[i]);
}

// Wave-wide reductions of the device library (DPP row shifts, no LDS).
extern "C" __device__ float __ockl_wfred_max_f32(float);
extern "C" __device__ float __ockl_wfred_add_f32(float);
extern "C" __device__ unsigned long long __ockl_wfred_max_u64(unsigned long long);

// Ranking key of (p, e) for p >= 0: the float bits order like the values, and
// ~e puts the lower expert first on equal p.  0 means "nothing left".
__device__ __forceinline__ unsigned long long rank_key(float p, int e) {
  return ((unsigned long long)__float_as_uint(p) << 32) | (uint32_t)~(uint32_t)e;
}

// One token by one wave.  Lane l holds experts l + 64 i, i < NV (NV = ceil(E/64));
// lane j < top_k returns pick j and its (normalized) score.
template <int L, int NV>
__device__ __forceinline__ void route_token(const void* logits, size_t row, int n_experts, int top_k, int normalize,
                                            int& pick, float& score) {
  const int lane = threadIdx.x & 63;
  float v[NV];
  bool live[NV];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = lane + 64 * i;
    live[i] = e < n_experts;
    v[i] = live[i] ? logit_at<L>(logits, row + e) : -INFINITY;
    m = fmaxf(m, v[i]);
  }
  m = __ockl_wfred_max_f32(m);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    v[i] = live[i] ? expf(v[i] - m) : 0.f;
    sum += v[i];
  }
  const float inv = 1.f / __ockl_wfred_add_f32(sum);
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] *= inv;

  // Lane j keeps pick j (top_k <= 16 < 64 lanes).
  float my_p = 0.f;
  int my_e = 0;
  for (int j = 0; j < top_k; ++j) {
    unsigned long long best = 0ull;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const unsigned long long key = live[i] ? rank_key(v[i], lane + 64 * i) : 0ull;
      best = key > best ? key : best;
    }
    best = __ockl_wfred_max_u64(best);
    const int be = (int)~(uint32_t)best;
    const float bp = __uint_as_float((uint32_t)(best >> 32));
    // The owner retires the winner.
    if ((be & 63) == lane) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i == (be >> 6)) live[i] = false;
    }
    if (lane == j) {
      my_p = bp;
      my_e = be;
    }
  }
  // The picks' sum in pick order (lane 0 .. k-1), the order a serial loop uses.
  float psum = 0.f;
  for (int j = 0; j < top_k; ++j) psum += __shfl(my_p, j, 64);
  pick = my_e;
  score = normalize ? my_p / psum : my_p;
}

// Over the wave by DPP: rows of 16 lanes, then from row to row; uniform.
template <typename F>
__device__ __forceinline__ uint32_t wave_u32(uint32_t v, F f) {
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));  // row_shr 1, 2, 4, 8
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));  // row_bcast 15, 31
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
// The lanes that have the largest of 64-bit keys: of the high words, and of the low words where
// several lanes share that.
__device__ __forceinline__ uint64_t wave_max_key(unsigned long long key) {
  auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  const uint32_t high = wave_u32((uint32_t)(key >> 32), larger);
  const uint64_t who = __ballot((uint32_t)(key >> 32) == high);
  if ((who & (who - 1)) == 0) return who;
  const bool in = who >> (threadIdx.x & 63) & 1;
  const uint32_t low = wave_u32(in ? (uint32_t)key : 0u, larger);
  return __ballot(in && (uint32_t)key == low);
}
__device__ __forceinline__ double lane_f64(double v, int lane) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v);
  return __longlong_as_double((long long)((unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), lane) << 32 |
                                          (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane)));
}

// moe_route_grouped, in fp64: a choice is a whole number, which near scores must not
// change with the order of a sum.  A group has `lanes` neighbouring lanes, each of them
// `per` neighbouring experts, up to NV, so that what lies before is the lower expert.  Bound
// by its instructions, a quarter of them five exponentials, a third the picks: 8191 tokens of
// 256 experts 15.5 us of the 22.7 that the call takes, the chip's vector pipes busy for 84 %.
struct GroupedRouter {
  cpq_moe_router r;
  bool chosen;           // of the groups some are left out
  int size, lanes, per;  // experts of a group (of all where none is left out), its lanes, experts of a lane
  GroupedRouter(const cpq_moe_router& router, int n_experts) : r(router) {
    chosen = r.top_groups < r.n_groups;
    const int groups = chosen ? (int)r.n_groups : 1;
    size = n_experts / groups;
    lanes = 64 / groups;
    per = (size + lanes - 1) / lanes;  // 33 lanes or more have experts: up to 32
  }
  // Orders like the values, NaN below all of them; 0: no choice.
  static __device__ __forceinline__ unsigned long long key_of(double v) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(v);
    return v != v ? 1ull : b >> 63 ? ~b : b | 1ull << 63;
  }
  static __device__ __forceinline__ double value_of(unsigned long long key) {
    return key == 1ull ? NAN : __longlong_as_double((long long)(key >> 63 ? key & ~(1ull << 63) : ~key));
  }
  // 1 / (1 + e^-x) of e = e^-|x|, by a reciprocal in steps: 1 + e is between 1 and 2.
  static __device__ __forceinline__ double logistic(float x, double e) {
    const double y = 1.0 + e;
    double q = __builtin_amdgcn_rcp(y);
    q = fma(fma(-y, q, 1.0), q, q);
    q = fma(fma(-y, q, 1.0), q, q);
    return x < 0.f ? e * q : q;
  }
  // A group's key by its two largest.
  __device__ __forceinline__ unsigned long long group_key(unsigned long long first, unsigned long long second) const {
    return r.group_best > 1 ? key_of(value_of(first) + value_of(second)) : first;
  }
  // The larger two of two pairs, each in order.
  static __device__ __forceinline__ void merge(unsigned long long& first, unsigned long long& second,
                                               unsigned long long a, unsigned long long b) {
    const unsigned long long low = first < a ? first : a, high = first < a ? b : second;
    first = first < a ? a : first;
    second = low > high ? low : high;
  }
  // A lane's keys with the places of their experts.  Up to four are in order (descending,
  // lower places first), so that the next is the first (8191 tokens of 256 experts: 27.4 us,
  // looked for each time 29.4); of more the largest is looked for, ordering them takes longer.
  template <int NV>
  struct Keys {
    static constexpr bool kSorted = NV <= 4;
    unsigned long long key[NV];
    int place[NV];
    unsigned long long head;
    int at;
    __device__ __forceinline__ void order(int i, int j) {
      const bool swap = key[i] < key[j] || (key[i] == key[j] && place[i] > place[j]);
      const unsigned long long k = key[i];
      const int p = place[i];
      key[i] = swap ? key[j] : k;
      place[i] = swap ? place[j] : p;
      key[j] = swap ? k : key[j];
      place[j] = swap ? p : place[j];
    }
    __device__ __forceinline__ void find() {
      if constexpr (kSorted) {
        head = key[0];
        at = place[0];
      } else {
        head = 0ull;
        at = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (key[i] > head) {
            head = key[i];
            at = i;
          }
      }
    }
    // Of keys at their own places.
    __device__ __forceinline__ void start() {
#pragma unroll
      for (int i = 0; i < NV; ++i) place[i] = i;
      if constexpr (NV == 2) order(0, 1);
      if constexpr (NV == 4) {
        order(0, 1);
        order(2, 3);
        order(0, 2);
        order(1, 3);
        order(1, 2);
      }
      find();
    }
    // The lowest expert of the wave's largest key, which is taken out (`base`: a lane's first).
    __device__ __forceinline__ int take(int base) {
      const int owner = __builtin_ctzll(wave_max_key(head));
      const int expert = __builtin_amdgcn_readlane(base + at, owner);
      const bool mine = (int)(threadIdx.x & 63) == owner;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if constexpr (kSorted) {
          key[i] = mine ? i + 1 < NV ? key[(i + 1) % NV] : 0ull : key[i];
          place[i] = mine && i + 1 < NV ? place[(i + 1) % NV] : place[i];
        } else {
          key[i] = mine && at == i ? 0ull : key[i];
        }
      }
      find();
      return expert;
    }
  };
  // Keys of groups that are not kept become 0; this lane is the at-th of `group`.
  template <int NV>
  __device__ __forceinline__ void keep_groups(Keys<NV>& k, int group, int at) const {
    const int lane = threadIdx.x & 63;
    unsigned long long first = k.key[0], second = NV > 1 ? k.key[NV > 1] : 0ull;
    if constexpr (!Keys<NV>::kSorted) {
      first = second = 0ull;
#pragma unroll
      for (int i = 0; i < NV; ++i) merge(first, second, k.key[i], 0ull);
    }
    for (int d = 1; d < lanes; d <<= 1) {  // over lanes at .. at + 2 d - 1 of the group
      const unsigned long long a = __shfl(first, (lane + d) & 63, 64), b = __shfl(second, (lane + d) & 63, 64);
      if (at + d < lanes) merge(first, second, a, b);
    }
    const unsigned long long of_group = group_key(first, second);  // in its first lane
    const unsigned long long mine = __shfl(of_group, (lane - at) & 63, 64);
    int before = 0;
    for (int g = 0; g < (int)r.n_groups; ++g) {
      const unsigned long long other =
          (unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(of_group >> 32), g * lanes) << 32 |
          (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)of_group, g * lanes);
      before += other > mine || (other == mine && g < group);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) k.key[i] = before < (int)r.top_groups ? k.key[i] : 0ull;
    k.find();
  }
  template <int L, int NV>
  __device__ __forceinline__ void route(const void* logits, size_t row, int n_experts, int top_k, int& pick,
                                        float& score) const {
    const int lane = threadIdx.x & 63;
    const int group = lane / lanes, at = lane - group * lanes, first = at * per, base = group * size + first;
    // Experts that a lane has: none past the groups' lanes.
    const int own = (group + 1) * size <= n_experts ? min(size - first, per) : 0;
    float x[NV];
    Keys<NV> k;
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = i < own ? logit_at<L>(logits, row + base + i) : -INFINITY;
    double most = 0.0, part = 1.0;  // of a softmax: its largest logit, 1 / its sum
    if (!r.sigmoid) {
      float m = x[0];
#pragma unroll
      for (int i = 1; i < NV; ++i) m = fmaxf(m, x[i]);
      most = (double)__ockl_wfred_max_f32(m);
    }
    // Four at a time, own or not: in one block they share their exponentials' constants and
    // hide each other's latency (8191 tokens of 256 experts 0.8 us less than one by one, 1500
    // of 160 1.4).
    constexpr int F = NV < 4 ? NV : 4;
    double v[NV], sum = 0.0;
#pragma unroll
    for (int i = 0; i < NV; i += F) {
      if (i >= F && i >= per) {  // (for the whole wave)
#pragma unroll
        for (int u = 0; u < F; ++u) v[i + u] = 0.0;
        continue;
      }
#pragma unroll
      for (int u = 0; u < F; ++u) v[i + u] = r.sigmoid ? -fabs((double)x[i + u]) : (double)x[i + u] - most;
#pragma unroll
      for (int u = 0; u < F; ++u) v[i + u] = exp(v[i + u]);
      if (r.sigmoid) {
#pragma unroll
        for (int u = 0; u < F; ++u) v[i + u] = logistic(x[i + u], v[i + u]);
      } else {
#pragma unroll
        for (int u = 0; u < F; ++u) sum += i + u < own ? v[i + u] : 0.0;
      }
    }
    if (!r.sigmoid) {
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
      part = 1.0 / sum;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const double s = v[i] * part;
      k.key[i] = i < own ? key_of(r.bias ? s + (double)r.bias[base + i] : s) : 0ull;
    }
    k.start();
    if (chosen) keep_groups<NV>(k, group, at);
    pick = 0;
    for (int j = 0; j < top_k; ++j) {
      const int e = k.take(base);
      if (lane == j) pick = e;
    }
    // Lane j's pick again, cheaper than every expert's score kept until here.
    const float own_logit = logit_at<L>(logits, row + pick);
    const double e = exp(r.sigmoid ? -fabs((double)own_logit) : (double)own_logit - most);
    double s = lane < top_k ? r.sigmoid ? logistic(own_logit, e) : e * part : 0.0;
    if (r.normalize) {
      double sum = 0.0;
      for (int j = 0; j < top_k; ++j) sum += lane_f64(s, j);
      s = sum == 0.0 ? 0.0 : s / sum;
    }
    score = (float)(s * (double)r.scale);
  }
};

// One wave per token.
template <int L, int NV>
__global__ __launch_bounds__(256) void route_kernel(const void* __restrict__ logits, int tokens, int n_experts,
                                                    int top_k, int normalize, uint32_t* __restrict__ experts,
                                                    float* __restrict__ scores) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= tokens) return;  // whole waves leave together
  int pick;
  float score;
  route_token<L, NV>(logits, (size_t)t * n_experts, n_experts, top_k, normalize, pick, score);
  if (lane < top_k) {
    experts[(size_t)t * top_k + lane] = (uint32_t)pick;
    scores[(size_t)t * top_k + lane] = score;
  }
}

// The grouped router, a token to a wave, with the histogram of the workgroup's tokens, which
// the sort starts from (a launch less: 8191 tokens of 256 experts 26.0 us instead of 27.4).
// (Null `counts`: none is asked for.)
// Small workgroups make more histograms, large ones leave CUs idle: four tokens each while that
// is one for a CU, then eight, then 16 (256 experts, 1000 tokens 13.4 us, 15.5 with 16 each; 1500
// 14.0, 15.6 with 16; 4000, in 16s either way, 16.2).
constexpr int most_tokens(int nv) { return nv > 8 ? 8 : 16; }  // by the registers of a wave
inline int grouped_tokens(int tokens, int nv, int cus) {
  int per = 4;
  while (per < most_tokens(nv) && tokens > cus * per) per *= 2;
  return per;
}
// A histogram's rows of bytes (a token picks an expert once, so counts are at most 16), where the
// sort takes them so: whole groups of 16.
constexpr int byte_row(int n_experts) { return (n_experts + 15) & ~15; }
template <int L, int NV>
__global__ __launch_bounds__(most_tokens(NV) * 64) void route_grouped_kernel(
    const void* __restrict__ logits, int tokens, int n_experts, int top_k, GroupedRouter router,
    uint32_t* __restrict__ experts, float* __restrict__ scores, uint32_t* __restrict__ counts, int bytes) {
  __shared__ uint32_t h[kMaxExperts];
  const int lane = threadIdx.x & 63, t = (int)((blockIdx.x * blockDim.x + threadIdx.x) >> 6);
  const int row = byte_row(n_experts);
  for (int e = threadIdx.x; e < row; e += blockDim.x) h[e] = 0u;
  __syncthreads();
  if (t < tokens) {
    int pick;
    float score;
    router.template route<L, NV>(logits, (size_t)t * n_experts, n_experts, top_k, pick, score);
    if (lane < top_k) {
      experts[(size_t)t * top_k + lane] = (uint32_t)pick;
      scores[(size_t)t * top_k + lane] = score;
      atomicAdd(&h[pick], 1u);
    }
  }
  if (!counts) return;
  __syncthreads();
  if (bytes) {
    for (int i = threadIdx.x; i < row / 4; i += blockDim.x)
      counts[(size_t)blockIdx.x * (row / 4) + i] = h[4 * i] | h[4 * i + 1] << 8 | h[4 * i + 2] << 16 | h[4 * i + 3] << 24;
    return;
  }
  for (int e = threadIdx.x; e < n_experts; e += blockDim.x) counts[(size_t)blockIdx.x * n_experts + e] = h[e];
}

// Rank of a lane among the earlier lanes of its wave with the same value, and
// how many lanes have it (64 lane reads, no LDS round trips).
__device__ __forceinline__ void lane_rank(uint32_t e, uint32_t& rank, uint32_t& same) {
  const int lane = threadIdx.x & 63;
  rank = same = 0;
#pragma unroll 8
  for (int i = 0; i < 64; ++i) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)e, i);
    const uint32_t eq = (o == e) ? 1u : 0u;
    same += eq;
    rank += (i < lane) ? eq : 0u;
  }
}

// Routing and sort of a few tokens (at most kFusedTokens, so at most 512 rows)
// by one workgroup in one launch: decode steps otherwise spend four launches
// and their gaps on a few hundred bytes.  16 waves route a token each at a
// time into LDS; then wave w ranks rows 64w .. 64w + 63, thread e adds the waves'
// counts of expert e, a scan over the experts gives the starts, and each row's
// position is its expert's start, the earlier waves' counts and its rank.
constexpr int kFusedTokens = 32;
template <int L, int NV>
__global__ __launch_bounds__(1024) void route_sort_kernel(const void* __restrict__ logits, int tokens, int n_experts,
                                                          int top_k, int normalize, uint32_t* __restrict__ experts,
                                                          float* __restrict__ scores, uint32_t* __restrict__ lhs,
                                                          uint32_t* __restrict__ rhs, uint32_t* __restrict__ inv,
                                                          uint32_t* __restrict__ offsets) {
  constexpr int ROWS = kFusedTokens * kMaxTopK, RW = ROWS / 64;
  __shared__ uint32_t pick_of[ROWS];
  __shared__ uint32_t start[kMaxExperts];
  __shared__ uint32_t wave_total[16];
  __shared__ __attribute__((aligned(4))) uint8_t cnt[RW][kMaxExperts];  // cleared by words
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int rows = tokens * top_k;
  for (int i = tid; i < RW * kMaxExperts / 4; i += 1024) reinterpret_cast<uint32_t*>(&cnt[0][0])[i] = 0u;
  for (int t = wave; t < tokens; t += 16) {
    int pick;
    float score;
    route_token<L, NV>(logits, (size_t)t * n_experts, n_experts, top_k, normalize, pick, score);
    if (lane < top_k) {
      const int r = t * top_k + lane;
      pick_of[r] = (uint32_t)pick;
      experts[r] = (uint32_t)pick;
      scores[r] = score;
    }
  }
  __syncthreads();  // picks in LDS, cnt cleared
  const bool live = tid < rows;
  const uint32_t e = live ? pick_of[tid] : 0xffffffffu;
  uint32_t rank = 0, same = 0;
  if (wave * 64 < rows) {
    lane_rank(e, rank, same);
    if (live && rank + 1 == same) cnt[wave][e] = (uint8_t)same;
  }
  __syncthreads();
  // Exclusive scan of the experts' totals: inside a wave, then over the waves.
  uint32_t total = 0;
#pragma unroll
  for (int w = 0; w < RW; ++w) total += cnt[w][tid];
  uint32_t upto = total;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(upto, d, 64);
    upto += lane >= d ? o : 0u;
  }
  if (lane == 63) wave_total[wave] = upto;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < wave; ++w) before += wave_total[w];
  start[tid] = before + upto - total;
  if (tid < n_experts) offsets[tid] = before + upto - total;
  if (tid == 0) offsets[n_experts] = (uint32_t)rows;
  __syncthreads();
  if (live) {
    uint32_t pos = start[e] + rank;
    for (int w = 0; w < wave; ++w) pos += cnt[w][e];
    lhs[pos] = (uint32_t)(tid / top_k);
    rhs[pos] = e;
    inv[tid] = pos;
  }
}

// The same for the grouped router, whose thousand instructions a token are spread over the
// chip: four tokens a workgroup, and the last workgroup to arrive sorts (16 tokens of 256
// experts 9.6 us, by one workgroup of 16 waves 13.6).  Picks go through to the memory side
// and come back from it; `counter` is zero between launches.
template <int L, int NV>
__global__ __launch_bounds__(256) void route_grouped_sort_kernel(const void* __restrict__ logits, int tokens,
                                                                 int n_experts, int top_k, GroupedRouter router,
                                                                 uint32_t* experts, float* __restrict__ scores,
                                                                 uint32_t* __restrict__ lhs, uint32_t* __restrict__ rhs,
                                                                 uint32_t* __restrict__ inv,
                                                                 uint32_t* __restrict__ offsets,
                                                                 unsigned int* counter) {
  constexpr int ROWS = kFusedTokens * kMaxTopK, RW = ROWS / 64, RT = ROWS / 256;
  __shared__ uint32_t start[kMaxExperts];
  __shared__ uint32_t wave_total[4];
  __shared__ unsigned int arrived;
  __shared__ __attribute__((aligned(4))) uint8_t cnt[RW][kMaxExperts];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int rows = tokens * top_k, t = blockIdx.x * 4 + wave;
  for (int i = tid; i < RW * kMaxExperts / 4; i += 256) reinterpret_cast<uint32_t*>(&cnt[0][0])[i] = 0u;
  if (t < tokens) {
    int pick;
    float score;
    router.template route<L, NV>(logits, (size_t)t * n_experts, n_experts, top_k, pick, score);
    if (lane < top_k) {
      __hip_atomic_store(experts + t * top_k + lane, (uint32_t)pick, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      scores[t * top_k + lane] = score;
    }
  }
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();  // the workgroup's picks are there, cnt cleared
  if (gridDim.x > 1) {
    if (tid == 0) arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (arrived != gridDim.x - 1) return;
    if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  // Wave w ranks rows 64 w .. and 64 (w + 4) ..
  uint32_t e[RT], rank[RT];
#pragma unroll
  for (int h = 0; h < RT; ++h) {
    const int r = 256 * h + tid;
    e[h] = r < rows ? __hip_atomic_load(experts + r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0xffffffffu;
  }
#pragma unroll
  for (int h = 0; h < RT; ++h) {
    if (256 * h + 64 * wave >= rows) break;
    uint32_t same;
    lane_rank(e[h], rank[h], same);
    if (256 * h + tid < rows && rank[h] + 1 == same) cnt[4 * h + wave][e[h]] = (uint8_t)same;
  }
  __syncthreads();
  // Thread t sums experts 4 t .. 4 t + 3.
  uint32_t t4[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int w = 0; w < RW; ++w) {
    const uint32_t c = reinterpret_cast<const uint32_t*>(cnt[w])[tid];
#pragma unroll
    for (int i = 0; i < 4; ++i) t4[i] += c >> (8 * i) & 255u;
  }
  const uint32_t sum = t4[0] + t4[1] + t4[2] + t4[3];
  uint32_t upto = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(upto, d, 64);
    upto += lane >= d ? o : 0u;
  }
  if (lane == 63) wave_total[wave] = upto;
  __syncthreads();
  uint32_t before = upto - sum;
  for (int w = 0; w < wave; ++w) before += wave_total[w];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = 4 * tid + i;
    start[at] = before;
    if (at < n_experts) offsets[at] = before;
    before += t4[i];
  }
  if (tid == 255) offsets[n_experts] = (uint32_t)rows;
  __syncthreads();
#pragma unroll
  for (int h = 0; h < RT; ++h) {
    const int r = 256 * h + tid;
    if (r >= rows) break;
    uint32_t pos = start[e[h]] + rank[h];
    for (int w = 0; w < 4 * h + wave; ++w) pos += cnt[w][e[h]];
    lhs[pos] = (uint32_t)(r / top_k);
    rhs[pos] = e[h];
    inv[r] = pos;
  }
}

// Per-block expert histograms: counts[b * E + e].
__global__ __launch_bounds__(64) void sort_count_kernel(const uint32_t* __restrict__ experts, int rows, int n_experts,
                                                        uint32_t* __restrict__ counts) {
  __shared__ uint32_t h[kMaxExperts];
  for (int e = threadIdx.x; e < n_experts; e += 64) h[e] = 0u;
  __syncthreads();
  const int r0 = blockIdx.x * kSortRows;
  for (int r = r0 + threadIdx.x; r < min(rows, r0 + kSortRows); r += 64) atomicAdd(&h[experts[r]], 1u);
  __syncthreads();
  for (int e = threadIdx.x; e < n_experts; e += 64) counts[(size_t)blockIdx.x * n_experts + e] = h[e];
}

// Turns the histograms of kScanExperts experts a workgroup into where each block's rows end
// within their expert (the last block's are the totals).  A thread sums a
// sixteenth of the blocks, 16 neighbouring lanes the experts of one.  (One thread an expert
// over all blocks, by one workgroup: 65528 rows of 256 experts 26 us; so 4.)
constexpr int kScanExperts = 16, kScanSlices = 16;
__global__ __launch_bounds__(kScanExperts * kScanSlices) void sort_scan_kernel(uint32_t* __restrict__ counts, int blocks,
                                                                              int n_experts) {
  __shared__ uint32_t sums[kScanSlices][kScanExperts];
  const int el = threadIdx.x % kScanExperts, slice = threadIdx.x / kScanExperts;
  const int e = blockIdx.x * kScanExperts + el;
  const int per = (blocks + kScanSlices - 1) / kScanSlices, b0 = slice * per, b1 = min(b0 + per, blocks);
  uint32_t sum = 0;
  if (e < n_experts) {
#pragma unroll 16
    for (int b = b0; b < b1; ++b) sum += counts[(size_t)b * n_experts + e];
  }
  sums[slice][el] = sum;
  __syncthreads();
  if (e >= n_experts) return;
  uint32_t end = 0;
#pragma unroll
  for (int i = 0; i < kScanSlices; ++i) end += i < slice ? sums[i][el] : 0u;
  constexpr int U = 16;  // loads in flight, which the stores between them would keep apart
  for (int b = b0; b < b1; b += U) {
    uint32_t c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) c[u] = b + u < b1 ? counts[(size_t)(b + u) * n_experts + e] : 0u;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      end += c[u];
      if (b + u < b1) counts[(size_t)(b + u) * n_experts + e] = end;
    }
  }
}

// Histograms of bytes that a workgroup sums itself: of experts 16 c .. 16 c + 15 a thread of
// column c takes every row of its slice, eight at a time in bytes (8 * 16 < 256), then in pairs
// of 16 bits, which go into LDS.  Pair 2 j + p of a column holds its experts 4 j + p and
// 4 j + p + 2.
struct ByteSums {
  uint32_t of[kMaxExperts / 2];
  __device__ __forceinline__ void clear() {
    for (int i = threadIdx.x; i < kMaxExperts / 2; i += blockDim.x) of[i] = 0u;
  }
  __device__ __forceinline__ uint32_t get(int e, int columns) const {
    const int k = e & 15;
    return of[(k >> 2 << 1 | (k & 1)) * columns + (e >> 4)] >> (k & 2 ? 16 : 0) & 0xffffu;
  }
  __device__ __forceinline__ void add(const uint32_t (&pairs)[8], int column, int columns) {
#pragma unroll
    for (int i = 0; i < 8; ++i) atomicAdd(&of[i * columns + column], pairs[i]);
  }
};
template <int U>  // loads in flight, summed by eight
__device__ __forceinline__ void sum_bytes(const u32x4* __restrict__ counts, int column, int columns, int b0, int b1,
                                          uint32_t (&pairs)[8]) {
  for (int b = b0; b < b1; b += U) {
    u32x4 c[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      c[u] = b + u < b1 ? counts[(size_t)(b + u) * columns + column] : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int h = 0; h < U; h += 8) {
#pragma unroll
      for (int u = 1; u < 8; ++u) c[h] += c[h + u];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        pairs[2 * j] += c[h][j] & 0x00ff00ffu;
        pairs[2 * j + 1] += c[h][j] >> 8 & 0x00ff00ffu;
      }
    }
  }
}
// Up to here (and below 65536 tokens) it does, which saves launches; past it counting and the
// scan read less (of 256 experts, 8 picks: 8191 tokens 22.7 us, 25.5 with the scan; 12000 31.6
// and 36.1; 16000, 250 KB, 38.3 and 39.2; 20480 51.4 and 47.3; 32000 77.1 and 67.4; 2 picks of
// 20480 33.6 and 35.4, 16 picks 71.3 and 57.4).
constexpr size_t kByteSums = 256 * 1024;
inline bool sums_bytes(int tokens, int blocks, int n_experts) {
  return tokens < 65536 && (size_t)blocks * byte_row(n_experts) <= kByteSums;
}

// Four waves per block of up to kSortRows rows, wave w on rows 64w .. 64w+63 of
// the block; the last lane of each (wave, expert) run publishes the run's
// length, and a lane's sorted position is its expert's start (every workgroup sums the
// experts' totals), plus the end of the block before within the expert, plus the counts of
// the earlier waves, plus its rank -- so equal experts keep row order.  SUMS: `ends` are
// histograms of bytes yet, `blocks` in all and `per` of a workgroup's rows.
constexpr int kSumThreads = 512;  // (8191 tokens of 256 experts 22.7 us; 256 threads 23.3, 1024 23.8)
template <bool SUMS>
__global__ __launch_bounds__(SUMS ? kSumThreads : 256) void sort_scatter_kernel(const uint32_t* __restrict__ experts, int rows,
                                                           int block_rows, int blocks, int per, int top_k,
                                                           int n_experts, const uint32_t* __restrict__ ends,
                                                           uint32_t* __restrict__ lhs, uint32_t* __restrict__ rhs,
                                                           uint32_t* __restrict__ inv, uint32_t* __restrict__ offsets) {
  __shared__ uint32_t cnt[4][kMaxExperts];
  __shared__ uint32_t first[kMaxExperts];
  constexpr int THREADS = SUMS ? kSumThreads : 256;
  __shared__ uint32_t wave_total[THREADS / 64];
  __shared__ ByteSums before_of, after_of;  // this workgroup's rows, and from them on
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, columns = byte_row(n_experts) / 16;
  for (int i = threadIdx.x; i < 4 * kMaxExperts; i += THREADS) (&cnt[0][0])[i] = 0u;
  const int r = blockIdx.x * block_rows + threadIdx.x;
  const bool live = (int)threadIdx.x < block_rows && r < rows;
  const uint32_t e = live ? experts[r] : 0xffffffffu;
  if constexpr (SUMS) {
    before_of.clear();
    after_of.clear();
    __syncthreads();
    const int slices = THREADS / columns, slice = threadIdx.x / columns, column = threadIdx.x - slice * columns;
    const int n = (blocks + slices - 1) / slices, mine = min((int)blockIdx.x * per, blocks);
    const int b0 = min(slice * n, blocks), b1 = slice < slices ? min(b0 + n, blocks) : b0;
    const u32x4* rows_of = reinterpret_cast<const u32x4*>(ends);
    uint32_t early[8] = {}, late[8] = {};
    if (n > 8) {
      sum_bytes<16>(rows_of, column, columns, b0, min(b1, mine), early);
      sum_bytes<16>(rows_of, column, columns, max(b0, mine), b1, late);
    } else {
      sum_bytes<8>(rows_of, column, columns, b0, min(b1, mine), early);
      sum_bytes<8>(rows_of, column, columns, max(b0, mine), b1, late);
    }
    if (b0 < min(b1, mine)) before_of.add(early, column, columns);
    if (max(b0, mine) < b1) after_of.add(late, column, columns);
    __syncthreads();
  }
  // Thread t sums experts 4 t .. 4 t + 3.
  uint32_t t4[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = 4 * (int)threadIdx.x + i;
    if constexpr (SUMS)
      t4[i] = at < n_experts ? before_of.get(at, columns) + after_of.get(at, columns) : 0u;
    else
      t4[i] = at < n_experts && blocks ? ends[(size_t)(blocks - 1) * n_experts + at] : 0u;
    sum += t4[i];
  }
  uint32_t upto = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(upto, d, 64);
    upto += lane >= d ? o : 0u;
  }
  if (lane == 63) wave_total[wave] = upto;
  uint32_t rank, same;
  lane_rank(e, rank, same);
  __syncthreads();  // cnt cleared, waves' totals
  uint32_t before = upto - sum;
  for (int w = 0; w < wave; ++w) before += wave_total[w];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = 4 * (int)threadIdx.x + i;
    if (at < kMaxExperts) first[at] = before;
    if (blockIdx.x == 0 && at < n_experts) offsets[at] = before;
    before += t4[i];
  }
  if (blockIdx.x == 0 && threadIdx.x == 255) offsets[n_experts] = before;
  if (live && rank + 1 == same) cnt[wave][e] = same;
  __syncthreads();
  if (live) {
    uint32_t pos = first[e] + rank;
    if constexpr (SUMS) pos += before_of.get((int)e, columns);
    else pos += blockIdx.x ? ends[(size_t)(blockIdx.x - 1) * n_experts + e] : 0u;
    for (int w = 0; w < wave; ++w) pos += cnt[w][e];
    lhs[pos] = (uint32_t)(r / top_k);
    rhs[pos] = e;
    inv[r] = pos;
  }
}

// out[t, c..c+7] = sum_j scores[t*k+j] * y[inv[t*k+j], c..c+7]; one thread per 8 columns.
// A position at or past rows (a corrupted inv) contributes nothing and is
// counted in *bad once per (token, slot).
template <typename TT>
__global__ __launch_bounds__(256) void combine_kernel(const uint16_t* __restrict__ y, const float* __restrict__ scores,
                                                      const uint32_t* __restrict__ inv, int tokens, int top_k, int n,
                                                      uint16_t* __restrict__ out, unsigned int* bad) {
  const int per_row = n / 8;
  const size_t total = (size_t)tokens * per_row;
  const size_t stride = (size_t)gridDim.x * blockDim.x;
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += stride) {
    const size_t t = i / per_row;
    const int c = (int)(i - t * per_row) * 8;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const uint32_t rows = (uint32_t)tokens * (uint32_t)top_k;
    for (int j = 0; j < top_k; ++j) {
      const uint32_t p = inv[t * top_k + j];
      if (p >= rows) {
        if (c == 0) atomicAdd(bad, 1u);
        continue;
      }
      const float w = scores[t * top_k + j];
      const u32x4 v = *reinterpret_cast<const u32x4*>(y + (size_t)p * n + c);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        acc[2 * h] = fmaf(w, TT::to_f32((uint16_t)(v[h] & 0xffffu)), acc[2 * h]);
        acc[2 * h + 1] = fmaf(w, TT::to_f32((uint16_t)(v[h] >> 16)), acc[2 * h + 1]);
      }
    }
    u32x4 o;
#pragma unroll
    for (int h = 0; h < 4; ++h) o[h] = TT::pack2(acc[2 * h], acc[2 * h + 1]);
    *reinterpret_cast<u32x4*>(out + t * n + c) = o;
  }
}

}  // namespace

size_t moe_sort_scratch_bytes(int rows, int n_experts) {
  const size_t blocks = (size_t)(rows + kSortRows - 1) / kSortRows;
  return blocks * (size_t)n_experts * 4;
}

// run(L, NV) as types of integral constants: the logits' type and at least nv of them a lane.
template <int MOST = 16, typename F>
hipError_t with_logits(int logits_dtype, int nv, F run) {
  auto typed = [&](auto l) {
    if (nv <= 1) run(l, std::integral_constant<int, 1>{});
    else if (nv <= 2) run(l, std::integral_constant<int, 2>{});
    else if (nv <= 4) run(l, std::integral_constant<int, 4>{});
    else if (nv <= 8) run(l, std::integral_constant<int, 8>{});
    else if (MOST == 16 || nv <= 16) run(l, std::integral_constant<int, 16>{});
    else run(l, std::integral_constant<int, MOST>{});
    return hipGetLastError();
  };
  if (logits_dtype == CPQ_DTYPE_F32) return typed(std::integral_constant<int, 0>{});
  if (logits_dtype == CPQ_DTYPE_F16) return typed(std::integral_constant<int, 1>{});
  return typed(std::integral_constant<int, 2>{});
}

bool moe_route_sort_fits(int tokens) { return tokens >= 1 && tokens <= kFusedTokens; }

hipError_t launch_moe_route(hipStream_t s, int logits_dtype, const void* logits, int tokens, int n_experts, int top_k,
                            int normalize, uint32_t* experts, float* scores) {
  if (tokens == 0) return hipSuccess;
  return with_logits(logits_dtype, (n_experts + 63) / 64, [&](auto l, auto nv) {
    hipLaunchKernelGGL((route_kernel<decltype(l)::value, decltype(nv)::value>), dim3((unsigned)((tokens + 3) / 4)),
                       dim3(256), 0, s, logits, tokens, n_experts, top_k, normalize, experts, scores);
  });
}

hipError_t launch_moe_route_sort(hipStream_t s, int logits_dtype, const void* logits, int tokens, int n_experts,
                                 int top_k, int normalize, uint32_t* experts, float* scores, uint32_t* lhs,
                                 uint32_t* rhs, uint32_t* inv, uint32_t* offsets) {
  if (!moe_route_sort_fits(tokens)) return hipErrorInvalidValue;
  return with_logits(logits_dtype, (n_experts + 63) / 64, [&](auto l, auto nv) {
    hipLaunchKernelGGL((route_sort_kernel<decltype(l)::value, decltype(nv)::value>), dim3(1), dim3(1024), 0, s, logits,
                       tokens, n_experts, top_k, normalize, experts, scores, lhs, rhs, inv, offsets);
  });
}

// From the histograms of blocks of block_rows rows to the sorted rows.
static hipError_t sort_blocks(hipStream_t s, const uint32_t* experts, int rows, int block_rows, int blocks, int top_k,
                              int n_experts, uint32_t* scratch, uint32_t* lhs, uint32_t* rhs, uint32_t* inv,
                              uint32_t* offsets) {
  hipLaunchKernelGGL(sort_scan_kernel, dim3((unsigned)((n_experts + kScanExperts - 1) / kScanExperts)),
                     dim3(kScanExperts * kScanSlices), 0, s, scratch, blocks, n_experts);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(sort_scatter_kernel<false>, dim3((unsigned)std::max(blocks, 1)), dim3(256), 0, s, experts, rows,
                     block_rows, blocks, 1, top_k, n_experts, scratch, lhs, rhs, inv, offsets);
  return hipGetLastError();
}

// Where histograms are scanned: whether they are the routing workgroups' own, of `rows` rows.
// Those of half a sort block or less are many, each with a scatter workgroup of its own: then
// the picks are counted again, a block at a time, a launch more (65536 tokens of 256 experts, 8
// picks 113 us, 129 with the routing kernel's histograms of 128 rows; 2 picks 79 and 109; 131072
// tokens of 64 experts, 1 pick 62 and 127; 65536 of 1024, 8 picks 389 and 450), in the scratch
// that moe_route takes.
inline bool keeps_counts(int rows) { return 2 * rows > kSortRows; }

size_t moe_grouped_scratch_bytes(int tokens, int n_experts, int top_k, const cpq_moe_router& r, int cus) {
  const int per = grouped_tokens(tokens, GroupedRouter(r, n_experts).per, cus), blocks = (tokens + per - 1) / per;
  if (sums_bytes(tokens, blocks, n_experts)) return (size_t)blocks * byte_row(n_experts);
  return keeps_counts(per * top_k) ? (size_t)blocks * n_experts * 4 : moe_sort_scratch_bytes(tokens * top_k, n_experts);
}

hipError_t launch_moe_route_grouped(hipStream_t s, int logits_dtype, const void* logits, int tokens, int n_experts,
                                    int top_k, const cpq_moe_router& r, int cus, uint32_t* experts, float* scores,
                                    uint32_t* scratch, uint32_t* lhs, uint32_t* rhs, uint32_t* inv, uint32_t* offsets) {
  const GroupedRouter router(r, n_experts);
  const int per = grouped_tokens(tokens, router.per, cus), blocks = (tokens + per - 1) / per;
  const bool bytes = sums_bytes(tokens, blocks, n_experts), counted = bytes || keeps_counts(per * top_k);
  if (blocks) {
    const hipError_t e = with_logits<32>(logits_dtype, router.per, [&](auto l, auto nv) {
      constexpr int NV = decltype(nv)::value;
      hipLaunchKernelGGL((route_grouped_kernel<decltype(l)::value, NV>), dim3((unsigned)blocks),
                         dim3(per * 64), 0, s, logits, tokens, n_experts, top_k, router, experts, scores,
                         counted ? scratch : nullptr, (int)bytes);
    });
    if (e != hipSuccess) return e;
  }
  if (!counted) return launch_moe_sort(s, experts, tokens * top_k, top_k, n_experts, scratch, lhs, rhs, inv, offsets);
  if (bytes) {
    const int rows = per * top_k, together = std::max(kSortRows / rows, 1);
    hipLaunchKernelGGL(sort_scatter_kernel<true>, dim3((unsigned)std::max((blocks + together - 1) / together, 1)),
                       dim3(kSumThreads), 0, s, experts, tokens * top_k, together * rows, blocks, together, top_k, n_experts,
                       scratch, lhs, rhs, inv, offsets);
    return hipGetLastError();
  }
  return sort_blocks(s, experts, tokens * top_k, per * top_k, blocks, top_k, n_experts, scratch, lhs, rhs, inv, offsets);
}

hipError_t launch_moe_route_grouped_sort(hipStream_t s, int logits_dtype, const void* logits, int tokens,
                                         int n_experts, int top_k, const cpq_moe_router& r, uint32_t* experts,
                                         float* scores, uint32_t* lhs, uint32_t* rhs, uint32_t* inv, uint32_t* offsets,
                                         unsigned int* counter) {
  if (!moe_route_sort_fits(tokens)) return hipErrorInvalidValue;
  const GroupedRouter router(r, n_experts);
  return with_logits<32>(logits_dtype, router.per, [&](auto l, auto nv) {
    hipLaunchKernelGGL((route_grouped_sort_kernel<decltype(l)::value, decltype(nv)::value>),
                       dim3((unsigned)((tokens + 3) / 4)), dim3(256), 0, s, logits, tokens, n_experts, top_k,
                       router, experts, scores, lhs, rhs, inv, offsets, counter);
  });
}

hipError_t launch_moe_sort(hipStream_t s, const uint32_t* experts, int rows, int top_k, int n_experts,
                           uint32_t* scratch, uint32_t* lhs, uint32_t* rhs, uint32_t* inv, uint32_t* offsets) {
  const int blocks = (rows + kSortRows - 1) / kSortRows;
  if (blocks) {
    hipLaunchKernelGGL(sort_count_kernel, dim3((unsigned)blocks), dim3(64), 0, s, experts, rows, n_experts, scratch);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return sort_blocks(s, experts, rows, kSortRows, blocks, top_k, n_experts, scratch, lhs, rhs, inv, offsets);
}

hipError_t launch_moe_combine(hipStream_t s, int dtype, const void* y, const float* scores, const uint32_t* inv,
                              int tokens, int top_k, int n, void* out, unsigned int* bad) {
  const size_t total = (size_t)tokens * (n / 8);
  if (total == 0) return hipSuccess;
  size_t blocks = (total + 255) / 256;
  if (blocks > 256 * 32) blocks = 256 * 32;
  if (dtype == CPQ_DTYPE_BF16)
    hipLaunchKernelGGL(combine_kernel<BF16>, dim3((unsigned)blocks), dim3(256), 0, s,
                       static_cast<const uint16_t*>(y), scores, inv, tokens, top_k, n, static_cast<uint16_t*>(out), bad);
  else
    hipLaunchKernelGGL(combine_kernel<F16>, dim3((unsigned)blocks), dim3(256), 0, s,
                       static_cast<const uint16_t*>(y), scores, inv, tokens, top_k, n, static_cast<uint16_t*>(out), bad);
  return hipGetLastError();
}

}  // namespace cpq
