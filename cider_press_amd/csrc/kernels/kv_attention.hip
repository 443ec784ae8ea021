// Attention of a step's queries over the 4-bit key/value cache (semantics:
// cpq_kv_attention in cpq.h).
//
// One wave per (query row, head) walks its sequence's keys 64 at a time: lane
// j scores key j in fp32, the running maximum and sum of the softmax are kept
// in registers, then lane d adds the weighted values of its dimensions.
#include "../cpq_internal.hpp"
#include "common.hpp"

namespace cpq {
namespace {

using namespace dev;

template <typename TT, int D>
__global__ __launch_bounds__(64) void kv_attention_rows_kernel(cpq_kv_cache c, cpq_kv_attention_args a,
                                                               unsigned int* bad) {
  constexpr int W = D / 8, DL = D / 64;
  __shared__ float qs[D];
  __shared__ float ps[64];
  __shared__ uint32_t blocks[64];
  const int lane = threadIdx.x;
  const uint32_t row = blockIdx.x, head = blockIdx.y, group = a.n_heads / c.n_kv_heads, kvh = head / group;
  uint32_t lo = 0, hi = a.n_seqs;  // starts[lo] <= row < starts[hi], if any
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (a.query_starts[mid] <= row) lo = mid;
    else hi = mid;
  }
  const uint32_t s0 = a.query_starts[lo], s1 = a.query_starts[lo + 1];
  if (row < s0 || row >= s1) return;
  if (s1 - s0 > a.max_q || s1 > a.n_tokens) {
    if (lane == 0 && head == 0 && row == s0) atomicAdd(bad, 1u);
    return;
  }
  const long n = a.kv_lens[lo], pos = n - (long)(s1 - s0) + (row - s0);
  const long first = a.window && pos + 1 > (long)a.window ? pos + 1 - (long)a.window : 0;
  // Keys past the table's row are masked.
  const uint32_t bs = c.block_size, shift = 31 - __builtin_clz(bs);
  const long room = (long)a.max_blocks << shift, end = min(a.causal ? pos + 1 : n, room);
  if (n > room && lane == 0 && head == 0 && row == s0) atomicAdd(bad, 1u);
  const uint16_t* q = static_cast<const uint16_t*>(a.q) + row * a.q_token_stride + head * a.q_head_stride;
  for (int d = lane; d < D; d += 64) qs[d] = TT::to_f32(q[d]);
  __syncthreads();
  const uint32_t gs = c.group_size, G = D / gs;
  float m = -INFINITY, l = 0.f, acc[DL] = {};
  for (long base = first; base < end; base += 64) {
    const long j = base + lane;
    float score = -INFINITY;
    uint32_t block = 0xffffffffu;
    if (j < end) {
      const long at = j >> shift;
      block = a.block_table[(size_t)lo * a.max_blocks + at];
      if (block >= c.n_blocks) {
        atomicAdd(bad, 1u);
      } else {
        const size_t krow = ((size_t)block * c.n_kv_heads + kvh) * bs + (j & (bs - 1));
        float dot = 0.f;
        for (int w = 0; w < W; ++w) {
          const uint32_t word = c.k_q[krow * W + w], sb = c.k_sb[krow * G + w * 8 / gs];
          const float s = TT::lo(sb), b = TT::hi(sb);
#pragma unroll
          for (int i = 0; i < 8; ++i) dot = fmaf(fmaf(s, (float)(word >> (4 * i) & 15u), b), qs[8 * w + i], dot);
        }
        score = dot * a.scale;
      }
    }
    float top = score;
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    const float m_new = fmaxf(m, top), ref = m_new == -INFINITY ? 0.f : m_new;
    const float keep = expf(m - ref), p = block < c.n_blocks ? expf(score - ref) : 0.f;
    l = l * keep + wave_sum(p);
    m = m_new;
    ps[lane] = p;
    blocks[lane] = block;
    __syncthreads();
    for (int i = 0; i < DL; ++i) acc[i] *= keep;
    for (int i = 0; i < 64; ++i) {
      if (blocks[i] >= c.n_blocks) continue;
      const uint32_t off = (uint32_t)(base + i) & (bs - 1);
      const size_t quad = ((size_t)blocks[i] * c.n_kv_heads + kvh) * bs + (off & ~3u);
      for (int e = 0; e < DL; ++e) {
        const uint32_t d = lane + 64 * e;
        const uint32_t word = c.v_q[quad * W + d / 8 * 4 + (off & 3)], sb = c.v_sb[quad * G + d / gs * 4 + (off & 3)];
        acc[e] = fmaf(ps[i], fmaf(TT::lo(sb), (float)(word >> (4 * (d & 7)) & 15u), TT::hi(sb)), acc[e]);
      }
    }
    __syncthreads();
  }
  uint16_t* out = static_cast<uint16_t*>(a.out) + row * a.out_token_stride + head * a.out_head_stride;
  for (int e = 0; e < DL; ++e) out[lane + 64 * e] = TT::from_f32(l == 0.f ? 0.f : acc[e] / l);
}

}  // namespace

hipError_t launch_kv_attention(const ExecCtx& ex, const cpq_kv_cache& c, const cpq_kv_attention_args& a,
                               unsigned int* bad) {
  if (a.max_q * (a.n_heads / c.n_kv_heads) <= kKvDecodeRows) return launch_kv_decode(ex, c, a, bad);
  const dim3 grid((uint32_t)a.n_tokens, (uint32_t)a.n_heads);
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(64), 0, ex.stream, c, a, bad);
    return hipGetLastError();
  };
  const bool bf16 = c.dtype == CPQ_DTYPE_BF16;
  switch (c.head_dim) {
    case 64: return bf16 ? run(kv_attention_rows_kernel<BF16, 64>) : run(kv_attention_rows_kernel<F16, 64>);
    case 128: return bf16 ? run(kv_attention_rows_kernel<BF16, 128>) : run(kv_attention_rows_kernel<F16, 128>);
    case 256: return bf16 ? run(kv_attention_rows_kernel<BF16, 256>) : run(kv_attention_rows_kernel<F16, 256>);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace cpq
