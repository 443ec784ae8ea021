// Entry points of the 4-bit key/value cache (cpq_kv_*): argument validation
// and launch.  No reference counterpart; semantics in cpq.h.
#include <climits>
#include <cstdint>
#include <string>

#include "cpq_internal.hpp"

using cpq::fail;

namespace {

cpq_status invalid(const char* op, const std::string& what) {
  return fail(CPQ_ERR_INVALID_ARGUMENT, std::string(op) + ": " + what);
}

bool mul(size_t a, size_t b, size_t* out) { return !__builtin_mul_overflow(a, b, out); }

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

cpq_status launched(hipError_t e, const char* what) { return e == hipSuccess ? CPQ_OK : cpq::hip_fail(e, what); }

bool block_size_ok(uint32_t b) { return b >= 16 && b <= 1024 && (b & (b - 1)) == 0; }

cpq_status geometry(const char* op, const cpq_kv_cache* c, size_t* q_words, size_t* sb_words) {
  if (!c) return invalid(op, "NULL cache descriptor");
  if (c->dtype != CPQ_DTYPE_BF16 && c->dtype != CPQ_DTYPE_F16) return invalid(op, "dtype must be BF16 or F16");
  if (!block_size_ok(c->block_size))
    return invalid(op, "block_size (" + std::to_string(c->block_size) + ") must be a power of two, 16 ..= 1024");
  if (c->n_kv_heads == 0 || c->n_kv_heads > 65535) return invalid(op, "n_kv_heads outside 1..=65535");
  size_t slots;
  if (!mul(c->n_blocks, c->block_size, &slots) || slots >= 0xffffffffull)
    return invalid(op, "n_blocks * block_size must stay below 2^32 - 1");
  if (c->head_dim == 0 || c->group_size == 0 || c->head_dim % c->group_size != 0)
    return invalid(op, "head_dim (" + std::to_string(c->head_dim) + ") must be a multiple of group_size (" +
                           std::to_string(c->group_size) + ")");
  if ((c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) ||
      (c->group_size != 32 && c->group_size != 64 && c->group_size != 128))
    return fail(CPQ_ERR_KERNEL_NOT_FOUND, std::string(op) + ": no kernel for head_dim " +
                                              std::to_string(c->head_dim) + ", group_size " +
                                              std::to_string(c->group_size));
  size_t rows;
  if (!mul(slots, c->n_kv_heads, &rows) || !mul(rows, c->head_dim / 8, q_words))
    return invalid(op, "cache size overflows usize");
  *sb_words = rows * (c->head_dim / c->group_size);  // no more than q_words
  return CPQ_OK;
}

cpq_status check_cache(const char* op, const cpq_kv_cache* c) {
  size_t q, sb;
  cpq_status st = geometry(op, c, &q, &sb);
  if (st != CPQ_OK) return st;
  if (c->k_q_len != q || c->v_q_len != q)
    return invalid(op, "k_q / v_q of " + std::to_string(c->k_q_len) + " / " + std::to_string(c->v_q_len) +
                           " words, expected " + std::to_string(q));
  if (c->k_sb_len != sb || c->v_sb_len != sb)
    return invalid(op, "k_sb / v_sb of " + std::to_string(c->k_sb_len) + " / " + std::to_string(c->v_sb_len) +
                           " words, expected " + std::to_string(sb));
  if (!c->k_q || !c->k_sb || !c->v_q || !c->v_sb) return invalid(op, "NULL cache buffer");
  if (!aligned(c->k_q, 16) || !aligned(c->k_sb, 16) || !aligned(c->v_q, 16) || !aligned(c->v_sb, 16))
    return invalid(op, "cache buffers must be 16-byte aligned");
  return CPQ_OK;
}

// [tokens, heads, dim] of T at token and head strides: 16-byte loads of
// every row, addresses within the address space.
cpq_status check_strided(const char* op, const char* name, const void* p, size_t tokens, size_t heads, size_t dim,
                         size_t token_stride, size_t head_stride) {
  if (token_stride % 8 != 0 || head_stride % 8 != 0)
    return invalid(op, std::string(name) + " strides must be multiples of 8 elements");
  size_t a, b, n;
  if (!mul(tokens - 1, token_stride, &a) || !mul(heads - 1, head_stride, &b) || __builtin_add_overflow(a, b, &n) ||
      n > (size_t(1) << 60) - dim)
    return invalid(op, std::string(name) + " strides overflow");
  if (!p) return invalid(op, std::string("NULL ") + name);
  if (!aligned(p, 16)) return invalid(op, std::string(name) + " must be 16-byte aligned");
  return CPQ_OK;
}

bool overlap(const void* a, size_t a_words, const void* b, size_t b_words) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a_words && b_words && x < y + 4 * b_words && y < x + 4 * a_words;
}

struct Words {
  const char* name;
  const void* p;
  size_t n;
};

// u32 arrays of one call: not NULL, 4-byte aligned, and no output (the last
// n_out of them) over another.
cpq_status check_words(const char* op, const Words* w, int n, int n_out) {
  for (int i = 0; i < n; ++i) {
    if (w[i].n && !w[i].p) return invalid(op, std::string("NULL ") + w[i].name);
    if (!aligned(w[i].p, 4)) return invalid(op, std::string(w[i].name) + " must be 4-byte aligned");
  }
  for (int i = n - n_out; i < n; ++i)
    for (int j = 0; j < i; ++j)
      if (overlap(w[i].p, w[i].n, w[j].p, w[j].n))
        return invalid(op, std::string(w[i].name) + " overlaps " + w[j].name);
  return CPQ_OK;
}

cpq_status check_table(const char* op, size_t n_seqs, size_t max_blocks, uint32_t block_size, size_t* entries) {
  if (n_seqs > cpq::kKvMaxSeqs) return invalid(op, "n_seqs outside 0..=" + std::to_string(cpq::kKvMaxSeqs));
  if (!block_size_ok(block_size))
    return invalid(op, "block_size (" + std::to_string(block_size) + ") must be a power of two, 16 ..= 1024");
  if (!mul(n_seqs, max_blocks, entries) || *entries >= (1ull << 31) || max_blocks >= (1ull << 31))
    return invalid(op, "n_seqs * max_blocks must stay below 2^31");
  return CPQ_OK;
}

}  // namespace

extern "C" {

cpq_status cpq_kv_cache_words(const cpq_kv_cache* cache, size_t* q_words, size_t* sb_words) {
  size_t q, sb;
  cpq_status st = geometry("kv_cache", cache, &q, &sb);
  if (st != CPQ_OK) return st;
  if (q_words) *q_words = q;
  if (sb_words) *sb_words = sb;
  return CPQ_OK;
}

cpq_status cpq_check_kv_cache(const cpq_kv_cache* cache) { return check_cache("kv_cache", cache); }

cpq_status cpq_kv_release(cpq_commands* cmds, const uint32_t* finished, const uint32_t* lens,
                          const uint32_t* block_table, size_t n_seqs, size_t max_blocks, uint32_t block_size,
                          uint32_t* free_list, size_t free_cap, const uint32_t* free_count, uint32_t* lens_out,
                          uint32_t* free_count_out) {
  const char* op = "kv_release";
  if (!cmds) return invalid(op, "NULL command session");
  size_t entries;
  cpq_status st = check_table(op, n_seqs, max_blocks, block_size, &entries);
  if (st != CPQ_OK) return st;
  if (free_cap >= (1ull << 31)) return invalid(op, "free_cap must stay below 2^31");
  const Words w[] = {{"finished", finished, n_seqs},   {"lens", lens, n_seqs},
                     {"block_table", block_table, entries}, {"free_count", free_count, 1},
                     {"free_list", free_list, free_cap},    {"lens_out", lens_out, n_seqs},
                     {"free_count_out", free_count_out, 1}};
  st = check_words(op, w, 7, 3);
  if (st != CPQ_OK) return st;
  return launched(cpq::launch_kv_release(cmds->stream, finished, lens, block_table, (uint32_t)n_seqs,
                                         (uint32_t)max_blocks, block_size, free_list, (uint32_t)free_cap, free_count,
                                         lens_out, free_count_out, cmds->status + 3),
                  "kv_release launch");
}

cpq_status cpq_kv_plan(cpq_commands* cmds, const uint32_t* lens, const uint32_t* new_lens, uint32_t* block_table,
                       size_t n_seqs, size_t max_blocks, uint32_t block_size, const uint32_t* free_list,
                       size_t free_cap, const uint32_t* free_count, uint32_t* query_starts, uint32_t* kv_lens,
                       uint32_t* slots, uint32_t* positions, size_t cap, uint32_t* free_count_out) {
  const char* op = "kv_plan";
  if (!cmds) return invalid(op, "NULL command session");
  size_t entries;
  cpq_status st = check_table(op, n_seqs, max_blocks, block_size, &entries);
  if (st != CPQ_OK) return st;
  if (free_cap >= (1ull << 31) || cap >= (1ull << 31)) return invalid(op, "free_cap and cap must stay below 2^31");
  const Words w[] = {{"lens", lens, n_seqs},
                     {"new_lens", new_lens, n_seqs},
                     {"free_list", free_list, free_cap},
                     {"free_count", free_count, 1},
                     {"block_table", block_table, entries},
                     {"query_starts", query_starts, n_seqs + 1},
                     {"kv_lens", kv_lens, n_seqs},
                     {"slots", slots, cap},
                     {"positions", positions, cap},
                     {"free_count_out", free_count_out, 1}};
  st = check_words(op, w, 10, 6);
  if (st != CPQ_OK) return st;
  return launched(cpq::launch_kv_plan(cmds->stream, lens, new_lens, block_table, (uint32_t)n_seqs,
                                      (uint32_t)max_blocks, block_size, free_list, (uint32_t)free_cap, free_count,
                                      query_starts, kv_lens, slots, positions, (uint32_t)cap, free_count_out,
                                      reinterpret_cast<unsigned long long*>(cmds->status + 4)),
                  "kv_plan launch");
}

cpq_status cpq_kv_append(cpq_commands* cmds, const cpq_kv_cache* cache, const void* k, size_t k_token_stride,
                         size_t k_head_stride, const void* v, size_t v_token_stride, size_t v_head_stride,
                         const uint32_t* slots, size_t n_tokens) {
  const char* op = "kv_append";
  if (!cmds) return invalid(op, "NULL command session");
  cpq_status st = check_cache(op, cache);
  if (st != CPQ_OK) return st;
  if (n_tokens > (size_t)INT_MAX) return invalid(op, "n_tokens must fit in i32");
  if (n_tokens == 0) return CPQ_OK;
  st = check_strided(op, "k", k, n_tokens, cache->n_kv_heads, cache->head_dim, k_token_stride, k_head_stride);
  if (st != CPQ_OK) return st;
  st = check_strided(op, "v", v, n_tokens, cache->n_kv_heads, cache->head_dim, v_token_stride, v_head_stride);
  if (st != CPQ_OK) return st;
  const Words w[] = {{"slots", slots, n_tokens}};
  st = check_words(op, w, 1, 0);
  if (st != CPQ_OK) return st;
  return launched(cpq::launch_kv_append(cmds->stream, *cache, k, k_token_stride, k_head_stride, v, v_token_stride,
                                        v_head_stride, slots, (uint32_t)n_tokens, cmds->status + 6),
                  "kv_append launch");
}

cpq_status cpq_kv_gather(cpq_commands* cmds, const cpq_kv_cache* cache, const uint32_t* slots, size_t n_rows,
                         void* k_out, void* v_out) {
  const char* op = "kv_gather";
  if (!cmds) return invalid(op, "NULL command session");
  cpq_status st = check_cache(op, cache);
  if (st != CPQ_OK) return st;
  if (n_rows > (size_t)INT_MAX) return invalid(op, "n_rows must fit in i32");
  if (n_rows == 0 || (!k_out && !v_out)) return CPQ_OK;
  if (!aligned(k_out, 16) || !aligned(v_out, 16)) return invalid(op, "k_out and v_out must be 16-byte aligned");
  const Words w[] = {{"slots", slots, n_rows}};
  st = check_words(op, w, 1, 0);
  if (st != CPQ_OK) return st;
  return launched(cpq::launch_kv_gather(cmds->stream, *cache, slots, (uint32_t)n_rows, k_out, v_out, cmds->status + 6),
                  "kv_gather launch");
}

cpq_status cpq_check_kv_attention_args(const cpq_kv_cache* cache, const cpq_kv_attention_args* a) {
  const char* op = "kv_attention";
  cpq_status st = check_cache(op, cache);
  if (st != CPQ_OK) return st;
  if (!a) return invalid(op, "NULL arguments");
  if (a->n_heads == 0 || a->n_heads > 65535 || a->n_heads % cache->n_kv_heads != 0)
    return invalid(op, "n_heads (" + std::to_string(a->n_heads) + ") must be a positive multiple of n_kv_heads (" +
                           std::to_string(cache->n_kv_heads) + "), up to 65535");
  if (a->n_seqs > 65535) return invalid(op, "n_seqs outside 0..=65535");
  size_t rows, entries;
  if (!mul(a->n_tokens, a->n_heads, &rows) || rows >= (1ull << 31))
    return invalid(op, "n_tokens * n_heads must stay below 2^31");
  if (!mul(a->n_seqs, a->max_blocks, &entries) || entries >= (1ull << 31) || a->max_blocks >= (1ull << 31))
    return invalid(op, "n_seqs * max_blocks must stay below 2^31");
  if (cache->n_blocks == 0 && a->n_tokens != 0) return invalid(op, "the cache has no blocks");
  if (a->n_seqs * cache->n_kv_heads * 4096 >= (1ull << 31)) return invalid(op, "n_seqs * n_kv_heads past 2^19");
  if (!(a->scale > 0.f) || a->scale > 3.4e38f) return invalid(op, "scale must be positive and finite");
  if (a->n_tokens == 0 || a->n_seqs == 0) return CPQ_OK;
  st = check_strided(op, "q", a->q, a->n_tokens, a->n_heads, cache->head_dim, a->q_token_stride, a->q_head_stride);
  if (st != CPQ_OK) return st;
  st = check_strided(op, "out", a->out, a->n_tokens, a->n_heads, cache->head_dim, a->out_token_stride,
                     a->out_head_stride);
  if (st != CPQ_OK) return st;
  // No two output rows share elements: heads within a token's row, or tokens within a head's.
  const size_t d = cache->head_dim, t = a->out_token_stride, h = a->out_head_stride;
  const bool inner_heads = (a->n_heads == 1 || h >= d) && (a->n_tokens == 1 || t >= (a->n_heads - 1) * h + d);
  const bool inner_tokens = (a->n_tokens == 1 || t >= d) && (a->n_heads == 1 || h >= (a->n_tokens - 1) * t + d);
  if (!inner_heads && !inner_tokens) return invalid(op, "out rows overlap at these strides");
  const Words w[] = {{"block_table", a->block_table, entries},
                     {"query_starts", a->query_starts, a->n_seqs + 1},
                     {"kv_lens", a->kv_lens, a->n_seqs}};
  return check_words(op, w, 3, 0);
}

cpq_status cpq_kv_attention(cpq_commands* cmds, const cpq_kv_cache* cache, const cpq_kv_attention_args* args) {
  if (!cmds) return invalid("kv_attention", "NULL command session");
  cpq_status st = cpq_check_kv_attention_args(cache, args);
  if (st != CPQ_OK) return st;
  if (args->n_tokens == 0 || args->n_seqs == 0) return CPQ_OK;
  return launched(cpq::launch_kv_attention(cpq::session_ctx(cmds), *cache, *args, cmds->status + 7),
                  "kv_attention launch");
}

}  // extern "C"
