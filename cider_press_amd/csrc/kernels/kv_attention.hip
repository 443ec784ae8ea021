// Attention over the 4-bit key/value cache.
#include "kv_attention.hpp"

namespace cpq {

hipError_t launch_kv_attention(const ExecCtx& ex, const cpq_kv_cache& c, const cpq_kv_attention_args& args,
                               unsigned int* bad) {
  return run_attention<dev::Scores::kPlain>(ex, c, args, KvScore{}, bad,
                              [&](const cpq_kv_attention_args& a, int rows_max, bool report) {
                                return launch_kv_decode(ex, c, a, rows_max, report, bad);
                              });
}

}  // namespace cpq
