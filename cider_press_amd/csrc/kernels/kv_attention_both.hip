// Attention over the 4-bit key/value cache, scores capped and with a bias, prefixes seen.
#include "kv_attention.hpp"

namespace cpq {

hipError_t launch_kv_attention_both(const ExecCtx& ex, const cpq_kv_cache& c, const cpq_kv_attention_args& args,
                                      const KvScore& score, unsigned int* bad) {
  return run_attention<dev::Scores::kBoth>(ex, c, args, score, bad,
                                          [&](const cpq_kv_attention_args& a, int rows_max, bool report) {
                                            return launch_kv_decode_both(ex, c, a, score, rows_max, report, bad);
                                          });
}

}  // namespace cpq
