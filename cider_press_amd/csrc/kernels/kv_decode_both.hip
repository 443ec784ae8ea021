// Attention over the 4-bit key/value cache for few query rows per sequence, scores
// capped and with a bias, prefixes seen.
#include "kv_decode.hpp"

namespace cpq {

hipError_t launch_kv_decode_both(const ExecCtx& ex, const cpq_kv_cache& c, const cpq_kv_attention_args& a,
                                   const KvScore& score, int rows_max, bool report, unsigned int* bad) {
  return run_decode<dev::Scores::kBoth>(ex, c, a, score, rows_max, report, bad);
}

}  // namespace cpq
