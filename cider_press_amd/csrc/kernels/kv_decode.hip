// Attention over the 4-bit key/value cache for few query rows per sequence.
#include "kv_decode.hpp"

namespace cpq {

hipError_t launch_kv_decode(const ExecCtx& ex, const cpq_kv_cache& c, const cpq_kv_attention_args& a, int rows_max,
                            bool report, unsigned int* bad) {
  return run_decode<dev::Scores::kPlain>(ex, c, a, KvScore{}, rows_max, report, bad);
}

}  // namespace cpq
