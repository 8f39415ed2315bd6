// Token log-probabilities and their gradient over bf16 logits.
#include "logp_dev.h"

namespace wc {
namespace learn {

size_t logp_scratch_bf16(const wc_logp_args& a, int cus) { return logp_plan<bf16>(a.rows, a.vocab, a.top, cus).bytes; }
void logp_bf16(const wc_logp_args& a, int cus, hipStream_t s) { logp<bf16>(a, cus, s); }
void logp_back_bf16(const wc_logp_back_args& a, hipStream_t s) { logp_back<bf16>(a, s); }

}  // namespace learn
}  // namespace wc
