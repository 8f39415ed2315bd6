// Token log-probabilities and their gradient over f32 logits.
#include "logp_dev.h"

namespace wc {
namespace learn {

size_t logp_scratch_f32(const wc_logp_args& a, int cus) { return logp_plan<float>(a.rows, a.vocab, a.top, cus).bytes; }
void logp_f32(const wc_logp_args& a, int cus, hipStream_t s) { logp<float>(a, cus, s); }
void logp_back_f32(const wc_logp_back_args& a, hipStream_t s) { logp_back<float>(a, s); }

}  // namespace learn
}  // namespace wc
