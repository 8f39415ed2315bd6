// The policy and preference losses over f16 logits.
#include "policy_dev.h"

namespace wc {
namespace learn {

void policy_f16(const wc_policy_args& a, hipStream_t s) { policy_of<f16>(a, s); }
void preference_f16(const wc_preference_args& a, hipStream_t s) { preference<f16>(a, s); }

}  // namespace learn
}  // namespace wc
