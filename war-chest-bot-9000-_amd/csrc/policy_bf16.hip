// The policy and preference losses over bf16 logits.
#include "policy_dev.h"

namespace wc {
namespace learn {

void policy_bf16(const wc_policy_args& a, hipStream_t s) { policy_of<bf16>(a, s); }
void preference_bf16(const wc_preference_args& a, hipStream_t s) { preference<bf16>(a, s); }

}  // namespace learn
}  // namespace wc
