// The policy and preference losses over f32 logits.
#include "policy_dev.h"

namespace wc {
namespace learn {

void policy_f32(const wc_policy_args& a, hipStream_t s) { policy_of<float>(a, s); }
void preference_f32(const wc_preference_args& a, hipStream_t s) { preference<float>(a, s); }

}  // namespace learn
}  // namespace wc
