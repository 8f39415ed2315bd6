// The losses' scratch sizes, and their launches by element type (policy_dev.h).
#include "policy_dev.h"

namespace wc {
namespace learn {

size_t policy_scratch(const wc_policy_args& a, int) {
    const size_t losses = pad256(size_t(a.rows) * sizeof(double));
    // the larger of both forms, with and without a reference's logits
    if (holds(a.dtype, a.vocab, true))
        return one_group(a.rows, lanes_of(a.vocab / (a.dtype == WC_DTYPE_F32 ? 4 : 8))) ? 0 : losses;
    return losses + pad256(size_t(a.rows) * sizeof(RowGrad)) +
           pad256(size_t(a.rows) * splits_of(a.vocab) * sizeof(Part));
}

size_t preference_scratch(const wc_preference_args& a, int) {
    const size_t base = pad256(size_t(a.rows) * sizeof(RowGrad)) + pad256(size_t(a.pairs) * sizeof(double));
    return holds(a.dtype, a.vocab, false) ? base : base + pad256(size_t(a.rows) * splits_of(a.vocab) * sizeof(Part));
}

void launch_policy(const wc_policy_args& a, int, hipStream_t s) {
    if (a.dtype == WC_DTYPE_F32) policy_f32(a, s);
    else if (a.dtype == WC_DTYPE_F16) policy_f16(a, s);
    else policy_bf16(a, s);
}

void launch_preference(const wc_preference_args& a, int, hipStream_t s) {
    if (a.dtype == WC_DTYPE_F32) preference_f32(a, s);
    else if (a.dtype == WC_DTYPE_F16) preference_f16(a, s);
    else preference_bf16(a, s);
}

}  // namespace learn
}  // namespace wc
