// The layers' and the log-probabilities' scratch sizes and launches by element type (linear_dev.h, logp_dev.h).
#include "learn.h"

namespace wc {
namespace learn {

#define BY_TYPE(call, ...)                                                                                     \
    (a.dtype == WC_DTYPE_F32 ? call##_f32(__VA_ARGS__) : a.dtype == WC_DTYPE_F16 ? call##_f16(__VA_ARGS__) \
                                                                                  : call##_bf16(__VA_ARGS__))

size_t linear_scratch(const wc_linear_args& a, int cus) { return BY_TYPE(linear_scratch, a, cus); }
size_t linear_back_scratch(const wc_linear_back_args& a, int cus) { return BY_TYPE(linear_back_scratch, a, cus); }
size_t logp_scratch(const wc_logp_args& a, int cus) { return BY_TYPE(logp_scratch, a, cus); }

void launch_linear(const wc_linear_args& a, int cus, hipStream_t s) { BY_TYPE(linear, a, cus, s); }
void launch_linear_back(const wc_linear_back_args& a, int cus, hipStream_t s) { BY_TYPE(linear_back, a, cus, s); }
void launch_logp(const wc_logp_args& a, int cus, hipStream_t s) { BY_TYPE(logp, a, cus, s); }
void launch_logp_back(const wc_logp_back_args& a, int, hipStream_t s) { BY_TYPE(logp_back, a, s); }

}  // namespace learn
}  // namespace wc
