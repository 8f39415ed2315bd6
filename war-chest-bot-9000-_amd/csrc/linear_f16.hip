// A layer's product and its gradients on f16 matrices.
#include "linear_dev.h"

namespace wc {
namespace learn {

size_t linear_scratch_f16(const wc_linear_args& a, int cus) { return linear_plan<f16>(a, cus).bytes; }
size_t linear_back_scratch_f16(const wc_linear_back_args& a, int cus) { return linear_back_plan<f16>(a, cus).bytes; }
void linear_f16(const wc_linear_args& a, int cus, hipStream_t s) { linear<f16>(a, cus, s); }
void linear_back_f16(const wc_linear_back_args& a, int cus, hipStream_t s) { linear_back<f16>(a, cus, s); }

}  // namespace learn
}  // namespace wc
