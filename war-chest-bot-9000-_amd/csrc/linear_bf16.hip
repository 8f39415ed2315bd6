// A layer's product and its gradients on bf16 matrices.
#include "linear_dev.h"

namespace wc {
namespace learn {

size_t linear_scratch_bf16(const wc_linear_args& a, int cus) { return linear_plan<bf16>(a, cus).bytes; }
size_t linear_back_scratch_bf16(const wc_linear_back_args& a, int cus) { return linear_back_plan<bf16>(a, cus).bytes; }
void linear_bf16(const wc_linear_args& a, int cus, hipStream_t s) { linear<bf16>(a, cus, s); }
void linear_back_bf16(const wc_linear_back_args& a, int cus, hipStream_t s) { linear_back<bf16>(a, cus, s); }

}  // namespace learn
}  // namespace wc
