// A layer's product and its gradients on f32 matrices.
#include "linear_dev.h"

namespace wc {
namespace learn {

size_t linear_scratch_f32(const wc_linear_args& a, int cus) { return linear_plan<float>(a, cus).bytes; }
size_t linear_back_scratch_f32(const wc_linear_back_args& a, int cus) { return linear_back_plan<float>(a, cus).bytes; }
void linear_f32(const wc_linear_args& a, int cus, hipStream_t s) { linear<float>(a, cus, s); }
void linear_back_f32(const wc_linear_back_args& a, int cus, hipStream_t s) { linear_back<float>(a, cus, s); }

}  // namespace learn
}  // namespace wc
