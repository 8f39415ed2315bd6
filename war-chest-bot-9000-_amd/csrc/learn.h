// The training operators' launches (include/wc_learn.h) and what their device
// code shares. The entry points check every argument first (capi_learn.cpp).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/wc_learn.h"

namespace wc {
namespace learn {

// Scratch bytes a call needs, given the device's compute units.
size_t policy_scratch(const wc_policy_args& a, int cus);
size_t preference_scratch(const wc_preference_args& a, int cus);
size_t norm_back_scratch(const wc_norm_back_args& a, int cus);
size_t ckpt_weight_scratch(const wc_ckpt_weight_args& a, int cus);

void launch_policy(const wc_policy_args& a, int cus, hipStream_t s);
void launch_preference(const wc_preference_args& a, int cus, hipStream_t s);
void launch_norm(const wc_norm_args& a, int cus, hipStream_t s);
void launch_norm_back(const wc_norm_back_args& a, int cus, hipStream_t s);
void launch_ckpt_write(const wc_ckpt_args& a, int cus, hipStream_t s);
void launch_ckpt_read(const wc_ckpt_args& a, int cus, hipStream_t s);
void launch_ckpt_act_back(const wc_ckpt_args& a, int cus, hipStream_t s);
void launch_ckpt_weight(const wc_ckpt_weight_args& a, int cus, hipStream_t s);

// The losses by element type.
void policy_f32(const wc_policy_args& a, hipStream_t s);
void policy_f16(const wc_policy_args& a, hipStream_t s);
void policy_bf16(const wc_policy_args& a, hipStream_t s);
void preference_f32(const wc_preference_args& a, hipStream_t s);
void preference_f16(const wc_preference_args& a, hipStream_t s);
void preference_bf16(const wc_preference_args& a, hipStream_t s);

inline size_t pad256(size_t x) { return (x + 255) & ~size_t(255); }

}  // namespace learn
}  // namespace wc
