// ops_internal.h -- what ops.hip (entry points, argument checks, choice of kernel) shares with the operators' kernel files.
#pragma once
#include "../../include/vadc_amd.h"

#include <hip/hip_runtime.h>

namespace vadc {
int fail(int code, const char *fmt, ...);                            // engine.hip: records the calling thread's message, returns code
namespace ops {
// A long call goes out in slices; `first` is its first slice, the largest, by which the form and the workspace of ALL of them are chosen (a shorter last one on its own might take another
// form, whose workspace the caller was not asked for).
void launch_linear(const vadc_amd_linear_args &slice, hipStream_t);
int64_t group_norm_workspace(const vadc_amd_group_norm_args &first);
void launch_group_norm(const vadc_amd_group_norm_args &slice, const vadc_amd_group_norm_args &first, hipStream_t);
int64_t gated_delta_workspace(const vadc_amd_gated_delta_args &first);
void launch_gated_delta(const vadc_amd_gated_delta_args &slice, const vadc_amd_gated_delta_args &first, hipStream_t);
}  // namespace ops
}  // namespace vadc
