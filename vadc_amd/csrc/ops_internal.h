// ops_internal.h -- what ops.hip (entry points, argument checks, choice of kernel) shares with the operators' kernel files.
#pragma once
#include "../../include/vadc_amd.h"

#include <hip/hip_runtime.h>

namespace vadc {
int fail(int code, const char *fmt, ...);                            // engine.hip: records the calling thread's message, returns code
namespace ops {
void launch_linear(const vadc_amd_linear_args &, hipStream_t);
int64_t group_norm_workspace(const vadc_amd_group_norm_args &);
void launch_group_norm(const vadc_amd_group_norm_args &, hipStream_t);
int64_t gated_delta_workspace(const vadc_amd_gated_delta_args &);
void launch_gated_delta(const vadc_amd_gated_delta_args &, hipStream_t);
}  // namespace ops
}  // namespace vadc
