// kernels_ops_norm.hip -- group norm with an activation, channels last: x [sequences][positions][channels], statistics over a sequence's positions and one group's channels.
#include "ops_internal.h"
#include "ops_prims.h"

namespace vadc {
namespace ops {

// Count, mean and sum of squared deviations of a set of values; two sets merge exactly (Chan, Golub and LeVeque's update), so that a mean far from zero
// costs no digits of the variance, as a sum of squares would.
struct Stats { float n, mean, m2; };
__device__ __forceinline__ Stats merge(const Stats &a, const Stats &b)
{
   const float n = a.n + b.n, d = b.mean - a.mean, w = n > 0.0f ? b.n / n : 0.0f;
   return {n, a.mean + d * w, a.m2 + b.m2 + d * d * (a.n * w)};
}
__device__ __forceinline__ Stats shuffle_xor(const Stats &s, int d) { return {__shfl_xor(s.n, d), __shfl_xor(s.mean, d), __shfl_xor(s.m2, d)}; }
// the set of the lanes that differ in the low bits; both partners of an exchange merge in the same order, so that every lane holds the same bits
__device__ __forceinline__ Stats merge_lanes(Stats s, int width, int lane)
{
   for (int d = 1; d < width; d <<= 1) {
      const Stats o = shuffle_xor(s, d);
      s = (lane & d) ? merge(o, s) : merge(s, o);
   }
   return s;
}

__device__ __forceinline__ int64_t live_positions(const vadc_amd_group_norm_args &a, int64_t seq)
{
   if (!a.lengths) return a.positions;
   const int64_t v = a.lengths[seq];
   return v < 0 ? 0 : v > a.positions ? a.positions : v;
}

// One workgroup per (sequence, group), any sizes: one pass for the statistics, one to normalise.
template <typename T>
__global__ __launch_bounds__(256) void k_group_norm(const vadc_amd_group_norm_args a)
{
   __shared__ Stats part[4];
   const int tid = threadIdx.x, lane = tid & 63;
   const int64_t seq = blockIdx.x / a.groups, size = a.channels / a.groups, c0 = (blockIdx.x % a.groups) * size;
   const int64_t count = live_positions(a, seq) * size;
   const T *x = (const T *)a.x + seq * a.x_stride[0] + c0;
   Stats s = {0, 0, 0};
   for (int64_t e = tid; e < count; e += 256) {
      const int64_t p = e / size;
      s = merge(s, {1.0f, (float)x[p * a.x_stride[1] + e - p * size], 0.0f});
   }
   s = merge_lanes(s, 64, lane);
   if (lane == 0) part[tid >> 6] = s;
   __syncthreads();
   s = merge(merge(part[0], part[1]), merge(part[2], part[3]));
   const float rstd = 1.0f / sqrtf(s.m2 / fmaxf(s.n, 1.0f) + a.eps);
   const T *w = (const T *)a.weight + c0, *b = (const T *)a.bias + c0, *gate = (const T *)a.gate + seq * a.gate_stride[0] + c0;
   T *out = (T *)a.out + seq * a.out_stride[0] + c0;
   for (int64_t e = tid; e < count; e += 256) {
      const int64_t p = e / size, c = e - p * size;
      float y = ((float)x[p * a.x_stride[1] + c] - s.mean) * rstd;
      if (a.weight) y *= (float)w[c];
      if (a.bias) y += (float)b[c];
      y = a.gate ? y * activate((float)gate[p * a.gate_stride[1] + c], a.activation) : activate(y, a.activation);
      out[p * a.out_stride[1] + c] = (T)y;
   }
}

template <typename T> static void launch(const vadc_amd_group_norm_args &a, hipStream_t s)
{
   hipLaunchKernelGGL(k_group_norm<T>, dim3((unsigned)(a.sequences * a.groups)), dim3(256), 0, s, a);
}

int64_t group_norm_workspace(const vadc_amd_group_norm_args &) { return 0; }

void launch_group_norm(const vadc_amd_group_norm_args &a, hipStream_t s)
{
   if (a.dtype == VADC_AMD_F32) launch<float>(a, s);
   else if (a.dtype == VADC_AMD_F16) launch<_Float16>(a, s);
   else launch<__bf16>(a, s);
}

}  // namespace ops
}  // namespace vadc
