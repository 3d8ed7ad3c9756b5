// ops_prims.h -- pieces shared by the operators on device tensors (linear, group_norm, gated_delta): element types, activations, wave reductions.
// Device code only; include inside a .hip translation unit.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vadc {
namespace ops {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

enum { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActSigmoid = 4 };

// 1 / (1 + e^-y): the reciprocal is v_rcp_f32 (1 ulp); e^-y = inf gives 0, as the division would
__device__ __forceinline__ float sigmoid_f32(float y) { return __builtin_amdgcn_rcpf(1.0f + expf(-y)); }

__device__ __forceinline__ float activate(float y, int act)
{
   switch (act) {
      case kActRelu:    return y < 0.0f ? 0.0f : y;          // NaN stays NaN
      case kActSilu:    return y * sigmoid_f32(y);
      case kActGelu:    return 0.5f * y * (1.0f + erff(y * 0.70710678118654752f));
      case kActSigmoid: return sigmoid_f32(y);
      default:          return y;
   }
}

// N consecutive elements; the pointer needs the element's alignment only (gfx950 serves unaligned vector accesses; an aligned address costs no more)
template <typename T, int N> struct __attribute__((packed)) Pack { T v[N]; };
template <typename T, int N> __device__ __forceinline__ void load_f32(const T *p, float (&f)[N])
{
   const Pack<T, N> u = *reinterpret_cast<const Pack<T, N> *>(p);
#pragma unroll
   for (int i = 0; i < N; ++i) f[i] = (float)u.v[i];
}
template <typename T, int N> __device__ __forceinline__ void store_f32(T *p, const float (&f)[N])
{
   Pack<T, N> u;
#pragma unroll
   for (int i = 0; i < N; ++i) u.v[i] = (T)f[i];             // round to nearest even, once
   *reinterpret_cast<Pack<T, N> *>(p) = u;
}

// sum over the 2^k lanes that differ in the low bits (k = log2(width)); every lane gets it, in the same order of additions
__device__ __forceinline__ float sum_lanes(float v, int width)
{
   for (int d = 1; d < width; d <<= 1) v += __shfl_xor(v, d);
   return v;
}

}  // namespace ops
}  // namespace vadc
