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

// 1 / (1 + e^-y) on the hardware's exponential and reciprocal (1 ulp each; the product -y log2(e) rounds once: e^-y is off by |y| 2^-24 relative, where it is as small as it
// counts); e^-y = inf gives 0, as the division would
__device__ __forceinline__ float sigmoid_f32(float y) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y * -1.4426950408889634f)); }

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

// ---- a value as a sum of bfloat16 parts ---------------------------------------------------------------------------------------------------------------------
// float32 = three parts (8 bits each, rounded to nearest: what is left out is below 2^-25 of the value), fp16 = two, bf16 = one: products of parts are exact in float32, so that a
// product of float32 accuracy runs on the bf16 matrix pipe.  Products of parts i, j with i + j > 2 are below 2^-24 of the whole and left out.  An infinity becomes (inf, NaN, NaN).
template <typename T> struct Parts;
template <> struct Parts<__bf16> { static constexpr int n = 1; };
template <> struct Parts<_Float16> { static constexpr int n = 2; };
template <> struct Parts<float> { static constexpr int n = 3; };
template <typename T> __device__ __forceinline__ void split8(const T (&x)[8], b8 (&p)[Parts<T>::n])
{
   if constexpr (Parts<T>::n == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[0][i] = x[i];
   } else {
      float rest[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) rest[i] = (float)x[i];
#pragma unroll
      for (int k = 0; k < Parts<T>::n; ++k)
#pragma unroll
         for (int i = 0; i < 8; ++i) { p[k][i] = (__bf16)rest[i]; rest[i] -= (float)p[k][i]; }
   }
}
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void split4(const f4 &x, b4 (&p)[3])
{
   f4 rest = x;
#pragma unroll
   for (int k = 0; k < 3; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) { p[k][i] = (__bf16)rest[i]; rest[i] -= (float)p[k][i]; }
}
// acc += a . b over 32 k's, operands in NA and NB parts: the small products first
template <int NA, int NB> __device__ __forceinline__ f4 mfma_parts(const b8 (&a)[NA], const b8 (&b)[NB], f4 acc)
{
#pragma unroll
   for (int o = 2; o >= 0; --o)
#pragma unroll
      for (int i = 0; i < NA; ++i)
         if (o - i >= 0 && o - i < NB) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[o - i], acc, 0, 0, 0);
   return acc;
}
// two of them at once, product by product: the matrix pipe has the other's while one's result is under way
template <int NA, int NB> __device__ __forceinline__ void mfma_parts2(const b8 (&a)[NA], const b8 (&b)[NB], f4 &x, const b8 (&c)[NA], const b8 (&d)[NB], f4 &y)
{
#pragma unroll
   for (int o = 2; o >= 0; --o)
#pragma unroll
      for (int i = 0; i < NA; ++i)
         if (o - i >= 0 && o - i < NB) {
            x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[o - i], x, 0, 0, 0);
            y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(c[i], d[o - i], y, 0, 0, 0);
         }
}

// LDS is ready for the other waves and theirs for this one; global loads stay in flight (__syncthreads would wait for them)
__device__ __forceinline__ void lds_barrier()
{
   asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
   __builtin_amdgcn_s_barrier();
   asm volatile("" ::: "memory");
}

// sum over the 2^k lanes that differ in the low bits (k = log2(width)); every lane gets it, in the same order of additions
__device__ __forceinline__ float sum_lanes(float v, int width)
{
   for (int d = 1; d < width; d <<= 1) v += __shfl_xor(v, d);
   return v;
}

}  // namespace ops
}  // namespace vadc
