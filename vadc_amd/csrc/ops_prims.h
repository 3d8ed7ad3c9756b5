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

// 1 / (1 + e^-y) on the hardware's exponential and reciprocal (1 ulp each), for an output of type T.  t = -y log2(e) rounded puts e^-y off by |y| 2^-24 relative.  Where the output is float32, t is
// carried in two parts: good to three float32 steps up to |y| = 80 (with one part 63 there, 16 at 20); from there on the second part is left out, since beside 1 the exponential is nothing, or
// its reciprocal is about to be.  An output of 16 bits has no use for it: up to |y| = 16 one part is off by 2^-20 of a value that is rounded by up to 2^-12 (fp16) or 2^-9 (49152 x 4096
// bfloat16 group norm with a SiLU gate: 232 us so, 248 with both parts).  e^-y = inf gives 0, as the division would
template <typename T> __device__ __forceinline__ float sigmoid_f32(float y)
{
   constexpr float log2e = 1.44269504f, rest = 1.92596299e-8f, ln2 = 0.693147181f;      // log2e + rest = log2(e)
   const float t = y * -log2e;
   float e = __builtin_amdgcn_exp2f(t);
   if constexpr (sizeof(T) == 4) {
      const float r = fmaf(y, -rest, fmaf(y, -log2e, -t));                              // t + r = -y log2(e)
      e = fabsf(y) < 80.0f ? fmaf(e, r * ln2, e) : e;
   }
   return __builtin_amdgcn_rcpf(1.0f + e);
}

// gelu by the complement: 1 + erf loses every digit of a negative tail (y = -5: a tenth of the value, y = -6: all of it).  What is left is the argument's rounding, y^2 2^-23 relative, and
// erfc's own.  (1111 x 1000 x 1537 bfloat16 with it: 13.95 us, with 1 + erf 13.75)
template <typename T> __device__ __forceinline__ float activate(float y, int act)
{
   switch (act) {
      case kActRelu:    return y < 0.0f ? 0.0f : y;          // NaN stays NaN
      case kActSilu:    return y * sigmoid_f32<T>(y);
      case kActGelu:    return 0.5f * y * erfcf(y * -0.70710678118654752f);
      case kActSigmoid: return sigmoid_f32<T>(y);
      default:          return y;
   }
}

template <typename T, int N> __device__ __forceinline__ void activate_all(float (&y)[N], int act)      // one branch for all
{
   if (act == kActNone) return;
   if (act == kActRelu) {
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = activate<T>(y[i], kActRelu);
   } else if (act == kActSilu) {
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = activate<T>(y[i], kActSilu);
   } else if (act == kActGelu) {
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = activate<T>(y[i], kActGelu);
   } else {
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = activate<T>(y[i], kActSigmoid);
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
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef u4 p8;                                                       // eight values' one part: an operand.  In whole words: the compiler takes vectors of 16 bits apart
typedef u2 p4;
// the next part of two values, packed, taken off them
__device__ __forceinline__ uint32_t next_part(f2 &rest)
{
   const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, b2));
   rest[0] -= __builtin_bit_cast(float, w << 16);
   rest[1] -= __builtin_bit_cast(float, w & 0xffff0000u);
   return w;
}
template <typename T> __device__ __forceinline__ void split8(const T (&x)[8], p8 (&p)[Parts<T>::n])
{
   if constexpr (Parts<T>::n == 1) {
      __builtin_memcpy(&p[0], x, sizeof(p8));
   } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
         f2 rest = {(float)x[2 * i], (float)x[2 * i + 1]};
#pragma unroll
         for (int k = 0; k < Parts<T>::n; ++k) p[k][i] = next_part(rest);
      }
   }
}
template <int N> __device__ __forceinline__ void split4(const f4 &x, p4 (&p)[N])
{
   f2 lo = {x[0], x[1]}, hi = {x[2], x[3]};
#pragma unroll
   for (int k = 0; k < N; ++k) p[k] = p4{next_part(lo), next_part(hi)};
}
__device__ __forceinline__ p8 join(const p4 &lo, const p4 &hi) { return p8{lo[0], lo[1], hi[0], hi[1]}; }
__device__ __forceinline__ f4 mfma16(const p8 &a, const p8 &b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0); }
// acc += a . b over 32 k's, operands in NA and NB parts: the small products first
template <int NA, int NB> __device__ __forceinline__ f4 mfma_parts(const p8 (&a)[NA], const p8 (&b)[NB], f4 acc)
{
#pragma unroll
   for (int o = 2; o >= 0; --o)
#pragma unroll
      for (int i = 0; i < NA; ++i)
         if (o - i >= 0 && o - i < NB) acc = mfma16(a[i], b[o - i], acc);
   return acc;
}
// two of them at once, product by product: the matrix pipe has the other's while one's result is under way
template <int NA, int NB, int NC, int ND>
__device__ __forceinline__ void mfma_parts2(const p8 (&a)[NA], const p8 (&b)[NB], f4 &x, const p8 (&c)[NC], const p8 (&d)[ND], f4 &y)
{
#pragma unroll
   for (int o = 2; o >= 0; --o)
#pragma unroll
      for (int i = 0; i <= o; ++i) {
         if (i < NA && o - i < NB) x = mfma16(a[i], b[o - i], x);
         if (i < NC && o - i < ND) y = mfma16(c[i], d[o - i], y);
      }
}

// LDS is ready for the other waves and theirs for this one; global loads stay in flight (__syncthreads would wait for them)
__device__ __forceinline__ void lds_barrier()
{
   asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
   __builtin_amdgcn_s_barrier();
   asm volatile("" ::: "memory");
}

// The same past the caches, for outputs larger than the L2s together (32 MB): none of it would be left when it is read, and it leaves them to the operands (6 x 20011 x 384 float32 group norm
// 64 -> 56 us, 98304 x 512 float32 outputs of linear 109 -> 101 us, 8192 x 4096 bfloat16 257 -> 251 us).  Smaller ones stay for whoever reads them next.
constexpr int64_t kStreamBytes = int64_t(32) << 20;
template <typename T, int N> __device__ __forceinline__ void stream_f32(T *p, const float (&f)[N])
{
   if constexpr (sizeof(T) * N == 16) {
      typedef uint32_t words __attribute__((ext_vector_type(4), aligned(2)));      // (as Pack: any element's alignment)
      T u[N];
#pragma unroll
      for (int i = 0; i < N; ++i) u[i] = (T)f[i];
      words w;
      __builtin_memcpy(&w, u, sizeof(w));
      __builtin_nontemporal_store(w, reinterpret_cast<words *>(p));
   } else store_f32<T, N>(p, f);
}

// sum over the 2^k lanes that differ in the low bits (k = log2(width)); every lane gets it, the same bits.  Inside 16 lanes a neighbour's value is an operand modifier (quad permutations,
// then mirrors, whose lanes hold the same sums as the ones eight and four away), between the rows of 16 a swap: a tenth of the time of six reads through the LDS crossbar
template <int CTRL> __device__ __forceinline__ float plus_dpp(float v)
{
   return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float plus_row(float v)                   // the row of 16 beside
{
   const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
   return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}
__device__ __forceinline__ float plus_half(float v)                  // the other 32 lanes
{
   const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
   return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}
__device__ __forceinline__ float sum_lanes(float v, int width)
{
   if (width > 1) v = plus_dpp<0xb1>(v);                             // quad_perm [1,0,3,2]
   if (width > 2) v = plus_dpp<0x4e>(v);                             // quad_perm [2,3,0,1]
   if (width > 4) v = plus_dpp<0x141>(v);                            // row_half_mirror
   if (width > 8) v = plus_dpp<0x140>(v);                            // row_mirror
   if (width > 16) v = plus_row(v);
   if (width > 32) v = plus_half(v);
   return v;
}

}  // namespace ops
}  // namespace vadc
