// kernels_ops_linear.hip -- out = act(x W^T + b) + r  (or act(x W^T + b + r)): matrix product with its epilogue, any sizes and row strides.
#include "ops_internal.h"
#include "ops_prims.h"

namespace vadc {
namespace ops {

// The epilogue of 4 consecutive output features of one row: bias, residual, activation in float32, one rounding at the end.
template <typename T>
__device__ __forceinline__ void finish4(const vadc_amd_linear_args &a, int64_t row, int64_t col, const f4 &acc)
{
   const int64_t left = a.out_features - col;
   if (row >= a.rows || left <= 0) return;
   const T *bias = (const T *)a.bias, *res = (const T *)a.residual + row * a.residual_stride;
   T *out = (T *)a.out + row * a.out_stride;
   float y[4] = {acc[0], acc[1], acc[2], acc[3]}, b[4] = {0, 0, 0, 0}, r[4] = {0, 0, 0, 0};
   if (left >= 4) {
      if (a.bias) load_f32<T, 4>(bias + col, b);
      if (a.residual) load_f32<T, 4>(res + col, r);
   } else {
      for (int i = 0; i < left; ++i) {
         if (a.bias) b[i] = (float)bias[col + i];
         if (a.residual) r[i] = (float)res[col + i];
      }
   }
#pragma unroll
   for (int i = 0; i < 4; ++i) {
      y[i] += b[i];
      if (a.residual && a.residual_first) y[i] += r[i];
      y[i] = activate(y[i], a.activation);
      if (a.residual && !a.residual_first) y[i] += r[i];
   }
   if (left >= 4) store_f32<T, 4>(out + col, y);
   else for (int i = 0; i < left; ++i) out[col + i] = (T)y[i];
}

// 64 x 64 outputs per workgroup of four waves, float32 matrix instructions on operands converted to float32 on their way into LDS.  The weight is the A operand,
// so that a lane's four accumulators are four consecutive features of one row.
constexpr int kPitch = 36;       // floats per LDS row of 32: 16-byte aligned, and eight consecutive rows start in different banks
template <typename T>
__global__ __launch_bounds__(256) void k_linear(const vadc_amd_linear_args a)
{
   __shared__ float sx[64 * kPitch], sw[64 * kPitch];
   const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
   const int64_t tiles_n = (a.out_features + 63) / 64;
   const int64_t row0 = (blockIdx.x / tiles_n) * 64, col0 = (blockIdx.x % tiles_n) * 64;
   const int r = tid >> 2, c = (tid & 3) * 8;                        // a thread stages 8 consecutive k of one row of each operand
   const T *px = (const T *)a.x + (row0 + r) * a.x_stride, *pw = (const T *)a.weight + (col0 + r) * a.weight_stride;
   const bool okx = row0 + r < a.rows, okw = col0 + r < a.out_features;
   f4 acc[2][2] = {};
   const int wr = (wave & 1) * 32, wc = (wave >> 1) * 32;
   for (int64_t k = 0; k < a.in_features; k += 32) {
      float fx[8] = {}, fw[8] = {};
      const int64_t left = a.in_features - (k + c);
      if (left >= 8) {
         if (okx) load_f32<T, 8>(px + k + c, fx);
         if (okw) load_f32<T, 8>(pw + k + c, fw);
      } else {
         for (int i = 0; i < left; ++i) {
            if (okx) fx[i] = (float)px[k + c + i];
            if (okw) fw[i] = (float)pw[k + c + i];
         }
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) { sx[r * kPitch + c + i] = fx[i]; sw[r * kPitch + c + i] = fw[i]; }
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < 32; kk += 4) {
         float fa[2], fb[2];
#pragma unroll
         for (int i = 0; i < 2; ++i) {
            fa[i] = sw[(wc + 16 * i + (lane & 15)) * kPitch + kk + (lane >> 4)];
            fb[i] = sx[(wr + 16 * i + (lane & 15)) * kPitch + kk + (lane >> 4)];
         }
#pragma unroll
         for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[i], fb[j], acc[i][j], 0, 0, 0);
      }
   }
#pragma unroll
   for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) finish4<T>(a, row0 + wr + 16 * j + (lane & 15), col0 + wc + 16 * i + (lane >> 4) * 4, acc[i][j]);
}

template <typename T> static void launch(const vadc_amd_linear_args &a, hipStream_t s)
{
   const int64_t tiles = ((a.rows + 63) / 64) * ((a.out_features + 63) / 64);
   hipLaunchKernelGGL(k_linear<T>, dim3((unsigned)tiles), dim3(256), 0, s, a);
}

void launch_linear(const vadc_amd_linear_args &a, hipStream_t s)
{
   if (a.dtype == VADC_AMD_F32) launch<float>(a, s);
   else if (a.dtype == VADC_AMD_F16) launch<_Float16>(a, s);
   else launch<__bf16>(a, s);
}

}  // namespace ops
}  // namespace vadc
