// kernels_ops_delta.hip -- the gated delta rule with one state [key_dim][value_dim] per stream and head:
//   S' = e^g S;  u = beta (v - S'^T k);  S = S' + k u^T;  o = scale S^T q
#include "ops_internal.h"
#include "ops_prims.h"

namespace vadc {
namespace ops {

__device__ __forceinline__ int64_t live_steps(const vadc_amd_gated_delta_args &a, int64_t stream)
{
   if (!a.lengths) return a.steps;
   const int64_t v = a.lengths[stream];
   return v < 0 ? 0 : v > a.steps ? a.steps : v;
}

// Step by step.  A workgroup holds 16 VEC columns of one state in registers: thread (r, c) the rows r, r + 16, ... of VEC columns.  S^T k and S^T q of the OLD state
// come out of one reduction, because S^T q = e^g S_old^T q + (k . q) u.  Unit length of q and k is a factor behind the sums.
template <typename T, int VEC, int ROWS>
__global__ __launch_bounds__(256) void k_delta_step(const vadc_amd_gated_delta_args a)
{
   constexpr int COLS = 16 * VEC;
   __shared__ float sq[2][16 * ROWS], sk[2][16 * ROWS], dots[2][4][3], part[2][4][2][COLS];
   const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = tid >> 4, c = (tid & 15) * VEC;
   const int64_t tiles = (a.value_dim + COLS - 1) / COLS;
   const int64_t tile = blockIdx.x % tiles, head = blockIdx.x / tiles % a.heads, stream = blockIdx.x / tiles / a.heads;
   const int64_t col = tile * COLS + c;
   const int kd = (int)a.key_dim;
   const bool live = col < a.value_dim;                              // VEC divides value_dim
   const int64_t kh = head / (a.heads / a.key_heads), steps = live_steps(a, stream);
   if (!steps) return;
   float *state = a.state + stream * a.state_stride + head * a.key_dim * a.value_dim + col;
   float s[ROWS][VEC];
#pragma unroll
   for (int i = 0; i < ROWS; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[i][j] = 0.0f;
      if (live && r + 16 * i < kd) load_f32<float, VEC>(state + (int64_t)(r + 16 * i) * a.value_dim, s[i]);
   }
   const T *q = (const T *)a.q + stream * a.q_stride[0] + kh * a.q_stride[2], *k = (const T *)a.k + stream * a.k_stride[0] + kh * a.k_stride[2];
   const T *v = (const T *)a.v + stream * a.v_stride[0] + head * a.v_stride[2] + col;
   T *out = (T *)a.out + stream * a.out_stride[0] + head * a.out_stride[2] + col;
   const float *pg = a.log_decay + stream * a.decay_stride[0] + head, *pb = a.beta + stream * a.beta_stride[0] + head;
   for (int64_t t = 0; t < steps; ++t) {
      const int at = t & 1;                                          // two sets of LDS buffers: two barriers a step
      const float decay = expf(pg[t * a.decay_stride[1]]), beta = pb[t * a.beta_stride[1]];
      float vv[VEC] = {};
      if (live) load_f32<T, VEC>(v + t * a.v_stride[1], vv);
      float qi = 0.0f, ki = 0.0f;
      if (tid < kd) { qi = (float)q[t * a.q_stride[1] + tid]; ki = (float)k[t * a.k_stride[1] + tid]; }
      if (tid < 16 * ROWS) { sq[at][tid] = qi; sk[at][tid] = ki; }
      const float qq = sum_lanes(qi * qi, 64), kk = sum_lanes(ki * ki, 64), qk = sum_lanes(qi * ki, 64);
      if (lane == 0) { dots[at][wave][0] = qq; dots[at][wave][1] = kk; dots[at][wave][2] = qk; }
      __syncthreads();
      float d[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) d[i] = (dots[at][0][i] + dots[at][1][i]) + (dots[at][2][i] + dots[at][3][i]);
      const float rq = a.normalize ? a.scale / sqrtf(d[0] + 1e-6f) : a.scale, rk = a.normalize ? 1.0f / sqrtf(d[1] + 1e-6f) : 1.0f;
      float ks[VEC] = {}, qs[VEC] = {};
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
#pragma unroll
         for (int j = 0; j < VEC; ++j) {
            ks[j] = fmaf(sk[at][r + 16 * i], s[i][j], ks[j]);
            qs[j] = fmaf(sq[at][r + 16 * i], s[i][j], qs[j]);
         }
#pragma unroll
      for (int j = 0; j < VEC; ++j) {                                // the wave's four rows of threads
         ks[j] += __shfl_xor(ks[j], 16); ks[j] += __shfl_xor(ks[j], 32);
         qs[j] += __shfl_xor(qs[j], 16); qs[j] += __shfl_xor(qs[j], 32);
      }
      if (lane < 16)
#pragma unroll
         for (int j = 0; j < VEC; ++j) { part[at][wave][0][c + j] = ks[j]; part[at][wave][1][c + j] = qs[j]; }
      __syncthreads();
      float o[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
         const float fk = (part[at][0][0][c + j] + part[at][1][0][c + j]) + (part[at][2][0][c + j] + part[at][3][0][c + j]);
         const float fq = (part[at][0][1][c + j] + part[at][1][1][c + j]) + (part[at][2][1][c + j] + part[at][3][1][c + j]);
         const float u = beta * (vv[j] - decay * rk * fk);
         o[j] = rq * (decay * fq + d[2] * rk * u);
         const float ku = rk * u;
#pragma unroll
         for (int i = 0; i < ROWS; ++i) s[i][j] = fmaf(sk[at][r + 16 * i], ku, decay * s[i][j]);
      }
      if (r == 0 && live) store_f32<T, VEC>(out + t * a.out_stride[1], o);
   }
#pragma unroll
   for (int i = 0; i < ROWS; ++i)
      if (live && r + 16 * i < kd) store_f32<float, VEC>(state + (int64_t)(r + 16 * i) * a.value_dim, s[i]);
}

template <typename T, int VEC, int ROWS> static void launch_step(const vadc_amd_gated_delta_args &a, hipStream_t s)
{
   const int64_t tiles = (a.value_dim + 16 * VEC - 1) / (16 * VEC);
   hipLaunchKernelGGL((k_delta_step<T, VEC, ROWS>), dim3((unsigned)(a.streams * a.heads * tiles)), dim3(256), 0, s, a);
}
template <typename T> static void launch(const vadc_amd_gated_delta_args &a, hipStream_t s)
{
   const bool four = a.value_dim % 4 == 0;
   if (a.key_dim <= 64) four ? launch_step<T, 4, 4>(a, s) : launch_step<T, 1, 4>(a, s);
   else if (a.key_dim <= 128) four ? launch_step<T, 4, 8>(a, s) : launch_step<T, 1, 8>(a, s);
   else four ? launch_step<T, 4, 16>(a, s) : launch_step<T, 1, 16>(a, s);
}

int64_t gated_delta_workspace(const vadc_amd_gated_delta_args &) { return 0; }

void launch_gated_delta(const vadc_amd_gated_delta_args &a, hipStream_t s)
{
   if (a.dtype == VADC_AMD_F32) launch<float>(a, s);
   else if (a.dtype == VADC_AMD_F16) launch<_Float16>(a, s);
   else launch<__bf16>(a, s);
}

}  // namespace ops
}  // namespace vadc
