// kernels_ops_delta.hip -- the gated delta rule with one state [key_dim][value_dim] per stream and head:
//   S' = e^g S;  u = beta (v - S'^T k);  S = S' + k u^T;  o = scale S^T q
#include "ops_internal.h"
#include "ops_prims.h"

#include <algorithm>

namespace vadc {
namespace ops {

__device__ __forceinline__ int64_t live_steps(const vadc_amd_gated_delta_args &a, int64_t stream)
{
   if (!a.lengths) return a.steps;
   const int64_t v = a.lengths[stream];
   return v < 0 ? 0 : v > a.steps ? a.steps : v;
}

// Step by step.  A workgroup holds 16 VEC columns of one state in registers: thread (r, c) the rows r, r + 16, ... of VEC columns.  S^T k and S^T q of the OLD state
// come out of one reduction, because S^T q = e^g S_old^T q + (k . q) u.  Unit length of q and k is a factor behind the sums.  What is not finite ends in u, in every column that it reaches, or,
// of a query, in its outputs: NaN is put there, as blocks put it, so that an infinity leaves the same whichever form a call takes.
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
   // a step's operands are fetched while the one before is computed; column and row are moved inside where they lie behind the end
   const int64_t krow = min(tid, kd - 1), vback = live ? 0 : col;
   T nq, nk, nv[VEC];
   float ng, nb;
   const auto fetch = [&](int64_t t) {
      nq = q[t * a.q_stride[1] + krow]; nk = k[t * a.k_stride[1] + krow];
      const Pack<T, VEC> u = *reinterpret_cast<const Pack<T, VEC> *>(v + t * a.v_stride[1] - vback);
#pragma unroll
      for (int j = 0; j < VEC; ++j) nv[j] = u.v[j];
      ng = pg[t * a.decay_stride[1]]; nb = pb[t * a.beta_stride[1]];
   };
   fetch(0);
   for (int64_t t = 0; t < steps; ++t) {
      const int at = t & 1;                                          // two sets of LDS buffers: two barriers a step
      const float decay = expf(ng), beta = nb, qi = tid < kd ? (float)nq : 0.0f, ki = tid < kd ? (float)nk : 0.0f;
      float vv[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) vv[j] = (float)nv[j];
      if (t + 1 < steps) fetch(t + 1);
      if (tid < 16 * ROWS) { sq[at][tid] = qi; sk[at][tid] = ki; }
      const float qq = sum_lanes(qi * qi, 64), kk = sum_lanes(ki * ki, 64), qk = sum_lanes(qi * ki, 64);
      if (lane == 0) { dots[at][wave][0] = qq; dots[at][wave][1] = kk; dots[at][wave][2] = qk; }
      lds_barrier();
      float d[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) d[i] = (dots[at][0][i] + dots[at][1][i]) + (dots[at][2][i] + dots[at][3][i]);
      const float rq = a.normalize ? a.scale * __builtin_amdgcn_rsqf(d[0] + 1e-6f) : a.scale, rk = a.normalize ? __builtin_amdgcn_rsqf(d[1] + 1e-6f) : 1.0f;      // 1 ulp
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
         ks[j] = plus_half(plus_row(ks[j]));
         qs[j] = plus_half(plus_row(qs[j]));
      }
      if (lane < 16)
#pragma unroll
         for (int j = 0; j < VEC; ++j) { part[at][wave][0][c + j] = ks[j]; part[at][wave][1][c + j] = qs[j]; }
      lds_barrier();
      float o[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
         const float fk = (part[at][0][0][c + j] + part[at][1][0][c + j]) + (part[at][2][0][c + j] + part[at][3][0][c + j]);
         const float fq = (part[at][0][1][c + j] + part[at][1][1][c + j]) + (part[at][2][1][c + j] + part[at][3][1][c + j]);
         float u = beta * (vv[j] - decay * rk * fk);
         u = fabsf(u) < INFINITY ? u : NAN;
         o[j] = rq * (decay * fq + d[2] * rk * u);
         if (!(d[0] < INFINITY)) o[j] = fabsf(o[j]) < INFINITY ? o[j] : NAN;
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

// ---- blocks of 64 steps ---------------------------------------------------------------------------------------------------------------------------------
// Inside a block, with G the running sum of log_decay, a = e^G, k and q of unit length where asked (factors rk, rq; rq holds the scale):
//   A[i][j] = beta_i e^(G_i - G_j) rk_i rk_j k_i.k_j  (j < i),  T = (I + A)^-1,  P[i][j] = e^(G_i - G_j) rq_i rk_j q_i.k_j  (j <= i)
//   u = T (beta v - beta a rk (K S)),   out = a rq (Q S) + P u,   S = a_63 S + K^T (e^(G_63 - G) rk u)
// k_delta_blocks computes T, P and the factors of all blocks at once, k_delta_scan walks the blocks with S in registers.  Every product runs on the bf16 matrix pipe with its float32
// operands in three parts (ops_prims.h): float32 accuracy at three products where k and q are bfloat16, against one sixteenth of the rate on the float32 pipe.
// Steps behind a stream's last enter as k = q = v = 0, beta = 0, log_decay = 0, which leaves S and the others alone.
//
// What is not finite stays where the recurrence puts it: in its column from its step on.  A product with zeros would carry a NaN to the steps BEFORE it, so it is taken out where it
// enters (k rows, gates in k_delta_blocks; beta v - c1 x in k_delta_scan, which every non-finite operand reaches in its own step) and the column is NaN from that step on.
constexpr int kBlock = 64;
constexpr int kTiles = 6;                                            // 16 x 32 tiles of a lower triangle: rows 0, 16 need columns 0 .. 31 only
// Three parts of P, u and S also where the outputs leave in 16 bits: they are float32 sums rounded once, whatever the type.  (With two, 2^-17 of a product was left out and ten times as many
// bfloat16 outputs were rounded to the other neighbour, 0.28 % against 0.03 %, for 4 % of the time.)
struct __align__(16) BlockData {
   p8 t[kTiles][3][64], p[kTiles][3][64];                            // operand order, in parts: lane (l4, l15) has row l15, columns 4 l4 .. and 16 + 4 l4 .. of the tile
   float c1[kBlock], beta[kBlock], c2[kBlock], c3[kBlock];           // beta a rk, beta, a rq, e^(G_63 - G) rk
   float end[32];                                                    // a_63, four times; the rest keeps the next block on a line of its own
};
static_assert(sizeof(BlockData) % 128 == 0, "a block's tiles start on a cache line");
__device__ __forceinline__ int tile_of(int mt, int ks) { return mt < 2 ? mt : 2 * mt - 2 + ks; }
// LDS rows of KD bfloat16 in 16-byte pieces, the piece index mixed with the row: 16 rows' pieces of one column (an operand) and two neighbouring pieces of 4 rows and of the 4 rows
// eight further (a transposing read) lie in different places of the 256 bytes of banks
template <int KD> __device__ __forceinline__ int place(int row, int piece)
{
   const int x = row >> 1;
   const int mix = KD == 64 ? (x & 1) << 1 | (x & 4) | (x >> 1 & 1) : (row & 3) << 1 | (row & 8) | (row >> 2 & 1);
   return row * KD + 8 * (piece ^ mix);
}

// Eight elements of a row from c on, in two halves: the load from min(c, kd - 8), which always goes out and is always inside the row, and, where the value is used, what does not count:
// elements behind the row's kd, and everything where `keep` is false.  A load under a branch or with its value touched at once would be waited for on the spot.
template <typename T> struct Raw8 { uint32_t w[2 * sizeof(T)]; };
template <typename T> __device__ __forceinline__ Raw8<T> load8(const T *p)
{
   const Pack<uint32_t, 2 * (int)sizeof(T)> u = *reinterpret_cast<const Pack<uint32_t, 2 * (int)sizeof(T)> *>(p);
   Raw8<T> r;
   __builtin_memcpy(&r, &u, sizeof(r));
   return r;
}
template <typename T> __device__ __forceinline__ void trim8(Raw8<T> &r, int c, int kd, bool keep)
{
   constexpr int W = 2 * (int)sizeof(T);
   {
      const int back = c + 8 - kd;                                   // elements the load was moved back by: the row's last ones come down to the front
      const bool moved = back > 0 && back < 8;
      if (kd & 7) {
         const int n = 8 - (kd & 7);
         uint32_t v[W];
#pragma unroll
         for (int i = 0; i < W; ++i) v[i] = r.w[i];
#pragma unroll
         for (int bit = 0; bit < 3; ++bit)
            if (n >> bit & 1) {
               const int by = sizeof(T) == 4 ? 1 << bit : bit ? 1 << (bit - 1) : 0;      // words
#pragma unroll
               for (int i = 0; i < W; ++i) {
                  if (by) v[i] = i + by < W ? v[i + by] : 0u;
                  else v[i] = v[i] >> 16 | (i + 1 < W ? v[i + 1] << 16 : 0u);
               }
            }
#pragma unroll
         for (int i = 0; i < W; ++i) r.w[i] = moved ? v[i] : r.w[i];
      }
      const bool in = keep && c < kd;
#pragma unroll
      for (int i = 0; i < W; ++i) r.w[i] = in ? r.w[i] : 0u;
   }
}
// its parts, through memory of the value's own type
template <typename T> __device__ __forceinline__ void split_raw(const Raw8<T> &r, p8 (&p)[Parts<T>::n])
{
   T x[8];
   __builtin_memcpy(x, &r, sizeof(x));
   split8<T>(x, p);
}
template <typename T> struct Raw4 { uint32_t w[sizeof(T)]; };
template <typename T> __device__ __forceinline__ Raw4<T> load4(const T *p)
{
   const Pack<uint32_t, (int)sizeof(T)> u = *reinterpret_cast<const Pack<uint32_t, (int)sizeof(T)> *>(p);
   Raw4<T> r;
   __builtin_memcpy(&r, &u, sizeof(r));
   return r;
}
template <typename T> __device__ __forceinline__ f4 values4(const Raw4<T> &r)
{
   T x[4];
   __builtin_memcpy(x, &r, sizeof(x));
   return f4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
}
// the values behind the first `back`, moved to the front; zeros follow
__device__ __forceinline__ f4 trim4(f4 x, int back)
{
   const f4 one = {x[1], x[2], x[3], 0.0f};
   x = back & 1 ? one : x;
   const f4 two = {x[2], x[3], 0.0f, 0.0f}, none = {0.0f, 0.0f, 0.0f, 0.0f};
   x = back & 2 ? two : x;
   return back >= 4 ? none : x;
}
// four lanes' four values, rows for columns: lane i of the four hands its j-th value to lane j
template <int CTRL> __device__ __forceinline__ void swap_lanes(float &keep, float &give, bool second)
{
   const int got = __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, second ? keep : give), CTRL, 0xf, 0xf, true);
   keep = second ? __builtin_bit_cast(float, got) : keep;
   give = second ? give : __builtin_bit_cast(float, got);
}
__device__ __forceinline__ void transpose4(f4 &x, int lane)
{
   constexpr int kNeighbour = 0xb1, kOpposite = 0x4e;                // quad_perm [1,0,3,2] and [2,3,0,1]
   float a = x[0], b = x[1], c = x[2], d = x[3];
   swap_lanes<kNeighbour>(a, b, lane & 1); swap_lanes<kNeighbour>(c, d, lane & 1);
   swap_lanes<kOpposite>(a, c, lane & 2); swap_lanes<kOpposite>(b, d, lane & 2);
   x = f4{a, b, c, d};
}
// The A fragment of k^T from rows of k in LDS: 16 columns from c0 on, this lane's 8 rows from row on.  The transposing read hands lane i of 16 the i-th column of the 4 x 16 elements
// whose rows lanes 4 m .. 4 m + 3 point at.
template <int KD> __device__ __forceinline__ p8 load_transposed(const __bf16 *rows, int row, int c0, int l15)
{
   typedef short s4 __attribute__((ext_vector_type(4)));
   typedef __attribute__((address_space(3))) s4 *lds_s4;
   const int c = c0 + 4 * (l15 & 3);
   const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(rows + place<KD>(row + (l15 >> 2), c >> 3) + (c & 7)));
   const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(rows + place<KD>(row + 4 + (l15 >> 2), c >> 3) + (c & 7)));
   return join(__builtin_bit_cast(p4, lo), __builtin_bit_cast(p4, hi));
}

// the tiles of rows 16 mt .. from the sixteen-column pieces a lane holds of its row
__device__ __forceinline__ void store_rows(p8 (&to)[kTiles][3][64], const f4 (&x)[4], int mt, int lane)
{
#pragma unroll
   for (int s = 0; s < 2; ++s)
      if (s == 0 || mt >= 2) {
         p4 lo[3], hi[3];
         split4(x[2 * s], lo);
         split4(x[2 * s + 1], hi);
#pragma unroll
         for (int n = 0; n < 3; ++n) to[tile_of(mt, s)][n][lane] = join(lo[n], hi[n]);
      }
}

struct Segment { int64_t from, blocks; };                            // the blocks from step `from` on that one pair of launches does

// One workgroup of four waves per block.  Everything is computed transposed -- k.k and q.k as (column, row), T through T[i][j] = -(sum_m T[i][m] A[m][j]) T[j][j] -- because an accumulator
// then holds four consecutive columns of a lane's row: what the scan wants as an operand (its k order is the same permutation of the columns on both sides), so that P and T go from
// registers to memory.  The inverse runs on the float32 pipe, whose operand is the accumulator as it is.
template <typename T, int KD>
__global__ __launch_bounds__(256) void k_delta_blocks(const vadc_amd_gated_delta_args a, const Segment seg)
{
   constexpr int NT = Parts<T>::n, PITCH = kBlock + 4, KS = KD / 32;
   __shared__ __attribute__((aligned(16))) __bf16 sk[NT][kBlock * KD];
   __shared__ __attribute__((aligned(16))) float sat[kBlock * PITCH], std_[kBlock * 20];      // A transposed; the diagonal blocks of T, each transposed
   __shared__ double sg[kBlock];
   __shared__ float sbeta[kBlock], srk[kBlock], srq[kBlock];
   const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, l4 = lane >> 4;
   const int64_t block = blockIdx.x % seg.blocks, head = blockIdx.x / seg.blocks % a.heads, stream = blockIdx.x / seg.blocks / a.heads;
   const int64_t t0 = seg.from + block * kBlock;
   const int live = (int)min((int64_t)kBlock, live_steps(a, stream) - t0), kd = (int)a.key_dim;
   if (live <= 0) return;
   const bool partial = live < kBlock || kd < KD;
   const int64_t kh = head / (a.heads / a.key_heads);
   const T *q = (const T *)a.q + stream * a.q_stride[0] + t0 * a.q_stride[1] + kh * a.q_stride[2], *k = (const T *)a.k + stream * a.k_stride[0] + t0 * a.k_stride[1] + kh * a.k_stride[2];
   BlockData &out = ((BlockData *)a.workspace)[blockIdx.x];
   const int mine = 16 * wave + l15;                                 // the row of the block that this lane holds of the wave's sixteen
   Raw8<T> xk[KS], xq[KS];
   {  // rows of q in operand order; k into LDS in its parts, four threads a row
      const int row = tid >> 2;
      const T *from = k + min(row, live - 1) * a.k_stride[1];
#pragma unroll
      for (int s = 0; s < KS; ++s) xk[s] = load8(from + min(8 * ((tid & 3) + 4 * s), kd - 8));
      const T *fromq = q + min(mine, live - 1) * a.q_stride[1];
#pragma unroll
      for (int s = 0; s < KS; ++s) xq[s] = load8(fromq + min(32 * s + 8 * l4, kd - 8));
   }
   if (wave == 0) {  // G in 64 bits and in powers of two: differences of neighbours far down the block keep their digits.  e^-200 is zero in float32, as e^-inf is
      const int64_t t = t0 + min(lane, live - 1);
      float g = a.log_decay[stream * a.decay_stride[0] + t * a.decay_stride[1] + head], beta = a.beta[stream * a.beta_stride[0] + t * a.beta_stride[1] + head];
      if (lane >= live) g = beta = 0.0f;
      const bool bad = !(g < INFINITY) || !(fabsf(beta) < INFINITY);
      g = bad ? 0.0f : fmaxf(g, -200.0f);
      double sum = g * 1.4426950408889634;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) { const double o = __shfl_up(sum, d); sum += lane >= d ? o : 0.0; }
      sg[lane] = sum;
      sbeta[lane] = bad ? 0.0f : beta;
      out.beta[lane] = bad ? NAN : beta;
   }
   {
      const int row = tid >> 2;
      float kk = 0.0f, odd = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
         if (partial) trim8<T>(xk[s], 8 * ((tid & 3) + 4 * s), kd, row < live);
         T x[8];
         __builtin_memcpy(x, &xk[s], sizeof(x));
#pragma unroll
         for (int i = 0; i < 8; ++i) { const float f = (float)x[i]; kk = fmaf(f, f, kk); odd = fmaf(f, 0.0f, odd); }
      }
      kk = sum_lanes(kk, 4); odd = sum_lanes(odd, 4);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
         if (odd != 0.0f) xk[s] = Raw8<T>{};                         // NaN: an element is not finite
         p8 p[NT];
         split_raw<T>(xk[s], p);
#pragma unroll
         for (int n = 0; n < NT; ++n) *reinterpret_cast<p8 *>(&sk[n][place<KD>(row, (tid & 3) + 4 * s)]) = p[n];
      }
      if ((tid & 3) == 0) srk[row] = a.normalize ? __builtin_amdgcn_rsqf((odd != 0.0f ? 1.0f : kk) + 1e-6f) : 1.0f;
      float qq = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
         if (partial) trim8<T>(xq[s], 32 * s + 8 * l4, kd, mine < live);
         T x[8];
         __builtin_memcpy(x, &xq[s], sizeof(x));
#pragma unroll
         for (int i = 0; i < 8; ++i) { const float f = (float)x[i]; qq = fmaf(f, f, qq); }
      }
      qq = plus_half(plus_row(qq));
      if (l4 == 0) srq[mine] = a.normalize ? a.scale * __builtin_amdgcn_rsqf(qq + 1e-6f) : a.scale;
   }
   __syncthreads();
   const double gi = sg[mine];
   {
      p8 fk[KS][NT], fq[KS][NT];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
         split_raw<T>(xq[s], fq[s]);
#pragma unroll
         for (int n = 0; n < NT; ++n) fk[s][n] = *reinterpret_cast<const p8 *>(&sk[n][place<KD>(mine, 4 * s + l4)]);
      }
      const float rowk = sbeta[mine] * srk[mine], rowq = srq[mine];
      f4 p[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {                                  // columns 16 j ..
         p[j] = (f4)(0.0f);
         if (j > wave) continue;
         f4 ck = {0, 0, 0, 0}, cq = {0, 0, 0, 0};
#pragma unroll
         for (int s = 0; s < KS; ++s) {
            p8 fa[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) fa[n] = *reinterpret_cast<const p8 *>(&sk[n][place<KD>(16 * j + l15, 4 * s + l4)]);
            mfma_parts2(fa, fk[s], ck, fa, fq[s], cq);
         }
#pragma unroll
         for (int r = 0; r < 4; ++r) {
            const int c = 16 * j + 4 * l4 + r;
            const float e = c <= mine ? __builtin_amdgcn_exp2f((float)(gi - sg[c])) * srk[c] : 0.0f;
            sat[c * PITCH + mine] = c < mine ? rowk * e * ck[r] : 0.0f;
            p[j][r] = c <= mine ? rowq * e * cq[r] : 0.0f;
         }
      }
      store_rows(out.p, p, wave, lane);
   }
   __syncthreads();
   {  // T[w][w] by substitution: lane = column (the four quarters of the wave do the same); row i of the transposed A holds what row i of T gives to the rows below
      float t[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) t[i] = i == l15 ? 1.0f : 0.0f;
#pragma unroll
      for (int i = 0; i < 15; ++i) {
#pragma unroll
         for (int m4 = (i + 1) & ~3; m4 < 16; m4 += 4) {
            const f4 col = *reinterpret_cast<const f4 *>(&sat[(16 * wave + i) * PITCH + 16 * wave + m4]);
#pragma unroll
            for (int m = 0; m < 4; ++m)
               if (m4 + m > i) t[m4 + m] = fmaf(-col[m], t[i], t[m4 + m]);
         }
      }
      if (lane < 16)
#pragma unroll
         for (int i = 0; i < 16; i += 4) *reinterpret_cast<f4 *>(&std_[mine * 20 + i]) = f4{t[i], t[i + 1], t[i + 2], t[i + 3]};
   }
   __syncthreads();
   {  // wave = block row
      f4 t[4];
#pragma unroll
      for (int j = 3; j >= 0; --j) {
         t[j] = (f4)(0.0f);
         if (j > wave) continue;
         if (j == wave) {
#pragma unroll
            for (int r = 0; r < 4; ++r) t[j][r] = std_[(16 * j + 4 * l4 + r) * 20 + l15];
            continue;
         }
         f4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
#pragma unroll
         for (int m = j + 1; m < 4; ++m) {
            if (m > wave) continue;
            const f4 f = *reinterpret_cast<const f4 *>(&sat[(16 * j + l15) * PITCH + 16 * m + 4 * l4]);
#pragma unroll
            for (int s = 0; s < 4; ++s) x = __builtin_amdgcn_mfma_f32_16x16x4f32(f[s], t[m][s], x, 0, 0, 0);
         }
         const f4 f = *reinterpret_cast<const f4 *>(&std_[(16 * j + l15) * 20 + 4 * l4]);
#pragma unroll
         for (int s = 0; s < 4; ++s) y = __builtin_amdgcn_mfma_f32_16x16x4f32(f[s], x[s], y, 0, 0, 0);
         t[j] = -y;
      }
      store_rows(out.t, t, wave, lane);
   }
   if (wave == 0) {
      const float g = __builtin_amdgcn_exp2f((float)sg[lane]);
      out.c1[lane] = sbeta[lane] * g * srk[lane];
      out.c2[lane] = g * srq[lane];
      out.c3[lane] = __builtin_amdgcn_exp2f((float)(sg[kBlock - 1] - sg[lane])) * srk[lane];
      if (lane < 4) out.end[lane] = __builtin_amdgcn_exp2f((float)sg[kBlock - 1]);
   }
}

// A workgroup of four or eight waves walks the blocks of one stream and head with 16 or 32 columns of S: wave (mt, nt) does rows 16 mt .. of the block's products and rows 16 mt .., 16 mt + 64 .. of S,
// columns 16 nt ...  k and q go through registers into LDS in their parts, a block ahead, each row read once as a run; T and P come from global memory in operand order; S, r, u and the
// scaled u pass through LDS in three parts, written as four consecutive k's from the accumulators; k^T is k's rows through the transposing LDS read.  Three barriers a block.
template <typename T, int KD, int COLS>
__global__ __launch_bounds__(16 * COLS) void k_delta_scan(const vadc_amd_gated_delta_args a, const Segment seg)
{
   constexpr int NT = Parts<T>::n, KS = KD / 32, ST = KD / 64, WAVES = COLS / 4;
   __shared__ __attribute__((aligned(16))) __bf16 sk[NT][kBlock * KD], sq[NT][kBlock * KD], ss[3][COLS * KD], sr[3][COLS * kBlock], su[3][COLS * kBlock], sw[3][COLS * kBlock];
   __shared__ int spoison[COLS];
   const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, l4 = lane >> 4, mt = wave & 3, nt = wave >> 2;
   // the workgroups of one state, which read the same k, q, T and P, lie eight apart: on one XCD, behind one L2
   const unsigned tiles = (unsigned)((a.value_dim + COLS - 1) / COLS), all = gridDim.x / tiles, group = blockIdx.x / (8 * tiles), in = blockIdx.x - group * 8 * tiles, wide = min(8u, all - 8 * group);
   const int64_t tile = in / wide, which = 8 * group + in % wide, head = which % a.heads, stream = which / a.heads;
   const int64_t steps = live_steps(a, stream) - seg.from;
   if (steps <= 0) return;
   const int blocks = (int)min(seg.blocks, (steps + kBlock - 1) / kBlock), kd = (int)a.key_dim;
   const int64_t kh = head / (a.heads / a.key_heads);
   const int col = 16 * nt + l15;                                    // of this workgroup's columns
   const int64_t column = tile * COLS + col;
   const bool there = column < a.value_dim;
   const T *q = (const T *)a.q + stream * a.q_stride[0] + seg.from * a.q_stride[1] + kh * a.q_stride[2], *k = (const T *)a.k + stream * a.k_stride[0] + seg.from * a.k_stride[1] + kh * a.k_stride[2];
   const T *v = (const T *)a.v + stream * a.v_stride[0] + seg.from * a.v_stride[1] + head * a.v_stride[2] + tile * COLS;
   T *o = (T *)a.out + stream * a.out_stride[0] + seg.from * a.out_stride[1] + head * a.out_stride[2] + tile * COLS;
   const BlockData *data = (const BlockData *)a.workspace + (stream * a.heads + head) * seg.blocks;
   float *state = a.state + stream * a.state_stride + head * a.key_dim * a.value_dim + column;
   f4 S[ST];
#pragma unroll
   for (int i = 0; i < ST; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
         const int row = 64 * i + 16 * mt + 4 * l4 + r;
         S[i][r] = there && row < kd ? state[(int64_t)row * a.value_dim] : 0.0f;
      }
   if (tid < COLS) spoison[tid] = kBlock;
   bool dead = false;

   // this lane's part of the wave's rows of k and q: one piece of eight columns in every PER-th row from row0 on
   constexpr int PER = 512 / KD, LOADS = kBlock / WAVES / PER;
   const int row0 = kBlock / WAVES * wave + lane / (KD / 8), piece = lane % (KD / 8);
   Raw8<T> xk[LOADS], xq[LOADS];
   // v and out: four columns of one row per lane, turned to one column of four rows (transpose4); a group of columns that ends behind the last is read from further left
   const int vrow = 16 * mt + 4 * l4 + (l15 & 3), vcol = 16 * nt + (l15 & 12), width = (int)min((int64_t)COLS, a.value_dim - tile * COLS), vback = max(0, vcol + 4 - width);
   Raw4<T> xv;
   int64_t atk[LOADS], atq[LOADS], atv;                              // from a block's first row
   const auto aim = [&](int live) {                                  // rows behind the last are copies of it
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
         const int64_t row = min(row0 + PER * i, live - 1);
         atk[i] = row * a.k_stride[1] + min(8 * piece, kd - 8);
         atq[i] = row * a.q_stride[1] + min(8 * piece, kd - 8);
      }
      atv = min(vrow, live - 1) * a.v_stride[1] + vcol - vback;
   };
   aim(kBlock);
   const auto fetch = [&](int b) {                                   // block b's k, q, v
      const int64_t t = (int64_t)b * kBlock;
      if (steps - t < kBlock) aim((int)(steps - t));                 // the last one
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
         xk[i] = load8(k + t * a.k_stride[1] + atk[i]);
         xq[i] = load8(q + t * a.q_stride[1] + atq[i]);
      }
      xv = load4(v + t * a.v_stride[1] + atv);
   };
   // T, P and the factors of a block are fetched behind the last use of the block before: each has the better part of a block to arrive
   const auto rows4 = [&](const float *f) { return *reinterpret_cast<const f4 *>(f + 16 * mt + 4 * l4); };
   const auto tiles2 = [&](const auto &from, auto &to) {
#pragma unroll
      for (int n = 0; n < 3; ++n) {
         to[0][n] = from[tile_of(mt, 0)][n][lane];
         to[1][n] = from[tile_of(mt, mt >= 2)][n][lane];             // rows 0 .. 31 have one tile
      }
   };
   const auto rows8 = [&](const __bf16 *from, int s) {                // of this lane's column, in the order of T's and P's columns
      const p4 lo = *reinterpret_cast<const p4 *>(from + place<kBlock>(col, 4 * s + (l4 >> 1)) + 4 * (l4 & 1)), hi = *reinterpret_cast<const p4 *>(from + place<kBlock>(col, 4 * s + 2 + (l4 >> 1)) + 4 * (l4 & 1));
      return join(lo, hi);
   };
   p8 ft[2][3], fp[2][3];
   // the first block's, in the order in which the loop fetches the next one's: the compiler's counts of what is still under way hold for both then
   const auto in_order = [] { asm volatile("" ::: "memory"); };
   f4 c1 = rows4(data->c1), beta = rows4(data->beta);
   in_order();
   fetch(0);
   in_order();
   tiles2(data->t, ft);
   in_order();
   f4 c3 = rows4(data->c3);
   float end = data->end[lane & 3];                                  // a vector load: a scalar one would be waited for at the next barrier, with the LDS
   f4 c2 = rows4(data->c2);
   in_order();
   tiles2(data->p, fp);
   in_order();
   for (int b = 0; b < blocks; ++b) {
      const BlockData &next = data[min(b + 1, blocks - 1)];
      const int live = (int)min((int64_t)kBlock, steps - (int64_t)b * kBlock);
      const bool partial = live < kBlock || kd < KD;
#pragma unroll
      for (int i = 0; i < ST; ++i) {
         p4 p[3];
         split4(S[i], p);
#pragma unroll
         for (int n = 0; n < 3; ++n) *reinterpret_cast<p4 *>(&ss[n][place<KD>(col, 8 * i + 2 * mt + (l4 >> 1)) + 4 * (l4 & 1)]) = p[n];
      }
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
         const int row = row0 + PER * i;
         if (partial) { trim8<T>(xk[i], 8 * piece, kd, row < live); trim8<T>(xq[i], 8 * piece, kd, row < live); }
         p8 p[NT];
         split_raw<T>(xk[i], p);
#pragma unroll
         for (int n = 0; n < NT; ++n) *reinterpret_cast<p8 *>(&sk[n][place<KD>(row, piece)]) = p[n];
         split_raw<T>(xq[i], p);
#pragma unroll
         for (int n = 0; n < NT; ++n) *reinterpret_cast<p8 *>(&sq[n][place<KD>(row, piece)]) = p[n];
      }
      lds_barrier();
      f4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
         p8 fs[3], fk[NT], fq[NT];
#pragma unroll
         for (int n = 0; n < 3; ++n) fs[n] = *reinterpret_cast<const p8 *>(&ss[n][place<KD>(col, 4 * s + l4)]);
#pragma unroll
         for (int n = 0; n < NT; ++n) {
            fk[n] = *reinterpret_cast<const p8 *>(&sk[n][place<KD>(16 * mt + l15, 4 * s + l4)]);
            fq[n] = *reinterpret_cast<const p8 *>(&sq[n][place<KD>(16 * mt + l15, 4 * s + l4)]);
         }
         mfma_parts2(fk, fs, x, fq, fs, y);
      }
      f4 r = values4<T>(xv);
      if (live < kBlock || width < COLS) r = trim4(r, vrow < live ? vback : 4);
      transpose4(r, l15);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
         r[i] = beta[i] * r[i] - c1[i] * x[i];
      }
      if (!(fabsf(r[0]) + fabsf(r[1]) + fabsf(r[2]) + fabsf(r[3]) < INFINITY))
#pragma unroll
         for (int i = 3; i >= 0; --i)
            if (!(fabsf(r[i]) < INFINITY)) { r[i] = 0.0f; atomicMin(&spoison[col], 16 * mt + 4 * l4 + i); }
      c1 = rows4(next.c1); beta = rows4(next.beta);
      fetch(min(b + 1, blocks - 1));
      p4 p[3];
      split4(r, p);
#pragma unroll
      for (int n = 0; n < 3; ++n) *reinterpret_cast<p4 *>(&sr[n][place<kBlock>(col, 2 * mt + (l4 >> 1)) + 4 * (l4 & 1)]) = p[n];
      lds_barrier();
      const int poison = dead ? 0 : spoison[col];
      f4 u = {0, 0, 0, 0};
      {
         p8 f[2][3];
#pragma unroll
         for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int n = 0; n < 3; ++n) f[s][n] = rows8(sr[n], s);
         if (mt >= 2) {
            f4 u2 = {0, 0, 0, 0};
            mfma_parts2(ft[0], f[0], u, ft[1], f[1], u2);
            u += u2;
         } else u = mfma_parts<3, 3>(ft[0], f[0], u);
      }
      tiles2(next.t, ft);
      p8 kt[2][ST][NT];                                              // k^T, before the next block's k may take its place
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
         for (int i = 0; i < ST; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) kt[s][i][n] = load_transposed<KD>(sk[n], 32 * s + 8 * l4, 64 * i + 16 * mt, l15);
      split4(u, p);
#pragma unroll
      for (int n = 0; n < 3; ++n) *reinterpret_cast<p4 *>(&su[n][place<kBlock>(col, 2 * mt + (l4 >> 1)) + 4 * (l4 & 1)]) = p[n];
      split4(c3 * u, p);
#pragma unroll
      for (int n = 0; n < 3; ++n) *reinterpret_cast<p4 *>(&sw[n][place<kBlock>(col, 2 * mt + (l4 >> 1)) + 4 * (l4 & 1)]) = p[n];
      lds_barrier();
      if (tid < COLS) spoison[tid] = kBlock;
      c3 = rows4(next.c3);
      {  // two chains of products at a time: the rows of S this wave holds, or one of them beside the outputs
         p8 fw[2][3];
#pragma unroll
         for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int n = 0; n < 3; ++n) fw[s][n] = *reinterpret_cast<const p8 *>(&sw[n][place<kBlock>(col, 4 * s + l4)]);
#pragma unroll
         for (int i = 0; i < ST; ++i) S[i] *= end;
         end = next.end[lane & 3];
#pragma unroll
         for (int s = 0; s < 2; ++s) {
            if constexpr (ST == 2) mfma_parts2(kt[s][0], fw[s], S[0], kt[s][ST - 1], fw[s], S[ST - 1]);
            else S[0] = mfma_parts<NT, 3>(kt[s][0], fw[s], S[0]);
         }
      }
      {
         p8 f[2][3];
#pragma unroll
         for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int n = 0; n < 3; ++n) f[s][n] = rows8(su[n], s);
         y *= c2;
         if (mt >= 2) {
            f4 y2 = {0, 0, 0, 0};
            mfma_parts2(fp[0], f[0], y, fp[1], f[1], y2);
            y += y2;
         } else y = mfma_parts<3, 3>(fp[0], f[0], y);
      }
      c2 = rows4(next.c2);
      tiles2(next.p, fp);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = 16 * mt + 4 * l4 + i < poison ? y[i] : NAN;
      transpose4(y, l15);
      if (vrow < live) {
         T *to = o + ((int64_t)b * kBlock + vrow) * a.out_stride[1] + vcol;
         const float f[4] = {y[0], y[1], y[2], y[3]};
         if (!vback) store_f32<T, 4>(to, f);
         else
#pragma unroll
            for (int i = 0; i < 3; ++i)
               if (vcol + i < width) to[i] = (T)f[i];
      }
      dead = dead || poison < kBlock;
   }
#pragma unroll
   for (int i = 0; i < ST; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
         const int row = 64 * i + 16 * mt + 4 * l4 + r;
         if (there && row < kd) state[(int64_t)row * a.value_dim] = dead ? NAN : S[i][r];
      }
}

// ---- choice ---------------------------------------------------------------------------------------------------------------------------------------------
// Blocks for keys of 8 to 128 and values of 4 and more, from as many steps on as they are the faster form.  One by one a step takes 1.1 us and, with many states, more; blocks take two
// launches and whole blocks of work: 1 stream, 16 heads of 128, bfloat16: 17 us up to 64 steps, against 13.5 for 8 steps, 18 for 12 and 76 for 64; 256 streams, 4 heads of 64: 56 us, against
// 38 for 16 steps, 51 for 24 and 58 for 28; 8 heads of 128: 250 us against 139 for 16, 199 for 24, 230 for 28 and 505 for 64.  Longer keys go one by one however many steps there are (1 stream,
// 8 heads of 256 x 128: 1.4 us a step; of 128 x 128 in blocks: 0.06).
static bool in_blocks(const vadc_amd_gated_delta_args &a)
{
   return a.steps >= (a.streams * a.heads <= 256 ? 12 : 28) && a.key_dim >= 8 && a.key_dim <= 128 && a.value_dim >= 4;
}
// Columns of S per workgroup: with keys of up to 64, 16 -- several workgroups a CU, one computes while another waits at its barriers (61 streams of up to 333 steps, 6 heads of 48 x 80,
// float32: 88 us a call against 103 with 32) --; with longer keys, where staging k and q again for every 16 columns costs more than that gains, 32 (2 x 8192 steps, 32 heads of 128 x 128,
// bfloat16: 540 us against 585 with 16)
template <int KD> constexpr int scan_columns() { return KD == 64 ? 16 : 32; }
// The workspace holds 4096 blocks of 37 KB, which stay in the last-level cache between the two launches; longer calls go out in segments of steps (2 x 8192 steps, 32 heads: 540 us so,
// 560 with 2048, 535 with 8192)
static int64_t segment_blocks(const vadc_amd_gated_delta_args &a)
{
   const int64_t blocks = (a.steps + kBlock - 1) / kBlock, most = std::max<int64_t>(1, 4096 / (a.streams * a.heads));
   return std::min(blocks, most);
}
template <typename T, int KD> static void launch_blocks(const vadc_amd_gated_delta_args &a, const vadc_amd_gated_delta_args &first, hipStream_t s)
{
   constexpr int cols = scan_columns<KD>();
   const int64_t step = segment_blocks(first), tiles = (a.value_dim + cols - 1) / cols;
   for (Segment seg = {0, 0}; seg.from < a.steps; seg.from += step * kBlock) {
      seg.blocks = std::min(step, (a.steps - seg.from + kBlock - 1) / kBlock);
      hipLaunchKernelGGL((k_delta_blocks<T, KD>), dim3((unsigned)(a.streams * a.heads * seg.blocks)), dim3(256), 0, s, a, seg);
      hipLaunchKernelGGL((k_delta_scan<T, KD, cols>), dim3((unsigned)(a.streams * a.heads * tiles)), dim3(16 * cols), 0, s, a, seg);
   }
}

template <typename T> static void launch(const vadc_amd_gated_delta_args &a, const vadc_amd_gated_delta_args &first, hipStream_t s)
{
   if (in_blocks(first)) return a.key_dim <= 64 ? launch_blocks<T, 64>(a, first, s) : launch_blocks<T, 128>(a, first, s);
   const bool four = a.value_dim % 4 == 0;
   if (a.key_dim <= 64) four ? launch_step<T, 4, 4>(a, s) : launch_step<T, 1, 4>(a, s);
   else if (a.key_dim <= 128) four ? launch_step<T, 4, 8>(a, s) : launch_step<T, 1, 8>(a, s);
   else four ? launch_step<T, 4, 16>(a, s) : launch_step<T, 1, 16>(a, s);
}

int64_t gated_delta_workspace(const vadc_amd_gated_delta_args &a)
{
   return in_blocks(a) ? a.streams * a.heads * segment_blocks(a) * (int64_t)sizeof(BlockData) : 0;
}

void launch_gated_delta(const vadc_amd_gated_delta_args &a, const vadc_amd_gated_delta_args &first, hipStream_t s)
{
   if (a.dtype == VADC_AMD_F32) launch<float>(a, first, s);
   else if (a.dtype == VADC_AMD_F16) launch<_Float16>(a, first, s);
   else launch<__bf16>(a, first, s);
}

}  // namespace ops
}  // namespace vadc
