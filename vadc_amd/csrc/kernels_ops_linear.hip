// kernels_ops_linear.hip -- out = act(x W^T + b) + r  (or act(x W^T + b + r)): matrix product with its epilogue, any sizes and row strides.
#include "ops_internal.h"
#include "ops_prims.h"

#include <algorithm>

namespace vadc {
namespace ops {

typedef float f16v __attribute__((ext_vector_type(16)));

// The epilogue of N consecutive output features of one row: bias, residual, activation in float32, one rounding at the end.  `left` features are left in the row.
template <typename T, int N> __device__ __forceinline__ void load_bias(const vadc_amd_linear_args &a, int64_t col, float (&b)[N])
{
#pragma unroll
   for (int i = 0; i < N; ++i) b[i] = 0.0f;
   const int64_t left = a.out_features - col;
   if (!a.bias || left <= 0) return;
   const T *bias = (const T *)a.bias + col;
   if (left >= N) load_f32<T, N>(bias, b);
   else
#pragma unroll
      for (int i = 0; i < N; ++i)
         if (i < left) b[i] = (float)bias[i];
}
template <typename T, int N>
__device__ __forceinline__ void finish(const vadc_amd_linear_args &a, int64_t row, int64_t col, float (&y)[N], const float (&b)[N])
{
   const int64_t left = a.out_features - col;
   if (row >= a.rows || left <= 0) return;
   const T *res = (const T *)a.residual + row * a.residual_stride + col;
   T *out = (T *)a.out + row * a.out_stride + col;
   float r[N];
#pragma unroll
   for (int i = 0; i < N; ++i) { r[i] = 0.0f; y[i] += b[i]; }
   if (a.residual) {
      if (left >= N) load_f32<T, N>(res, r);
      else
#pragma unroll
         for (int i = 0; i < N; ++i)
            if (i < left) r[i] = (float)res[i];
      if (a.residual_first)
#pragma unroll
         for (int i = 0; i < N; ++i) y[i] += r[i];
   }
   activate_all<N>(y, a.activation);
   if (a.residual && !a.residual_first)
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] += r[i];
   if (left >= N) store_f32<T, N>(out, y);
   else
#pragma unroll
      for (int i = 0; i < N; ++i)
         if (i < left) out[i] = (T)y[i];
}

// ---- operands in LDS: rows of RB = 64 or 128 bytes, 16-byte pieces, the piece index mixed with the row so that the rows of a fragment lie in different banks
template <int RB> __device__ __forceinline__ int mixed(int row, int piece) { return RB == 128 ? piece ^ ((row >> 1) & 7) : piece ^ ((row >> 2) & 3); }
template <int RB> __device__ __forceinline__ int piece_at(int row, int piece) { return row * RB + (mixed<RB>(row, piece) << 4); }

// one product step: 16 k's of a 32 x 32 tile (float32: in three bfloat16 parts, ops_prims.h)
template <typename T> struct Frag;
template <> struct Frag<__bf16> { b8 v; };
template <> struct Frag<_Float16> { h8 v; };
template <> struct Frag<float> { p8 p[3]; };
template <typename T, int RB> __device__ __forceinline__ Frag<T> load_frag(const char *tile, int row, int step, int half)
{
   Frag<T> f;
   if constexpr (sizeof(T) == 2) f.v = *reinterpret_cast<const decltype(f.v) *>(tile + piece_at<RB>(row, 2 * step + half));
   else {
      const f4 lo = *reinterpret_cast<const f4 *>(tile + piece_at<RB>(row, 4 * step + 2 * half)), hi = *reinterpret_cast<const f4 *>(tile + piece_at<RB>(row, 4 * step + 2 * half + 1));
      const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      split8<float>(x, f.p);
   }
   return f;
}
__device__ __forceinline__ f16v product(const Frag<__bf16> &a, const Frag<__bf16> &b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0); }
__device__ __forceinline__ f16v product(const Frag<_Float16> &a, const Frag<_Float16> &b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.v, b.v, c, 0, 0, 0); }
__device__ __forceinline__ f16v product(const Frag<float> &a, const Frag<float> &b, f16v c)
{
#pragma unroll
   for (int o = 2; o >= 0; --o)
#pragma unroll
      for (int i = 0; i <= o; ++i) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a.p[i]), __builtin_bit_cast(b8, b.p[o - i]), c, 0, 0, 0);
   return c;
}

// 1024 bytes (eight LDS rows) from global memory straight into LDS, 16 bytes a lane, no registers between.  The caller waits with vm_wait before a barrier; M0 is written and
// read in one statement.
__device__ __forceinline__ void dma(uint32_t lds, uint32_t offset, const void *base)
{
   asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(lds), "v"(offset), "s"(base) : "memory");
}
// the same for all lanes, and the compiler may know: a scalar register
__device__ __forceinline__ const void *uniform(const void *p)
{
   const uint64_t v = (uint64_t)(uintptr_t)p;
   const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
   return (const void *)(uintptr_t)((uint64_t)hi << 32 | lo);
}
template <int N> __device__ __forceinline__ void vm_wait() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }

// BM rows x BN features per tile, WR x WC waves of (BM / WR) x (BN / WC) outputs in 32 x 32 tiles.  The weight is the A operand: a lane's accumulators are groups of four consecutive
// features of one row.  STAGES tiles of k are in LDS or on their way there: with DMA (16-byte aligned rows) a wave waits for the oldest with a counted vmcnt -- an operation the count does
// not know of can only make it wait longer -- and one barrier a tile lets everybody read it and the next one overwrite the last; without, tiles pass through registers.
// A workgroup does every gridDim-th output tile; the next one's first tiles of k are fetched before this one's outputs leave, which takes as long as a few tiles of k.
// Outputs leave through LDS, 32 rows of 64 or 32 of the wave's features at a time in float32, so that a row's features leave (and its residuals come) as one run, 16 bytes to a lane: a
// lane's own accumulators lie in pieces of four features of 32 different rows (8192 x 4096 x 4096 bfloat16 with a residual: 340 us with stores straight from them, 260 us so).
template <typename T, int BM, int BN, int WR, int WC, int RB, int STAGES, bool DMA>
__global__ __launch_bounds__(64 * WR * WC, 512 / (64 * WR * WC)) void k_linear_tile(const vadc_amd_linear_args a)
{
   constexpr int WAVES = WR * WC, KT = RB / (int)sizeof(T), TM = BM / WR / 32, TN = BN / WC / 32, BYTES = (BM + BN) * RB, PER = 16 / (int)sizeof(T);
   constexpr int ROWS = 1024 / RB, XP = BM / ROWS / WAVES, PIECES = (BM + BN) / ROWS / WAVES;      // LDS rows of a DMA instruction; a wave's instructions for x, for both
   static_assert(BM % (ROWS * WAVES) == 0 && BN % (ROWS * WAVES) == 0, "every wave does the same");
   __shared__ __attribute__((aligned(16))) char lds[STAGES * BYTES];
   const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
   const int64_t tiles_m = (a.rows + BM - 1) / BM, tiles_n = (a.out_features + BN - 1) / BN;
   const unsigned tiles = (unsigned)(tiles_m * tiles_n);
   const int wr = wave % WR * (BM / WR), wc = wave / WR * (BN / WC);
   const int64_t whole = a.in_features / KT;                          // full tiles of k

   // this wave's instructions: of x's tile, then of the weight's, each ROWS of its rows; rows behind the last are copies of it, their outputs are dropped
   int64_t row0, col0;
   int lastx, lastw;
   const T *srcx, *srcw;
   uint32_t offset[PIECES];
   const auto row_in = [&](int p) { return ((p < XP ? p : p - XP) * WAVES + wave) * ROWS + lane / (RB / 16); };
   const auto row_of = [&](int p) { return min(row_in(p), p < XP ? lastx : lastw); };
   const auto piece_of = [&](int p) { return mixed<RB>(row_in(p), lane % (RB / 16)); };
   const auto aim = [&](unsigned index) {
      // launch order -> tile: the workgroups of one XCD (every eighth) take consecutive tiles, which go down eight row tiles before the next feature tile: their operands stay in its L2
      const unsigned x = index % 8, q = tiles / 8, r = tiles % 8;
      const int64_t id = x * q + min(x, r) + index / 8, group = id / (8 * tiles_n), first = group * 8, high = min((int64_t)8, tiles_m - first), in = id - group * 8 * tiles_n;
      row0 = (first + in % high) * BM;
      col0 = in / high * BN;
      lastx = (int)min(a.rows - 1 - row0, (int64_t)BM);
      lastw = (int)min(a.out_features - 1 - col0, (int64_t)BN);
      srcx = (const T *)a.x + row0 * a.x_stride;
      srcw = (const T *)a.weight + col0 * a.weight_stride;
      if constexpr (DMA)
#pragma unroll
         for (int p = 0; p < PIECES; ++p) offset[p] = (uint32_t)(row_of(p) * (int)((p < XP ? a.x_stride : a.weight_stride) * sizeof(T)) + 16 * piece_of(p));
   };
   const auto issue = [&](int64_t kt, int stage) {
      const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds + (uint32_t)stage * BYTES + wave * 1024;
      const void *fromx = uniform(srcx + kt * KT), *fromw = uniform(srcw + kt * KT);
#pragma unroll
      for (int p = 0; p < PIECES; ++p) dma(to + p * WAVES * 1024, offset[p], p < XP ? fromx : fromw);
   };
   const auto fetch = [&](int64_t kt, auto &h) {                      // through registers: any alignment, zeros behind the last k
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
         const int64_t k = kt * KT + piece_of(p) * PER, left = a.in_features - k;
         const T *from = p < XP ? srcx + row_of(p) * a.x_stride + k : srcw + row_of(p) * a.weight_stride + k;
         if (left >= PER) {
            const Pack<T, PER> u = *reinterpret_cast<const Pack<T, PER> *>(from);
#pragma unroll
            for (int i = 0; i < PER; ++i) h[p][i] = u.v[i];
         } else
#pragma unroll
            for (int i = 0; i < PER; ++i) h[p][i] = i < left ? from[i] : (T)0.0f;
      }
   };
   const auto place = [&](int stage, const auto &h) {
#pragma unroll
      for (int p = 0; p < PIECES; ++p) __builtin_memcpy(__builtin_assume_aligned(lds + stage * BYTES + (p * WAVES + wave) * 1024 + lane * 16, 16), &h[p], 16);
   };
   f16v acc[TN][TM];
   const auto compute = [&](int stage) {
      const char *sx = lds + stage * BYTES, *sw = sx + BM * RB;
#pragma unroll
      for (int s = 0; s < KT / 16; ++s) {
         Frag<T> fa[TN], fb[TM];
#pragma unroll
         for (int i = 0; i < TN; ++i) fa[i] = load_frag<T, RB>(sw, wc + 32 * i + (lane & 31), s, lane >> 5);
#pragma unroll
         for (int j = 0; j < TM; ++j) fb[j] = load_frag<T, RB>(sx, wr + 32 * j + (lane & 31), s, lane >> 5);
#pragma unroll
         for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) acc[i][j] = product(fa[i], fb[j], acc[i][j]);
      }
   };
   constexpr int FEATS = BN / WC >= 64 && BYTES >= WAVES * 32 * 64 * 4 ? 64 : 32, PP = FEATS / 4, OUT = PER, LPR = FEATS / OUT, RPI = 64 / LPR;      // OUT features (16 bytes) to a lane, LPR lanes to a row
   static_assert(BYTES >= WAVES * 32 * FEATS * 4, "the outputs leave through one stage");
   const auto leave = [&](int stage, int64_t row0, int64_t col0) {
      f4 *mine = reinterpret_cast<f4 *>(lds + stage * BYTES) + wave * 32 * PP;
      const auto slot = [&](int row, int piece) { return row * PP + (piece ^ (PP == 8 ? (row >> 1) & 7 : row & (PP - 1))); };
#pragma unroll
      for (int h = 0; h < TN * 32 / FEATS; ++h) {
         const int64_t col = col0 + wc + h * FEATS + OUT * (lane % LPR);
         float bias[OUT];
         load_bias<T, OUT>(a, col, bias);
#pragma unroll
         for (int j = 0; j < TM; ++j) {
#pragma unroll
            for (int i = 0; i < FEATS / 32; ++i)
#pragma unroll
               for (int g = 0; g < 4; ++g) {
                  const f16v &c = acc[h * (FEATS / 32) + i][j];
                  mine[slot(lane & 31, 8 * i + 2 * g + (lane >> 5))] = f4{c[4 * g], c[4 * g + 1], c[4 * g + 2], c[4 * g + 3]};
               }
#pragma unroll
            for (int k = 0; k < 32 / RPI; ++k) {
               const int row = k * RPI + lane / LPR;
               float y[OUT];
#pragma unroll
               for (int p = 0; p < OUT / 4; ++p) {
                  const f4 c = mine[slot(row, OUT / 4 * (lane % LPR) + p)];
#pragma unroll
                  for (int e = 0; e < 4; ++e) y[4 * p + e] = c[e];
               }
               finish<T, OUT>(a, row0 + wr + 32 * j + row, col, y, bias);
            }
         }
      }
   };

   unsigned index = blockIdx.x;
   aim(index);
   int stage = 0;                                                     // of the next tile of k
   const auto step = [](int stage, int by) { const int s = stage + by; return s < STAGES ? s : s - STAGES; };
   const int ahead = (int)min(whole, (int64_t)(STAGES - 1));
   if constexpr (DMA)
      for (int i = 0; i < ahead; ++i) issue(i, step(stage, i));
   for (;;) {
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
         for (int j = 0; j < TM; ++j) acc[i][j] = (f16v)(0.0f);
      if constexpr (DMA) {
         if (a.in_features % KT) {                                    // the part of a tile at the end comes first, through registers, into the stage that is free
            T part[PIECES][PER];
            fetch(whole, part);
            lds_barrier();
            place(step(stage, STAGES - 1), part);
            lds_barrier();
            compute(step(stage, STAGES - 1));
         }
         for (int64_t kt = 0; kt < whole; ++kt) {
            if (whole - kt >= STAGES - 1) vm_wait<PIECES * (STAGES - 2)>(); else vm_wait<0>();
            lds_barrier();
            if (kt + STAGES - 1 < whole) issue(kt + STAGES - 1, step(stage, STAGES - 1));
            compute(stage);
            stage = step(stage, 1);
         }
      } else {
         const int64_t all = (a.in_features + KT - 1) / KT;
         T held[PIECES][PER];
         if (all) { fetch(0, held); lds_barrier(); place(0, held); }
         for (int64_t kt = 0; kt < all; ++kt) {
            if (kt + 1 < all) fetch(kt + 1, held);
            lds_barrier();
            compute((int)(kt & 1));
            if (kt + 1 < all) place((int)((kt + 1) & 1), held);       // its readers are behind the barrier above
         }
      }
      if constexpr (sizeof(T) == 4) {
         // An infinity times a part that is zero makes a NaN, and a value whose first part rounds to infinity one too: a wave that finds one does its outputs again, on the float32
         // pipe, straight from memory.  Every NaN of the definition ends here as well and stays one.
         bool nan = false;
#pragma unroll
         for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j)
#pragma unroll
               for (int e = 0; e < 16; ++e) nan |= acc[i][j][e] != acc[i][j][e];
         if (__any(nan)) {
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
               for (int j = 0; j < TM; ++j) {
                  const float *px = (const float *)a.x + min(row0 + wr + 32 * j + (lane & 31), a.rows - 1) * a.x_stride;
                  const float *pw = (const float *)a.weight + min(col0 + wc + 32 * i + (lane & 31), a.out_features - 1) * a.weight_stride;
                  acc[i][j] = (f16v)(0.0f);
#pragma unroll 1
                  for (int64_t k = lane >> 5; k - (lane >> 5) < a.in_features; k += 2) {
                     const bool in = k < a.in_features;
                     acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(in ? pw[k] : 0.0f, in ? px[k] : 0.0f, acc[i][j], 0, 0, 0);
                  }
               }
         }
      }
      lds_barrier();                                                  // everybody has read the last tile of k: its stage is free
      const int64_t row = row0, col = col0;
      index += gridDim.x;
      const bool more = index < tiles;
      if (more) {
         aim(index);
         if constexpr (DMA)
            for (int i = 0; i < ahead; ++i) issue(i, step(stage, i));
      }
      leave(DMA ? step(stage, STAGES - 1) : 0, row, col);
      if (!more) break;
   }
}

// ---- few rows: the weight goes once through registers, nothing is shared -------------------------------------------------------------------------------
// A workgroup does 16 features of up to 16 TM rows; its eight waves take every eighth 64 k's and add up in LDS in a fixed order.  A lane reads 32 (float32: 64) consecutive bytes of its
// row, so that the four lanes of a row read a run: the k's of an operand fragment may come in any order that both operands share.
template <typename T, int TM>
__global__ __launch_bounds__(512) void k_linear_narrow(const vadc_amd_linear_args a)
{
   constexpr int WAVES = 8;
   __shared__ __attribute__((aligned(16))) f4 part[WAVES][TM][64];
   const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l15 = lane & 15, l4 = lane >> 4;
   const int64_t tiles_n = (a.out_features + 15) / 16, row0 = blockIdx.x / tiles_n * (16 * TM), col0 = blockIdx.x % tiles_n * 16;
   const T *pw = (const T *)a.weight + min(col0 + l15, a.out_features - 1) * a.weight_stride, *px[TM];
#pragma unroll
   for (int j = 0; j < TM; ++j) px[j] = (const T *)a.x + min(row0 + 16 * j + l15, a.rows - 1) * a.x_stride;
   f4 acc[TM];
#pragma unroll
   for (int j = 0; j < TM; ++j) acc[j] = (f4)(0.0f);
   const auto load16 = [&](const T *p, int64_t k, T (&x)[16]) {
      const int64_t left = a.in_features - k;
      if (left >= 16) {
         const Pack<T, 16> u = *reinterpret_cast<const Pack<T, 16> *>(p + k);
#pragma unroll
         for (int i = 0; i < 16; ++i) x[i] = u.v[i];
      } else
#pragma unroll
         for (int i = 0; i < 16; ++i) x[i] = i < left ? p[k + i] : (T)0.0f;
   };
   for (int64_t k = 64 * wave; k < a.in_features; k += 64 * WAVES) {
      T w[16], x[TM][16];
      load16(pw, k + 16 * l4, w);
#pragma unroll
      for (int j = 0; j < TM; ++j) load16(px[j], k + 16 * l4, x[j]);
#pragma unroll
      for (int j = 0; j < TM; ++j) {
         if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int s = 0; s < 16; ++s) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[s], x[j][s], acc[j], 0, 0, 0);
         } else {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
               Frag<T> fa, fb;
#pragma unroll
               for (int i = 0; i < 8; ++i) { fa.v[i] = w[8 * s + i]; fb.v[i] = x[j][8 * s + i]; }
               if constexpr (__is_same(T, __bf16)) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa.v, fb.v, acc[j], 0, 0, 0);
               else acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa.v, fb.v, acc[j], 0, 0, 0);
            }
         }
      }
   }
#pragma unroll
   for (int j = 0; j < TM; ++j) part[wave][j][lane] = acc[j];
   __syncthreads();
   for (int j = wave; j < TM; j += WAVES) {
      f4 sum = part[0][j][lane];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) sum += part[w][j][lane];
      float y[4] = {sum[0], sum[1], sum[2], sum[3]}, bias[4];
      load_bias<T, 4>(a, col0 + 4 * l4, bias);
      finish<T, 4>(a, row0 + 16 * j + l15, col0 + 4 * l4, y, bias);
   }
}

// ---- choice ---------------------------------------------------------------------------------------------------------------------------------------------
template <typename T, int BM, int BN, int WR, int WC, int RB, int STAGES> static void launch_tile(const vadc_amd_linear_args &a, hipStream_t s, bool dma)
{
   constexpr int64_t slots = 256 * (512 / (64 * WR * WC));             // 512 threads a CU at a time
   const dim3 grid((unsigned)std::min(slots, ((a.rows + BM - 1) / BM) * ((a.out_features + BN - 1) / BN)));
   if (dma) hipLaunchKernelGGL((k_linear_tile<T, BM, BN, WR, WC, RB, STAGES, true>), grid, dim3(64 * WR * WC), 0, s, a);
   else hipLaunchKernelGGL((k_linear_tile<T, BM, BN, WR, WC, RB, 2, false>), grid, dim3(64 * WR * WC), 0, s, a);
}
template <typename T, int TM> static void launch_narrow(const vadc_amd_linear_args &a, hipStream_t s)
{
   hipLaunchKernelGGL((k_linear_narrow<T, TM>), dim3((unsigned)(((a.rows + 16 * TM - 1) / (16 * TM)) * ((a.out_features + 15) / 16))), dim3(512), 0, s, a);
}
template <typename T> static void launch(const vadc_amd_linear_args &a, hipStream_t s)
{
   if (a.rows <= 16) return launch_narrow<T, 1>(a, s);
   if (a.rows <= 64) return launch_narrow<T, 4>(a, s);
   constexpr int64_t per = 16 / sizeof(T);
   const bool dma = ((uintptr_t)a.x | (uintptr_t)a.weight) % 16 == 0 && a.x_stride % per == 0 && a.weight_stride % per == 0 &&
                    std::max(a.x_stride, a.weight_stride) * (int64_t)sizeof(T) < (int64_t(1) << 31) / 256;      // a tile's rows within 32-bit offsets
   const auto tiles = [&](int64_t t) { return ((a.rows + t - 1) / t) * ((a.out_features + t - 1) / t); };
   if constexpr (sizeof(T) == 2) if (tiles(256) >= 200) return launch_tile<T, 256, 256, 2, 4, 128, 2>(a, s, dma);
   if (tiles(128) >= 200) return launch_tile<T, 128, 128, 2, 2, 128, 2>(a, s, dma);
   launch_tile<T, 64, 64, 2, 2, 128, 4>(a, s, dma);
}

void launch_linear(const vadc_amd_linear_args &a, hipStream_t s)
{
   if (a.dtype == VADC_AMD_F32) launch<float>(a, s);
   else if (a.dtype == VADC_AMD_F16) launch<_Float16>(a, s);
   else launch<__bf16>(a, s);
}

}  // namespace ops
}  // namespace vadc
