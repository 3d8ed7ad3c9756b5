// kernels_ops_linear.hip -- out = act(x W^T + b) + r  (or act(x W^T + b + r)): matrix product with its epilogue, any sizes and row strides.
#include "ops_internal.h"
#include "ops_prims.h"

#include <algorithm>
#include <type_traits>

namespace vadc {
namespace ops {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef unsigned __int128 u128;

// N pieces of 16 bytes of rows of n values: left(i) values of piece i are in its row from from(i) on (none: that points behind the row), zeros behind.  A piece that passes the end is the
// row's last 16 bytes, shifted; the loads stand together, before any branch (1111 x 1000 x 1537 bfloat16 with a load per value: 17.9 us, with a wait per piece 12.8 us, so 10.9 us)
template <typename T, int N, typename From, typename Left> __device__ __forceinline__ void load_ends(int64_t n, const From &from, const Left &left, u128 (&u)[N])
{
   constexpr int PER = 16 / (int)sizeof(T), BITS = 8 * (int)sizeof(T);
   typedef std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t> bits;
   if (n >= PER) {
#pragma unroll
      for (int i = 0; i < N; ++i) __builtin_memcpy(&u[i], from(i) - max(PER - left(i), 0), 16);
      if (n % PER)                                                    // pieces of other rows are whole or empty
#pragma unroll
         for (int i = 0; i < N; ++i) u[i] >>= min(max(PER - left(i), 0), PER - 1) * BITS;
#pragma unroll
      for (int i = 0; i < N; ++i) u[i] = left(i) <= 0 ? (u128)0 : u[i];
   } else
#pragma unroll
      for (int i = 0; i < N; ++i) {
         u[i] = 0;
#pragma unroll 1
         for (int e = min(left(i), PER) - 1; e >= 0; --e) u[i] = u[i] << BITS | __builtin_bit_cast(bits, from(i)[e]);
      }
}

// 16 values in one run.  ODD: two-byte values may begin within a dword, where a wide load takes about four times as long: whole dwords are loaded and shifted; the last dword is the one
// that the last value lies in (16 x 4095 x 4095 bfloat16: 27 us with loads from where the values begin, 11 us so; rows that need no shift lose 3 of 10 us by it)
template <typename T, bool ODD> __device__ __forceinline__ void load16(const T *from, T (&x)[16])
{
   if constexpr (!ODD) __builtin_memcpy(x, from, sizeof(x));
   else {
      static_assert(sizeof(T) == 2, "a float begins where a dword does");
      const uint32_t in = (uint32_t)(uintptr_t)from & 3;
      const char *base = (const char *)from - in;
      uint32_t d[9];
      __builtin_memcpy(d, __builtin_assume_aligned(base, 4), 32);
      __builtin_memcpy(&d[8], __builtin_assume_aligned(base + 28 + 2 * in, 4), 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = __builtin_amdgcn_alignbyte(d[i + 1], d[i], in);
      __builtin_memcpy(x, d, sizeof(x));
   }
}

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
__device__ __forceinline__ void finish(const vadc_amd_linear_args &a, const T *res, T *out, int left, float (&y)[N], const float (&b)[N])
{
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
   activate_all<T, N>(y, a.activation);
   if (a.residual && !a.residual_first)
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] += r[i];
   if (left < N) {
#pragma unroll
      for (int i = 0; i < N; ++i)
         if (i < left) out[i] = (T)y[i];
   } else if (a.rows * a.out_features * (int64_t)sizeof(T) >= kStreamBytes) stream_f32<T, N>(out, y);
   else store_f32<T, N>(out, y);
}

// Outputs leave through LDS, 32 rows of FEATS of the wave's features at a time in float32, so that a row's features leave (and its residuals come) as one run, 16 bytes to a lane: a
// lane's own accumulators lie in pieces of four features of 32 different rows (8192 x 4096 x 4096 bfloat16 with a residual: 340 us with stores straight from them, 260 us so).
// row, col: the wave's first; mine: 32 FEATS floats of its own.  KG > 1: as many waves hold sums over their part of the k's, `apart` further in LDS each; all write, and each does its
// share of the rows from the sums of all.
template <typename T, int TN, int TM, int FEATS, int KG>
__device__ __forceinline__ void leave(const vadc_amd_linear_args &a, f4 *mine, int kg, int apart, const f16v (&acc)[TN][TM], int64_t row, int64_t col, int lane)
{
   static_assert(KG == 1 || (TN == 1 && TM == 1 && FEATS == 32), "one round: the sums of all are there behind one barrier");
   constexpr int OUT = 16 / (int)sizeof(T), PP = FEATS / 4, LPR = FEATS / OUT, RPI = 64 / LPR;      // OUT features to a lane, LPR lanes to a row
   const auto slot = [&](int r, int piece) { return r * PP + (piece ^ (PP == 8 ? (r >> 1) & 7 : r & (PP - 1))); };
   const int64_t from = row + kg * RPI + lane / LPR;
#pragma unroll
   for (int h = 0; h < TN * 32 / FEATS; ++h) {
      const int64_t c = col + h * FEATS + OUT * (lane % LPR);
      const int left = (int)min((int64_t)OUT, a.out_features - c);
      float bias[OUT];
      load_bias<T, OUT>(a, c, bias);
      const T *res = (const T *)a.residual + from * a.residual_stride + c;
      T *out = (T *)a.out + from * a.out_stride + c;
#pragma unroll
      for (int j = 0; j < TM; ++j) {
#pragma unroll
         for (int i = 0; i < FEATS / 32; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
               const f16v &v = acc[h * (FEATS / 32) + i][j];
               mine[kg * apart + slot(lane & 31, 8 * i + 2 * g + (lane >> 5))] = f4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
            }
         if constexpr (KG > 1) lds_barrier();
#pragma unroll
         for (int k = 0; k < 32 / RPI / KG; ++k) {
            const int r = (k * KG + kg) * RPI + lane / LPR;
            float y[OUT];
#pragma unroll
            for (int p = 0; p < OUT / 4; ++p) {
               f4 v = mine[slot(r, OUT / 4 * (lane % LPR) + p)];
#pragma unroll
               for (int g = 1; g < KG; ++g) v += mine[g * apart + slot(r, OUT / 4 * (lane % LPR) + p)];
#pragma unroll
               for (int e = 0; e < 4; ++e) y[4 * p + e] = v[e];
            }
            if (from + 32 * j + k * KG * RPI < a.rows && left > 0) finish<T, OUT>(a, res, out, left, y, bias);
            res += KG * RPI * a.residual_stride;
            out += KG * RPI * a.out_stride;
         }
      }
   }
}

// Output tile of a launch's index: the workgroups of one XCD (every eighth) take consecutive tiles, which go down eight row tiles before the next feature tile: their operands stay in its L2
__device__ __forceinline__ void tile_of(unsigned index, unsigned tiles, int64_t tiles_m, int64_t tiles_n, int64_t &tm, int64_t &tn)
{
   const unsigned x = index % 8, q = tiles / 8, r = tiles % 8;
   const int64_t id = x * q + min(x, r) + index / 8, group = id / (8 * tiles_n), first = group * 8, high = min((int64_t)8, tiles_m - first), in = id - group * 8 * tiles_n;
   tm = first + in % high;
   tn = in / high;
}

// ---- operands in LDS: rows of RB = 64, 128 or 256 bytes, 16-byte pieces, the piece index mixed with the row so that the rows of a fragment lie in different banks
template <int RB> __device__ __forceinline__ int mixed(int row, int piece) { return RB == 256 ? piece ^ (row & 15) : RB == 128 ? piece ^ ((row >> 1) & 7) : piece ^ ((row >> 2) & 3); }
template <int RB> __device__ __forceinline__ int piece_at(int row, int piece) { return row * RB + (mixed<RB>(row, piece) << 4); }

// one product step: 16 k's of a 32 x 32 tile
__device__ __forceinline__ f16v product(const p8 &a, const p8 &b, f16v c, __bf16) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0); }
__device__ __forceinline__ f16v product(const p8 &a, const p8 &b, f16v c, _Float16) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0); }

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
   return (const void *)(const __attribute__((address_space(1))) char *)(uintptr_t)((uint64_t)hi << 32 | lo);      // global: a generic pointer's loads would count with those of LDS
}
__device__ __forceinline__ void vm_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// BM rows x BN features per tile, WR x WC waves of (BM / WR) x (BN / WC) outputs in 32 x 32 tiles.  The weight is the A operand: a lane's accumulators are groups of four consecutive
// features of one row.  Two tiles of k are in LDS, one that is read and one on its way there: with DMA (16-byte aligned rows) a wave waits for all that it has on its way -- the next tile of k,
// and, in the first step behind outputs, their stores -- and one barrier a tile lets everybody read it and the one after overwrite the last; without, tiles pass through registers.
// A workgroup does every gridDim-th output tile; the next one's first tiles of k are fetched before this one's outputs leave, which takes as long as a few tiles of k.
// KG groups of waves take every KG-th tile of k each, where there are too few output tiles to fill the device with work.
template <typename T, int BM, int BN, int WR, int WC, int RB, int KG, bool DMA>
__global__ __launch_bounds__(64 * WR * WC * KG, (512 + 64 * WR * WC * KG - 1) / (64 * WR * WC * KG)) void k_linear_tile(const vadc_amd_linear_args a)
{
   constexpr int WAVES = WR * WC, KT = RB / (int)sizeof(T), TM = BM / WR / 32, TN = BN / WC / 32, BYTES = (BM + BN) * RB, PER = 16 / (int)sizeof(T);
   constexpr int ROWS = 1024 / RB, XP = BM / ROWS / WAVES, PIECES = (BM + BN) / ROWS / WAVES;      // LDS rows of a DMA instruction; a wave's instructions for x, for both
   static_assert(BM % (ROWS * WAVES) == 0 && BN % (ROWS * WAVES) == 0, "every wave does the same");
   __shared__ __attribute__((aligned(16))) char lds[2 * KG * BYTES];
   const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6) % WAVES, kg = __builtin_amdgcn_readfirstlane(tid >> 6) / WAVES;
   const int64_t tiles_m = (a.rows + BM - 1) / BM, tiles_n = (a.out_features + BN - 1) / BN;
   const unsigned tiles = (unsigned)(tiles_m * tiles_n);
   const int wr = wave % WR * (BM / WR), wc = wave / WR * (BN / WC);
   const int64_t full = a.in_features / KT, rounds = (full + KG - 1) / KG, whole = (full - kg + KG - 1) / KG;      // full tiles of k; this group's are kg, kg + KG, ...

   // this wave's instructions: of x's tile, then of the weight's, each ROWS of its rows; rows behind the last are copies of it, their outputs are dropped
   int64_t row0, col0;
   int lastx, lastw;
   const T *srcx, *srcw;
   uint32_t offset[PIECES];
   const auto row_in = [&](int p) { return ((p < XP ? p : p - XP) * WAVES + wave) * ROWS + lane / (RB / 16); };
   const auto row_of = [&](int p) { return min(row_in(p), p < XP ? lastx : lastw); };
   const auto piece_of = [&](int p) { return mixed<RB>(row_in(p), lane % (RB / 16)); };
   const auto aim = [&](unsigned index) {
      int64_t tm, tn;
      tile_of(index, tiles, tiles_m, tiles_n, tm, tn);
      row0 = tm * BM;
      col0 = tn * BN;
      lastx = (int)min(a.rows - 1 - row0, (int64_t)BM);
      lastw = (int)min(a.out_features - 1 - col0, (int64_t)BN);
      srcx = (const T *)a.x + row0 * a.x_stride;
      srcw = (const T *)a.weight + col0 * a.weight_stride;
#pragma unroll
      for (int p = 0; p < PIECES; ++p) offset[p] = (uint32_t)(row_of(p) * (int)((p < XP ? a.x_stride : a.weight_stride) * sizeof(T)) + 16 * piece_of(p));
   };
   const auto issue = [&](int64_t kt, int stage) {
      const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds + (uint32_t)(stage * KG + kg) * BYTES + wave * 1024;
      const void *fromx = uniform(srcx + (kt * KG + kg) * KT), *fromw = uniform(srcw + (kt * KG + kg) * KT);
#pragma unroll
      for (int p = 0; p < PIECES; ++p) dma(to + p * WAVES * 1024, offset[p], p < XP ? fromx : fromw);
   };
   const auto fetch = [&](int64_t kt, auto &h) {                      // a full tile through registers, any alignment
      const char *fromx = (const char *)uniform(srcx + (kt * KG + kg) * KT), *fromw = (const char *)uniform(srcw + (kt * KG + kg) * KT);
#pragma unroll
      for (int p = 0; p < PIECES; ++p) __builtin_memcpy(&h[p], (p < XP ? fromx : fromw) + offset[p], 16);
   };
   const auto fetch_part = [&](auto &h) {                             // the part of a tile at the end, zeros behind the last k
      const char *fromx = (const char *)uniform(srcx + full * KT), *fromw = (const char *)uniform(srcw + full * KT);
      const int rest = (int)(a.in_features - full * KT);
      u128 u[PIECES];
      load_ends<T, PIECES>(a.in_features, [&](int p) { return (const T *)((p < XP ? fromx : fromw) + offset[p]); }, [&](int p) { return rest - piece_of(p) * PER; }, u);
      __builtin_memcpy(&h, &u, sizeof(u));
   };
   const auto place = [&](int stage, const auto &h) {
#pragma unroll
      for (int p = 0; p < PIECES; ++p) __builtin_memcpy(__builtin_assume_aligned(lds + (stage * KG + kg) * BYTES + (p * WAVES + wave) * 1024 + lane * 16, 16), &h[p], 16);
   };
   f16v acc[TN][TM];
   const auto compute = [&](int stage) {
      const char *sx = lds + (stage * KG + kg) * BYTES, *sw = sx + BM * RB;
#pragma unroll
      for (int s = 0; s < KT / 16; ++s) {
         p8 fa[TN], fb[TM];
#pragma unroll
         for (int i = 0; i < TN; ++i) fa[i] = *reinterpret_cast<const p8 *>(sw + piece_at<RB>(wc + 32 * i + (lane & 31), 2 * s + (lane >> 5)));
#pragma unroll
         for (int j = 0; j < TM; ++j) fb[j] = *reinterpret_cast<const p8 *>(sx + piece_at<RB>(wr + 32 * j + (lane & 31), 2 * s + (lane >> 5)));
#pragma unroll
         for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) acc[i][j] = product(fa[i], fb[j], acc[i][j], T());
      }
   };
   constexpr int FEATS = BN / WC >= 64 && BYTES >= WAVES * 32 * 64 * 4 ? 64 : 32;
   static_assert(BYTES >= WAVES * 32 * FEATS * 4, "the outputs leave through one stage");

   unsigned index = blockIdx.x;
   aim(index);
   int stage = 0;                                                     // of the next tile of k; the other one is free, or about to be
   if constexpr (DMA)
      if (whole) issue(0, stage);
   const bool part = a.in_features % KT != 0, parts_mine = kg == KG - 1;      // the part of a tile at the end comes first, while no sums are held; the last group has the least else
   const auto clear = [&] {
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
         for (int j = 0; j < TM; ++j) acc[i][j] = (f16v)(0.0f);
   };
   for (;;) {
      T held[PIECES][PER];
      if constexpr (DMA) {
         if (part) {                                                  // through registers, into the stage that is free
            if (parts_mine) fetch_part(held);
            lds_barrier();
            if (parts_mine) place(stage ^ 1, held);
            lds_barrier();
         }
         clear();
         if (part && parts_mine) compute(stage ^ 1);
         for (int64_t kt = 0; kt < rounds; ++kt) {
            vm_wait();
            lds_barrier();
            if (kt + 1 < whole) issue(kt + 1, stage ^ 1);
            if (KG == 1 || kt < whole) compute(stage);
            stage ^= 1;
         }
      } else {
         if (part && parts_mine) fetch_part(held);
         lds_barrier();
         if (part && parts_mine) place(1, held);
         if (whole) {
            fetch(0, held);
            place(0, held);
         }
         if (whole > 1) fetch(1, held);
         clear();
         if (part) {
            lds_barrier();
            if (parts_mine) compute(1);
         }
         for (int64_t kt = 0; kt < rounds; ++kt) {
            lds_barrier();
            if (kt + 1 < whole) place((int)((kt + 1) & 1), held);     // its readers are behind the barrier above; written under the products, and the loads have a whole step to arrive
            if (kt + 2 < whole) fetch(kt + 2, held);
            if (KG == 1 || kt < whole) compute((int)(kt & 1));
         }
      }
      lds_barrier();                                                  // everybody has read the last tile of k: its stage is free
      const int64_t row = row0, col = col0;
      index += gridDim.x;
      const bool more = index < tiles;
      if (more) {
         aim(index);
         if constexpr (DMA)
            if (whole) issue(0, stage);
      }
      leave<T, TN, TM, FEATS, KG>(a, reinterpret_cast<f4 *>(lds + (DMA ? stage ^ 1 : 0) * KG * BYTES) + wave * 8 * FEATS, kg, BYTES / 16, acc, row + wr, col + wc, lane);
      if (!more) break;
   }
}

// float32, BM x BN outputs per tile, four waves: operands go through registers into LDS in three bfloat16 parts (ops_prims.h), 32 k's at a time, six products for one.  Splitting on the
// way in costs a value 5.5 instructions once; split where a wave reads them, every value was split twice (98304 x 128 x 512: 110 us so, 105 us this way).  One set of tiles, two barriers a
// step: two workgroups share a CU and fill each other's gaps (a third would cost 30 spilled registers: 118 us).
template <int BM, int BN, int WR, int WC>
__global__ __launch_bounds__(256, 2) void k_linear_parts(const vadc_amd_linear_args a)
{
   constexpr int WAVES = WR * WC, KT = 32, TM = BM / WR / 32, TN = BN / WC / 32, PLANE = (BM + BN) * 64, XP = BM / 16 / WAVES, PIECES = (BM + BN) / 16 / WAVES;
   static_assert(WAVES == 4 && BM % (16 * WAVES) == 0 && BN % (16 * WAVES) == 0, "every wave does the same");
   __shared__ __attribute__((aligned(16))) char lds[3 * PLANE];
   const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
   const int64_t tiles_m = (a.rows + BM - 1) / BM, tiles_n = (a.out_features + BN - 1) / BN;
   const unsigned tiles = (unsigned)(tiles_m * tiles_n);
   const int wr = wave % WR * (BM / WR), wc = wave / WR * (BN / WC);
   const int64_t all = (a.in_features + KT - 1) / KT;
   const auto row_in = [&](int p) { return ((p < XP ? p : p - XP) * WAVES + wave) * 16 + (lane >> 2); };      // a lane's eight k's of this row of its operand, lane % 4 of the four eights
   int64_t row0, col0;
   const float *from[PIECES];
   const auto aim = [&](unsigned index) {
      int64_t tm, tn;
      tile_of(index, tiles, tiles_m, tiles_n, tm, tn);
      row0 = tm * BM;
      col0 = tn * BN;
#pragma unroll
      for (int p = 0; p < PIECES; ++p)                                // rows behind the last are copies of it: their outputs are dropped
         from[p] = (p < XP ? (const float *)a.x + min(row0 + row_in(p), a.rows - 1) * a.x_stride : (const float *)a.weight + min(col0 + row_in(p), a.out_features - 1) * a.weight_stride) + 8 * (lane & 3);
   };
   float held[PIECES][8];
   const auto fetch = [&](int64_t kt) {
      const int64_t k = kt * KT;
      if (k + KT <= a.in_features) {
#pragma unroll
         for (int p = 0; p < PIECES; ++p) load_f32<float, 8>(from[p] + k, held[p]);
      } else {
         const int left = (int)(a.in_features - k) - 8 * (lane & 3);
#pragma unroll
         for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int i = 0; i < 8; ++i) held[p][i] = i < left ? from[p][k + i] : 0.0f;
      }
   };
   const auto place = [&] {
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
         p8 w[3];
         split8<float>(held[p], w);
#pragma unroll
         for (int n = 0; n < 3; ++n) *reinterpret_cast<p8 *>(lds + n * PLANE + (p < XP ? 0 : BM * 64) + piece_at<64>(row_in(p), lane & 3)) = w[n];
      }
   };
   constexpr int FEATS = BN / WC >= 64 ? 64 : 32;
   static_assert(3 * PLANE >= WAVES * 32 * FEATS * 4, "the outputs leave through the same LDS");

   unsigned index = blockIdx.x;
   aim(index);
   if (all) fetch(0);
   for (;;) {
      f16v acc[TN][TM];
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
         for (int j = 0; j < TM; ++j) acc[i][j] = (f16v)(0.0f);
      for (int64_t kt = 0; kt < all; ++kt) {
         lds_barrier();                                               // everybody is through with the last tiles, or with the last outputs
         place();
         if (kt + 1 < all) fetch(kt + 1);
         lds_barrier();
#pragma unroll
         for (int s = 0; s < 2; ++s) {
            p8 fb[TM][3];
#pragma unroll
            for (int n = 0; n < 3; ++n)
#pragma unroll
               for (int j = 0; j < TM; ++j) fb[j][n] = *reinterpret_cast<const p8 *>(lds + n * PLANE + piece_at<64>(wr + 32 * j + (lane & 31), 2 * s + (lane >> 5)));
#pragma unroll
            for (int i = 0; i < TN; ++i) {
               p8 fa[3];
#pragma unroll
               for (int n = 0; n < 3; ++n) fa[n] = *reinterpret_cast<const p8 *>(lds + n * PLANE + BM * 64 + piece_at<64>(wc + 32 * i + (lane & 31), 2 * s + (lane >> 5)));
#pragma unroll
               for (int o = 2; o >= 0; --o)                           // the small products first
#pragma unroll
                  for (int n = 0; n <= o; ++n)
#pragma unroll
                     for (int j = 0; j < TM; ++j) acc[i][j] = product(fa[n], fb[j][o - n], acc[i][j], __bf16());
            }
         }
      }
      // An infinity times a part that is zero makes a NaN, and a value whose first part rounds to infinity one too: a wave that finds one does its outputs again, on the float32 pipe,
      // straight from memory.  Every NaN of the definition ends here as well and stays one.
      f16v sum = (f16v)(0.0f);
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
         for (int j = 0; j < TM; ++j) sum += acc[i][j] * 0.0f;
      float nan = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) nan += sum[e];
      if (__any(nan != 0.0f)) {
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
      const int64_t row = row0, col = col0;
      index += gridDim.x;
      const bool more = index < tiles;
      if (more) {
         aim(index);
         if (all) fetch(0);
      }
      lds_barrier();                                                  // everybody has read the last tiles
      leave<float, TN, TM, FEATS, 1>(a, reinterpret_cast<f4 *>(lds) + wave * 8 * FEATS, 0, 0, acc, row + wr, col + wc, lane);
      if (!more) break;
   }
}

// ---- few rows: the weight goes once through registers, nothing is shared -------------------------------------------------------------------------------
// A workgroup does 16 TN features of up to 16 TM rows; its eight waves take every eighth 64 k's and add up in LDS in a fixed order.  A lane reads 32 (float32: 64) consecutive bytes of its
// row, so that the four lanes of a row read a run: the k's of an operand fragment may come in any order that both operands share.
template <typename T, int TN, int TM, bool ODD>
__global__ __launch_bounds__(512) void k_linear_narrow(const vadc_amd_linear_args a)
{
   constexpr int WAVES = 8;
   __shared__ __attribute__((aligned(16))) f4 part[WAVES][TN * TM][64];
   const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, l4 = lane >> 4;
   const int64_t tiles_n = (a.out_features + 16 * TN - 1) / (16 * TN), row0 = blockIdx.x / tiles_n * (16 * TM), col0 = blockIdx.x % tiles_n * (16 * TN);
   const T *pw[TN], *px[TM];
#pragma unroll
   for (int i = 0; i < TN; ++i) pw[i] = (const T *)a.weight + min(col0 + 16 * i + l15, a.out_features - 1) * a.weight_stride;
#pragma unroll
   for (int j = 0; j < TM; ++j) px[j] = (const T *)a.x + min(row0 + 16 * j + l15, a.rows - 1) * a.x_stride;
   f4 acc[TN * TM];
#pragma unroll
   for (int j = 0; j < TN * TM; ++j) acc[j] = (f4)(0.0f);
   struct Held { T w[TN][16], x[TM][16]; };
   const auto products = [&](const Held &h) {
#pragma unroll
      for (int t = 0; t < TN * TM; ++t) {
         const int i = t / TM, j = t % TM;
         if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int s = 0; s < 16; ++s) acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(h.w[i][s], h.x[j][s], acc[t], 0, 0, 0);
         } else {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
               p8 fa, fb;
               __builtin_memcpy(&fa, &h.w[i][8 * s], sizeof(fa));
               __builtin_memcpy(&fb, &h.x[j][8 * s], sizeof(fb));
               if constexpr (__is_same(T, __bf16)) acc[t] = mfma16(fa, fb, acc[t]);
               else acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, fa), __builtin_bit_cast(h8, fb), acc[t], 0, 0, 0);
            }
         }
      }
   };
   // Whole pieces of 64 k's in a loop of their own; at most one wave has the part at the end
   const auto load = [&](int64_t k, Held &h) {
#pragma unroll
      for (int i = 0; i < TN; ++i) load16<T, ODD>(pw[i] + k + 16 * l4, h.w[i]);
#pragma unroll
      for (int j = 0; j < TM; ++j) load16<T, ODD>(px[j] + k + 16 * l4, h.x[j]);
   };
   Held even, odd;
   int64_t k = 64 * wave;
   if constexpr (TM == 1) {                                           // the next piece's loads are on their way under a piece's products (1 x 4096 x 4096 float32: 20.0 us without, 16.7 us so)
      if (k + 64 <= a.in_features) load(k, even);
      while (k + 64 <= a.in_features) {
         k += 64 * WAVES;
         const bool more = k + 64 <= a.in_features;
         if (more) load(k, odd);
         products(even);
         if (!more) break;
         k += 64 * WAVES;
         if (k + 64 <= a.in_features) load(k, even);
         products(odd);
      }
   } else                                                             // there is enough on its way (64 x 4096 x 4096 float32: 39.7 us so, 46.5 us as above)
      for (; k + 64 <= a.in_features; k += 64 * WAVES) {
         load(k, even);
         products(even);
      }
   if (k < a.in_features) {
      const int left = (int)(a.in_features - k) - 16 * l4;
      k += 16 * l4;
      constexpr int PER = 16 / (int)sizeof(T), PP = 16 / PER;
      u128 u[(TN + TM) * PP];
      load_ends<T, (TN + TM) * PP>(a.in_features, [&](int i) { return (i < TN * PP ? pw[i / PP] : px[(i - TN * PP) / PP]) + k + i % PP * PER; }, [&](int i) { return left - i % PP * PER; }, u);
      __builtin_memcpy(&even, &u, sizeof(u));
      products(even);
   }
#pragma unroll
   for (int t = 0; t < TN * TM; ++t) part[wave][t][lane] = acc[t];
   __syncthreads();
   for (int t = wave; t < TN * TM; t += WAVES) {
      f4 sum = part[0][t][lane];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) sum += part[w][t][lane];
      const int64_t row = row0 + 16 * (t % TM) + l15, col = col0 + 16 * (t / TM) + 4 * l4;
      float y[4] = {sum[0], sum[1], sum[2], sum[3]}, bias[4];
      load_bias<T, 4>(a, col, bias);
      const int left = (int)min((int64_t)4, a.out_features - col);
      if (row < a.rows && left > 0) finish<T, 4>(a, (const T *)a.residual + row * a.residual_stride + col, (T *)a.out + row * a.out_stride + col, left, y, bias);
   }
}

// ---- choice ---------------------------------------------------------------------------------------------------------------------------------------------
template <typename T, int BM, int BN, int WR, int WC, int RB, int KG> static void launch_tile(const vadc_amd_linear_args &a, hipStream_t s, bool dma)
{
   constexpr int threads = 64 * WR * WC * KG;
   constexpr int64_t slots = 256 * std::max(1, 512 / threads);         // 512 threads a CU at a time
   const dim3 grid((unsigned)std::min(slots, ((a.rows + BM - 1) / BM) * ((a.out_features + BN - 1) / BN)));
   if (dma) hipLaunchKernelGGL((k_linear_tile<T, BM, BN, WR, WC, RB, KG, true>), grid, dim3(threads), 0, s, a);
   else hipLaunchKernelGGL((k_linear_tile<T, BM, BN, WR, WC, RB, KG, false>), grid, dim3(threads), 0, s, a);
}
template <typename T, int TN, int TM> static void launch_narrow(const vadc_amd_linear_args &a, hipStream_t s)
{
   const dim3 grid((unsigned)(((a.rows + 16 * TM - 1) / (16 * TM)) * ((a.out_features + 16 * TN - 1) / (16 * TN))));
   if constexpr (sizeof(T) == 2)
      if (((uintptr_t)a.x | (uintptr_t)a.weight) % 4 || a.x_stride % 2 || a.weight_stride % 2) {
         hipLaunchKernelGGL((k_linear_narrow<T, TN, TM, true>), grid, dim3(512), 0, s, a);
         return;
      }
   hipLaunchKernelGGL((k_linear_narrow<T, TN, TM, false>), grid, dim3(512), 0, s, a);
}
template <int BM, int BN> static void launch_parts(const vadc_amd_linear_args &a, hipStream_t s)
{
   const dim3 grid((unsigned)std::min<int64_t>(256 * 2, ((a.rows + BM - 1) / BM) * ((a.out_features + BN - 1) / BN)));
   hipLaunchKernelGGL((k_linear_parts<BM, BN, 2, 2>), grid, dim3(256), 0, s, a);
}
template <typename T> static void launch(const vadc_amd_linear_args &a, hipStream_t s)
{
   if (a.rows <= 16) return launch_narrow<T, 1, 1>(a, s);
   const auto tiles = [&](int64_t t) { return ((a.rows + t - 1) / t) * ((a.out_features + t - 1) / t); };
   if constexpr (sizeof(T) == 4) {
      const int64_t blocks = (a.rows + 63) / 64 * ((a.out_features + 15) / 16);
      // 64 x 4096 x 4096: 39 us, in tiles 95 us; 2048 x 512 x 128: 9.7, 14.3 us.  Twice as many: 256 x 2048 x 2048 34, 50 us; but rows that two workgroups read far apart: 8192 x 512 x 64
      // 20.6, 15.4 us
      if (blocks <= 256) launch_narrow<T, 1, 4>(a, s);
      else if (blocks <= 512 && a.rows <= 2048) launch_narrow<T, 2, 4>(a, s);
      else if (tiles(128) >= 200) launch_parts<128, 128>(a, s);
      else launch_parts<64, 64>(a, s);
   } else {
      // 32 x 4096 x 4096: 13.2 us, in tiles 16.6 us; 64 rows: 20.4 us.  The other case: a tile's rows are not within 32-bit offsets
      if (a.rows <= 32 || std::max(a.x_stride, a.weight_stride) * (int64_t)sizeof(T) >= (int64_t(1) << 31) / 256) return launch_narrow<T, 1, 2>(a, s);
      const bool dma = ((uintptr_t)a.x | (uintptr_t)a.weight) % 16 == 0 && a.x_stride % 8 == 0 && a.weight_stride % 8 == 0;
      if (tiles(256) >= 200) launch_tile<T, 256, 256, 2, 4, 128, 1>(a, s, dma);
      else if (tiles(128) >= 200) launch_tile<T, 128, 128, 2, 2, 128, 1>(a, s, dma);
      else if (tiles(64) > 256 || a.in_features < 512) launch_tile<T, 64, 64, 2, 2, 256, 1>(a, s, dma);
      else launch_tile<T, 64, 64, 2, 2, 256, 2>(a, s, dma);
   }
}

void launch_linear(const vadc_amd_linear_args &a, hipStream_t s)
{
   if (a.dtype == VADC_AMD_F32) launch<float>(a, s);
   else if (a.dtype == VADC_AMD_F16) launch<_Float16>(a, s);
   else launch<__bf16>(a, s);
}

}  // namespace ops
}  // namespace vadc
