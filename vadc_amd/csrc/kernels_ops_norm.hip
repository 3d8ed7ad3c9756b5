// kernels_ops_norm.hip -- group norm with an activation, channels last: x [sequences][positions][channels], statistics over a sequence's positions and one group's channels.
#include "ops_internal.h"
#include "ops_prims.h"

#include <algorithm>

namespace vadc {
namespace ops {

// Count, mean and sum of squared deviations of a set of values; two sets merge exactly (Chan, Golub and LeVeque's update), so that a mean far from zero
// costs no digits of the variance, as a sum of squares would.
struct Stats { float n, mean, m2; };
__device__ __forceinline__ Stats merge(const Stats &a, const Stats &b)
{
   const float n = a.n + b.n, d = b.mean - a.mean, w = n > 0.0f ? b.n * __builtin_amdgcn_rcpf(n) : 0.0f;      // a step of the reciprocal is one of the mean's distance, no more
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


// y = (x - mean) rstd w + b of VEC consecutive channels of one position, with the gate or activation behind it
template <typename T, int VEC>
__device__ __forceinline__ void apply(const vadc_amd_group_norm_args &a, const float (&x)[VEC], float mean, float rstd, const float (&w)[VEC], const float (&b)[VEC], const T *gate, T *out)
{
   float y[VEC], g[VEC];
   if (a.gate) load_f32<T, VEC>(gate, g);
#pragma unroll
   for (int i = 0; i < VEC; ++i) y[i] = fmaf((x[i] - mean) * rstd, w[i], b[i]);
   if (a.gate) {
      activate_all<T, VEC>(g, a.activation);
#pragma unroll
      for (int i = 0; i < VEC; ++i) y[i] *= g[i];
   } else activate_all<T, VEC>(y, a.activation);
   if (a.sequences * a.positions * a.channels * (int64_t)sizeof(T) >= kStreamBytes) stream_f32<T, VEC>(out, y);
   else store_f32<T, VEC>(out, y);
}
template <typename T, int VEC>
__device__ __forceinline__ void affine(const vadc_amd_group_norm_args &a, int64_t c, float (&w)[VEC], float (&b)[VEC])
{
#pragma unroll
   for (int i = 0; i < VEC; ++i) { w[i] = 1.0f; b[i] = 0.0f; }
   if (a.weight) load_f32<T, VEC>((const T *)a.weight + c, w);
   if (a.bias) load_f32<T, VEC>((const T *)a.bias + c, b);
}

// ---- one position per sequence: a norm per token and group ---------------------------------------------------------------------------------------------
// LANES lanes (a power of two) hold one group in registers, R vectors of VEC channels each: x is read once, mean and squared deviations are two sums over registers and lanes.
template <typename T, int VEC, int R>
__global__ __launch_bounds__(256) void k_norm_token(const vadc_amd_group_norm_args a, int lanes, unsigned items)
{
   const unsigned item = (blockIdx.x * 256u + threadIdx.x) / lanes, at = threadIdx.x & (lanes - 1);
   const unsigned groups = (unsigned)a.groups, size = (unsigned)(a.channels / a.groups);
   const unsigned token = item / groups, c0 = (item - token * groups) * size;
   const bool live = item < items && (!a.lengths || a.lengths[token] > 0);
   const T *x = (const T *)a.x + (int64_t)token * a.x_stride[0] + c0;
   float v[R][VEC];
   float sum = 0.0f;
#pragma unroll
   for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[r][i] = 0.0f;
      const unsigned c = (r * lanes + at) * VEC;
      if (live && c < size) load_f32<T, VEC>(x + c, v[r]);
   }
#pragma unroll
   for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += v[r][i];
   const float mean = sum_lanes(sum, lanes) / (float)size;
   float m2 = 0.0f;
#pragma unroll
   for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
         const float d = (unsigned)(r * lanes + at) * VEC < size ? v[r][i] - mean : 0.0f;
         m2 = fmaf(d, d, m2);
      }
   const float rstd = 1.0f / sqrtf(sum_lanes(m2, lanes) / (float)size + a.eps);
#pragma unroll
   for (int r = 0; r < R; ++r) {
      const unsigned c = (r * lanes + at) * VEC;
      if (live && c < size) {
         float w[VEC], b[VEC];
         affine<T, VEC>(a, c0 + c, w, b);
         apply<T, VEC>(a, v[r], mean, rstd, w, b, (const T *)a.gate + (int64_t)token * a.gate_stride[0] + c0 + c, (T *)a.out + (int64_t)token * a.out_stride[0] + c0 + c);
      }
   }
}

// ---- many positions: columns of VEC channels, positions down the workgroup -----------------------------------------------------------------------------
// A workgroup takes gb whole groups (width columns) of one sequence and a span of its positions; `across` threads lie along the columns, `down` along the positions, so that a
// position's channels are read as one run.  kPartial leaves each group's set of this span in the workspace, kApply merges the sets of all spans and normalises its own,
// kWhole (one span) does both.  Two launches read x twice, the second time out of the caches where the tensor fits them.
enum { kPartial, kApply, kWhole };
struct Shape { int gb, chunks, width, across, down, spans, apply_spans; int64_t span, apply_span; };

constexpr int kUnroll = 4;                                           // positions a thread has in flight
template <typename T, int VEC, int MODE>
__global__ __launch_bounds__(256) void k_norm_columns(const vadc_amd_group_norm_args a, const Shape h)
{
   __shared__ Stats part[256], whole[256];
   const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
   const int chunk = blockIdx.x % h.chunks;
   const unsigned rest = blockIdx.x / h.chunks;
   const int spans = MODE == kApply ? h.apply_spans : h.spans;
   const int64_t span = MODE == kApply ? h.apply_span : h.span;
   const int64_t seq = rest / spans, at = rest % spans;
   const int size = (int)(a.channels / a.groups), g0 = chunk * h.gb, gb = min(h.gb, (int)a.groups - g0);
   const int width = gb * (size / VEC), c0 = g0 * size;
   const int64_t length = live_positions(a, seq), from = at * span, to = min(from + span, length);
   const int tx = tid % h.across, ty = tid / h.across;
   const bool busy = ty < h.down;
   const T *x = (const T *)a.x + seq * a.x_stride[0] + c0;
   float3 *sets = (float3 *)a.workspace;
   if (MODE != kApply) {
      Stats s = {0, 0, 0};
      if (busy)
         for (int col = tx; col < width; col += h.across) {          // more than one turn only where a single group is wider than the workgroup
            const T *px = x + (int64_t)col * VEC;
            int64_t p = from + ty;
            for (; p + (kUnroll - 1) * h.down < to; p += kUnroll * h.down) {
               float v[kUnroll][VEC], sum = 0.0f, m2 = 0.0f;
#pragma unroll
               for (int u = 0; u < kUnroll; ++u) load_f32<T, VEC>(px + (p + u * h.down) * a.x_stride[1], v[u]);
#pragma unroll
               for (int u = 0; u < kUnroll; ++u)
#pragma unroll
                  for (int i = 0; i < VEC; ++i) sum += v[u][i];
               const float mean = sum * (1.0f / (kUnroll * VEC));
#pragma unroll
               for (int u = 0; u < kUnroll; ++u)
#pragma unroll
                  for (int i = 0; i < VEC; ++i) { const float d = v[u][i] - mean; m2 = fmaf(d, d, m2); }
               s = merge(s, {(float)(kUnroll * VEC), mean, m2});
            }
            for (; p < to; p += h.down) {
               float v[VEC], sum = 0.0f, m2 = 0.0f;
               load_f32<T, VEC>(px + p * a.x_stride[1], v);
#pragma unroll
               for (int i = 0; i < VEC; ++i) sum += v[i];
               const float mean = sum * (1.0f / VEC);
#pragma unroll
               for (int i = 0; i < VEC; ++i) { const float d = v[i] - mean; m2 = fmaf(d, d, m2); }
               s = merge(s, {(float)VEC, mean, m2});
            }
         }
      part[tid] = s;
      __syncthreads();
      const int per = gb == 1 ? h.across : size / VEC;               // threads along the columns that hold one group
      for (int g = wave; g < gb; g += 4) {
         Stats t = {0, 0, 0};
         for (int i = lane; i < per * h.down; i += 64) t = merge(t, part[(i / per) * h.across + g * per + i % per]);
         t = merge_lanes(t, 64, lane);
         if (lane == 0) {
            if (MODE == kWhole) whole[g] = t;
            else sets[(seq * h.spans + at) * a.groups + g0 + g] = make_float3(t.n, t.mean, t.m2);
         }
      }
      if (MODE == kPartial) return;
   } else {
      if (from >= to) return;                                        // the whole workgroup: nothing of this sequence lies here
      for (int g = wave; g < gb; g += 4) {
         Stats t = {0, 0, 0};
         for (int i = lane; i < h.spans; i += 64) {
            const float3 f = sets[(seq * h.spans + i) * a.groups + g0 + g];
            t = merge(t, {f.x, f.y, f.z});
         }
         t = merge_lanes(t, 64, lane);
         if (lane == 0) whole[g] = t;
      }
   }
   __syncthreads();
   if (!busy) return;
   for (int col = tx; col < width; col += h.across) {
      const int64_t c = c0 + (int64_t)col * VEC;
      const Stats s = whole[col * VEC / size];
      const float mean = s.mean, rstd = 1.0f / sqrtf(s.m2 / fmaxf(s.n, 1.0f) + a.eps);
      float w[VEC], b[VEC];
      affine<T, VEC>(a, c, w, b);
      const T *px = (const T *)a.x + seq * a.x_stride[0] + c, *gate = (const T *)a.gate + seq * a.gate_stride[0] + c;
      T *out = (T *)a.out + seq * a.out_stride[0] + c;
#pragma unroll 2
      for (int64_t p = from + ty; p < to; p += h.down) {
         float v[VEC];
         load_f32<T, VEC>(px + p * a.x_stride[1], v);
         apply<T, VEC>(a, v, mean, rstd, w, b, gate + p * a.gate_stride[1], out + p * a.out_stride[1]);
      }
   }
}

// ---- choice ---------------------------------------------------------------------------------------------------------------------------------------------
// channels a thread takes at once: the most that divide a group, up to 16 bytes
static int vector_of(const vadc_amd_group_norm_args &a)
{
   const int64_t size = a.channels / a.groups;
   for (int v = a.dtype == VADC_AMD_F32 ? 4 : 8; v > 1; v /= 2)
      if (size % v == 0) return v;
   return 1;
}
static Shape shape_of(const vadc_amd_group_norm_args &a, int vec)
{
   Shape h;
   const int per = (int)(a.channels / a.groups) / vec;               // columns of a group
   h.gb = per >= 256 ? 1 : (int)std::min<int64_t>(a.groups, 256 / per);
   h.chunks = (int)((a.groups + h.gb - 1) / h.gb);
   h.gb = (int)((a.groups + h.chunks - 1) / h.chunks);
   h.chunks = (int)((a.groups + h.gb - 1) / h.gb);
   h.width = h.gb * per;
   h.across = std::min(h.width, 256);
   h.down = 256 / h.across;
   // spans: enough workgroups to fill the device, none with less than 4 rounds of its positions in flight; at most 256 sets to merge
   const int64_t others = a.sequences * h.chunks, most = std::max<int64_t>(1, a.positions / (4 * kUnroll * h.down));
   h.spans = (int)std::max<int64_t>(1, std::min<int64_t>({256, most, (1024 + others - 1) / others}));
   h.span = (a.positions + h.spans - 1) / h.spans;
   h.apply_spans = (int)std::max<int64_t>(1, std::min<int64_t>(most, (2048 + others - 1) / others));
   h.apply_span = (a.positions + h.apply_spans - 1) / h.apply_spans;
   return h;
}

template <typename T, int VEC> static void launch_columns(const vadc_amd_group_norm_args &a, const vadc_amd_group_norm_args &first, hipStream_t s)
{
   const Shape h = shape_of(first, VEC);
   const int64_t others = a.sequences * h.chunks;
   if (h.spans == 1) {
      hipLaunchKernelGGL((k_norm_columns<T, VEC, kWhole>), dim3((unsigned)others), dim3(256), 0, s, a, h);
   } else {
      hipLaunchKernelGGL((k_norm_columns<T, VEC, kPartial>), dim3((unsigned)(others * h.spans)), dim3(256), 0, s, a, h);
      hipLaunchKernelGGL((k_norm_columns<T, VEC, kApply>), dim3((unsigned)(others * h.apply_spans)), dim3(256), 0, s, a, h);
   }
}
template <typename T, int VEC> static void launch_vec(const vadc_amd_group_norm_args &a, const vadc_amd_group_norm_args &first, hipStream_t s)
{
   const int64_t per = a.channels / a.groups / VEC, items = a.sequences * a.groups;
   if (a.positions > 1 || per > 512) return launch_columns<T, VEC>(a, first, s);     // a group of more than 512 vectors does not fit a wave's registers
   int lanes = 1;
   while (lanes < 64 && lanes < per) lanes *= 2;
   const int r = (int)((per + lanes - 1) / lanes);
   const dim3 grid((unsigned)((items * lanes + 255) / 256));
   if (r == 1) hipLaunchKernelGGL((k_norm_token<T, VEC, 1>), grid, dim3(256), 0, s, a, lanes, (unsigned)items);
   else if (r == 2) hipLaunchKernelGGL((k_norm_token<T, VEC, 2>), grid, dim3(256), 0, s, a, lanes, (unsigned)items);
   else if (r <= 4) hipLaunchKernelGGL((k_norm_token<T, VEC, 4>), grid, dim3(256), 0, s, a, lanes, (unsigned)items);
   else hipLaunchKernelGGL((k_norm_token<T, VEC, 8>), grid, dim3(256), 0, s, a, lanes, (unsigned)items);
}
template <typename T> static void launch(const vadc_amd_group_norm_args &a, const vadc_amd_group_norm_args &first, hipStream_t s)
{
   const int v = vector_of(a);
   if constexpr (sizeof(T) == 2) if (v == 8) return launch_vec<T, 8>(a, first, s);
   if (v == 4) launch_vec<T, 4>(a, first, s);
   else if (v == 2) launch_vec<T, 2>(a, first, s);
   else launch_vec<T, 1>(a, first, s);
}

int64_t group_norm_workspace(const vadc_amd_group_norm_args &a)
{
   if (a.positions <= 1) return 0;
   const Shape h = shape_of(a, vector_of(a));
   return h.spans == 1 ? 0 : a.sequences * h.spans * a.groups * (int64_t)sizeof(float3);
}

void launch_group_norm(const vadc_amd_group_norm_args &a, const vadc_amd_group_norm_args &first, hipStream_t s)
{
   if (a.dtype == VADC_AMD_F32) launch<float>(a, first, s);
   else if (a.dtype == VADC_AMD_F16) launch<_Float16>(a, first, s);
   else launch<__bf16>(a, first, s);
}

}  // namespace ops
}  // namespace vadc
