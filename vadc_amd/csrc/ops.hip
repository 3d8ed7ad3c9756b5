// ops.hip -- entry points of the operators on device tensors (include/vadc_amd.h): argument checks, the device, the launch.  The kernels: kernels_ops_*.hip.
#include "ops_internal.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>

using vadc::fail;

namespace {

constexpr int64_t kMaxSize = int64_t(1) << 40;        // every size and stride; products of two stay inside 64 bits by the checks below
constexpr int64_t kMaxBlocks = (int64_t(1) << 32) / 1024;      // a launch has fewer than 2^32 threads, in workgroups of up to 1024: longer calls go out in slices

bool ranged(std::initializer_list<int64_t> vs)
{
   for (int64_t v : vs) if (v < 0 || v > kMaxSize) return false;
   return true;
}
// a * b * c > limit, without overflow (all >= 0)
bool product_over(int64_t limit, std::initializer_list<int64_t> vs)
{
   int64_t p = 1;
   for (int64_t v : vs) { if (v == 0) return false; }
   for (int64_t v : vs) { if (p > limit / v) return true; p *= v; }
   return false;
}
bool aligned(const void *p, int64_t to) { return ((uintptr_t)p % (uintptr_t)to) == 0; }
int64_t width(int32_t dtype) { return dtype == VADC_AMD_F32 ? 4 : 2; }

// Makes `device` (< 0: the current one) current for the launch and the caller's device current again afterwards.
class OnDevice {
public:
   int enter(int device, const char *what)
   {
      if (hipGetDevice(&before_) != hipSuccess) { (void)hipGetLastError(); return fail(VADC_AMD_ENODEVICE, "%s: no HIP device available (this backend has no CPU fallback)", what); }
      if (device < 0) device = before_;
      if (device >= kDevices) return fail(VADC_AMD_ENODEVICE, "%s: device %d out of range", what, device);
      static std::atomic<int> known[kDevices];                       // 0: not asked yet, 1: gfx950, 2: another part
      int k = known[device].load(std::memory_order_relaxed);
      if (!k) {
         hipDeviceProp_t prop;
         if (hipGetDeviceProperties(&prop, device) != hipSuccess) { (void)hipGetLastError(); return fail(VADC_AMD_ENODEVICE, "%s: device %d out of range", what, device); }
         k = strncmp(prop.gcnArchName, "gfx950", 6) == 0 ? 1 : 2;
         known[device].store(k, std::memory_order_relaxed);
      }
      if (k != 1) return fail(VADC_AMD_ENODEVICE, "%s: device %d is no gfx950; this library carries gfx950 code only", what, device);
      if (device != before_) {
         if (hipSetDevice(device) != hipSuccess) { (void)hipGetLastError(); return fail(VADC_AMD_ENODEVICE, "%s: device %d cannot be used", what, device); }
         moved_ = true;
      }
      (void)hipGetLastError();                                       // an error of an earlier call is not this one's
      return VADC_AMD_OK;
   }
   int left(const char *what)
   {
      const hipError_t e = hipGetLastError();
      return e == hipSuccess ? VADC_AMD_OK : fail(VADC_AMD_EHIP, "%s: %s", what, hipGetErrorString(e));
   }
   ~OnDevice() { if (moved_) (void)hipSetDevice(before_); }

private:
   static constexpr int kDevices = 64;
   int before_ = 0;
   bool moved_ = false;
};

int check_linear(const vadc_amd_linear_args *a)
{
   if (!a) return fail(VADC_AMD_EINVAL, "linear: NULL arguments");
   if (a->dtype < VADC_AMD_F32 || a->dtype > VADC_AMD_BF16) return fail(VADC_AMD_EINVAL, "linear: unknown dtype %d", a->dtype);
   if (a->activation < VADC_AMD_ACT_NONE || a->activation > VADC_AMD_ACT_SIGMOID) return fail(VADC_AMD_EINVAL, "linear: unknown activation %d", a->activation);
   if (!ranged({a->rows, a->in_features, a->out_features, a->x_stride, a->weight_stride, a->residual_stride, a->out_stride}))
      return fail(VADC_AMD_EINVAL, "linear: a size or stride is negative or over 2^40");
   if (a->rows == 0 || a->out_features == 0) return VADC_AMD_OK;
   if (!a->out || (a->in_features && (!a->x || !a->weight))) return fail(VADC_AMD_EINVAL, "linear: NULL tensor");
   if (a->rows > 1 && a->out_stride < a->out_features) return fail(VADC_AMD_EINVAL, "linear: rows of the output overlap (stride %lld)", (long long)a->out_stride);
   const int64_t w = width(a->dtype);
   if (!aligned(a->x, w) || !aligned(a->weight, w) || !aligned(a->bias, w) || !aligned(a->residual, w) || !aligned(a->out, w))
      return fail(VADC_AMD_EINVAL, "linear: a tensor is not aligned to its element");
   if (a->out_features > (1 << 24)) return fail(VADC_AMD_EINVAL, "linear: out_features over 2^24");
   if (product_over(kMaxSize, {a->rows, std::max({a->x_stride, a->residual_stride, a->out_stride, a->out_features})}) || product_over(kMaxSize, {a->out_features, a->weight_stride}))
      return fail(VADC_AMD_EINVAL, "linear: a tensor spans over 2^40 elements");
   return VADC_AMD_OK;
}

int check_norm(const vadc_amd_group_norm_args *a)
{
   if (!a) return fail(VADC_AMD_EINVAL, "group_norm: NULL arguments");
   if (a->dtype < VADC_AMD_F32 || a->dtype > VADC_AMD_BF16) return fail(VADC_AMD_EINVAL, "group_norm: unknown dtype %d", a->dtype);
   if (a->activation < VADC_AMD_ACT_NONE || a->activation > VADC_AMD_ACT_SIGMOID) return fail(VADC_AMD_EINVAL, "group_norm: unknown activation %d", a->activation);
   if (!ranged({a->sequences, a->positions, a->channels, a->groups, a->x_stride[0], a->x_stride[1], a->gate_stride[0], a->gate_stride[1], a->out_stride[0], a->out_stride[1]}))
      return fail(VADC_AMD_EINVAL, "group_norm: a size or stride is negative or over 2^40");
   if (a->groups < 1 || a->channels % a->groups) return fail(VADC_AMD_EINVAL, "group_norm: %lld channels do not divide into %lld groups", (long long)a->channels, (long long)a->groups);
   if (!(a->eps >= 0.0f) || !std::isfinite(a->eps)) return fail(VADC_AMD_EINVAL, "group_norm: eps must be finite and not negative");
   if (a->sequences == 0 || a->positions == 0 || a->channels == 0) return VADC_AMD_OK;
   if (a->channels > (1 << 20)) return fail(VADC_AMD_EINVAL, "group_norm: more than 2^20 channels");
   for (const int64_t *st : {a->x_stride, a->gate_stride, a->out_stride})
      if (product_over(kMaxSize, {a->sequences, st[0]}) || product_over(kMaxSize, {a->positions, std::max(st[1], a->channels)})) return fail(VADC_AMD_EINVAL, "group_norm: a tensor spans over 2^40 elements");
   return VADC_AMD_OK;
}

int check_delta(const vadc_amd_gated_delta_args *a)
{
   if (!a) return fail(VADC_AMD_EINVAL, "gated_delta: NULL arguments");
   if (a->dtype < VADC_AMD_F32 || a->dtype > VADC_AMD_BF16) return fail(VADC_AMD_EINVAL, "gated_delta: unknown dtype %d", a->dtype);
   if (!ranged({a->streams, a->steps, a->key_heads, a->heads, a->key_dim, a->value_dim, a->state_stride, a->decay_stride[0], a->decay_stride[1], a->beta_stride[0], a->beta_stride[1]}))
      return fail(VADC_AMD_EINVAL, "gated_delta: a size or stride is negative or over 2^40");
   for (int i = 0; i < 3; ++i)
      if (!ranged({a->q_stride[i], a->k_stride[i], a->v_stride[i], a->out_stride[i]})) return fail(VADC_AMD_EINVAL, "gated_delta: a size or stride is negative or over 2^40");
   if (a->key_dim < 1 || a->key_dim > 256) return fail(VADC_AMD_EINVAL, "gated_delta: key_dim %lld is not in 1 ... 256", (long long)a->key_dim);
   if (a->key_heads < 1 || a->heads % a->key_heads) return fail(VADC_AMD_EINVAL, "gated_delta: %lld heads are no multiple of %lld key heads", (long long)a->heads, (long long)a->key_heads);
   if (!std::isfinite(a->scale)) return fail(VADC_AMD_EINVAL, "gated_delta: scale must be finite");
   if (a->streams == 0 || a->steps == 0 || a->heads == 0 || a->value_dim == 0) return VADC_AMD_OK;
   if (a->value_dim > (1 << 20) || a->heads > (1 << 20) || product_over(1 << 20, {a->heads, (a->value_dim + 15) / 16})) return fail(VADC_AMD_EINVAL, "gated_delta: heads and value_dim over 2^24 values a step");
   if (a->steps > (1 << 26)) return fail(VADC_AMD_EINVAL, "gated_delta: more than 2^26 steps");
   for (const int64_t *st : {a->q_stride, a->k_stride, a->v_stride, a->out_stride})
      if (product_over(kMaxSize, {a->streams, st[0]}) || product_over(kMaxSize, {a->steps, st[1]}) || product_over(kMaxSize, {a->heads, st[2]})) return fail(VADC_AMD_EINVAL, "gated_delta: a tensor spans over 2^40 elements");
   for (const int64_t *st : {a->decay_stride, a->beta_stride})
      if (product_over(kMaxSize, {a->streams, st[0]}) || product_over(kMaxSize, {a->steps, st[1]})) return fail(VADC_AMD_EINVAL, "gated_delta: a tensor spans over 2^40 elements");
   if (product_over(kMaxSize, {a->streams, a->state_stride})) return fail(VADC_AMD_EINVAL, "gated_delta: a tensor spans over 2^40 elements");
   return VADC_AMD_OK;
}

const void *ahead(const void *p, int64_t elements, int64_t w) { return p ? (const char *)p + elements * w : nullptr; }

// ---- slices: of rows, sequences or streams, as many as one launch takes; launches of one stream follow each other, so that all slices may use one workspace
int64_t rows_per_launch(const vadc_amd_linear_args &a) { return std::max<int64_t>(1, kMaxBlocks / ((a.out_features + 15) / 16)); }
vadc_amd_group_norm_args first_slice(const vadc_amd_group_norm_args &a)
{
   vadc_amd_group_norm_args s = a;
   s.sequences = std::min(a.sequences, std::max<int64_t>(1, kMaxBlocks / a.groups));
   return s;
}
vadc_amd_gated_delta_args first_slice(const vadc_amd_gated_delta_args &a)
{
   const int64_t most = kMaxBlocks / (a.heads * ((a.value_dim + 15) / 16));
   vadc_amd_gated_delta_args s = a;
   s.streams = std::min(a.streams, std::max<int64_t>(1, a.steps > 1 ? std::min(most, 8192 / a.heads) : most));      // many steps: a slice's workspace has a block of each head at once
   return s;
}

}  // namespace

extern "C" int vadc_amd_linear(const vadc_amd_linear_args *a, void *hip_stream)
{
   if (int rc = check_linear(a)) return rc;
   if (a->rows == 0 || a->out_features == 0) return VADC_AMD_OK;
   const int64_t w = width(a->dtype);
   OnDevice d;
   if (int rc = d.enter(a->device, "linear")) return rc;
   for (int64_t from = 0, most = rows_per_launch(*a); from < a->rows; from += most) {
      vadc_amd_linear_args s = *a;
      s.rows = std::min(most, a->rows - from);
      s.x = ahead(a->x, from * a->x_stride, w); s.residual = ahead(a->residual, from * a->residual_stride, w); s.out = (void *)ahead(a->out, from * a->out_stride, w);
      vadc::ops::launch_linear(s, (hipStream_t)hip_stream);
   }
   return d.left("linear");
}

extern "C" int64_t vadc_amd_group_norm_workspace(const vadc_amd_group_norm_args *a)
{
   if (int rc = check_norm(a)) return rc;
   if (a->sequences == 0 || a->positions == 0 || a->channels == 0) return 0;
   return vadc::ops::group_norm_workspace(first_slice(*a));
}

extern "C" int vadc_amd_group_norm(const vadc_amd_group_norm_args *a, void *hip_stream)
{
   if (int rc = check_norm(a)) return rc;
   if (a->sequences == 0 || a->positions == 0 || a->channels == 0) return VADC_AMD_OK;
   if (!a->x || !a->out) return fail(VADC_AMD_EINVAL, "group_norm: NULL tensor");
   if ((a->positions > 1 && a->out_stride[1] < a->channels) || (a->sequences > 1 && a->out_stride[0] < a->channels))
      return fail(VADC_AMD_EINVAL, "group_norm: rows of the output overlap (strides %lld, %lld)", (long long)a->out_stride[0], (long long)a->out_stride[1]);
   const int64_t w = width(a->dtype);
   if (!aligned(a->x, w) || !aligned(a->weight, w) || !aligned(a->bias, w) || !aligned(a->gate, w) || !aligned(a->out, w) || !aligned(a->lengths, 4))
      return fail(VADC_AMD_EINVAL, "group_norm: a tensor is not aligned to its element");
   const int64_t need = vadc_amd_group_norm_workspace(a);
   if (need && (!a->workspace || a->workspace_bytes < need || !aligned(a->workspace, 16)))
      return fail(VADC_AMD_EINVAL, "group_norm: the workspace must be 16-byte aligned and hold %lld bytes", (long long)need);
   OnDevice d;
   if (int rc = d.enter(a->device, "group_norm")) return rc;
   const vadc_amd_group_norm_args first = first_slice(*a);
   for (int64_t from = 0, most = first.sequences; from < a->sequences; from += most) {
      vadc_amd_group_norm_args s = *a;
      s.sequences = std::min(most, a->sequences - from);
      s.x = ahead(a->x, from * a->x_stride[0], w); s.gate = ahead(a->gate, from * a->gate_stride[0], w); s.out = (void *)ahead(a->out, from * a->out_stride[0], w);
      s.lengths = (const int32_t *)ahead(a->lengths, from, 4);
      vadc::ops::launch_group_norm(s, first, (hipStream_t)hip_stream);
   }
   return d.left("group_norm");
}

extern "C" int64_t vadc_amd_gated_delta_workspace(const vadc_amd_gated_delta_args *a)
{
   if (int rc = check_delta(a)) return rc;
   if (a->streams == 0 || a->steps == 0 || a->heads == 0 || a->value_dim == 0) return 0;
   return vadc::ops::gated_delta_workspace(first_slice(*a));
}

extern "C" int vadc_amd_gated_delta(const vadc_amd_gated_delta_args *a, void *hip_stream)
{
   if (int rc = check_delta(a)) return rc;
   if (a->streams == 0 || a->steps == 0 || a->heads == 0 || a->value_dim == 0) return VADC_AMD_OK;
   if (!a->q || !a->k || !a->v || !a->log_decay || !a->beta || !a->state || !a->out) return fail(VADC_AMD_EINVAL, "gated_delta: NULL tensor");
   if ((a->heads > 1 && a->out_stride[2] < a->value_dim) || (a->steps > 1 && a->out_stride[1] < a->value_dim) || (a->streams > 1 && a->out_stride[0] < a->value_dim))
      return fail(VADC_AMD_EINVAL, "gated_delta: rows of the output overlap (strides %lld, %lld, %lld)", (long long)a->out_stride[0], (long long)a->out_stride[1], (long long)a->out_stride[2]);
   if (a->streams > 1 && a->state_stride < a->heads * a->key_dim * a->value_dim) return fail(VADC_AMD_EINVAL, "gated_delta: states of two streams overlap (stride %lld)", (long long)a->state_stride);
   const int64_t w = width(a->dtype);
   if (!aligned(a->q, w) || !aligned(a->k, w) || !aligned(a->v, w) || !aligned(a->out, w) || !aligned(a->log_decay, 4) || !aligned(a->beta, 4) || !aligned(a->state, 4) || !aligned(a->lengths, 4))
      return fail(VADC_AMD_EINVAL, "gated_delta: a tensor is not aligned to its element");
   const int64_t need = vadc_amd_gated_delta_workspace(a);
   if (need && (!a->workspace || a->workspace_bytes < need || !aligned(a->workspace, 16)))
      return fail(VADC_AMD_EINVAL, "gated_delta: the workspace must be 16-byte aligned and hold %lld bytes", (long long)need);
   OnDevice d;
   if (int rc = d.enter(a->device, "gated_delta")) return rc;
   const vadc_amd_gated_delta_args first = first_slice(*a);
   for (int64_t from = 0, most = first.streams; from < a->streams; from += most) {
      vadc_amd_gated_delta_args s = *a;
      s.streams = std::min(most, a->streams - from);
      s.q = ahead(a->q, from * a->q_stride[0], w); s.k = ahead(a->k, from * a->k_stride[0], w); s.v = ahead(a->v, from * a->v_stride[0], w);
      s.out = (void *)ahead(a->out, from * a->out_stride[0], w);
      s.log_decay = a->log_decay + from * a->decay_stride[0]; s.beta = a->beta + from * a->beta_stride[0]; s.state = a->state + from * a->state_stride;
      s.lengths = (const int32_t *)ahead(a->lengths, from, 4);
      vadc::ops::launch_gated_delta(s, first, (hipStream_t)hip_stream);
   }
   return d.left("gated_delta");
}
