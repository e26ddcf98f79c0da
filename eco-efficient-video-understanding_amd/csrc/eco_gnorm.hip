// eco_gnorm.hip -- group norm with an activation over channels-last positions (include/eco_hip.h, ABI v20).
//
//   y = act((x - mean) / sqrt(var + eps) * gamma + beta),  mean / var over an image's valid positions x c/groups channels
#include <math.h>

#include "eco_common.h"

namespace eco {

constexpr int kGnThreads = 256;

struct GnArgs {
  const void* x;
  void* y;
  const int* lengths;
  const float* gamma;
  const float* beta;
  long x_image, x_row, y_image, y_row;   // strides in elements
  long s;
  int c, groups, cg;
  int act;
  float eps;
};

template <typename T>
__device__ __forceinline__ float gn_load(const T* p);
template <>
__device__ __forceinline__ float gn_load<float>(const float* p) { return ld(p); }
template <>
__device__ __forceinline__ float gn_load<unsigned short>(const unsigned short* p) { return bf16_bits_to_f32(ld(p)); }
__device__ __forceinline__ void gn_store(float* p, float v) { st(p, v); }
__device__ __forceinline__ void gn_store(unsigned short* p, float v) { st(p, (unsigned short)f32_to_bf16_bits(v)); }

__device__ __forceinline__ float gn_act(float v, int act) {
  if (act == ECO_ACT_RELU) return v < 0.0f ? 0.0f : v;      // (a NaN stays)
  if (act == ECO_ACT_SILU) return silu(v);
  return v;
}

// Sum over the workgroup, every thread gets it; the order is fixed.
__device__ __forceinline__ float gn_block_sum(float v, float* red) {
  v = wave_sum(v);
  if (lane_id() == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  const float t = (red[0] + red[1]) + (red[2] + red[3]);
  __syncthreads();
  return t;
}

// One workgroup per (image, group): mean, then the sum of squared differences, then the result, each a pass over the
// group's values.
template <typename T>
__global__ __launch_bounds__(256) void group_norm_kernel(const GnArgs a) {
  __shared__ float red[4];
  const int g = (int)(blockIdx.x % (unsigned)a.groups);
  const long img = (long)(blockIdx.x / (unsigned)a.groups);
  long rows = a.s;
  if (a.lengths) {
    const long len = ld(a.lengths + img);
    rows = len < 0 ? 0 : len > a.s ? a.s : len;
  }
  const T* x = (const T*)a.x + img * a.x_image + (long)g * a.cg;
  T* y = (T*)a.y + img * a.y_image + (long)g * a.cg;
  const long count = rows * a.cg;
  float sum = 0.0f;
  for (long i = threadIdx.x; i < count; i += kGnThreads) sum += gn_load(x + (i / a.cg) * a.x_row + i % a.cg);
  const float mean = gn_block_sum(sum, red) / (float)count;
  float sq = 0.0f;
  for (long i = threadIdx.x; i < count; i += kGnThreads) {
    const float d = gn_load(x + (i / a.cg) * a.x_row + i % a.cg) - mean;
    sq += d * d;
  }
  const float rstd = 1.0f / sqrtf(gn_block_sum(sq, red) / (float)count + a.eps);
  for (long i = threadIdx.x; i < count; i += kGnThreads) {
    const int ch = (int)(i % a.cg);
    const float scale = rstd * (a.gamma ? ld(a.gamma + g * a.cg + ch) : 1.0f);
    const float v = (gn_load(x + (i / a.cg) * a.x_row + ch) - mean) * scale + (a.beta ? ld(a.beta + g * a.cg + ch) : 0.0f);
    gn_store(y + (i / a.cg) * a.y_row + ch, gn_act(v, a.act));
  }
}

}  // namespace eco

using namespace eco;

extern "C" int eco_group_norm_plan_create(int64_t n, int64_t s, int32_t c, int32_t groups, int32_t dt, int32_t num_cu,
                                          eco_group_norm_plan* plan) {
  clear_error();
  ECO_REQUIRE(plan != nullptr, "group_norm: null plan");
  ECO_REQUIRE(n >= 0 && s >= 0, "group_norm: negative shape");
  ECO_REQUIRE(c > 0 && groups > 0 && c % groups == 0, "group_norm: %d groups do not divide %d channels", groups, c);
  ECO_REQUIRE(dt == ECO_DT_F32 || dt == ECO_DT_BF16, "group_norm: unknown type %d", dt);
  ECO_REQUIRE(num_cu >= 0, "group_norm: negative num_cu");
  ECO_REQUIRE(s <= 2147483647l && n <= 2147483647l / groups, "group_norm: too many positions or images for one launch");
  memset(plan, 0, sizeof(*plan));
  plan->n = n; plan->s = s; plan->c = c; plan->groups = groups; plan->dt = dt;
  plan->num_cu = num_cu ? num_cu : current_device_num_cu();
  plan->chunks = 1;
  return ECO_OK;
}

extern "C" int eco_group_norm_forward(const eco_group_norm_plan* plan, const void* x, int64_t x_image_stride,
                                      int64_t x_row_stride, const int32_t* lengths, const float* gamma, const float* beta,
                                      float eps, int32_t act, void* y, int64_t y_image_stride, int64_t y_row_stride,
                                      void* workspace, void* stream) {
  clear_error();
  ECO_REQUIRE(plan != nullptr, "group_norm: null plan");
  eco_group_norm_plan same;
  if (int rc = eco_group_norm_plan_create(plan->n, plan->s, plan->c, plan->groups, plan->dt, plan->num_cu, &same)) return rc;
  ECO_REQUIRE(memcmp(&same, plan, sizeof(same)) == 0, "group_norm: the plan is not one of eco_group_norm_plan_create");
  ECO_REQUIRE(act == ECO_ACT_NONE || act == ECO_ACT_RELU || act == ECO_ACT_SILU, "group_norm: unknown activation %d", act);
  ECO_REQUIRE(eps >= 0.0f && eps <= 3.4e38f, "group_norm: eps must be finite and not negative");
  if (plan->n == 0 || plan->s == 0) return ECO_OK;
  ECO_REQUIRE(x && y, "group_norm: null argument");
  const size_t es = plan->dt == ECO_DT_F32 ? 4 : 2;
  ECO_REQUIRE((uintptr_t)x % es == 0 && (uintptr_t)y % es == 0, "group_norm: x or y is not aligned to its type");
  GnArgs a;
  a.x = x; a.y = y; a.lengths = lengths; a.gamma = gamma; a.beta = beta;
  a.x_row = x_row_stride ? x_row_stride : plan->c;
  a.y_row = y_row_stride ? y_row_stride : plan->c;
  ECO_REQUIRE(a.x_row >= plan->c && a.y_row >= plan->c, "group_norm: a row stride is smaller than %d channels", plan->c);
  ECO_REQUIRE(extent_fits(plan->s + 1, a.x_row, 0) && extent_fits(plan->s + 1, a.y_row, 0), "group_norm: row stride too large");
  a.x_image = x_image_stride ? x_image_stride : plan->s * a.x_row;
  a.y_image = y_image_stride ? y_image_stride : plan->s * a.y_row;
  const long x_ext = (plan->s - 1) * a.x_row + plan->c, y_ext = (plan->s - 1) * a.y_row + plan->c;   // elements of one image
  ECO_REQUIRE(a.x_image >= 0 && a.y_image >= y_ext, "group_norm: an image stride is too small");
  ECO_REQUIRE(extent_fits(plan->n, a.x_image, x_ext) && extent_fits(plan->n, a.y_image, y_ext), "group_norm: image stride too large");
  ECO_REQUIRE(plan->ws_bytes == 0 || workspace, "group_norm: this plan needs %ld bytes of workspace", (long)plan->ws_bytes);
  a.s = plan->s; a.c = plan->c; a.groups = plan->groups; a.cg = plan->c / plan->groups; a.act = act; a.eps = eps;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(plan->n * plan->groups)), block(kGnThreads);
  if (plan->dt == ECO_DT_F32) hipLaunchKernelGGL((group_norm_kernel<float>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((group_norm_kernel<unsigned short>), grid, block, 0, st, a);
  return check_launch("eco_group_norm_forward");
}
