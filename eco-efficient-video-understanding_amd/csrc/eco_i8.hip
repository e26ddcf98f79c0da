// eco_i8.hip -- rows to 8-bit integers and the inner product of such rows (include/eco_hip.h, ABI v20).
#include <math.h>

#include "eco_common.h"

namespace eco {

constexpr int kI8Threads = 256;

__device__ __forceinline__ float i8_load(const float* p) { return ld(p); }
__device__ __forceinline__ float i8_load(const unsigned short* p) { return bf16_bits_to_f32(ld(p)); }

__device__ __forceinline__ unsigned f32_bits(float v) {
  unsigned u;
  __builtin_memcpy(&u, &v, 4);
  return u;
}
__device__ __forceinline__ float bits_f32(unsigned u) {
  float v;
  __builtin_memcpy(&v, &u, 4);
  return v;
}

// The integer nearest to 127 v / top (ties to even), 0 <= |v| <= top, top > 0 and finite.  inv = fp32(127 / top): the product
// is off by at most 127 * 2^-23 = 1.6e-5, so its rounding is right unless it lies within 1e-4 of a half; there the sides of
// the comparison |v| * 254 <> (2 k + 1) * top are products of a 24-bit and an 8-bit number, exact in fp64.
__device__ __forceinline__ int i8_quant(float v, float top, float inv) {
  const float t = v * inv;
  const float r = rintf(t);
  if (fabsf(fabsf(t - r) - 0.5f) > 1e-4f) return (int)r;
  const float k = floorf(fabsf(t));
  const double lhs = fabs((double)v) * 254.0, rhs = (double)(2.0f * k + 1.0f) * (double)top;
  const int n = (int)k + ((lhs > rhs || (lhs == rhs && ((int)k & 1))) ? 1 : 0);
  return v < 0.0f ? -n : n;
}

// One wave per row: the largest magnitude as bits (a NaN or an infinity has the largest), then the integers.
template <typename T>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T* x, long ldx, signed char* q, long ldq, float* scale,
                                                         long m, long k) {
  const int lane = lane_id();
  const int wave = uniform((int)(threadIdx.x >> 6));
  for (long i = (long)blockIdx.x * 4 + wave; i < m; i += (long)gridDim.x * 4) {
    const T* xr = x + i * ldx;
    unsigned top_bits = 0u;
    for (long j = lane; j < k; j += kWave) {
      const unsigned b = f32_bits(i8_load(xr + j)) & 0x7fffffffu;
      top_bits = b > top_bits ? b : top_bits;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      const unsigned o = f32_bits(shfl_xor(bits_f32(top_bits), d));
      top_bits = o > top_bits ? o : top_bits;
    }
    const bool finite = top_bits < 0x7f800000u;
    float top = bits_f32(top_bits);
    if (lane == 0) st(scale + i, finite ? top / 127.0f : bits_f32(0x7fc00000u));
    // rows of tiny values are scaled up by a power of two first: 127 / top must be finite
    const float up = top < 1e-30f ? 1.2676506e30f : 1.0f;   // 2^100
    top *= up;
    const float inv = 127.0f / top;
    for (long j = lane; j < k; j += kWave)
      st(q + i * ldq + j, (signed char)(finite && top > 0.0f ? i8_quant(i8_load(xr + j) * up, top, inv) : 0));
  }
}

struct I8Args {
  const signed char* x;
  const signed char* w;
  const float* sx;
  const float* sw;
  const float* bias;
  void* y;
  long ldx, ldw, ldy;
  long m;
  int n, k, act;
};

__device__ __forceinline__ float i8_epilogue(int acc, float sx, float sw, float bias, int act) {
  float v = (float)acc * sx * sw + bias;
  if (act == ECO_ACT_RELU) v = v < 0.0f ? 0.0f : v;
  else if (act == ECO_ACT_SILU) v = v / (1.0f + expf(-v));
  return v;
}
__device__ __forceinline__ void i8_store(float* p, float v) { st(p, v); }
__device__ __forceinline__ void i8_store(unsigned short* p, float v) { st(p, (unsigned short)f32_to_bf16_bits(v)); }

// One thread per output.
template <typename T>
__global__ __launch_bounds__(256) void inner_product_i8_kernel(const I8Args a) {
  const long total = a.m * a.n;
  for (long o = (long)blockIdx.x * kI8Threads + threadIdx.x; o < total; o += (long)gridDim.x * kI8Threads) {
    const long i = o / a.n;
    const int j = (int)(o - i * a.n);
    const signed char* xr = a.x + i * a.ldx;
    const signed char* wr = a.w + j * a.ldw;
    int acc = 0;
    for (int l = 0; l < a.k; ++l) acc += (int)ld(xr + l) * (int)ld(wr + l);
    i8_store((T*)a.y + i * a.ldy + j, i8_epilogue(acc, ld(a.sx + i), ld(a.sw + j), a.bias ? ld(a.bias + j) : 0.0f, a.act));
  }
}

static inline unsigned i8_grid(long count, long per_block) {
  const long g = ceil_div(count, per_block);
  return (unsigned)(g > 1048576 ? 1048576 : g);   // grid-stride beyond this
}

}  // namespace eco

using namespace eco;

extern "C" int eco_quant_rows_forward(const void* x, int32_t dt, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
                                      int64_t m, int64_t k, void* stream) {
  clear_error();
  ECO_REQUIRE(dt == ECO_DT_F32 || dt == ECO_DT_BF16, "quant_rows: unknown type %d", dt);
  ECO_REQUIRE(m >= 0 && k > 0, "quant_rows: bad shape");
  ECO_REQUIRE(m <= 2147483647l && k <= 2147483647l, "quant_rows: too many rows or columns");
  if (m == 0) return ECO_OK;
  ECO_REQUIRE(x && q && scale, "quant_rows: null argument");
  const size_t es = dt == ECO_DT_F32 ? 4 : 2;
  ECO_REQUIRE((uintptr_t)x % es == 0, "quant_rows: x is not aligned to its type");
  if (ldx == 0) ldx = k;
  if (ldq == 0) ldq = k;
  ECO_REQUIRE(ldx >= k && ldq >= k, "quant_rows: a row stride is smaller than %ld", (long)k);
  ECO_REQUIRE(extent_fits(m, ldx, k) && extent_fits(m, ldq, k), "quant_rows: a row stride is too large");
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid(i8_grid(m, 4)), block(kI8Threads);
  if (dt == ECO_DT_F32)
    hipLaunchKernelGGL((quant_rows_kernel<float>), grid, block, 0, st, (const float*)x, (long)ldx, (signed char*)q, (long)ldq,
                       scale, (long)m, (long)k);
  else
    hipLaunchKernelGGL((quant_rows_kernel<unsigned short>), grid, block, 0, st, (const unsigned short*)x, (long)ldx,
                       (signed char*)q, (long)ldq, scale, (long)m, (long)k);
  return check_launch("eco_quant_rows_forward");
}

extern "C" int eco_inner_product_i8_plan_create(int64_t m, int64_t n, int64_t k, int32_t dt, int32_t num_cu,
                                                eco_inner_product_i8_plan* plan) {
  clear_error();
  ECO_REQUIRE(plan != nullptr, "inner_product_i8: null plan");
  ECO_REQUIRE(m >= 0 && n > 0 && k > 0, "inner_product_i8: bad shape");
  ECO_REQUIRE(k <= ECO_I8_MAX_K, "inner_product_i8: sums of %ld products can leave 32 bits (at most %d)", (long)k, ECO_I8_MAX_K);
  ECO_REQUIRE(m <= 2147483647l && n <= 2147483647l, "inner_product_i8: too many rows");
  ECO_REQUIRE(dt == ECO_DT_F32 || dt == ECO_DT_BF16, "inner_product_i8: unknown type %d", dt);
  ECO_REQUIRE(num_cu >= 0, "inner_product_i8: negative num_cu");
  memset(plan, 0, sizeof(*plan));
  plan->m = m; plan->n = (int32_t)n; plan->k = (int32_t)k; plan->dt = dt;
  plan->num_cu = num_cu ? num_cu : current_device_num_cu();
  plan->bm = plan->bn = 1; plan->ksplit = 1;
  return ECO_OK;
}

extern "C" int eco_inner_product_i8_forward(const eco_inner_product_i8_plan* plan, const int8_t* x, int64_t ldx,
                                            const float* sx, const int8_t* w, int64_t ldw, const float* sw,
                                            const float* bias, int32_t act, void* y, int64_t ldy, void* workspace,
                                            void* stream) {
  clear_error();
  ECO_REQUIRE(plan != nullptr, "inner_product_i8: null plan");
  eco_inner_product_i8_plan same;
  if (int rc = eco_inner_product_i8_plan_create(plan->m, plan->n, plan->k, plan->dt, plan->num_cu, &same)) return rc;
  ECO_REQUIRE(memcmp(&same, plan, sizeof(same)) == 0, "inner_product_i8: the plan is not one of eco_inner_product_i8_plan_create");
  ECO_REQUIRE(act == ECO_ACT_NONE || act == ECO_ACT_RELU || act == ECO_ACT_SILU, "inner_product_i8: unknown activation %d", act);
  if (plan->m == 0) return ECO_OK;
  ECO_REQUIRE(x && sx && w && sw && y, "inner_product_i8: null argument");
  ECO_REQUIRE((uintptr_t)y % (plan->dt == ECO_DT_F32 ? 4 : 2) == 0, "inner_product_i8: y is not aligned to its type");
  I8Args a;
  a.x = (const signed char*)x; a.w = (const signed char*)w; a.sx = sx; a.sw = sw; a.bias = bias; a.y = y;
  a.ldx = ldx ? ldx : plan->k; a.ldw = ldw ? ldw : plan->k; a.ldy = ldy ? ldy : plan->n;
  ECO_REQUIRE(a.ldx >= plan->k && a.ldw >= plan->k && a.ldy >= plan->n, "inner_product_i8: a row stride is smaller than a row");
  ECO_REQUIRE(extent_fits(plan->m, a.ldx, plan->k) && extent_fits(plan->n, a.ldw, plan->k) && extent_fits(plan->m, a.ldy, plan->n),
              "inner_product_i8: a row stride is too large");
  ECO_REQUIRE(plan->ws_bytes == 0 || workspace, "inner_product_i8: this plan needs %ld bytes of workspace", (long)plan->ws_bytes);
  a.m = plan->m; a.n = plan->n; a.k = plan->k; a.act = act;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid(i8_grid(a.m * a.n, kI8Threads)), block(kI8Threads);
  if (plan->dt == ECO_DT_F32) hipLaunchKernelGGL((inner_product_i8_kernel<float>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((inner_product_i8_kernel<unsigned short>), grid, block, 0, st, a);
  return check_launch("eco_inner_product_i8_forward");
}
