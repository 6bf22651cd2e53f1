// Residual addition and RMSNorm in one launch, with an optional output in
// 8 bits: what stands between two projections of a decoder layer
// (RmsNorm::forward, qwen model.rs:98-108, and the residual sums of
// Qwen3_5Layer::forward, model.rs:348-365).
//
//   s = x + r                        rounded to the residual's type and stored
//   y = s / sqrt(mean(s^2) + eps) * w1          w1 = 1 + w; s as it is stored
//   out = y                          bf16 or f32, rounded once, or
//   out = e4m3(y / scale), scale = max(max|y| / 448, 2^-100)   per row
//
// Sums, means and y are f32.  The floor of the scale keeps a row of zeros
// finite; a row that holds a NaN or an infinity gets NaNs, as the formula
// does: max|y| propagates NaN.
//
// One CTA per row.
#include <cuda_fp8.h>

#include "common.cuh"

namespace mtn {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kMinScale = 7.888609052210118e-31f;  // 2^-100
constexpr int kMaxHidden = 32768;
constexpr int kNormThreads = 256;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct NormParams {
  const void* x;
  const void* res;  // or null
  void* sum;
  const float* w1;  // or null
  void* out;
  float* scales;
  int64_t x_stride, res_stride, sum_stride, out_stride;
  int hidden;
  float eps;
};

template <typename T>
__device__ __forceinline__ float ld_elem(const void* p, int64_t i) {
  if constexpr (sizeof(T) == 2)
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  else
    return static_cast<const float*>(p)[i];
}

template <bool kMax>
__device__ __forceinline__ float block_reduce(float v, float* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = kMax ? max_nan(v, u) : v + u;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (lane == 0) buf[warp] = v;
  __syncthreads();
  v = buf[0];
  for (int w = 1; w < kNormThreads / 32; ++w) v = kMax ? max_nan(v, buf[w]) : v + buf[w];
  return v;
}

template <typename X, typename R>
__global__ void __launch_bounds__(kNormThreads) add_rms_norm_kernel(const NormParams p, int out_dtype) {
  __shared__ float buf[kNormThreads / 32];
  const int64_t row = blockIdx.x;
  const int64_t xo = row * p.x_stride, ro = row * p.res_stride, so = row * p.sum_stride, oo = row * p.out_stride;
  float ss = 0.0f;
  for (int i = threadIdx.x; i < p.hidden; i += kNormThreads) {
    float s = ld_elem<X>(p.x, xo + i);
    if (p.res != nullptr) {
      s += ld_elem<R>(p.res, ro + i);
      if constexpr (sizeof(R) == 2) {
        const __nv_bfloat16 h = __float2bfloat16_rn(s);
        static_cast<__nv_bfloat16*>(p.sum)[so + i] = h;
        s = __bfloat162float(h);
      } else {
        static_cast<float*>(p.sum)[so + i] = s;
      }
    }
    ss = fmaf(s, s, ss);
  }
  ss = block_reduce<false>(ss, buf);
  const float rstd = 1.0f / sqrtf(ss / static_cast<float>(p.hidden) + p.eps);
  // every thread reads back the elements it wrote itself
  auto value = [&](int i) {
    const float s = p.res != nullptr ? ld_elem<R>(p.sum, so + i) : ld_elem<X>(p.x, xo + i);
    return s * rstd * (p.w1 != nullptr ? p.w1[i] : 1.0f);
  };
  float inv = 1.0f;
  if (out_dtype == MTN_DTYPE_E4M3) {
    float m = 0.0f;
    for (int i = threadIdx.x; i < p.hidden; i += kNormThreads) m = max_nan(m, fabsf(value(i)));
    m = block_reduce<true>(m, buf);
    const float scale = max_nan(m / kE4m3Max, kMinScale);
    if (threadIdx.x == 0) p.scales[row] = scale;
    inv = 1.0f / scale;
  }
  for (int i = threadIdx.x; i < p.hidden; i += kNormThreads) {
    const float y = value(i);
    if (out_dtype == MTN_DTYPE_E4M3)
      static_cast<uint8_t*>(p.out)[oo + i] = __nv_cvt_float_to_fp8(y * inv, __NV_SATFINITE, __NV_E4M3);
    else if (out_dtype == MTN_DTYPE_BF16)
      static_cast<__nv_bfloat16*>(p.out)[oo + i] = __float2bfloat16_rn(y);
    else
      static_cast<float*>(p.out)[oo + i] = y;
  }
}

}  // namespace
}  // namespace mtn

extern "C" {

int mtn_add_rms_norm(const void* x, int32_t x_dtype, int64_t x_stride, const void* residual, int64_t res_stride,
                     void* sum, int64_t sum_stride, int32_t res_dtype, const float* w1, float eps, int64_t n_rows,
                     int32_t hidden, void* out, int32_t out_dtype, int64_t out_stride, float* scales, void* stream) {
  MTN_CHECK_ARG(n_rows >= 0 && n_rows <= INT32_MAX, "mtn_add_rms_norm: bad row count");
  MTN_CHECK_ARG(hidden > 0 && hidden <= mtn::kMaxHidden, "mtn_add_rms_norm: hidden %d not in 1..%d", hidden,
                mtn::kMaxHidden);
  MTN_CHECK_ARG(x_dtype == MTN_DTYPE_BF16 || x_dtype == MTN_DTYPE_F32, "mtn_add_rms_norm: bad x dtype");
  MTN_CHECK_ARG(res_dtype == MTN_DTYPE_BF16 || res_dtype == MTN_DTYPE_F32, "mtn_add_rms_norm: bad residual dtype");
  MTN_CHECK_ARG(out_dtype == MTN_DTYPE_BF16 || out_dtype == MTN_DTYPE_F32 || out_dtype == MTN_DTYPE_E4M3,
                "mtn_add_rms_norm: bad out dtype");
  MTN_CHECK_ARG(eps >= 0.0f, "mtn_add_rms_norm: eps must not be negative");
  if (n_rows == 0) return MTN_OK;
  MTN_CHECK_ARG(x && out, "mtn_add_rms_norm: null pointer");
  MTN_CHECK_ARG((residual == nullptr) == (sum == nullptr), "mtn_add_rms_norm: residual and sum come together");
  MTN_CHECK_ARG((out_dtype == MTN_DTYPE_E4M3) == (scales != nullptr),
                "mtn_add_rms_norm: scales go with an e4m3 output, and only with one");
  MTN_CHECK_ARG(out != x && out != residual && out != sum && sum != x, "mtn_add_rms_norm: outputs overlap the inputs");
  MTN_CHECK_ARG(x_stride >= hidden && out_stride >= hidden &&
                    (residual == nullptr || (res_stride >= hidden && sum_stride >= hidden)),
                "mtn_add_rms_norm: row strides shorter than a row");
  mtn::NormParams p{x, residual, sum, w1, out, scales, x_stride, res_stride, sum_stride, out_stride, hidden, eps};
  auto s = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(n_rows);
  const bool xb = x_dtype == MTN_DTYPE_BF16, rb = res_dtype == MTN_DTYPE_BF16;
  if (xb && rb)
    mtn::add_rms_norm_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, mtn::kNormThreads, 0, s>>>(p, out_dtype);
  else if (xb)
    mtn::add_rms_norm_kernel<__nv_bfloat16, float><<<grid, mtn::kNormThreads, 0, s>>>(p, out_dtype);
  else if (rb)
    mtn::add_rms_norm_kernel<float, __nv_bfloat16><<<grid, mtn::kNormThreads, 0, s>>>(p, out_dtype);
  else
    mtn::add_rms_norm_kernel<float, float><<<grid, mtn::kNormThreads, 0, s>>>(p, out_dtype);
  return mtn::check_launch("add_rms_norm_kernel");
}

}  // extern "C"
