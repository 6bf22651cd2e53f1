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
// Sums, means, y and y / scale are f32.  The floor of the scale keeps a row of zeros
// finite; a row that holds a NaN or an infinity gets NaNs, as the formula
// does: max|y| propagates NaN.
//
// A row is read once and stays in registers, 8 elements (one or two 16-byte
// vectors) times kVecs a thread: a warp per row up to 1024 elements, else a
// CTA whose threads the row fills; one pass for the sum of squares, one over
// the registers for the maximum and the output.  (Rows of more than 16384
// elements have 32 a thread in 1024 threads of 64 registers, and spill up to 372
// bytes a thread: 4096 x 18944 bf16 to e4m3 125 us, 0.66 of the copy rate.)  Many rows are bound by the
// bytes of x, residual, sum and output (16384 x 3584 bf16 to e4m3: 71 us, 5.8
// TB/s, 0.88 of the copy rate; 16384 x 896 f32: 38 us, 0.94), a few by the
// latency of one load and the block's two reductions (1 x 896: 1.9 us).  Rows
// that allow no vectors are bound by their many small loads and stores: 16384 x
// 3581 bf16 to e4m3 381 us, 16384 x 895 f32 92 us.
#include <algorithm>
#include <type_traits>

#include <cuda_fp8.h>

#include "common.cuh"

namespace mtn {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kMinScale = 7.888609052210118e-31f;  // 2^-100
constexpr int kMaxHidden = 32768;
constexpr int kWarpRows = 4;  // rows of a CTA, a warp each

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two quotients y / scale from the scale's reciprocal, in packed f32: the product
// is off by up to two steps, the remainder y - q * scale (one fma) says by how
// much, and its own quotient makes up for it, all but 2^-22 of a step (Markstein,
// IBM J. Res. Dev. 34, 1990).  The product alone gives 7 % of the values halfway
// between two codes the wrong code.  16384 x 3584 bf16 takes 71 us with the
// product alone as with the remainder (73 where these and the products of the
// row are not packed), and 86 with divisions.
__device__ __forceinline__ float2 quotients(float a, float b, uint64_t inv2, uint64_t neg_scale2) {
  float2 r;
  asm("{\n\t.reg .b64 y, q, e;\n\t"
      "mov.b64 y, {%2, %3};\n\t"
      "mul.rn.f32x2 q, y, %4;\n\t"
      "fma.rn.f32x2 e, q, %5, y;\n\t"
      "fma.rn.f32x2 q, e, %4, q;\n\t"
      "mov.b64 {%0, %1}, q;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a), "f"(b), "l"(inv2), "l"(neg_scale2));
  return r;
}

__device__ __forceinline__ uint64_t twice(float x) {
  const uint64_t b = __float_as_uint(x);
  return b << 32 | b;
}

// (a, b) * by * (wa, wb), each product rounded.
__device__ __forceinline__ float2 products(float a, float b, uint64_t by2, float wa, float wb) {
  float2 r;
  asm("{\n\t.reg .b64 v, w;\n\t"
      "mov.b64 v, {%2, %3};\n\t"
      "mov.b64 w, {%5, %6};\n\t"
      "mul.rn.f32x2 v, v, %4;\n\t"
      "mul.rn.f32x2 v, v, w;\n\t"
      "mov.b64 {%0, %1}, v;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a), "f"(b), "l"(by2), "f"(wa), "f"(wb));
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
  int64_t n_rows;
  int hidden;
  float eps;
};

// Reduction over the threads of one row: a warp, or the CTA's warps.
template <bool kWarp, bool kMax>
__device__ __forceinline__ float row_reduce(float v, float* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = kMax ? max_nan(v, u) : v + u;
  }
  if constexpr (!kWarp) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) buf[warp] = v;
    __syncthreads();
    v = lane < warps ? buf[lane] : 0.0f;  // 0 changes neither a sum nor a maximum of magnitudes
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float u = __shfl_xor_sync(0xffffffffu, v, o);
      v = kMax ? max_nan(v, u) : v + u;
    }
  }
  return v;
}

struct NoRes {};  // no residual

template <typename T>
struct Raw8 {  // eight elements as loaded
  uint4 w[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ void load8(const void* p, int64_t at, Raw8<T>& r) {
  const uint4* q = reinterpret_cast<const uint4*>(static_cast<const T*>(p) + at);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.w[i] = q[i];
}

template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
    const uint32_t u[4] = {r.w[i].x, r.w[i].y, r.w[i].z, r.w[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 2) {
        v[2 * j] = bf2_to_f2(u[j]).x;
        v[2 * j + 1] = bf2_to_f2(u[j]).y;
      } else {
        v[4 * i + j] = __uint_as_float(u[j]);
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (sizeof(T) == 2)
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  else
    return static_cast<const float*>(p)[i];
}

// X, R: types of x and the residual (NoRes: none).  kVec: every row allows
// 16-byte vectors; else elements are loaded one by one, neighbouring threads
// next to each other.  kThreads: the most of a CTA (128: a warp per row).
template <typename X, typename R, int kVecs, bool kVec, int kThreads>
__global__ void __launch_bounds__(kThreads) add_rms_norm_kernel(const NormParams p, int out_dtype) {
  constexpr bool kWarp = kThreads == 32 * kWarpRows, kRes = !std::is_same<R, NoRes>::value;
  using RT = typename std::conditional<kRes, R, X>::type;
  __shared__ float buf[2][32];
  pdl_enter();
  const int64_t row = kWarp ? static_cast<int64_t>(blockIdx.x) * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
  if (kWarp && row >= p.n_rows) return;
  const int tid = kWarp ? threadIdx.x & 31 : threadIdx.x, threads = kWarp ? 32 : blockDim.x;
  const int64_t xo = row * p.x_stride, ro = row * p.res_stride, so = row * p.sum_stride, oo = row * p.out_stride;
  // element e of the thread's vector j
  auto place = [&](int j, int e) { return kVec ? (tid + j * threads) * 8 + e : tid + (j * 8 + e) * threads; };
  float v[kVecs][8];
  if constexpr (kVec) {
    Raw8<X> rx[kVecs];
    Raw8<RT> rr[kVecs];
#pragma unroll
    for (int j = 0; j < kVecs; ++j)
      if (place(j, 0) < p.hidden) {
        load8<X>(p.x, xo + place(j, 0), rx[j]);
        if constexpr (kRes) load8<RT>(p.res, ro + place(j, 0), rr[j]);
      }
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      if (place(j, 0) < p.hidden) {
        unpack8<X>(rx[j], v[j]);
        if constexpr (kRes) {
          float r[8];
          unpack8<RT>(rr[j], r);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[j][e] += r[e];
          if constexpr (sizeof(RT) == 2) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              w[e] = f2_to_bf2(v[j][2 * e], v[j][2 * e + 1]);
              v[j][2 * e] = bf2_to_f2(w[e]).x;
              v[j][2 * e + 1] = bf2_to_f2(w[e]).y;
            }
            *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.sum) + so + place(j, 0)) =
                make_uint4(w[0], w[1], w[2], w[3]);
          } else {
            float4* q = reinterpret_cast<float4*>(static_cast<float*>(p.sum) + so + place(j, 0));
            q[0] = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
            q[1] = make_float4(v[j][4], v[j][5], v[j][6], v[j][7]);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] = 0.0f;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < kVecs; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] = place(j, e) < p.hidden ? load1<X>(p.x, xo + place(j, e)) : 0.0f;
    if constexpr (kRes) {
#pragma unroll
      for (int j = 0; j < kVecs; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = place(j, e);
          if (i >= p.hidden) continue;
          v[j][e] += load1<RT>(p.res, ro + i);
          if constexpr (sizeof(RT) == 2) {
            const __nv_bfloat16 h = __float2bfloat16_rn(v[j][e]);
            static_cast<__nv_bfloat16*>(p.sum)[so + i] = h;
            v[j][e] = __bfloat162float(h);
          } else {
            static_cast<float*>(p.sum)[so + i] = v[j][e];
          }
        }
    }
  }
  float ss = 0.0f;
#pragma unroll
  for (int j = 0; j < kVecs; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(v[j][e], v[j][e], ss);
  ss = row_reduce<kWarp, false>(ss, buf[0]);
  const float rstd = 1.0f / sqrtf(ss / static_cast<float>(p.hidden) + p.eps);
  const uint64_t rstd2 = twice(rstd);
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 1.0f;
    if (p.w1 != nullptr) {
      if (kVec && place(j, 0) < p.hidden) {
        const float4 a = *reinterpret_cast<const float4*>(p.w1 + place(j, 0));
        const float4 b = *reinterpret_cast<const float4*>(p.w1 + place(j, 0) + 4);
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
      } else if (!kVec) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (place(j, e) < p.hidden) w[e] = p.w1[place(j, e)];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float2 y = products(v[j][e], v[j][e + 1], rstd2, w[e], w[e + 1]);
      v[j][e] = y.x;
      v[j][e + 1] = y.y;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (place(j, e) < p.hidden) top = max_nan(top, fabsf(v[j][e]));
  }
  if (out_dtype == MTN_DTYPE_E4M3) {
    top = row_reduce<kWarp, true>(top, buf[1]);
    const float scale = max_nan(top / kE4m3Max, kMinScale), inv = 1.0f / scale;
    if (tid == 0) p.scales[row] = scale;
    // an infinite scale: quotients of 0, and NaN for an infinite y
    const uint64_t inv2 = twice(inv), neg_scale2 = twice(scale < INFINITY ? -scale : 0.0f);
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      if (kVec && place(j, 0) >= p.hidden) continue;
      uint16_t c[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        c[e] = __nv_cvt_float2_to_fp8x2(quotients(v[j][2 * e], v[j][2 * e + 1], inv2, neg_scale2), __NV_SATFINITE, __NV_E4M3);
      uint8_t* o = static_cast<uint8_t*>(p.out) + oo;
      if constexpr (kVec) {
        *reinterpret_cast<uint2*>(o + place(j, 0)) = make_uint2(c[0] | static_cast<uint32_t>(c[1]) << 16,
                                                                c[2] | static_cast<uint32_t>(c[3]) << 16);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (place(j, e) < p.hidden) o[place(j, e)] = static_cast<uint8_t>(c[e >> 1] >> (8 * (e & 1)));
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    if (kVec) {
      if (place(j, 0) >= p.hidden) continue;
      if (out_dtype == MTN_DTYPE_BF16) {
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + oo + place(j, 0)) =
            make_uint4(f2_to_bf2(v[j][0], v[j][1]), f2_to_bf2(v[j][2], v[j][3]), f2_to_bf2(v[j][4], v[j][5]),
                       f2_to_bf2(v[j][6], v[j][7]));
      } else {
        float4* q = reinterpret_cast<float4*>(static_cast<float*>(p.out) + oo + place(j, 0));
        q[0] = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
        q[1] = make_float4(v[j][4], v[j][5], v[j][6], v[j][7]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (place(j, e) >= p.hidden) continue;
        if (out_dtype == MTN_DTYPE_BF16)
          static_cast<__nv_bfloat16*>(p.out)[oo + place(j, e)] = __float2bfloat16_rn(v[j][e]);
        else
          static_cast<float*>(p.out)[oo + place(j, e)] = v[j][e];
      }
    }
  }
}

using NormKernel = void (*)(const NormParams, int);

template <typename X, typename R, bool kVec>
NormKernel norm_kernel(int vecs, bool warp) {
  constexpr int kW = 32 * kWarpRows;
  if (warp)
    return vecs <= 1   ? add_rms_norm_kernel<X, R, 1, kVec, kW>
           : vecs <= 2 ? add_rms_norm_kernel<X, R, 2, kVec, kW>
                       : add_rms_norm_kernel<X, R, 4, kVec, kW>;
  if (vecs <= 1) return add_rms_norm_kernel<X, R, 1, kVec, 1024>;
  if (vecs <= 2) return add_rms_norm_kernel<X, R, 2, kVec, 1024>;
  return add_rms_norm_kernel<X, R, 4, kVec, 1024>;
}

template <typename X, typename R>
NormKernel norm_kernel(int vecs, bool vec, bool warp) {
  return vec ? norm_kernel<X, R, true>(vecs, warp) : norm_kernel<X, R, false>(vecs, warp);
}

template <typename X>
NormKernel norm_kernel(const NormParams& p, bool res_bf16, int vecs, bool vec, bool warp) {
  if (p.res == nullptr) return norm_kernel<X, NoRes>(vecs, vec, warp);
  return res_bf16 ? norm_kernel<X, __nv_bfloat16>(vecs, vec, warp) : norm_kernel<X, float>(vecs, vec, warp);
}

bool rows_aligned(const void* p, int64_t stride, int64_t n_rows, int elem, int64_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (n_rows == 1 || stride * elem % bytes == 0);
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
  MTN_CHECK_ARG(residual == nullptr || sum != residual || sum_stride == res_stride || n_rows == 1,
                "mtn_add_rms_norm: a sum in the residual's place needs equal strides");
  MTN_CHECK_ARG(mtn::elem_aligned(x, x_dtype) && mtn::elem_aligned(out, out_dtype) &&
                    mtn::elem_aligned(residual, res_dtype) && mtn::elem_aligned(sum, res_dtype) &&
                    mtn::elem_aligned(w1, MTN_DTYPE_F32) && mtn::elem_aligned(scales, MTN_DTYPE_F32),
                "mtn_add_rms_norm: a pointer is not aligned to its elements");
  MTN_CHECK_ARG(x_stride >= hidden && out_stride >= hidden &&
                    (residual == nullptr || (res_stride >= hidden && sum_stride >= hidden)),
                "mtn_add_rms_norm: row strides shorter than a row");
  mtn::NormParams p{x,          residual,   sum,        w1,         out,    scales, x_stride,
                    res_stride, sum_stride, out_stride, n_rows,     hidden, eps};
  const bool xb = x_dtype == MTN_DTYPE_BF16, rb = res_dtype == MTN_DTYPE_BF16;
  const int xe = xb ? 2 : 4, re = rb ? 2 : 4;
  const int oe = out_dtype == MTN_DTYPE_BF16 ? 2 : out_dtype == MTN_DTYPE_F32 ? 4 : 1;
  const bool vec = hidden % 8 == 0 && mtn::rows_aligned(x, x_stride, n_rows, xe, 16) &&
                   mtn::rows_aligned(out, out_stride, n_rows, oe, oe == 1 ? 8 : 16) &&
                   (residual == nullptr || (mtn::rows_aligned(residual, res_stride, n_rows, re, 16) &&
                                            mtn::rows_aligned(sum, sum_stride, n_rows, re, 16))) &&
                   (w1 == nullptr || reinterpret_cast<uintptr_t>(w1) % 16 == 0);
  // Vectors of 8 elements.  A warp takes a row of up to 4 a lane.  A CTA has a
  // thread per vector where the rows are few (latency) or not aligned, and one
  // per two where they are many: 16384 x 3584 bf16 to e4m3 took 82, 72 and 75
  // us with 1, 2 and 4 vectors a thread.
  const int vectors = (hidden + 7) / 8;
  const bool few = n_rows <= 2 * mtn::sm_count();
  const bool warp = vectors <= (few ? 32 : 128);
  int per = warp ? (vectors + 31) / 32 : few || !vec ? 1 : 2;
  while (!warp && (vectors + per - 1) / per > 1024) per *= 2;
  per = per == 3 ? 4 : per;
  const int threads = warp ? 32 * mtn::kWarpRows : ((vectors + per - 1) / per + 31) / 32 * 32;
  const int64_t grid = warp ? (n_rows + mtn::kWarpRows - 1) / mtn::kWarpRows : n_rows;
  const mtn::NormKernel kern = xb ? mtn::norm_kernel<__nv_bfloat16>(p, rb, per, vec, warp)
                                  : mtn::norm_kernel<float>(p, rb, per, vec, warp);
  return mtn::launch_pdl(kern, dim3(static_cast<unsigned>(grid)), dim3(static_cast<unsigned>(threads)), 0,
                         static_cast<cudaStream_t>(stream), "add_rms_norm_kernel", p, static_cast<int>(out_dtype));
}

}  // extern "C"
