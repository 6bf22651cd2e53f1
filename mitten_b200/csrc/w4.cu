// Products with 4-bit weights and group scales for the few rows of a decode
// step, and the weights' layout.  The reference computes its projections in
// f32 (MyLinear, qwen model.rs:110-130); a decode step reads every weight
// once for a handful of rows, so the weights' bytes bound it.
//
//   y[m][n] = sx[m] * sum_k x[m][k] * q[n][k] * s[n][k / G]
//
// q: integers -8..7; s: bf16, one per G = 32, 64 or 128 consecutive k of a
// row; x: bf16, f32, or e4m3 with one f32 scale sx per row (else sx = 1).
// q and bf16 s are exact, so y's error is x's products and f32 sums only.
// The codes enter the sums as q / 8, so that no product exceeds |x| before
// it meets its scale, and the result is multiplied by 8 (both exact).
//
// Layout.  Rows are padded to a multiple of 16 and k to a multiple of 128
// (codes 0, scales 0).  The unit is 16 rows x 64 k = 512 bytes, one 16-byte
// vector per lane of a warp: lane 4 g + t holds four words,
//   word 0: row g,     k = 8 t + 0..7       word 1: row g,     k = 32 + 8 t + 0..7
//   word 2: row g + 8, k = 8 t + 0..7       word 3: row g + 8, k = 32 + 8 t + 0..7
// and element j of a word's eight sits in nibble (j >> 1) + 4 (j & 1), two's
// complement: shifted right by 4 p and masked with 0x000f000f a word gives
// the neighbours k = 2p, 2p + 1 in its two halves.  Units follow one another
// along k, then along the rows.  Scales: [row unit][k / G][8] words, word g
// holding row g's scale in its low half and row g + 8's in its high half.
#include <algorithm>

#include <cuda_fp8.h>

#include "common.cuh"

namespace mtn {
namespace {

constexpr int kRowUnit = 16;
constexpr int kKPad = 128;
constexpr int64_t kMaxK = 65536;

__host__ __device__ __forceinline__ int64_t pad_k(int64_t k) { return (k + kKPad - 1) / kKPad * kKPad; }
__host__ __device__ __forceinline__ int64_t row_units(int64_t n) { return (n + kRowUnit - 1) / kRowUnit; }

__device__ __forceinline__ float ld_any(const void* p, int64_t i, int dtype) {
  if (dtype == MTN_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == MTN_DTYPE_F32) return static_cast<const float*>(p)[i];
  __nv_fp8_e4m3 v;
  v.__x = static_cast<const uint8_t*>(p)[i];
  return static_cast<float>(v);
}

// The word of eight codes (each -8..7) in k order.
__device__ __forceinline__ uint32_t pack_word(const int8_t* c) {
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) w |= (static_cast<uint32_t>(c[j]) & 15u) << (4 * ((j >> 1) + 4 * (j & 1)));
  return w;
}

// Element j of a word.
__device__ __forceinline__ int code_of(uint32_t w, int j) {
  return static_cast<int>(w << (28 - 4 * ((j >> 1) + 4 * (j & 1)))) >> 28;
}

// Packs 16 rows x 128 k per CTA of 128 threads: thread j owns column j of
// every row.  From float weights (codes == null) it first quantises: per
// group s = bf16(max|w| / 7), q = round(w / s) to -8..7, so that the codes
// are those of the scale as stored; a group of zeros has scale 0, one that
// holds a NaN or an infinity a NaN scale (its products then are NaN).
__global__ void __launch_bounds__(128) w4_pack_kernel(const void* w, int dtype, int64_t stride, const int8_t* codes,
                                                      int64_t code_stride, const __nv_bfloat16* in_scales,
                                                      int64_t scale_stride, int64_t n, int64_t k, int group,
                                                      uint4* packed, uint32_t* scales) {
  __shared__ int8_t q[kRowUnit][kKPad];
  __shared__ uint16_t sc[kRowUnit][kKPad / 32];
  const int64_t ksteps = pad_k(k) / kKPad;
  const int64_t ru = blockIdx.x / ksteps, ks = blockIdx.x - ru * ksteps;
  const int j = threadIdx.x, lane = j & 31;
  const int64_t col = ks * kKPad + j;
  const int gpw = kKPad / group;  // groups in this block
  __shared__ float wm[4];
  for (int r = 0; r < kRowUnit; ++r) {
    const int64_t row = ru * kRowUnit + r;
    const bool in = row < n && col < k;
    if (codes != nullptr) {
      const int c = in ? codes[row * code_stride + col] : 0;
      q[r][j] = static_cast<int8_t>(max(-8, min(7, c)));
      if (j < gpw) {
        const int64_t g = ks * gpw + j;
        sc[r][j] = row < n && g * group < k ? __bfloat16_as_ushort(in_scales[row * scale_stride + g]) : 0;
      }
      continue;
    }
    const float v = in ? ld_any(w, row * stride + col, dtype) : 0.0f;
    // max |w| of the group, NaN and infinity included as infinity
    float m = v - v == 0.0f ? fabsf(v) : INFINITY;
    m = warp_max(m);
    __syncthreads();
    if (lane == 0) wm[j >> 5] = m;
    __syncthreads();
    const int first = (j / group) * (group / 32);
    m = wm[first];
    for (int i = 1; i < group / 32; ++i) m = fmaxf(m, wm[first + i]);
    const __nv_bfloat16 s = __float2bfloat16_rn(m == INFINITY ? __int_as_float(0x7fc00000) : __fdiv_rn(m, 7.0f));
    const float sf = __bfloat162float(s);
    int c = 0;
    if (sf > 0.0f) c = static_cast<int>(fminf(7.0f, fmaxf(-8.0f, rintf(__fdiv_rn(v, sf)))));
    q[r][j] = static_cast<int8_t>(c);
    if (j % group == 0) sc[r][j / group] = __bfloat16_as_ushort(s);
  }
  __syncthreads();
  if (j < 64) {
    const int u = j >> 5, g = lane >> 2, t = lane & 3, k0 = 64 * u + 8 * t;
    uint4 o;
    o.x = pack_word(&q[g][k0]);
    o.y = pack_word(&q[g][k0 + 32]);
    o.z = pack_word(&q[g + 8][k0]);
    o.w = pack_word(&q[g + 8][k0 + 32]);
    packed[((ru * ksteps + ks) * 2 + u) * 32 + lane] = o;
  }
  for (int i = j; i < gpw * 8; i += 128) {
    const int g = i >> 3, r = i & 7;
    scales[((ru * ksteps + ks) * gpw + g) * 8 + r] =
        static_cast<uint32_t>(sc[r][g]) | static_cast<uint32_t>(sc[r + 8][g]) << 16;
  }
}

// Row-major values q * s of 16 rows x 128 k per CTA; the product of a 4-bit
// integer and a bf16 scale is exact in f32 and rounded once for bf16.
__global__ void __launch_bounds__(128) w4_dequantize_kernel(const uint4* packed, const uint32_t* scales, int64_t n,
                                                            int64_t k, int group, void* out, int dtype,
                                                            int64_t stride) {
  const int64_t ksteps = pad_k(k) / kKPad;
  const int64_t ru = blockIdx.x / ksteps, ks = blockIdx.x - ru * ksteps;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(packed + (ru * ksteps + ks) * 64);
  const int j = threadIdx.x;
  const int64_t col = ks * kKPad + j;
  if (col >= k) return;
  const int gpw = kKPad / group;
  const int u = j >> 6, h = (j >> 5) & 1, t = (j >> 3) & 3;
  for (int r = 0; r < kRowUnit; ++r) {
    const int64_t row = ru * kRowUnit + r;
    if (row >= n) return;
    const int g = r & 7;
    const uint32_t w = words[(u * 32 + 4 * g + t) * 4 + (r >> 3) * 2 + h];
    const uint32_t s2 = scales[((ru * ksteps + ks) * gpw + j / group) * 8 + g];
    const float s = __uint_as_float(r >= 8 ? s2 & 0xffff0000u : s2 << 16);
    const float v = static_cast<float>(code_of(w, j & 7)) * s;
    if (dtype == MTN_DTYPE_BF16)
      static_cast<__nv_bfloat16*>(out)[row * stride + col] = __float2bfloat16_rn(v);
    else
      static_cast<float*>(out)[row * stride + col] = v;
  }
}

struct W4Params {
  const void* x;
  int x_dtype;
  int64_t x_stride;
  const float* x_scales;
  int64_t m;
  const uint4* packed;
  const uint32_t* scales;
  int64_t n, k;
  int group;
  void* out;
  int out_dtype;
  int64_t out_stride;
};

__device__ __forceinline__ void store_out(const W4Params& p, int64_t m, int64_t n, float v) {
  v *= 8.0f;
  if (p.x_scales != nullptr) v *= p.x_scales[m];
  if (p.out_dtype == MTN_DTYPE_BF16)
    static_cast<__nv_bfloat16*>(p.out)[m * p.out_stride + n] = __float2bfloat16_rn(v);
  else
    static_cast<float*>(p.out)[m * p.out_stride + n] = v;
}

// One warp per output row and x row: lane l takes the words of its row in
// turn, eight products each.
__global__ void __launch_bounds__(256) w4_matvec_kernel(const W4Params p) {
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> 5;
  if (row >= p.n) return;
  const int64_t m = blockIdx.y;
  const int lane = threadIdx.x & 31;
  const int64_t kp = pad_k(p.k), ru = row / kRowUnit;
  const int r = static_cast<int>(row - ru * kRowUnit), g = r & 7;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(p.packed + ru * (kp / 64) * 32);
  const uint32_t* sc = p.scales + ru * (kp / p.group) * 8;
  float acc = 0.0f;
  for (int64_t c = lane; c * 8 < p.k; c += 32) {  // chunk c: k = 8 c .. 8 c + 7
    const int64_t unit = c >> 3;
    const int h = static_cast<int>(c >> 2) & 1, t = static_cast<int>(c) & 3;
    const uint32_t w = words[(unit * 32 + 4 * g + t) * 4 + (r >> 3) * 2 + h];
    const uint32_t s2 = sc[(c * 8 / p.group) * 8 + g];
    float part = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c * 8 + j < p.k)
        part = fmaf(ld_any(p.x, m * p.x_stride + c * 8 + j, p.x_dtype), static_cast<float>(code_of(w, j)) * 0.125f, part);
    acc = fmaf(part, __uint_as_float(r >= 8 ? s2 & 0xffff0000u : s2 << 16), acc);
  }
  acc = warp_sum(acc);
  if (lane == 0) store_out(p, m, row, acc);
}

int check_sizes(const char* who, int64_t n, int64_t k, int32_t group) {
  MTN_CHECK_ARG(n > 0 && n <= INT32_MAX && k > 0 && k <= kMaxK, "%s: n %lld or k %lld out of range", who,
                static_cast<long long>(n), static_cast<long long>(k));
  MTN_CHECK_ARG(group == 32 || group == 64 || group == 128, "%s: group %d not in {32,64,128}", who, group);
  MTN_CHECK_ARG(row_units(n) * (pad_k(k) / kKPad) <= INT32_MAX, "%s: matrix too large", who);
  return MTN_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace mtn

extern "C" {

size_t mtn_w4_packed_bytes(int64_t n, int64_t k) {
  if (n <= 0 || k <= 0 || k > mtn::kMaxK || n > INT32_MAX) return 0;
  return static_cast<size_t>(mtn::row_units(n)) * mtn::kRowUnit * mtn::pad_k(k) / 2;
}

size_t mtn_w4_scales_bytes(int64_t n, int64_t k, int32_t group) {
  if (n <= 0 || k <= 0 || k > mtn::kMaxK || n > INT32_MAX || (group != 32 && group != 64 && group != 128)) return 0;
  return static_cast<size_t>(mtn::row_units(n)) * mtn::kRowUnit * (mtn::pad_k(k) / group) * 2;
}

int mtn_w4_quantize(const void* weight, int32_t dtype, int64_t stride, int64_t n, int64_t k, int32_t group,
                    void* packed, void* scales, void* stream) {
  const int st = mtn::check_sizes("mtn_w4_quantize", n, k, group);
  if (st != MTN_OK) return st;
  MTN_CHECK_ARG(weight && packed && scales, "mtn_w4_quantize: null pointer");
  MTN_CHECK_ARG(dtype == MTN_DTYPE_BF16 || dtype == MTN_DTYPE_F32, "mtn_w4_quantize: bad dtype");
  MTN_CHECK_ARG(stride >= k, "mtn_w4_quantize: row stride shorter than a row");
  MTN_CHECK_ARG(mtn::aligned16(packed) && mtn::aligned16(scales), "mtn_w4_quantize: packed and scales must be 16-byte aligned");
  const int64_t blocks = mtn::row_units(n) * (mtn::pad_k(k) / mtn::kKPad);
  mtn::w4_pack_kernel<<<static_cast<unsigned>(blocks), 128, 0, static_cast<cudaStream_t>(stream)>>>(
      weight, dtype, stride, nullptr, 0, nullptr, 0, n, k, group, static_cast<uint4*>(packed),
      static_cast<uint32_t*>(scales));
  return mtn::check_launch("w4_pack_kernel");
}

int mtn_w4_pack(const int8_t* codes, int64_t code_stride, const void* code_scales, int64_t scale_stride, int64_t n,
                int64_t k, int32_t group, void* packed, void* scales, void* stream) {
  const int st = mtn::check_sizes("mtn_w4_pack", n, k, group);
  if (st != MTN_OK) return st;
  MTN_CHECK_ARG(codes && code_scales && packed && scales, "mtn_w4_pack: null pointer");
  MTN_CHECK_ARG(code_stride >= k && scale_stride >= (k + group - 1) / group, "mtn_w4_pack: row stride shorter than a row");
  MTN_CHECK_ARG(mtn::aligned16(packed) && mtn::aligned16(scales), "mtn_w4_pack: packed and scales must be 16-byte aligned");
  const int64_t blocks = mtn::row_units(n) * (mtn::pad_k(k) / mtn::kKPad);
  mtn::w4_pack_kernel<<<static_cast<unsigned>(blocks), 128, 0, static_cast<cudaStream_t>(stream)>>>(
      nullptr, MTN_DTYPE_F32, 0, codes, code_stride, static_cast<const __nv_bfloat16*>(code_scales), scale_stride, n, k,
      group, static_cast<uint4*>(packed), static_cast<uint32_t*>(scales));
  return mtn::check_launch("w4_pack_kernel");
}

int mtn_w4_dequantize(const void* packed, const void* scales, int64_t n, int64_t k, int32_t group, void* out,
                      int32_t dtype, int64_t stride, void* stream) {
  const int st = mtn::check_sizes("mtn_w4_dequantize", n, k, group);
  if (st != MTN_OK) return st;
  MTN_CHECK_ARG(packed && scales && out, "mtn_w4_dequantize: null pointer");
  MTN_CHECK_ARG(dtype == MTN_DTYPE_BF16 || dtype == MTN_DTYPE_F32, "mtn_w4_dequantize: bad dtype");
  MTN_CHECK_ARG(stride >= k, "mtn_w4_dequantize: row stride shorter than a row");
  MTN_CHECK_ARG(mtn::aligned16(packed) && mtn::aligned16(scales), "mtn_w4_dequantize: packed and scales must be 16-byte aligned");
  const int64_t blocks = mtn::row_units(n) * (mtn::pad_k(k) / mtn::kKPad);
  mtn::w4_dequantize_kernel<<<static_cast<unsigned>(blocks), 128, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint4*>(packed), static_cast<const uint32_t*>(scales), n, k, group, out, dtype, stride);
  return mtn::check_launch("w4_dequantize_kernel");
}

int mtn_w4_matvec(const void* x, int32_t x_dtype, int64_t x_stride, const float* x_scales, int64_t n_rows,
                  const void* packed, const void* scales, int64_t n, int64_t k, int32_t group, void* out,
                  int32_t out_dtype, int64_t out_stride, void* stream) {
  const int st = mtn::check_sizes("mtn_w4_matvec", n, k, group);
  if (st != MTN_OK) return st;
  MTN_CHECK_ARG(n_rows >= 0 && n_rows <= 65535, "mtn_w4_matvec: row count out of range");
  MTN_CHECK_ARG(x_dtype == MTN_DTYPE_BF16 || x_dtype == MTN_DTYPE_F32 || x_dtype == MTN_DTYPE_E4M3,
                "mtn_w4_matvec: bad x dtype");
  MTN_CHECK_ARG(out_dtype == MTN_DTYPE_BF16 || out_dtype == MTN_DTYPE_F32, "mtn_w4_matvec: bad out dtype");
  if (n_rows == 0) return MTN_OK;
  MTN_CHECK_ARG(x && packed && scales && out, "mtn_w4_matvec: null pointer");
  MTN_CHECK_ARG((x_dtype == MTN_DTYPE_E4M3) == (x_scales != nullptr),
                "mtn_w4_matvec: x_scales go with e4m3 rows, and only with them");
  MTN_CHECK_ARG(x_stride >= k && out_stride >= n, "mtn_w4_matvec: row strides shorter than a row");
  MTN_CHECK_ARG(mtn::aligned16(packed) && mtn::aligned16(scales), "mtn_w4_matvec: packed and scales must be 16-byte aligned");
  MTN_CHECK_ARG(out != x, "mtn_w4_matvec: out overlaps x");
  mtn::W4Params p{x, x_dtype, x_stride, x_scales, n_rows, static_cast<const uint4*>(packed),
                  static_cast<const uint32_t*>(scales), n, k, group, out, out_dtype, out_stride};
  const dim3 grid(static_cast<unsigned>((n + 7) / 8), static_cast<unsigned>(n_rows));
  mtn::w4_matvec_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return mtn::check_launch("w4_matvec_kernel");
}

}  // extern "C"
