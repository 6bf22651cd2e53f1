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
// the neighbours k = 2p, 2p + 1 in its two halves (integers made floats by an
// exponent set beside them: Kim, Henry, Fahim, Awadalla, 2022).  Units follow one another
// along k, then along the rows.  Scales: [row unit][k / G][8] words, word g
// holding row g's scale in its low half and row g + 8's in its high half.
#include <algorithm>
#include <atomic>

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
// holds a NaN or an infinity a NaN scale (its products then are NaN).  Runs once
// a weight and was not made faster: 18944 x 3584 takes 430 us from floats (two
// barriers a row) and 160 from codes.
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

// Row-major values q * s, 16 rows x 128 k at a time, kDequantSteps of them per
// CTA; a thread has eight consecutive k of a row.  The product of a 4-bit
// integer and a bf16 scale is exact in f32 and rounded once for bf16.  Bound by
// the bytes written: 18944 x 3584 to bf16 34 us, 5.1 TB/s.
constexpr int kDequantSteps = 4;

__global__ void __launch_bounds__(256) w4_dequantize_kernel(const uint32_t* packed, const uint32_t* scales, int64_t n,
                                                            int64_t k, int group, void* out, int dtype, int64_t stride,
                                                            bool vec) {
  const int64_t ksteps = pad_k(k) / kKPad, blocks = (ksteps + kDequantSteps - 1) / kDequantSteps;
  const int64_t ru = blockIdx.x / blocks, first = (blockIdx.x - ru * blocks) * kDequantSteps;
  const int r = threadIdx.x >> 4, c = threadIdx.x & 15, g = r & 7;
  const int64_t row = ru * kRowUnit + r;
  if (row >= n) return;
  const int word = (((c >> 3) * 32 + 4 * g + (c & 3)) * 4) + (r >> 3) * 2 + ((c >> 2) & 1), gpw = kKPad / group;
  uint32_t w[kDequantSteps], s2[kDequantSteps];
#pragma unroll
  for (int i = 0; i < kDequantSteps; ++i) {
    const int64_t at = ru * ksteps + first + i;
    if (first + i < ksteps) {
      w[i] = packed[at * 256 + word];
      s2[i] = scales[(at * gpw + c * 8 / group) * 8 + g];
    }
  }
#pragma unroll
  for (int i = 0; i < kDequantSteps; ++i) {
    const int64_t col = (first + i) * kKPad + c * 8;
    if (col >= k) return;
    const float s = __uint_as_float(r >= 8 ? s2[i] & 0xffff0000u : s2[i] << 16);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(code_of(w[i], j)) * s;
    const int64_t to = row * stride + col;
    if (vec && col + 8 <= k) {
      if (dtype == MTN_DTYPE_BF16) {
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + to) =
            make_uint4(f2_to_bf2(v[0], v[1]), f2_to_bf2(v[2], v[3]), f2_to_bf2(v[4], v[5]), f2_to_bf2(v[6], v[7]));
      } else {
        float4* q = reinterpret_cast<float4*>(static_cast<float*>(out) + to);
        q[0] = make_float4(v[0], v[1], v[2], v[3]);
        q[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
      continue;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (col + j >= k) break;
      if (dtype == MTN_DTYPE_BF16)
        static_cast<__nv_bfloat16*>(out)[to + j] = __float2bfloat16_rn(v[j]);
      else
        static_cast<float*>(out)[to + j] = v[j];
    }
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

// ------------------------------------------------------------------ matvec
//
// The weights are the A operand of mma.m16n8k16 (16 output rows x 16 k), the
// x rows its B operand, so up to 8 x rows cost no more than one, and the
// kernel is bound by the weights' bytes.  A lane's 16-byte vector of a unit
// is its A fragment of four such products (k in an order of the layout's own,
// which the x fragments follow): per word and pair of neighbours one shift,
// one lop3 that masks, flips the sign bit and sets the exponent of 16 --
// bf16(17 + q / 8) -- and one subtraction of 17, exact.  A group's products
// add up in f32 and meet the group's scale once, in f32.
//
// What bounds it (device time, weights from HBM): 1 x 152064 x 3584 takes 50.7
// us, 5.6 TB/s or 0.85 of the copy rate -- the loads alone and the unpacking
// alone would each take about 48, so the two no longer hide each other
// entirely.  A matrix of 34 MB (18944 x 3584) takes 10.0 us against 5.3 for
// its bytes: start (instructions, x, the first weights) 2 us, join and drain
// 1.5.  16 rows take 78 us for the 152064 rows (16.3 for 18944) and no unit is
// full: issue slots are 55 % used, ALUs 40 %, the tensor pipe 24 %, DRAM 21 %, and
// a version without the unpacking, without x loads or without the weights' loads
// took 66, 66 and 65 us (of 76).  Warps wait for fixed latencies (1.8 of 7.3 warps
// a cycle) and for math pipes (1.3): 16 warps of 128 registers, with 36 to 68 bytes
// spilled, hide too little of chains of two dependent products.
//
// f32 rows are cut into three bf16 parts of 8 bits each, which hold all 24
// bits, and multiplied part by part into the same sums.
//
// Work.  A cluster of S CTAs takes a contiguous range of row units, each CTA
// an S-th of k, whose x rows it stages in shared memory once.  Inside the CTA
// the (row unit, 128 k) steps are laid end to end and each of the 16 warps
// streams an equal contiguous part of them through a ring of its own, a few
// steps of asynchronous copies ahead of its products: no barrier until the
// end, and no warp has more than one step more than another.  With S = 1 a
// warp stores the units it has whole; the at most two it shares with its
// neighbours, and with S > 1 every unit, are left in shared memory as partial
// sums and added at the end in warp order, over the cluster's CTAs in rank
// order, so results do not depend on timing.

constexpr int kMvWarps = 16;
constexpr int kMvThreads = kMvWarps * 32;
constexpr int kXPad = 32;              // elements: rows 64 bytes apart modulo 128, no bank conflicts
constexpr int kMinUnits = 8;    // row units of a round that the slots of a split have room for at least
constexpr int kJoinSteps = 16;
constexpr int kSmemMax = 225 * 1024;

// Row units of a step: one, or two that share their x fragments where those
// are many, or where the steps of a warp are (kSteps2): 1 x 152064 x 3584 took
// 55.7 us with one and 51.9 with two, 8 x 3584 x 18944 13.9 and 15.2.
constexpr int mv_units(int parts, int nt, bool many) { return parts * nt > 1 || many ? 2 : 1; }  // kR
constexpr int mv_depth(int r) { return r > 1 ? 2 : 5; }                                          // kD
constexpr int64_t kSteps2 = 32;
constexpr int mv_stage(int r, int groups) { return r * (1024 + 32 * groups); }         // bytes of a step
constexpr int mv_slot(int r, int nt) { return 16 * r * 8 * nt; }                       // floats of a slot

struct MvPlan {
  int cluster;     // CTAs along k
  int clusters;
  int per, extra;  // row units of a cluster; the first `extra` have one more
  int tile;        // x rows of one pass
  int units_cap;   // row units of one round
  int x_stride;    // elements between staged rows
  int units;       // row units of a step
  int x_vec;       // x rows allow vector loads
  size_t smem, ring_off, slots_off;
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with c = 0.
__device__ __forceinline__ void mma_bf16_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// Neighbours k = 2 p, 2 p + 1 of a word as bf16x2 of q / 8.
template <int p>
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x41884188, 0x6a;" : "=r"(r) : "r"(w >> (4 * p)));  // (a & b) ^ c
  asm("sub.bf16x2 %0, %0, %1;" : "+r"(r) : "r"(0x41884188u));
  return r;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// The first `bytes` of 16, zeros for the rest.
__device__ __forceinline__ void cp_async16_fill(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds4(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// f32 at offset `off` of CTA `rank`'s shared memory.
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
  float v;
  asm volatile(
      "{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}"
      : "=f"(v)
      : "r"(addr), "r"(rank));
  return v;
}

// Three bf16 parts of an f32 value, cut (not rounded) so that no part
// overflows: hi + mid + lo == x for every finite x (below the range of
// bf16's subnormals the last bits are lost).
__device__ __forceinline__ void split3(float x, uint16_t (&h)[3]) {
  if (!(fabsf(x) < INFINITY)) {  // infinity or NaN: one part
    h[0] = static_cast<uint16_t>(x != x ? 0x7fc0u : __float_as_uint(x) >> 16);
    h[1] = h[2] = 0;
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const uint32_t b = __float_as_uint(x) & 0xffff0000u;
    h[i] = static_cast<uint16_t>(b >> 16);
    x -= __uint_as_float(b);
  }
}

__device__ __forceinline__ void store_out(const W4Params& p, int64_t m, int64_t n, float v) {
  v *= 8.0f;
  if (p.x_scales != nullptr) v *= p.x_scales[m];
  if (p.out_dtype == MTN_DTYPE_BF16)
    static_cast<__nv_bfloat16*>(p.out)[m * p.out_stride + n] = __float2bfloat16_rn(v);
  else
    static_cast<float*>(p.out)[m * p.out_stride + n] = v;
}

// Eight consecutive elements of an x row as loaded, zeros beyond k: two words
// of e4m3, four of bf16, eight of f32.  `vec`: the row allows vector loads.
struct Raw8 {
  uint32_t w[8];
};

template <int kParts>
__device__ __forceinline__ void load_raw(const W4Params& p, int64_t at, int64_t k, bool vec, Raw8& r) {
  if (vec && k + 8 <= p.k) {
    if constexpr (kParts == 3) {
      const uint4* q = reinterpret_cast<const uint4*>(static_cast<const float*>(p.x) + at);
      const uint4 a = q[0], b = q[1];
      r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w, r.w[4] = b.x, r.w[5] = b.y, r.w[6] = b.z, r.w[7] = b.w;
    } else {  // e4m3; aligned bf16 rows are copied as they are
      const uint2 a = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(p.x) + at);
      r.w[0] = a.x, r.w[1] = a.y;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) r.w[i] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (k + i >= p.k) break;
    if constexpr (kParts == 3)
      r.w[i] = static_cast<const uint32_t*>(p.x)[at + i];
    else if (p.x_dtype == MTN_DTYPE_BF16)
      r.w[i / 2] |= static_cast<uint32_t>(static_cast<const uint16_t*>(p.x)[at + i]) << (16 * (i & 1));
    else
      r.w[i / 4] |= static_cast<uint32_t>(static_cast<const uint8_t*>(p.x)[at + i]) << (8 * (i & 3));
  }
}

// Two e4m3 values of a word's half as bf16x2 (exact).
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w, int half) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * half)), __NV_E4M3);
  const float2 f = __half22float2(__half2(h));
  return f2_to_bf2(f.x, f.y);
}

// A thread's part of staged rows of `len` elements: the vector of 8 at `first`
// of every `rows`-th row from `row` on (rows longer than the CTA's vectors:
// every row, and the vectors kMvThreads apart).
struct RowSplit {
  int first, row, rows;
  __device__ __forceinline__ explicit RowSplit(int len) {
    const int per = len / 8, tid = static_cast<int>(threadIdx.x);
    rows = per > 0 && per < kMvThreads ? kMvThreads / per : 1;
    row = rows > 1 ? tid / per : 0;
    first = (tid - row * per) * 8;
    if (row >= rows) first = len;  // the threads left over
  }
};

// Copies x rows m0 .. m0 + mt, k0 .. k0 + len, to shared memory as they are
// (aligned bf16 rows), zeros beyond k; asynchronous.
__device__ __forceinline__ void copy_rows(const W4Params& p, const MvPlan& plan, uint32_t xs, int64_t m0, int mt,
                                          int64_t k0, int len) {
  const uint16_t* x = static_cast<const uint16_t*>(p.x) + m0 * p.x_stride + k0;
  const RowSplit t(len);
  for (int v = t.first; v < len; v += kMvThreads * 8) {
    const int64_t left = (p.k - k0 - v) * 2;
    const uint32_t bytes = left >= 16 ? 16u : left > 0 ? static_cast<uint32_t>(left) : 0u;
    const uint16_t* src = bytes > 0 ? x + v : x;
    for (int m = t.row; m < mt; m += t.rows)
      cp_async16_fill(xs + (m * plan.x_stride + v) * 2, src + m * p.x_stride, bytes);
  }
}

// The same through registers, for every other row: f32 cut into three bf16
// parts, e4m3 exact in bf16, unaligned rows.  kBatch rows are in flight;
// then() runs once, behind the last of this thread's loads.
template <int kParts, typename F>
__device__ __forceinline__ void convert_rows(const W4Params& p, const MvPlan& plan, uint16_t* xs, int64_t m0, int mt,
                                             int64_t k0, int len, F then) {
  constexpr int kBatch = kParts == 3 ? 4 : 8;
  const int step = kMvThreads * 8;
  const RowSplit t(len);
  bool done = false;
  for (int e = t.first; e < len; e += step) {
    for (int mb = t.row; mb < mt; mb += kBatch * t.rows) {
      Raw8 v[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        if (mb + b * t.rows < mt)
          load_raw<kParts>(p, (m0 + mb + b * t.rows) * p.x_stride + k0 + e, k0 + e, plan.x_vec != 0, v[b]);
      if (e + step >= len && mb + kBatch * t.rows >= mt) {
        then();
        done = true;
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (mb + b * t.rows >= mt) continue;
        uint16_t* dst = xs + (mb + b * t.rows) * plan.x_stride + e;
        const uint32_t* w = v[b].w;
        if constexpr (kParts == 1) {
          *reinterpret_cast<uint4*>(dst) =
              p.x_dtype == MTN_DTYPE_BF16
                  ? make_uint4(w[0], w[1], w[2], w[3])
                  : make_uint4(e4m3_pair(w[0], 0), e4m3_pair(w[0], 1), e4m3_pair(w[1], 0), e4m3_pair(w[1], 1));
        } else {
          uint16_t h[8][3];
#pragma unroll
          for (int j = 0; j < 8; ++j) split3(__uint_as_float(w[j]), h[j]);
#pragma unroll
          for (int q = 0; q < 3; ++q) {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = h[2 * j][q] | static_cast<uint32_t>(h[2 * j + 1][q]) << 16;
            *reinterpret_cast<uint4*>(dst + q * plan.tile * plan.x_stride) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
      }
    }
  }
  if (!done) then();
}

// kParts: bf16 parts of an x value (1, or 3 for f32).  kNT: 8-row tiles of
// x.  kR: 16-row units of one step, sharing its x fragments.  kGroups:
// scale groups in a step of 128 k.  kD: steps loaded ahead.
template <int kParts, int kNT, int kR, int kGroups, int kD>
__global__ void __launch_bounds__(kMvThreads, 1) w4_matvec_kernel(const W4Params p, const MvPlan plan) {
  extern __shared__ __align__(128) uint8_t smem[];
  uint16_t* xs = reinterpret_cast<uint16_t*>(smem);
  float* slots = reinterpret_cast<float*>(smem + plan.slots_off);
  constexpr int kSlot = mv_slot(kR, kNT);  // [x row][output row]
  constexpr int kStage = mv_stage(kR, kGroups);
  static_assert(kD * kStage >= kSlot * 4, "a warp's ring also holds a slot");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int S = plan.cluster;
  const int rank = S > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int cl = static_cast<int>(blockIdx.x) / S;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * plan.tile;
  const int mt = static_cast<int>(min(static_cast<int64_t>(plan.tile), p.m - m0));
  const int ksteps = static_cast<int>(pad_k(p.k) / kKPad);
  const int runits = static_cast<int>(row_units(p.n));
  const int cu0 = cl * plan.per + min(cl, plan.extra), cu1 = cu0 + plan.per + (cl < plan.extra ? 1 : 0);
  const int s0 = rank * ksteps / S, L = (rank + 1) * ksteps / S - s0;

  // The lane's x fragments: row g of each tile, 8 t elements into a half
  // unit.  Rows beyond the tile read its last row: their sums are not stored.
  const uint16_t* xf[kNT];
#pragma unroll
  for (int j = 0; j < kNT; ++j) xf[j] = xs + min(8 * j + g, mt - 1) * plan.x_stride + 8 * t;
  const int plane = plan.tile * plan.x_stride;

  uint8_t* ring_ptr = smem + plan.ring_off + warp * (kD * kStage);
  const uint32_t ring = smem_u32(ring_ptr);
  const bool direct = kParts == 1 && p.x_dtype == MTN_DTYPE_BF16 && plan.x_vec != 0;
  const int64_t k0 = static_cast<int64_t>(s0) * kKPad;

  for (int u0 = cu0; u0 < cu1; u0 += plan.units_cap) {
    const int nu = min(cu1 - u0, plan.units_cap);
    const int total = nu * L;
    const int i0 = warp * total / kMvWarps;
    const int n_items = (warp + 1) * total / kMvWarps - i0;
    // load cursor and compute cursor: (unit of the round, step of the slice)
    int lu = L > 0 ? i0 / L : 0, ls = i0 - lu * L;
    int cu = lu, cs = ls;
    const uint4* wp[kR];
    const uint4* sp[kR];
    auto seek = [&]() {  // an odd last unit reads its first half twice; its rows are not stored
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        const int64_t at = static_cast<int64_t>(min((u0 + lu) * kR + r, runits - 1)) * ksteps + s0 + ls;
        wp[r] = p.packed + at * 64 + lane;
        sp[r] = reinterpret_cast<const uint4*>(p.scales) + at * (kGroups * 2) + lane;
      }
    };
    auto load = [&](uint32_t at) {
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        cp_async16(at + r * 1024 + lane * 16, wp[r]);
        cp_async16(at + r * 1024 + 512 + lane * 16, wp[r] + 32);
        wp[r] += 64;
        if (lane < 2 * kGroups) cp_async16(at + kR * 1024 + r * (kGroups * 32) + lane * 16, sp[r]);
        sp[r] += kGroups * 2;
      }
      if (++ls == L) {
        ls = 0;
        ++lu;
        seek();
      }
    };
    auto fill = [&]() {
      seek();
#pragma unroll
      for (int d = 0; d < kD; ++d) {
        if (d < n_items) load(ring + d * kStage);
        cp_async_commit();
      }
    };
    if (u0 == cu0) {
      pdl_enter();
      // x before the weights: behind them it would wait for all their bytes.  (Asking for the weights in L2
      // before the wait above did as much harm as good: with add_rms_norm before it 8 x 18944 x 3584 took
      // 13.9 us against 14.3 for both, 1 x 18944 x 3584 11.6 against 11.2.)
      if (direct) {
        copy_rows(p, plan, smem_u32(xs), m0, mt, k0, L * kKPad);
        cp_async_commit();
        fill();
      } else {
        convert_rows<kParts>(p, plan, xs, m0, mt, k0, L * kKPad, fill);
      }
      if (direct) cp_async_wait<kD>();  // the copied rows, not the weights behind them
      __syncthreads();
    } else {
      fill();
    }

    float acc[kR][kNT][4] = {};
    // The lane holds output rows g, g + 8 of x rows 2 t, 2 t + 1 of each tile.
    auto leave = [&](float* sl) {
#pragma unroll
      for (int r = 0; r < kR; ++r)
#pragma unroll
        for (int j = 0; j < kNT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sl[(8 * j + 2 * t + (e & 1)) * (16 * kR) + 16 * r + g + 8 * (e >> 1)] = acc[r][j][e];
            acc[r][j][e] = 0.0f;
          }
    };
    auto finish = [&]() {  // at a unit's end
      if (S > 1) {
        leave(slots + (cu + warp) * kSlot);
      } else if (cu * L < i0) {  // its beginning is the warp before's
        leave(slots + warp * kSlot);
      } else {
#pragma unroll
        for (int r = 0; r < kR; ++r)
#pragma unroll
          for (int j = 0; j < kNT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int m = 8 * j + 2 * t + (e & 1);
              const int64_t n = static_cast<int64_t>((u0 + cu) * kR + r) * 16 + g + 8 * (e >> 1);
              if (m < mt && n < p.n) store_out(p, m0 + m, n, acc[r][j][e]);
              acc[r][j][e] = 0.0f;
            }
      }
    };
    uint32_t at = ring;
    for (int i = 0; i < n_items; ++i) {
      cp_async_wait<kD - 1>();
      __syncwarp();  // the scales came through other lanes
      const int xo = cs * kKPad;
      float cg[kR][kNT][4];
      uint4 w[kR];
#pragma unroll
      for (int h = 0; h < 4; ++h) {  // 32 k: half h & 1 of unit h >> 1
        constexpr int kPer = 4 / kGroups;  // halves in a group
        if ((h & 1) == 0) {
#pragma unroll
          for (int r = 0; r < kR; ++r) w[r] = lds16(at + r * 1024 + (h >> 1) * 512 + lane * 16);
        }
#pragma unroll
        for (int q = 0; q < kParts; ++q) {
          uint4 xv[kNT];
#pragma unroll
          for (int j = 0; j < kNT; ++j) xv[j] = *reinterpret_cast<const uint4*>(xf[j] + q * plane + xo + 32 * h);
#pragma unroll
          for (int r = 0; r < kR; ++r) {
            const uint32_t lo = h & 1 ? w[r].y : w[r].x, hi = h & 1 ? w[r].w : w[r].z;
            const uint32_t a0 = code_pair<0>(lo), a1 = code_pair<0>(hi), a2 = code_pair<1>(lo), a3 = code_pair<1>(hi);
            const uint32_t b0 = code_pair<2>(lo), b1 = code_pair<2>(hi), b2 = code_pair<3>(lo), b3 = code_pair<3>(hi);
#pragma unroll
            for (int j = 0; j < kNT; ++j) {
              if (h % kPer == 0 && q == 0)
                mma_bf16_zero(cg[r][j], a0, a1, a2, a3, xv[j].x, xv[j].y);
              else
                mma_bf16(cg[r][j], a0, a1, a2, a3, xv[j].x, xv[j].y);
              mma_bf16(cg[r][j], b0, b1, b2, b3, xv[j].z, xv[j].w);
            }
          }
        }
        if ((h + 1) % kPer == 0) {  // end of a group
#pragma unroll
          for (int r = 0; r < kR; ++r) {
            const uint32_t s2 = lds4(at + kR * 1024 + (r * kGroups + h / kPer) * 32 + g * 4);
            const float slo = __uint_as_float(s2 << 16), shi = __uint_as_float(s2 & 0xffff0000u);
#pragma unroll
            for (int j = 0; j < kNT; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[r][j][e] = fmaf(cg[r][j][e], e < 2 ? slo : shi, acc[r][j][e]);
          }
        }
      }
      // every lane has read the stage: refill it
      __syncwarp();
      if (i + kD < n_items) load(at);
      cp_async_commit();
      at = at + kStage == ring + kD * kStage ? ring : at + kStage;
      if (++cs == L) {
        finish();
        cs = 0;
        ++cu;
      }
    }
    if (n_items > 0 && cs != 0) {  // the unit goes on in the next warp
      if (S > 1)
        leave(slots + (cu + warp) * kSlot);
      else if (cu * L < i0)
        leave(slots + warp * kSlot);
      else
        leave(reinterpret_cast<float*>(ring_ptr));  // the ring is empty by now
    }

    constexpr int kUnitRows = 16 * kR;
    if (S > 1) {
      // Join the warps' slots of each unit into the space of the rings, then
      // those of the cluster's CTAs.
      float* part = reinterpret_cast<float*>(smem + plan.ring_off);
      __syncthreads();
      const int per_unit = mt * kUnitRows;
      for (int i = tid; i < nu * per_unit; i += kMvThreads) {
        const int q = i / per_unit, off = i - q * per_unit;
        float v = 0.0f;
        if (L > 0) {  // first to last warp with a step of unit q
          const int wa = ((q * L + 1) * kMvWarps - 1) / total, wb = ((q + 1) * L * kMvWarps - 1) / total;
          for (int w = wa; w <= wb; ++w)
            if (w * total / kMvWarps != (w + 1) * total / kMvWarps) v += slots[(q + w) * kSlot + off];
        }
        part[q * kSlot + off] = v;
      }
      cluster_sync();
      const uint32_t part_at = smem_u32(part);
      for (int i = rank * kMvThreads + tid; i < nu * per_unit; i += S * kMvThreads) {
        const int q = i / per_unit, off = i - q * per_unit;
        float v[8];
#pragma unroll
        for (int rk = 0; rk < 8; ++rk)
          if (rk < S) v[rk] = ld_cluster(part_at + (q * kSlot + off) * 4, rk);
        float sum = 0.0f;
#pragma unroll
        for (int rk = 0; rk < 8; ++rk)
          if (rk < S) sum += v[rk];
        const int64_t n = static_cast<int64_t>(u0 + q) * kUnitRows + off % kUnitRows;
        if (n < p.n) store_out(p, m0 + off / kUnitRows, n, sum);
      }
      cluster_sync();
    } else {
      // Join the units that begin in a warp and go on in the next ones.
      __shared__ int tail_of[kMvWarps];
      const int i1 = i0 + n_items, tail = i1 / L;
      if (lane == 0) tail_of[warp] = n_items > 0 && i1 != tail * L && tail * L >= i0 ? tail : -1;
      __syncthreads();
      const int per_unit = mt * kUnitRows;
      for (int e = tid; e < (kMvWarps - 1) * per_unit; e += kMvThreads) {
        const int w = e / per_unit, i = e - w * per_unit, q = tail_of[w], m = i / kUnitRows;
        if (q < 0) continue;
        float v = reinterpret_cast<const float*>(smem + plan.ring_off + w * (kD * kStage))[i];
        for (int z = w + 1; z < kMvWarps && z * total / kMvWarps < (q + 1) * L; ++z)
          if (z * total / kMvWarps != (z + 1) * total / kMvWarps) v += slots[z * kSlot + i];
        const int64_t n = static_cast<int64_t>(u0 + q) * kUnitRows + i % kUnitRows;
        if (n < p.n) store_out(p, m0 + m, n, v);
      }
      if (u0 + nu < cu1) __syncthreads();
    }
  }
}

using MvKernel = void (*)(const W4Params, const MvPlan);

template <int kParts, int kNT, int kR>
MvKernel mv_kernel(int group) {
  constexpr int kD = mv_depth(kR);
  switch (group) {
    case 32: return w4_matvec_kernel<kParts, kNT, kR, 4, kD>;
    case 64: return w4_matvec_kernel<kParts, kNT, kR, 2, kD>;
    default: return w4_matvec_kernel<kParts, kNT, kR, 1, kD>;
  }
}

MvKernel mv_kernel(int parts, int nt, int r, int group) {
  if (parts == 3) return nt > 1 ? mv_kernel<3, 2, 2>(group) : mv_kernel<3, 1, 2>(group);
  if (nt > 1) return mv_kernel<1, 2, 2>(group);
  return r > 1 ? mv_kernel<1, 1, 2>(group) : mv_kernel<1, 1, 1>(group);
}

// Clusters of `size` CTAs that the device holds at once (one CTA per SM).
int max_clusters(int size) {
  constexpr int kDevices = 64;
  static std::atomic<int> cached[kDevices][4];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) return std::max(1, 128 / size);
  const int slot = size == 1 ? 0 : size == 2 ? 1 : size == 4 ? 2 : 3;
  if (cached[dev][slot] == 0) {
    int n = sm_count();
    if (size > 1) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(static_cast<unsigned>(size));
      cfg.blockDim = dim3(kMvThreads);
      cfg.dynamicSmemBytes = kSmemMax;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = static_cast<unsigned>(size);
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      const MvKernel kern = mv_kernel(1, 1, 1, 128);
      if (allow_smem(reinterpret_cast<const void*>(kern), kSmemMax) != cudaSuccess ||
          cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
        cudaGetLastError();
        n = std::max(1, 128 / size);
      }
    }
    cached[dev][slot] = n;
  }
  return cached[dev][slot];
}

// The x rows of one pass and the split of k: as many rows (up to 16) as the
// slices of a cluster of at most 8 CTAs can hold in shared memory, then the
// split whose CTAs have the fewest steps, a join of slots counted as
// kJoinSteps of them.
MvPlan mv_plan(int64_t m, int64_t n, int64_t k, int group, int parts) {
  const int ksteps = static_cast<int>(pad_k(k) / kKPad);
  MvPlan pl{};
  pl.tile = static_cast<int>(std::min<int64_t>(m, 16));
  int nt, r;
  size_t ring, slot;
  const bool many = row_units(n) * ksteps >= kSteps2 * kMvWarps * sm_count();
  auto sizes = [&]() {
    nt = pl.tile > 8 ? 2 : 1;
    r = mv_units(parts, nt, many);
    ring = static_cast<size_t>(kMvWarps) * mv_depth(r) * mv_stage(r, kKPad / group);
    slot = static_cast<size_t>(mv_slot(r, nt)) * 4;
  };
  auto x_bytes = [&](int s) {
    const size_t b = static_cast<size_t>(parts) * pl.tile * ((ksteps + s - 1) / s * kKPad + kXPad) * 2;
    return (b + 127) / 128 * 128;
  };
  // slots that fit beside the rest: one a warp, and with a split one more for every row unit of a round
  auto fits = [&](int s) { return x_bytes(s) + ring + (kMvWarps + (s > 1 ? kMinUnits : 0)) * slot <= kSmemMax; };
  sizes();
  while (pl.tile > 1 && !fits(8)) {
    pl.tile = (pl.tile + 1) / 2;
    sizes();
  }
  const int64_t units = (row_units(n) + r - 1) / r;
  int64_t best = INT64_MAX;
  for (int s = 1; s <= 8; s *= 2) {
    if (!fits(s)) continue;
    const int64_t c = std::min<int64_t>(units, max_clusters(s));
    const int64_t per = (units + c - 1) / c;
    // a round's units: slots for them and for the warps, and the joined units in the rings
    const int64_t room =
        std::min(static_cast<int64_t>((kSmemMax - x_bytes(s) - ring) / slot) - kMvWarps, static_cast<int64_t>(ring / slot));
    const int64_t cap = s == 1 ? 4096 : room;  // 4096: steps x warps stay within 32 bits
    const int64_t rounds = (per + cap - 1) / cap;
    const int64_t cost = per * ((ksteps + s - 1) / s) + (s == 1 ? 0 : rounds * kJoinSteps);
    if (cost < best) {
      best = cost;
      pl.cluster = s;
      pl.clusters = static_cast<int>(c);
      pl.per = static_cast<int>(units / c);
      pl.extra = static_cast<int>(units % c);
      pl.units_cap = static_cast<int>((per + rounds - 1) / rounds);
    }
  }
  pl.units = r;
  pl.x_stride = (ksteps + pl.cluster - 1) / pl.cluster * kKPad + kXPad;
  pl.ring_off = x_bytes(pl.cluster);
  pl.slots_off = pl.ring_off + ring;
  pl.smem = pl.slots_off + (kMvWarps + (pl.cluster > 1 ? pl.units_cap : 0)) * slot;
  return pl;
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
  MTN_CHECK_ARG(mtn::elem_aligned(weight, dtype), "mtn_w4_quantize: weight is not aligned to its elements");
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
  MTN_CHECK_ARG(mtn::elem_aligned(code_scales, MTN_DTYPE_BF16), "mtn_w4_pack: code_scales is not aligned to its elements");
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
  MTN_CHECK_ARG(mtn::elem_aligned(out, dtype), "mtn_w4_dequantize: out is not aligned to its elements");
  const int64_t ksteps = mtn::pad_k(k) / mtn::kKPad;
  const int64_t blocks = mtn::row_units(n) * ((ksteps + mtn::kDequantSteps - 1) / mtn::kDequantSteps);
  const int elem = dtype == MTN_DTYPE_BF16 ? 2 : 4;
  const bool vec = mtn::aligned16(out) && (n == 1 || stride * elem % 16 == 0);
  mtn::w4_dequantize_kernel<<<static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint32_t*>(packed), static_cast<const uint32_t*>(scales), n, k, group, out, dtype, stride, vec);
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
  MTN_CHECK_ARG(mtn::elem_aligned(x, x_dtype) && mtn::elem_aligned(out, out_dtype) &&
                    mtn::elem_aligned(x_scales, MTN_DTYPE_F32),
                "mtn_w4_matvec: a pointer is not aligned to its elements");
  MTN_CHECK_ARG(out != x, "mtn_w4_matvec: out overlaps x");
  mtn::W4Params p{x, x_dtype, x_stride, x_scales, n_rows, static_cast<const uint4*>(packed),
                  static_cast<const uint32_t*>(scales), n, k, group, out, out_dtype, out_stride};
  const int parts = x_dtype == MTN_DTYPE_F32 ? 3 : 1;
  mtn::MvPlan plan = mtn::mv_plan(n_rows, n, k, group, parts);
  const int elem = x_dtype == MTN_DTYPE_F32 ? 4 : x_dtype == MTN_DTYPE_BF16 ? 2 : 1;
  const int64_t vec = elem == 1 ? 8 : 16;  // bytes of one vector load
  plan.x_vec = reinterpret_cast<uintptr_t>(x) % vec == 0 && (n_rows == 1 || x_stride * elem % vec == 0);
  const mtn::MvKernel kern = mtn::mv_kernel(parts, plan.tile > 8 ? 2 : 1, plan.units, group);
  MTN_CUDA_TRY(mtn::allow_smem(reinterpret_cast<const void*>(kern), mtn::kSmemMax), "mtn_w4_matvec");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(plan.clusters * plan.cluster),
                     static_cast<unsigned>((n_rows + plan.tile - 1) / plan.tile));
  cfg.blockDim = dim3(mtn::kMvThreads);
  cfg.dynamicSmemBytes = plan.smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(plan.cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  MTN_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p, plan), "w4_matvec_kernel");
  return mtn::check_launch("w4_matvec_kernel");
}

}  // extern "C"
