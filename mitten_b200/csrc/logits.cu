// What a request asks of its logits before a token is picked (sample_token,
// inference-engine/src/scheduler.rs:186-223, takes them as they are): for
// every row, token v with c_all occurrences in the row's history and c_gen
// in its generated part,
//   x = c_all > 0 ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - frequency * c_gen
//   x = x - (c_gen > 0 ? presence : 0)
//   x = x + bias[v]                    a token listed twice: its last entry
//   x = mask bit v set ? x : -inf
// in f32, every operation rounded by itself and in this order, so the values
// are those of the formula evaluated step by step.  Optionally the greedy
// token of the processed row: its first strict maximum (NaN never wins, a
// row of nothing but -inf gives 0, as scheduler.rs:187-199).
//
// One CTA per (row, chunk of the vocabulary).  It counts the row's history
// tokens that fall into its chunk in shared memory (integer atomics, so the
// counts do not depend on their order), then passes over its logits once.
// The chunks of a row join their maxima as 64-bit keys (value, then lowest
// index) with an atomic maximum; the last chunk to arrive writes the token
// and leaves the workspace zeroed.
#include "common.cuh"

namespace mtn {
namespace {

constexpr int kLogitsThreads = 256;
constexpr int kLogitsChunk = 8192;
constexpr uint32_t kSeen = 0x80000000u;  // in the history at all; the low bits count the generated part

struct LogitsParams {
  const void* logits;
  int64_t row_stride;
  int64_t vocab;
  mtn_logits_rules r;
  float* out;
  int64_t out_stride;
  int32_t* tokens;
  unsigned long long* keys;  // [rows] maxima, then [rows] arrival counters
  int64_t n_rows;
  int chunks;
  int* err;
};

// Entries [beg, end) of row r of a list: a malformed index pointer gives an
// empty row and a device error.
__device__ __forceinline__ void row_range(const int32_t* indptr, int64_t r, int64_t n_entries, int64_t& beg,
                                          int64_t& end, int* err) {
  beg = indptr[r];
  end = indptr[r + 1];
  if (beg < 0 || end < beg || end > n_entries) {
    if (threadIdx.x == 0) record_error(err, kDevErrBadLogitRule, static_cast<int>(r));
    beg = end = 0;
  }
}

// Order-preserving key of a processed logit: larger values first, then the
// lower index.  0 for what never wins (-inf, NaN).  x + 0 turns -0 into +0.
__device__ __forceinline__ unsigned long long arg_key(float x, int64_t v) {
  if (!(x > -INFINITY)) return 0ull;
  const uint32_t b = __float_as_uint(__fadd_rn(x, 0.0f));
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return static_cast<unsigned long long>(o) << 32 | (0xffffffffu - static_cast<uint32_t>(v));
}

template <typename T>
__global__ void __launch_bounds__(kLogitsThreads) process_logits_kernel(const LogitsParams p) {
  extern __shared__ uint32_t smem[];
  const int64_t row = blockIdx.x / p.chunks;
  const int chunk = static_cast<int>(blockIdx.x - row * p.chunks);
  const int64_t v0 = static_cast<int64_t>(chunk) * kLogitsChunk;
  const int nv = static_cast<int>(min(static_cast<int64_t>(kLogitsChunk), p.vocab - v0));
  const int tid = threadIdx.x;
  uint32_t* count = p.r.hist_indptr != nullptr ? smem : nullptr;
  uint32_t* bias = p.r.bias_indptr != nullptr ? smem + (count != nullptr ? kLogitsChunk : 0) : nullptr;
  for (int i = tid; i < nv; i += kLogitsThreads) {
    if (count != nullptr) count[i] = 0;
    if (bias != nullptr) bias[i] = 0;
  }
  __syncthreads();
  if (count != nullptr) {
    int64_t beg, end;
    row_range(p.r.hist_indptr, row, p.r.n_hist, beg, end, p.err);
    const int64_t gen = beg + (p.r.prompt_lens != nullptr ? max(p.r.prompt_lens[row], 0) : 0);
    for (int64_t i = beg + tid; i < end; i += kLogitsThreads) {
      const int64_t t = p.r.hist_tokens[i];
      if (t < 0 || t >= p.vocab) {
        record_error(p.err, kDevErrBadLogitRule, static_cast<int>(row));
        continue;
      }
      const int64_t k = t - v0;
      if (k < 0 || k >= nv) continue;
      atomicOr(&count[k], kSeen);
      if (i >= gen) atomicAdd(&count[k], 1u);
    }
  }
  int64_t bias_beg = 0;
  if (bias != nullptr) {
    int64_t end;
    row_range(p.r.bias_indptr, row, p.r.n_bias, bias_beg, end, p.err);
    for (int64_t i = bias_beg + tid; i < end; i += kLogitsThreads) {
      const int64_t t = p.r.bias_tokens[i];
      if (t < 0 || t >= p.vocab) {
        record_error(p.err, kDevErrBadLogitRule, static_cast<int>(row));
        continue;
      }
      const int64_t k = t - v0;
      if (k >= 0 && k < nv) atomicMax(&bias[k], static_cast<uint32_t>(i - bias_beg + 1));
    }
  }
  const float rep = p.r.repetition != nullptr ? p.r.repetition[row] : 1.0f;
  const float freq = p.r.frequency != nullptr ? p.r.frequency[row] : 0.0f;
  const float pres = p.r.presence != nullptr ? p.r.presence[row] : 0.0f;
  const uint32_t* mask = nullptr;
  if (p.r.mask != nullptr) {
    const int mr = p.r.mask_rows != nullptr ? p.r.mask_rows[row] : static_cast<int>(row);
    if (mr >= 0 && mr < p.r.n_masks)
      mask = p.r.mask + static_cast<int64_t>(mr) * p.r.mask_stride;
    else if (mr != -1 && tid == 0)
      record_error(p.err, kDevErrBadLogitRule, static_cast<int>(row));
  }
  __syncthreads();
  unsigned long long best = 0;
  for (int i = tid; i < nv; i += kLogitsThreads) {
    const int64_t v = v0 + i;
    float x;
    if constexpr (sizeof(T) == 2)
      x = __bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[row * p.row_stride + v]);
    else
      x = static_cast<const float*>(p.logits)[row * p.row_stride + v];
    if (count != nullptr && count[i] != 0) {
      const uint32_t c = count[i] & ~kSeen;
      x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      x = __fsub_rn(x, __fmul_rn(freq, static_cast<float>(c)));
      if (c != 0) x = __fsub_rn(x, pres);
    }
    if (bias != nullptr && bias[i] != 0) x = __fadd_rn(x, p.r.bias_values[bias_beg + bias[i] - 1]);
    if (mask != nullptr && !(mask[v >> 5] >> (v & 31) & 1u)) x = -INFINITY;
    p.out[row * p.out_stride + v] = x;
    best = max(best, arg_key(x, v));
  }
  if (p.tokens == nullptr) return;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  __shared__ unsigned long long wbest[kLogitsThreads / 32];
  if ((tid & 31) == 0) wbest[tid >> 5] = best;
  __syncthreads();
  if (tid != 0) return;
  for (int w = 1; w < kLogitsThreads / 32; ++w) best = max(best, wbest[w]);
  atomicMax(&p.keys[row], best);
  __threadfence();
  if (atomicAdd(&p.keys[p.n_rows + row], 1ull) != static_cast<unsigned long long>(p.chunks - 1)) return;
  __threadfence();
  best = atomicExch(&p.keys[row], 0ull);
  p.keys[p.n_rows + row] = 0ull;
  p.tokens[row] = best == 0 ? 0 : static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(best));
}

}  // namespace
}  // namespace mtn

extern "C" {

size_t mtn_process_logits_workspace_bytes(int64_t n_rows) {
  return n_rows <= 0 ? 0 : static_cast<size_t>(n_rows) * 16;
}

int mtn_process_logits(const void* logits, int32_t dtype, int64_t row_stride, int64_t n_rows, int64_t vocab,
                       const mtn_logits_rules* rules, float* out, int64_t out_stride, int32_t* tokens, void* workspace,
                       size_t workspace_bytes, void* stream) {
  MTN_CHECK_ARG(n_rows >= 0 && n_rows <= INT32_MAX && vocab > 0 && vocab <= INT32_MAX, "mtn_process_logits: bad sizes");
  MTN_CHECK_ARG(dtype == MTN_DTYPE_BF16 || dtype == MTN_DTYPE_F32, "mtn_process_logits: bad dtype");
  if (n_rows == 0) return MTN_OK;
  MTN_CHECK_ARG(logits && rules && out, "mtn_process_logits: null pointer");
  MTN_CHECK_ARG(row_stride >= vocab && out_stride >= vocab, "mtn_process_logits: row strides shorter than a row");
  MTN_CHECK_ARG(static_cast<const void*>(out) != logits || (dtype == MTN_DTYPE_F32 && row_stride == out_stride),
                "mtn_process_logits: in place needs f32 logits and equal strides");
  const mtn_logits_rules& r = *rules;
  MTN_CHECK_ARG(r.n_hist >= 0 && r.n_hist <= INT32_MAX && r.n_bias >= 0 && r.n_bias <= INT32_MAX,
                "mtn_process_logits: bad list sizes");
  MTN_CHECK_ARG(r.hist_indptr == nullptr || r.hist_tokens != nullptr || r.n_hist == 0,
                "mtn_process_logits: hist_indptr without hist_tokens");
  MTN_CHECK_ARG(r.hist_indptr != nullptr || (r.prompt_lens == nullptr && r.repetition == nullptr &&
                                             r.presence == nullptr && r.frequency == nullptr),
                "mtn_process_logits: penalties without a history");
  MTN_CHECK_ARG(r.bias_indptr == nullptr || (r.bias_tokens != nullptr && r.bias_values != nullptr) || r.n_bias == 0,
                "mtn_process_logits: bias_indptr without bias_tokens and bias_values");
  MTN_CHECK_ARG(r.mask == nullptr || (r.n_masks >= 0 && r.mask_stride >= (vocab + 31) / 32),
                "mtn_process_logits: mask rows shorter than the vocabulary");
  MTN_CHECK_ARG(r.mask == nullptr || r.mask_rows != nullptr || r.n_masks >= n_rows,
                "mtn_process_logits: fewer mask rows than rows, and no mask_rows");
  MTN_CHECK_ARG(r.mask != nullptr || r.mask_rows == nullptr, "mtn_process_logits: mask_rows without a mask");
  const size_t need = mtn_process_logits_workspace_bytes(n_rows);
  MTN_CHECK_ARG(tokens == nullptr || (workspace != nullptr && workspace_bytes >= need &&
                                      (reinterpret_cast<uintptr_t>(workspace) & 7) == 0),
                "mtn_process_logits: tokens need an 8-byte aligned workspace of %zu bytes", need);
  const int64_t chunks = (vocab + mtn::kLogitsChunk - 1) / mtn::kLogitsChunk;
  MTN_CHECK_ARG(chunks * n_rows <= INT32_MAX, "mtn_process_logits: batch too large");
  mtn::LogitsParams p{logits, row_stride, vocab, r, out, out_stride, tokens,
                      static_cast<unsigned long long*>(workspace), n_rows, static_cast<int>(chunks),
                      mtn::device_error_ptr()};
  size_t smem = 0;
  if (r.hist_indptr != nullptr) smem += mtn::kLogitsChunk * 4;
  if (r.bias_indptr != nullptr) smem += mtn::kLogitsChunk * 4;
  auto kern = dtype == MTN_DTYPE_BF16 ? mtn::process_logits_kernel<__nv_bfloat16> : mtn::process_logits_kernel<float>;
  MTN_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, mtn::kLogitsChunk * 8),
               "mtn_process_logits");
  kern<<<static_cast<unsigned>(chunks * n_rows), mtn::kLogitsThreads, smem, static_cast<cudaStream_t>(stream)>>>(p);
  return mtn::check_launch("process_logits_kernel");
}

}  // extern "C"
