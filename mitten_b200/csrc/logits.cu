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
// counts do not depend on their order) and marks the touched ones in a
// bitmap, then passes over its logits once, 16 bytes a load and four loads in
// flight, the first four already before the counting; only touched elements
// look their count up.  The chunks of a row join their maxima as 64-bit keys
// (value, then lowest index) with an atomic maximum; the last chunk to arrive
// writes the token and leaves the workspace zeroed.
#include "common.cuh"

namespace mtn {
namespace {

constexpr int kLogitsThreads = 256;
// Elements of a chunk: large ones re-read a row's history less often, small
// ones spread few rows over the SMs.
constexpr int kChunkLarge = 8192, kChunkSmall = 2048;
constexpr int kBatchVecs = 4;            // 16-byte loads of a thread in flight
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
  int chunks, chunk;
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

// Calls f(position, token) for entries [beg, end) of an int32 list, 16 bytes
// a load where the list's address allows.
template <typename F>
__device__ __forceinline__ void for_tokens(const int32_t* list, int64_t beg, int64_t end, F f) {
  const int tid = threadIdx.x;
  const int64_t head = min(end, beg + static_cast<int64_t>((0u - (reinterpret_cast<uintptr_t>(list + beg) >> 2)) & 3u));
  if (beg + tid < head) f(beg + tid, list[beg + tid]);
  const int4* vec = reinterpret_cast<const int4*>(list + head);
  const int n = static_cast<int>((end - head) >> 2);
  for (int i = tid; i < n; i += 2 * kLogitsThreads) {
    const bool two = i + kLogitsThreads < n;
    const int4 a = vec[i], b = two ? vec[i + kLogitsThreads] : a;
    const int64_t at = head + 4 * static_cast<int64_t>(i);
    f(at, a.x), f(at + 1, a.y), f(at + 2, a.z), f(at + 3, a.w);
    if (two) {
      const int64_t bt = at + 4 * kLogitsThreads;
      f(bt, b.x), f(bt + 1, b.y), f(bt + 2, b.z), f(bt + 3, b.w);
    }
  }
  const int64_t rest = head + 4 * static_cast<int64_t>(n) + tid;
  if (rest < end) f(rest, list[rest]);
}

// Bits i .. i + 31 of a bit array of n words (zeros behind its end are not needed).
__device__ __forceinline__ uint32_t bits_at(const uint32_t* words, int64_t n, int64_t i) {
  const int64_t w = i >> 5;
  return __funnelshift_r(words[w], words[min(w + 1, n - 1)], static_cast<uint32_t>(i) & 31u);
}

template <typename T>
struct Vec {  // 16 bytes of logits
  static constexpr int kN = 16 / sizeof(T);
  uint4 w;
  __device__ __forceinline__ float get(int i) const {
    const uint32_t u = (&w.x)[sizeof(T) == 2 ? i >> 1 : i];
    if constexpr (sizeof(T) == 2) return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
    return __uint_as_float(u);
  }
};

template <typename T>
__device__ __forceinline__ float ld_logit(const T* p) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(*p);
  else return *p;
}

template <typename T>
__global__ void __launch_bounds__(kLogitsThreads) process_logits_kernel(const LogitsParams p) {
  extern __shared__ __align__(16) uint32_t smem[];
  constexpr int kN = Vec<T>::kN;
  const int row = static_cast<int>(blockIdx.x) / p.chunks;
  const int chunk = static_cast<int>(blockIdx.x) - row * p.chunks;
  const int tid = threadIdx.x;
  const T* in = static_cast<const T*>(p.logits) + row * p.row_stride;
  float* out = p.out + row * p.out_stride;
  // Chunks begin where a 16-byte load may: `head` elements into the row.
  const int head = static_cast<int>((0u - (reinterpret_cast<uintptr_t>(in) / sizeof(T))) & (kN - 1u));
  const bool vec = ((reinterpret_cast<uintptr_t>(out + head)) & 15u) == 0;
  const int64_t v0 = chunk == 0 ? 0 : static_cast<int64_t>(chunk) * p.chunk + head;
  const int64_t v1 = chunk == p.chunks - 1 ? p.vocab : min(p.vocab, static_cast<int64_t>(chunk + 1) * p.chunk + head);
  const int nv = static_cast<int>(max(v1 - v0, static_cast<int64_t>(0)));
  // vectors: elements body .. body + kN * nvec of the row; the rest one by one
  const int64_t body = chunk == 0 ? min(static_cast<int64_t>(head), v1) : v0;
  const int nvec = vec && v1 > body ? static_cast<int>((v1 - body) / kN) : 0;
  const uint4* vin = reinterpret_cast<const uint4*>(in + body);

  Vec<T> x[kBatchVecs];
#pragma unroll
  for (int b = 0; b < kBatchVecs; ++b)
    if (tid + b * kLogitsThreads < nvec) x[b].w = vin[tid + b * kLogitsThreads];

  // shared memory: touched bits of the chunk's words, then counts, then bias entries
  const int64_t w0 = v0 >> 5;
  const int nwords = p.chunk / 32 + 2;
  const bool hist = p.r.hist_indptr != nullptr, biased = p.r.bias_indptr != nullptr, rules = hist || biased;
  uint32_t* touched = smem;
  uint32_t* count = smem + (nwords + 3) / 4 * 4;
  uint32_t* bias = count + (hist ? p.chunk + 8 : 0);
  int64_t bias_beg = 0;
  if (rules) {
    int64_t hbeg = 0, hend = 0, bend = 0;
    if (hist) row_range(p.r.hist_indptr, row, p.r.n_hist, hbeg, hend, p.err);
    if (biased) row_range(p.r.bias_indptr, row, p.r.n_bias, bias_beg, bend, p.err);
    const int words = static_cast<int>(bias - touched) + (biased ? p.chunk + 8 : 0);
    for (int i = tid; i < words / 4; i += kLogitsThreads) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    auto slot = [&](int32_t t, int& k) {  // the token's place in the chunk
      if (t < 0 || t >= p.vocab) {
        record_error(p.err, kDevErrBadLogitRule, row);
        return false;
      }
      k = static_cast<int>(t - v0);
      if (t < v0 || t >= v1) return false;
      const int64_t w = (t >> 5) - w0;
      const uint32_t bit = 1u << (t & 31);
      if (!(touched[w] & bit)) atomicOr(&touched[w], bit);
      return true;
    };
    if (hist) {
      const int64_t gen = hbeg + (p.r.prompt_lens != nullptr ? max(p.r.prompt_lens[row], 0) : 0);
      for_tokens(p.r.hist_tokens, hbeg, hend, [&](int64_t i, int32_t t) {
        int k;
        if (!slot(t, k)) return;
        if (i >= gen)
          atomicAdd(&count[k], 1u);
        if (!(count[k] & kSeen)) atomicOr(&count[k], kSeen);
      });
    }
    if (biased)
      for_tokens(p.r.bias_tokens, bias_beg, bend, [&](int64_t i, int32_t t) {
        int k;
        if (slot(t, k)) atomicMax(&bias[k], static_cast<uint32_t>(i - bias_beg + 1));
      });
  }
  const float rep = p.r.repetition != nullptr ? p.r.repetition[row] : 1.0f;
  const float freq = p.r.frequency != nullptr ? p.r.frequency[row] : 0.0f;
  const float pres = p.r.presence != nullptr ? p.r.presence[row] : 0.0f;
  const uint32_t* mask = nullptr;
  const int64_t mask_words = (p.vocab + 31) >> 5;
  if (p.r.mask != nullptr) {
    const int mr = p.r.mask_rows != nullptr ? p.r.mask_rows[row] : row;
    if (mr >= 0 && mr < p.r.n_masks)
      mask = p.r.mask + mr * p.r.mask_stride;
    else if (mr != -1 && tid == 0)
      record_error(p.err, kDevErrBadLogitRule, row);
  }
  if (rules) __syncthreads();

  auto ruled = [&](float y, int64_t v) {  // a touched element's penalties and bias
    const int k = static_cast<int>(v - v0);
    if (hist && count[k] != 0) {
      const uint32_t c = count[k] & ~kSeen;
      y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
      y = __fsub_rn(y, __fmul_rn(freq, static_cast<float>(c)));
      if (c != 0) y = __fsub_rn(y, pres);
    }
    if (biased && bias[k] != 0) y = __fadd_rn(y, p.r.bias_values[bias_beg + bias[k] - 1]);
    return y;
  };
  // A thread sees rising indices, so a strict comparison keeps the first maximum.
  float best = -INFINITY;
  int64_t best_v = 0;
  auto scalar = [&](int64_t v) {
    float y = ld_logit(in + v);
    if (rules && touched[(v >> 5) - w0] >> (v & 31) & 1u) y = ruled(y, v);
    if (mask != nullptr && !(mask[v >> 5] >> (v & 31) & 1u)) y = -INFINITY;
    out[v] = y;
    if (y > best) best = y, best_v = v;
  };
  if (!vec) {
    for (int i = tid; i < nv; i += kLogitsThreads) scalar(v0 + i);
  } else {
    if (v0 + tid < body) scalar(v0 + tid);
    for (int base = tid; base < nvec; base += kBatchVecs * kLogitsThreads) {
      uint32_t allow[kBatchVecs];
#pragma unroll
      for (int b = 0; b < kBatchVecs; ++b) {
        const int i = base + b * kLogitsThreads;
        allow[b] = ~0u;
        if (mask != nullptr && i < nvec) allow[b] = bits_at(mask, mask_words, body + static_cast<int64_t>(i) * kN);
      }
#pragma unroll
      for (int b = 0; b < kBatchVecs; ++b) {
        const int i = base + b * kLogitsThreads;
        if (i >= nvec) break;
        const int64_t v = body + static_cast<int64_t>(i) * kN;
        float y[kN];
#pragma unroll
        for (int e = 0; e < kN; ++e) y[e] = x[b].get(e);
        if (rules) {
          const uint32_t hit = bits_at(touched, nwords, v - (w0 << 5)) & ((1u << kN) - 1u);
          if (hit != 0) {
#pragma unroll
            for (int e = 0; e < kN; ++e)
              if (hit >> e & 1u) y[e] = ruled(y[e], v + e);
          }
        }
#pragma unroll
        for (int e = 0; e < kN; ++e)
          if (!(allow[b] >> e & 1u)) y[e] = -INFINITY;
        float top = y[0];
#pragma unroll
        for (int e = 1; e < kN; ++e) top = fmaxf(top, y[e]);
        if (top > best) {
          best = top;
#pragma unroll
          for (int e = kN - 1; e >= 0; --e)
            if (y[e] == top) best_v = v + e;
        }
#pragma unroll
        for (int e = 0; e < kN; e += 4)
          *reinterpret_cast<float4*>(out + v + e) = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
        const int next = i + kBatchVecs * kLogitsThreads;
        if (next < nvec) x[b].w = vin[next];
      }
    }
    const int64_t rest = body + static_cast<int64_t>(nvec) * kN + tid;
    if (rest < v1) scalar(rest);
  }
  if (p.tokens == nullptr) return;
  unsigned long long key = arg_key(best, best_v);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
  __shared__ unsigned long long wkey[kLogitsThreads / 32];
  if ((tid & 31) == 0) wkey[tid >> 5] = key;
  __syncthreads();
  if (tid != 0) return;
#pragma unroll
  for (int w = 1; w < kLogitsThreads / 32; ++w) key = max(key, wkey[w]);
  atomicMax(&p.keys[row], key);
  __threadfence();
  if (atomicAdd(&p.keys[p.n_rows + row], 1ull) != static_cast<unsigned long long>(p.chunks - 1)) return;
  __threadfence();
  key = atomicExch(&p.keys[row], 0ull);
  p.keys[p.n_rows + row] = 0ull;
  p.tokens[row] = key == 0 ? 0 : static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(key));
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
  // Few rows: small chunks, so that every SM has some.
  int chunk = mtn::kChunkLarge;
  if (n_rows * ((vocab + chunk - 1) / chunk) < 2 * mtn::sm_count()) chunk = mtn::kChunkSmall;
  const int64_t chunks = (vocab + chunk - 1) / chunk;
  MTN_CHECK_ARG(chunks * n_rows <= INT32_MAX, "mtn_process_logits: batch too large");
  mtn::LogitsParams p{logits, row_stride, vocab, r, out, out_stride, tokens,
                      static_cast<unsigned long long*>(workspace), n_rows, static_cast<int>(chunks), chunk,
                      mtn::device_error_ptr()};
  const size_t table = static_cast<size_t>(chunk + 8) * 4;
  size_t smem = 0;
  if (r.hist_indptr != nullptr || r.bias_indptr != nullptr) smem += (static_cast<size_t>(chunk) / 32 + 2 + 3) / 4 * 16;
  if (r.hist_indptr != nullptr) smem += table;
  if (r.bias_indptr != nullptr) smem += table;
  auto kern = dtype == MTN_DTYPE_BF16 ? mtn::process_logits_kernel<__nv_bfloat16> : mtn::process_logits_kernel<float>;
  if (smem > 48 * 1024)
    MTN_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)),
                 "mtn_process_logits");
  kern<<<static_cast<unsigned>(chunks * n_rows), mtn::kLogitsThreads, smem, static_cast<cudaStream_t>(stream)>>>(p);
  return mtn::check_launch("process_logits_kernel");
}

}  // extern "C"
