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
// Two launches.  sort_rules_kernel, one CTA per row, sorts the row's history
// and biases by the chunk of the vocabulary they fall into (a counting sort;
// the order inside a chunk does not matter).  process_logits_kernel, one CTA
// per (row, chunk), passes over the logits with the mask alone, 16 bytes a
// load; that pass is bound by memory and needs nothing of the first kernel,
// which therefore runs beside it (programmatic dependent launch).  Then it
// waits, counts its entries in a table in shared memory (integer atomics, so
// nothing depends on their order), and the first entry to claim a token
// applies its penalties to the original logit; the biases go the same way over
// the same table.  A thread whose maximum is a touched element looks its
// elements over again.  The
// chunks of a row join their maxima as 64-bit keys (value, then lowest index)
// with an atomic maximum; the last one to arrive writes the token and leaves
// the workspace zeroed.
//
// 64 x 152064 f32 with histories of 2048 tokens on average, 32 biases and a
// mask takes 32 us, the mask alone 18 (4.4 TB/s, 0.67 of the copy rate); the
// difference is the chain of small loads behind the pass, of which a wave of
// CTAs has one.  128 x 256000 bf16 with 8192 tokens: 81 us, the mask alone 41.
//
// Not kept, for 64 x 152064 with everything on: every chunk counting over the
// whole history (50 us: most warp steps met a hit for a lane or two), counting
// over a cluster's distributed shared memory (56-70 us: a frequent token's
// remote atomics queue up), one CTA per row making a list of different tokens
// in a hash table (45 us; 170 us for 128 x 256000, where a row's 13 k different
// tokens keep one SM busy for 100 us), the rules in a third kernel of a small
// CTA per 4096 tokens (51 us: its chains of small loads take longer than the
// pass over the logits that they hide behind here).
#include <algorithm>

#include "common.cuh"

namespace mtn {
namespace {

constexpr int kLogitsThreads = 256;
// CTAs an SM holds, by registers.  With rules, 64 x 152064 took 32.2, 32.7 and
// 36.4 us with 8, 6 and 4 (and more loads ahead); with a mask alone 21.9, 18.0
// and 19.5.
constexpr int logits_resident(bool rules) { return rules ? 8 : 6; }
constexpr int kChunkStep = 1024, kChunkMax = 32768;
constexpr int kChunkMaxRuled = 8192;  // tables of 32 KB
constexpr int kChunkFixed = 2048;
constexpr int kBatchVecs = 2;         // 16-byte loads of a thread ahead of the ones in work
constexpr int kAhead = 4;             // list entries of a thread in flight
constexpr int kSortThreads = 1024;
constexpr int kBuckets = 512;         // a row's chunks, or groups of 2^k of them
constexpr uint32_t kGenerated = 0x80000000u;

// Scratch between the two kernels: the entries of each list, sorted by bucket
// within a row, a row's from its index pointer on, and where the buckets begin.
struct SortedRules {
  uint2* bias;          // token, index in the row's list
  uint32_t* hist;       // token | kGenerated
  int32_t* hist_starts;  // [rows][kBuckets + 1]
  int32_t* bias_starts;
};

struct LogitsParams {
  const void* logits;
  int64_t row_stride;
  int64_t vocab;
  mtn_logits_rules r;
  SortedRules sorted;
  float* out;
  int64_t out_stride;
  int32_t* tokens;
  unsigned long long* keys;  // [rows] maxima, then [rows] arrival counters
  int64_t n_rows;
  int chunks, size;  // chunks a row, elements of a chunk
  int elem;          // bytes of a logit
  int bucket_shift;  // log2 of the chunks of a bucket
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

// Elements of row `row` before the first that a 16-byte load may start at.
// Chunk 0 of a row has them and the `size` elements behind them.
__device__ __forceinline__ int row_head(const LogitsParams& p, int row) {
  const uint64_t at = reinterpret_cast<uintptr_t>(p.logits) + row * p.row_stride * p.elem;
  return static_cast<int>((16u - (static_cast<uint32_t>(at) & 15u)) % 16u) / p.elem;
}

// One row's list, tokens[beg .. end), counted and placed by bucket; place(i, t,
// to) stores entry i.  All threads of the CTA.
template <typename F>
__device__ __forceinline__ void sort_list(const LogitsParams& p, int row, int head, const int32_t* tokens, int64_t beg,
                                          int64_t end, int32_t* starts, int* count, F place) {
  const int tid = threadIdx.x, lane = tid & 31;
  const uint32_t vocab = static_cast<uint32_t>(p.vocab);
  auto bucket_of = [&](int32_t t) {
    return static_cast<int>(static_cast<uint32_t>(max(t - head, 0)) / static_cast<uint32_t>(p.size)) >> p.bucket_shift;
  };
  auto each = [&](auto f) {
    for (int64_t i = beg + tid; i < end; i += kAhead * kSortThreads) {
      int32_t t[kAhead];
#pragma unroll
      for (int b = 0; b < kAhead; ++b) t[b] = i + b * kSortThreads < end ? tokens[i + b * kSortThreads] : -1;
#pragma unroll
      for (int b = 0; b < kAhead; ++b)
        if (i + b * kSortThreads < end) f(i + b * kSortThreads, t[b]);
    }
  };
  if (tid < kBuckets) count[tid] = 0;
  __syncthreads();
  each([&](int64_t, int32_t t) {
    if (static_cast<uint32_t>(t) < vocab)
      atomicAdd(&count[bucket_of(t)], 1);
    else
      record_error(p.err, kDevErrBadLogitRule, row);
  });
  __syncthreads();
  if (tid < 32) {  // exclusive sums, 16 buckets a lane
    constexpr int kPer = kBuckets / 32;
    int sum = 0;
    for (int i = 0; i < kPer; ++i) sum += count[lane * kPer + i];
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    int run = upto - sum;
    for (int i = 0; i < kPer; ++i) {
      const int n = count[lane * kPer + i];
      count[lane * kPer + i] = run;
      run += n;
    }
    if (lane == 31) starts[kBuckets] = upto;
  }
  __syncthreads();
  if (tid < kBuckets) starts[tid] = count[tid];
  __syncthreads();
  each([&](int64_t i, int32_t t) {
    if (static_cast<uint32_t>(t) < vocab) place(i, t, beg + atomicAdd(&count[bucket_of(t)], 1));
  });
}

__global__ void __launch_bounds__(kSortThreads) sort_rules_kernel(const LogitsParams p) {
  __shared__ int count[kBuckets];
  // the next kernel's first pass reads nothing of this one
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int row = static_cast<int>(blockIdx.x), head = row_head(p, row);
  const int64_t at = static_cast<int64_t>(row) * (kBuckets + 1);
  if (p.r.hist_indptr != nullptr) {
    int64_t beg, end;
    row_range(p.r.hist_indptr, row, p.r.n_hist, beg, end, p.err);
    const int64_t gen = beg + (p.r.prompt_lens != nullptr ? max(p.r.prompt_lens[row], 0) : 0);
    sort_list(p, row, head, p.r.hist_tokens, beg, end, p.sorted.hist_starts + at, count,
              [&](int64_t i, int32_t t, int64_t to) {
                p.sorted.hist[to] = static_cast<uint32_t>(t) | (i >= gen ? kGenerated : 0u);
              });
    __syncthreads();
  }
  if (p.r.bias_indptr != nullptr) {
    int64_t beg, end;
    row_range(p.r.bias_indptr, row, p.r.n_bias, beg, end, p.err);
    sort_list(p, row, head, p.r.bias_tokens, beg, end, p.sorted.bias_starts + at, count,
              [&](int64_t i, int32_t t, int64_t to) {
                p.sorted.bias[to] = make_uint2(static_cast<uint32_t>(t), static_cast<uint32_t>(i - beg));
              });
  }
}

// Order-preserving key of a processed logit: larger values first, then the
// lower index.  0 for what never wins (-inf, NaN).  x + 0 turns -0 into +0.
__device__ __forceinline__ unsigned long long arg_key(float x, int v) {
  if (!(x > -INFINITY)) return 0ull;
  const uint32_t b = __float_as_uint(__fadd_rn(x, 0.0f));
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return static_cast<unsigned long long>(o) << 32 | (0xffffffffu - static_cast<uint32_t>(v));
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

// kHist, kBias: a history, biases are given, and sort_rules_kernel went before.
template <typename T, bool kHist, bool kBias>
__global__ void __launch_bounds__(kLogitsThreads, logits_resident(kHist || kBias)) process_logits_kernel(const LogitsParams p) {
  extern __shared__ __align__(16) uint32_t smem[];
  constexpr int kN = Vec<T>::kN;
  constexpr bool kRules = kHist || kBias;
  const int tid = threadIdx.x;
  // The first chunks of all rows first: a tokenizer's frequent tokens come
  // early, and so do the chunks with the most entries.
  const int chunk = static_cast<int>(blockIdx.x / static_cast<uint32_t>(p.n_rows));
  const int row = static_cast<int>(blockIdx.x - static_cast<uint32_t>(chunk) * p.n_rows), vocab = static_cast<int>(p.vocab);
  const T* in = static_cast<const T*>(p.logits) + row * p.row_stride;
  float* out = p.out + row * p.out_stride;
  // Chunks begin where a 16-byte load may: `head` elements into the row; the
  // first one has the elements before that too.
  const int head = row_head(p, row);
  const bool vec = (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(out + head)) & 15u) == 0;
  auto start_of = [&](int c) {
    return c == 0 ? 0 : c >= p.chunks ? vocab : static_cast<int>(min(static_cast<int64_t>(vocab), static_cast<int64_t>(c) * p.size + head));
  };
  const int v0 = start_of(chunk), nv = start_of(chunk + 1) - v0;
  in += v0;
  out += v0;  // from here on elements count from the chunk's first
  const int body = chunk == 0 ? min(head, nv) : 0;  // vectors: body .. body + kN * nvec; the rest one by one
  const int nvec = vec ? (nv - body) / kN : 0;
  const uint4* vin = reinterpret_cast<const uint4*>(in + body);
  float4* vout = reinterpret_cast<float4*>(out + body);

  // The mask's words from the chunk's first element's on, and that element's bit.
  const uint32_t* mask = nullptr;
  const int mask_bit = v0 & 31, mask_last = ((vocab - 1) >> 5) - (v0 >> 5);
  if (p.r.mask != nullptr) {
    const int mr = p.r.mask_rows != nullptr ? p.r.mask_rows[row] : row;
    if (mr >= 0 && mr < p.r.n_masks)
      mask = p.r.mask + mr * p.r.mask_stride + (v0 >> 5);
    else if (mr != -1 && tid == 0)
      record_error(p.err, kDevErrBadLogitRule, row);
  }
  auto allowed = [&](int k) { return mask == nullptr || (mask[(k + mask_bit) >> 5] >> ((k + mask_bit) & 31) & 1u) != 0; };

  // A thread sees rising places, so a strict comparison keeps the first maximum.
  float best = -INFINITY;
  int best_k = 0;
  auto scalar = [&](int k) {
    float y = ld_logit(in + k);
    if (!allowed(k)) y = -INFINITY;
    out[k] = y;
    if (y > best) best = y, best_k = k;
  };
  if (vec) {
    if (tid < body) scalar(tid);
    // A step of 256 vectors is a whole number of mask words, so a thread's
    // bits lie at the same place of a word every time.
    const int bit = body + tid * kN + mask_bit, sh = bit & 31;
    const uint32_t* mw = mask + (bit >> 5);
    constexpr int kWords = kLogitsThreads * kN / 32;
    const int wlast = mask_last - (bit >> 5);
    Vec<T> x[kBatchVecs];
    uint32_t m[kBatchVecs];
    auto load = [&](int b, int i, int step) {
      if (i < nvec) {
        x[b].w = vin[i];
        m[b] = mask != nullptr ? mw[step * kWords] : ~0u;
      }
    };
#pragma unroll
    for (int b = 0; b < kBatchVecs; ++b) load(b, tid + b * kLogitsThreads, b);
    for (int i = tid, step = 0; i < nvec; i += kBatchVecs * kLogitsThreads, step += kBatchVecs) {
#pragma unroll
      for (int b = 0; b < kBatchVecs; ++b) {
        const int j = i + b * kLogitsThreads;
        if (j < nvec) {
          uint32_t allow = ~0u;
          if (mask != nullptr) {
            allow = m[b] >> sh;
            if (sh > 32 - kN) allow |= mw[min((step + b) * kWords + 1, wlast)] << (32 - sh);
          }
          float y[kN];
#pragma unroll
          for (int e = 0; e < kN; ++e) y[e] = allow & (1u << e) ? x[b].get(e) : -INFINITY;
          load(b, j + kBatchVecs * kLogitsThreads, step + b + kBatchVecs);
#pragma unroll
          for (int e = 0; e < kN; e += 4) vout[j * (kN / 4) + e / 4] = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
          float top = y[0];
#pragma unroll
          for (int e = 1; e < kN; ++e) top = fmaxf(top, y[e]);
          if (top > best) {
            best = top;
#pragma unroll
            for (int e = kN - 1; e >= 0; --e)
              if (y[e] == top) best_k = body + j * kN + e;
          }
        }
      }
    }
    const int rest = body + nvec * kN + tid;
    if (rest < nv) scalar(rest);
  } else {
    for (int k = tid; k < nv; k += kLogitsThreads) scalar(k);
  }

  unsigned long long key = 0;
  if constexpr (kRules) {
    // shared memory: bitmaps of touched elements and of those with a bias; a
    // table of times generated, and kGenerated for being in the history at
    // all, then of index + 1 of a token's last bias
    const int map_words = p.size / 32 + 4;
    uint32_t* touched = smem;
    uint32_t* biased = touched + map_words;
    uint32_t* table = biased + (kBias ? map_words : 0);
    const int vecs = static_cast<int>(table - smem + p.size + 8) / 4;
    for (int i = tid; i < vecs; i += kLogitsThreads) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    int64_t hbeg = 0, bbeg = 0, end;
    if constexpr (kHist) row_range(p.r.hist_indptr, row, p.r.n_hist, hbeg, end, p.err);
    if constexpr (kBias) row_range(p.r.bias_indptr, row, p.r.n_bias, bbeg, end, p.err);
    const float rep = kHist && p.r.repetition != nullptr ? p.r.repetition[row] : 1.0f;
    const float freq = kHist && p.r.frequency != nullptr ? p.r.frequency[row] : 0.0f;
    const float pres = kHist && p.r.presence != nullptr ? p.r.presence[row] : 0.0f;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the lists are sorted
    const int64_t bucket = static_cast<int64_t>(row) * (kBuckets + 1) + (chunk >> p.bucket_shift);
    const uint32_t* hist_list = nullptr;
    const uint2* bias_list = nullptr;
    int n_hist = 0, n_bias = 0;
    if constexpr (kHist) {
      const int from = p.sorted.hist_starts[bucket];
      n_hist = p.sorted.hist_starts[bucket + 1] - from;
      hist_list = p.sorted.hist + hbeg + from;
    }
    if constexpr (kBias) {
      const int from = p.sorted.bias_starts[bucket];
      n_bias = p.sorted.bias_starts[bucket + 1] - from;
      bias_list = p.sorted.bias + bbeg + from;
    }
    // Calls f for kAhead history entries at a time: places of the chunk, and
    // kNone where there is no entry or it is another chunk's of the bucket;
    // kGenerated with a place as with its entry.
    constexpr uint32_t kNone = ~kGenerated;
    auto entries = [&](auto f) {
      for (int i = tid; i < n_hist; i += kAhead * kLogitsThreads) {
        uint32_t k[kAhead];
#pragma unroll
        for (int b = 0; b < kAhead; ++b) k[b] = i + b * kLogitsThreads < n_hist ? hist_list[i + b * kLogitsThreads] : kNone;
#pragma unroll
        for (int b = 0; b < kAhead; ++b) {
          const uint32_t at = (k[b] & ~kGenerated) - static_cast<uint32_t>(v0);
          k[b] = k[b] != kNone && at < static_cast<uint32_t>(nv) ? at | (k[b] & kGenerated) : kNone;
        }
        f(k);
      }
    };
    __syncthreads();  // the tables, and the first pass's stores
    entries([&](const uint32_t(&k)[kAhead]) {
#pragma unroll
      for (int b = 0; b < kAhead; ++b) {
        if (k[b] == kNone) continue;
        uint32_t* slot = &table[k[b] & ~kGenerated];
        if (!(*slot & kGenerated)) atomicOr(slot, kGenerated);
        if (k[b] & kGenerated) atomicAdd(slot, 1u);
      }
    });
    for (int i = tid; i < n_bias; i += kLogitsThreads) {
      const uint32_t k = bias_list[i].x - static_cast<uint32_t>(v0);
      if (k < static_cast<uint32_t>(nv)) atomicOr(&biased[k >> 5], 1u << (k & 31));
    }
    __syncthreads();
    // The first entry to take a token's count out of the table applies it.
    entries([&](const uint32_t(&e)[kAhead]) {
      uint32_t c[kAhead];
      float y[kAhead];
#pragma unroll
      for (int b = 0; b < kAhead; ++b) {
        const uint32_t k = e[b] & ~kGenerated;
        c[b] = e[b] != kNone && table[k] != 0 ? atomicExch(&table[k], 0u) : 0u;
        if (c[b] == 0) continue;
        atomicOr(&touched[k >> 5], 1u << (k & 31));
        if (!allowed(static_cast<int>(k))) c[b] = 0;
      }
#pragma unroll
      for (int b = 0; b < kAhead; ++b)
        if (c[b] != 0) y[b] = ld_logit(in + (e[b] & ~kGenerated));
#pragma unroll
      for (int b = 0; b < kAhead; ++b) {
        if (c[b] == 0) continue;
        const uint32_t k = e[b] & ~kGenerated, n = c[b] & ~kGenerated;
        float z = y[b] > 0.0f ? __fdiv_rn(y[b], rep) : __fmul_rn(y[b], rep);
        z = __fsub_rn(z, __fmul_rn(freq, static_cast<float>(n)));
        if (n != 0) z = __fsub_rn(z, pres);
        out[k] = z;
        if (!kBias || !(biased[k >> 5] >> (k & 31) & 1u)) key = max(key, arg_key(z, v0 + static_cast<int>(k)));
      }
    });
    if constexpr (kBias) {
      __syncthreads();  // the table is zero again, the penalties are stored
      if (n_bias > 0) {
        for (int i = tid; i < n_bias; i += kLogitsThreads) {
          const uint32_t k = bias_list[i].x - static_cast<uint32_t>(v0);
          if (k < static_cast<uint32_t>(nv)) atomicMax(&table[k], bias_list[i].y + 1u);
        }
        __syncthreads();
        for (int i = tid; i < n_bias; i += kLogitsThreads) {
          const uint32_t k = bias_list[i].x - static_cast<uint32_t>(v0);
          if (k >= static_cast<uint32_t>(nv)) continue;
          const uint32_t last = atomicExch(&table[k], 0u);
          if (last == 0) continue;
          const bool penalised = (atomicOr(&touched[k >> 5], 1u << (k & 31)) >> (k & 31) & 1u) != 0;
          if (!allowed(static_cast<int>(k))) continue;
          // a malformed index pointer may have rows that share entries, and another row's index here
          const float bias = p.r.bias_values[min(bbeg + last, p.r.n_bias) - 1];
          const float y = __fadd_rn(penalised ? out[k] : ld_logit(in + k), bias);
          out[k] = y;
          key = max(key, arg_key(y, v0 + static_cast<int>(k)));
        }
      }
    }
    __syncthreads();
    auto is_touched = [&](int k) { return (touched[k >> 5] >> (k & 31) & 1u) != 0; };
    if (p.tokens != nullptr && best > -INFINITY && is_touched(best_k)) {
      // this thread's maximum is a touched element: look for another (untouched
      // elements of `out` are final)
      best = -INFINITY;
      auto again = [&](int k) {
        const float y = out[k];
        if (y > best && !is_touched(k)) best = y, best_k = k;
      };
      if (vec) {
        if (tid < body) again(tid);
        for (int i = tid; i < nvec; i += kLogitsThreads)
          for (int e = 0; e < kN; ++e) again(body + i * kN + e);
        if (body + nvec * kN + tid < nv) again(body + nvec * kN + tid);
      } else {
        for (int k = tid; k < nv; k += kLogitsThreads) again(k);
      }
    }
  }
  if (p.tokens == nullptr) return;
  key = max(key, arg_key(best, v0 + best_k));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
  __shared__ unsigned long long wkey[kLogitsThreads / 32];
  if ((tid & 31) == 0) wkey[tid >> 5] = key;
  __syncthreads();
  if (tid != 0) return;
#pragma unroll
  for (int w = 1; w < kLogitsThreads / 32; ++w) key = max(key, wkey[w]);
  atomicMax(&p.keys[row], key);
  unsigned long long before;  // release: the maximum above; acquire: the other chunks'
  asm volatile("atom.acq_rel.gpu.global.add.u64 %0, [%1], 1;" : "=l"(before) : "l"(&p.keys[p.n_rows + row]) : "memory");
  if (before != static_cast<unsigned long long>(p.chunks - 1)) return;
  key = atomicExch(&p.keys[row], 0ull);
  p.keys[p.n_rows + row] = 0ull;
  p.tokens[row] = key == 0 ? 0 : static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(key));
}

using LogitsKernel = void (*)(const LogitsParams);

template <typename T>
LogitsKernel logits_kernel(bool hist, bool biased) {
  if (hist) return biased ? process_logits_kernel<T, true, true> : process_logits_kernel<T, true, false>;
  return biased ? process_logits_kernel<T, false, true> : process_logits_kernel<T, false, false>;
}

// Shared memory of a chunk of `size` elements, bytes.
constexpr int logits_smem(int size, bool hist, bool biased) {
  return hist || biased ? ((size / 32 + 4) * (biased ? 2 : 1) + size + 8) * 4 : 0;
}

}  // namespace
}  // namespace mtn

extern "C" {

size_t mtn_process_logits_workspace_bytes(int64_t n_rows) {
  return n_rows <= 0 ? 0 : static_cast<size_t>(n_rows) * 16;
}

size_t mtn_process_logits_scratch_bytes(int64_t n_rows, int64_t n_hist, int64_t n_bias) {
  if (n_rows <= 0 || n_hist < 0 || n_bias < 0 || n_hist + n_bias == 0) return 0;
  // sorted biases and history, and where each row's buckets begin in both
  return static_cast<size_t>(n_bias) * 8 + static_cast<size_t>(n_hist) * 4 +
         static_cast<size_t>(n_rows) * (mtn::kBuckets + 1) * 8;
}

int mtn_process_logits(const void* logits, int32_t dtype, int64_t row_stride, int64_t n_rows, int64_t vocab,
                       const mtn_logits_rules* rules, float* out, int64_t out_stride, int32_t* tokens, void* workspace,
                       size_t workspace_bytes, void* scratch, size_t scratch_bytes, void* stream) {
  MTN_CHECK_ARG(n_rows >= 0 && n_rows <= INT32_MAX && vocab > 0 && vocab <= INT32_MAX - 65536, "mtn_process_logits: bad sizes");
  MTN_CHECK_ARG(dtype == MTN_DTYPE_BF16 || dtype == MTN_DTYPE_F32, "mtn_process_logits: bad dtype");
  if (n_rows == 0) return MTN_OK;
  MTN_CHECK_ARG(logits && rules && out, "mtn_process_logits: null pointer");
  MTN_CHECK_ARG(row_stride >= vocab && out_stride >= vocab, "mtn_process_logits: row strides shorter than a row");
  MTN_CHECK_ARG(static_cast<const void*>(out) != logits || (dtype == MTN_DTYPE_F32 && row_stride == out_stride),
                "mtn_process_logits: in place needs f32 logits and equal strides");
  MTN_CHECK_ARG(mtn::elem_aligned(logits, dtype) && mtn::elem_aligned(out, MTN_DTYPE_F32),
                "mtn_process_logits: a pointer is not aligned to its elements");
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
  for (const void* q : {static_cast<const void*>(r.hist_indptr), static_cast<const void*>(r.hist_tokens),
                        static_cast<const void*>(r.prompt_lens), static_cast<const void*>(r.repetition),
                        static_cast<const void*>(r.presence), static_cast<const void*>(r.frequency),
                        static_cast<const void*>(r.bias_indptr), static_cast<const void*>(r.bias_tokens),
                        static_cast<const void*>(r.bias_values), static_cast<const void*>(r.mask),
                        static_cast<const void*>(r.mask_rows), static_cast<const void*>(tokens)})
    MTN_CHECK_ARG(reinterpret_cast<uintptr_t>(q) % 4 == 0, "mtn_process_logits: a rule's array or tokens is not aligned to its elements");
  const size_t need = mtn_process_logits_workspace_bytes(n_rows);
  MTN_CHECK_ARG(tokens == nullptr || (workspace != nullptr && workspace_bytes >= need &&
                                      (reinterpret_cast<uintptr_t>(workspace) & 7) == 0),
                "mtn_process_logits: tokens need an 8-byte aligned workspace of %zu bytes", need);
  const int64_t n_hist = r.hist_indptr != nullptr ? r.n_hist : 0, n_bias = r.bias_indptr != nullptr ? r.n_bias : 0;
  const bool ruled = n_hist + n_bias > 0;
  const size_t lists = mtn_process_logits_scratch_bytes(n_rows, n_hist, n_bias);
  MTN_CHECK_ARG(!ruled || (scratch != nullptr && scratch_bytes >= lists && (reinterpret_cast<uintptr_t>(scratch) & 7) == 0),
                "mtn_process_logits: a history or biases need an 8-byte aligned scratch of %zu bytes", lists);
  // The chunk whose waves of resident CTAs have the fewest elements to pass,
  // a CTA's fixed part counted as kChunkFixed of them.
  int size = 0;
  int64_t chunks = 0, best = INT64_MAX;
  const bool hist = n_hist > 0, biased = n_bias > 0;
  for (int sz = mtn::kChunkStep; sz <= (ruled ? mtn::kChunkMaxRuled : mtn::kChunkMax); sz += mtn::kChunkStep) {
    const int64_t c = (vocab + sz - 1) / sz;
    const int most = mtn::logits_resident(ruled);
    const int fit = ruled ? std::min(most, 227 * 1024 / (mtn::logits_smem(sz, hist, biased) + 1024)) : most;
    const int64_t slots = static_cast<int64_t>(mtn::sm_count()) * fit;
    const int64_t cost = (n_rows * c + slots - 1) / slots * (sz + mtn::kChunkFixed);
    if (cost < best) {
      best = cost;
      size = sz;
      chunks = c;
    }
  }
  MTN_CHECK_ARG(chunks * n_rows <= INT32_MAX, "mtn_process_logits: batch too large");
  mtn::SortedRules l{};
  if (ruled) {
    l.bias = static_cast<uint2*>(scratch);
    l.hist = reinterpret_cast<uint32_t*>(l.bias + n_bias);
    l.hist_starts = reinterpret_cast<int32_t*>(l.hist + n_hist);
    l.bias_starts = l.hist_starts + n_rows * (mtn::kBuckets + 1);
  }
  int bucket_shift = 0;
  while ((chunks - 1) >> bucket_shift >= mtn::kBuckets) ++bucket_shift;
  const bool bf16 = dtype == MTN_DTYPE_BF16;
  mtn::LogitsParams p{logits, row_stride, vocab, r, l, out, out_stride, tokens, static_cast<unsigned long long*>(workspace),
                      n_rows, static_cast<int>(chunks), size, bf16 ? 2 : 4, bucket_shift, mtn::device_error_ptr()};
  if (!hist) p.r.hist_indptr = nullptr;
  if (!biased) p.r.bias_indptr = nullptr;
  auto s = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(chunks * n_rows);
  const mtn::LogitsKernel kern =
      bf16 ? mtn::logits_kernel<__nv_bfloat16>(hist, biased) : mtn::logits_kernel<float>(hist, biased);
  if (!ruled) {
    kern<<<grid, mtn::kLogitsThreads, 0, s>>>(p);
    return mtn::check_launch("process_logits_kernel");
  }
  mtn::sort_rules_kernel<<<static_cast<unsigned>(n_rows), mtn::kSortThreads, 0, s>>>(p);
  const int st = mtn::check_launch("sort_rules_kernel");
  if (st != MTN_OK) return st;
  const int smem = mtn::logits_smem(size, hist, biased);
  MTN_CUDA_TRY(mtn::allow_smem(reinterpret_cast<const void*>(kern), mtn::logits_smem(mtn::kChunkMaxRuled, true, true)),
               "mtn_process_logits");
  return mtn::launch_pdl(kern, dim3(grid), dim3(mtn::kLogitsThreads), smem, s, "process_logits_kernel", p);
}

}  // extern "C"
