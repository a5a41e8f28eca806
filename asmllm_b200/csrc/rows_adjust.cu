// asmllm_b200/csrc/rows_adjust.cu -- what is done to logits before a word is
// chosen: penalties for words that have come already, biases of some words,
// and a mask of the allowed ones.
//
// For word w of a row, seen `all` times among the row's tokens and c times
// among those behind its prompt, in fp32, each step rounded:
//   1. all > 0:  x = x > 0 ? x * (1 / repetition) : x * repetition
//   2. c > 0:    x = (x - frequency * c) - presence
//   3. x = x + the sum of the word's biases (added up in 64 bits in their order)
//   4. not allowed: -inf
// and one rounding to the logits' type; other words are copied.
//
// Bound by HBM: logits are read and written once.  A slice of a row's words has
// a counter for each in shared memory, and looks at all of the row's tokens
// (integer atomics count: their order does not matter).  The few biased words
// are marked in their counters and left to a thread each, which reads the logit
// before it stores the new one, so that `out` may be the logits themselves.
// The penalties are computed without a branch a word: in a long history nearly
// every warp has a word that has come.
//   A large batch: one CTA an SM with an equal share of the slices, a quarter of
//     its threads counting for the next slice while the others stream this
//     one's logits (asked for a slice ahead), two sets of counters in turn.
//   A small batch: a CTA a slice of 2048 words, as many as there are.
// Measured on one B200, 128 rows of 128256 words, 8192 tokens, 64 biases and a
// mask: 44 us (the copy alone takes 21); instructions, of which the words'
// penalties are the most, issue in 58 % of the cycles.  56 where every CTA
// counts and then streams; 49 with a row's tokens in a hash table that is
// applied to a copy of the logits (its scattered accesses take one cycle of an
// SM each, three a word); 150 and more where the counting threads change the
// words that have come by themselves.  32 rows of bf16, 1024 tokens, 300
// biases: 15 us.  One row of 32000 words: 4 us.  Rows that are not aligned in
// fours of words (a dense vocabulary of 50257) go by slices of 2048 with single
// accesses, each of which looks at all of the row's tokens: 128 rows of 50257
// words 32 us where 50256 take 23, of 128257 words 73 where 128256 take 45.
#include "matvec.cuh"
#include "serving_q8.cuh"

namespace asmllm {

namespace {

// A word's counter: in the prompt; has a bias, has several; and how often it comes behind the prompt.
constexpr unsigned kSeen = 1u << 31, kBiased = 1u << 30, kSeveral = 1u << 29, kCount = kSeveral - 1;

template <class T> __device__ __forceinline__ float load1(const T* p) {
  if constexpr (sizeof(T) == 4) return __ldcg(p);
  else {
    const unsigned short w = __ldcg(reinterpret_cast<const unsigned short*>(p));
    return to_f32(*reinterpret_cast<const T*>(&w));
  }
}
template <class T> __device__ __forceinline__ void store1(T* p, float v) {
  if constexpr (sizeof(T) == 4) *p = v;
  else *reinterpret_cast<unsigned short*>(p) = (unsigned short)pack16<T>(v, 0.0f);
}

struct Penalty {
  float repetition, inverse, frequency, presence;
  __device__ __forceinline__ float operator()(float x, unsigned n) const {
    const unsigned c = n & kCount;
    const float r = __fmul_rn(x, x > 0.0f ? inverse : repetition);
    const float f = __fsub_rn(__fsub_rn(r, __fmul_rn(frequency, (float)c)), presence);
    return c ? f : n & kSeen ? r : x;
  }
};

// Four words as they are in memory, and as floats.
template <class T> struct Raw4Of { using type = uint2; };
template <> struct Raw4Of<float> { using type = float4; };
template <class T> using Raw4 = typename Raw4Of<T>::type;
template <class T>
__device__ __forceinline__ void unpack4(const Raw4<T>& f, float (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
    const float2 lo = unpack16<T>(f.x), hi = unpack16<T>(f.y);
    v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
  }
}
// Four words from x on, n of which exist; VEC: they are aligned.
template <class T, bool VEC>
__device__ __forceinline__ void load4(const T* x, int n, float (&v)[4]) {
  if (VEC && n >= 4) {
    unpack4<T>(__ldcg(reinterpret_cast<const Raw4<T>*>(x)), v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < n ? load1(x + e) : 0.0f;
  }
}
template <class T, bool VEC>
__device__ __forceinline__ void store4(T* y, int n, const float (&v)[4], unsigned keep) {
  if (VEC && n >= 4 && keep == 15u) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(y) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<uint2*>(y) = make_uint2(pack16<T>(v[0], v[1]), pack16<T>(v[2], v[3]));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n && (keep >> e & 1u)) store1(y + e, v[e]);
  }
}

struct Row {  // a row's penalties and tokens
  Penalty p;
  const int32_t* tokens;
  int held, prompt;
  __device__ __forceinline__ Row() {}
  __device__ __forceinline__ Row(const AdjustArgs& a, int row, bool report, unsigned* err) {
    p.repetition = a.repetition ? __ldcg(a.repetition + row) : 1.0f;
    p.inverse = __frcp_rn(p.repetition);
    p.frequency = a.frequency ? __ldcg(a.frequency + row) : 0.0f;
    p.presence = a.presence ? __ldcg(a.presence + row) : 0.0f;
    tokens = a.tokens + (long long)row * a.token_stride;
    held = !a.tokens ? 0 : a.n_tokens ? __ldcg(a.n_tokens + row) : a.held;
    prompt = a.n_prompt ? __ldcg(a.n_prompt + row) : 0;
    if (held < 0 || held > a.held) {
      if (report) atomicOr(err, kErrDecodeRange);
      held = held < 0 ? 0 : a.held;
    }
  }
  // f(place, token) for all of them, by `threads` threads; four loads of four under way at a time
  template <class F>
  __device__ __forceinline__ void each(int tid, int threads, F f) const {
    const int first = (reinterpret_cast<uintptr_t>(tokens) & 15u) == 0 ? held & ~3 : 0;
    for (int i0 = 4 * tid; i0 < first; i0 += 16 * threads) {
      int4 t[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) t[q] = four(i0 + 4 * threads * q, first);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = i0 + 4 * threads * q;
        f(i, t[q].x);
        f(i + 1, t[q].y);
        f(i + 2, t[q].z);
        f(i + 3, t[q].w);
      }
    }
    for (int i = first + tid; i < held; i += threads) f(i, __ldca(tokens + i));
  }
  __device__ __forceinline__ int4 four(int i, int end) const {
    return i < end ? __ldca(reinterpret_cast<const int4*>(tokens + i)) : make_int4(-1, -1, -1, -1);
  }
};

__device__ __forceinline__ bool is_allowed(const AdjustArgs& a, int row, int w) {
  return !a.allowed || (__ldcg(a.allowed + (long long)row * a.allowed_stride + (w >> 5)) >> (w & 31) & 1);
}

// The mask's bits of words w .. w + 3, w a multiple of 4.
__device__ __forceinline__ unsigned mask4(const AdjustArgs& a, int row, int w, bool live) {
  return a.allowed && live ? (unsigned)__ldcg(a.allowed + (long long)row * a.allowed_stride + (w >> 5)) >> (w & 31) : 15u;
}

// The sum of word w's biases, in their order: entry i is one of them, `several` says that there are more.
__device__ __forceinline__ float bias_of(const int* word, const float* bias, int n_list, int i, int w, bool several) {
  double sum = 0.0;
  if (!several) return bias[i];
  for (int j = 0; j < n_list; j += 4) {
    const int4 z = *reinterpret_cast<const int4*>(word + j);
    if (z.x == w) sum += (double)bias[j];
    if (z.y == w) sum += (double)bias[j + 1];
    if (z.z == w) sum += (double)bias[j + 2];
    if (z.w == w) sum += (double)bias[j + 3];
  }
  return (float)sum;
}

// The list of biased words [n_bias, to a multiple of 4] into shared memory.
__device__ __forceinline__ void load_list(const AdjustArgs& a, int row, int n_list, int* word, float* bias, int tid,
                                          int threads) {
  for (int i = tid; i < n_list; i += threads) {
    const bool live = i < a.n_bias;
    const int w = live ? __ldcg(a.bias_tokens + (long long)row * a.n_bias + i) : -1;
    word[i] = (unsigned)w < (unsigned)a.n ? w : -1;
    bias[i] = live ? __ldcg(a.bias + (long long)row * a.n_bias + i) : 0.0f;
  }
}

// Counts the tokens that fall into words [w0, w0 + n), and marks the biased words among them: bit k of the result, this
// thread is the one to find the new logit of entry tid + k threads.
template <int THREADS>
__device__ __forceinline__ unsigned count_slice(const Row& r, int w0, int n, unsigned* count, const int* word, int n_list,
                                                int tid) {
  r.each(tid, THREADS, [&](int i, int token) {
    const unsigned w = (unsigned)token - (unsigned)w0;
    if (w < (unsigned)n) {
      if (i < r.prompt) atomicOr(count + w, kSeen);
      else atomicAdd(count + w, 1u);
    }
  });
  unsigned mine = 0u;
  for (int i = tid, k = 0; i < n_list; i += THREADS, ++k) {
    const int w = word[i];
    if (w < w0 || w >= w0 + n) continue;
    if (atomicOr(count + (w - w0), kBiased) & kBiased) atomicOr(count + (w - w0), kSeveral);
    else mine |= 1u << k;
  }
  return mine;
}

// The new logits of the entries in `mine`, once the slice's tokens are counted.
template <class T, int THREADS>
__device__ __forceinline__ void store_biased(const AdjustArgs& a, const Row& r, int row, int w0, const unsigned* count,
                                             const int* word, const float* bias, int n_list, unsigned mine, int tid) {
  const T* x = static_cast<const T*>(a.logits) + (long long)row * a.stride;
  T* y = static_cast<T*>(a.out) + (long long)row * a.out_stride;
  for (int i = tid; mine; i += THREADS, mine >>= 1) {
    if (!(mine & 1u)) continue;
    const int w = word[i];
    const unsigned c = count[w - w0];
    const float v = __fadd_rn(r.p(load1(x + w), c), bias_of(word, bias, n_list, i, w, c & kSeveral));
    store1(y + w, is_allowed(a, row, w) ? v : -INFINITY);
  }
}

// Four words with their counters (CLEAR: which are zero again then) and bits of the mask, into y; biased ones are left.
template <class T, bool VEC, bool CLEAR>
__device__ __forceinline__ void put4(T* y, int n, float (&v)[4], unsigned* count, unsigned bits, const Penalty& p) {
  const uint4 c4 = *reinterpret_cast<const uint4*>(count);
  unsigned keep = 15u;
  if (c4.x | c4.y | c4.z | c4.w) {
    const unsigned c[4] = {c4.x, c4.y, c4.z, c4.w};
    keep = 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = p(v[e], c[e]);
      keep |= c[e] & kBiased ? 0u : 1u << e;
    }
    if (CLEAR) *reinterpret_cast<uint4*>(count) = make_uint4(0u, 0u, 0u, 0u);
  }
  if ((bits & 15u) != 15u) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (!(bits >> e & 1u)) v[e] = -INFINITY;
  }
  store4<T, VEC>(y, n, v, keep);
}

// A small batch: a slice of kSmallSlice words a CTA.  VEC: rows whose groups of four words are aligned.
constexpr int kSmallSlice = 2048;
template <class T, bool VEC>
__global__ void __launch_bounds__(256) rows_adjust_slice_kernel(const AdjustArgs a, unsigned* __restrict__ err) {
  constexpr int kThreads = 256, kGroups = kSmallSlice / 4 / kThreads;
  __shared__ __align__(16) unsigned s_count[kSmallSlice];
  __shared__ __align__(16) int s_word[kAdjustMaxBias];
  __shared__ float s_bias[kAdjustMaxBias];
  pdl_trigger();
  const int tid = threadIdx.x, row = blockIdx.y, w0 = blockIdx.x * kSmallSlice, n = min(kSmallSlice, a.n - w0);
  const int n_list = (a.n_bias + 3) & ~3;
  for (int i = tid; i < kSmallSlice / 4; i += kThreads) reinterpret_cast<uint4*>(s_count)[i] = make_uint4(0u, 0u, 0u, 0u);
  pdl_wait();
  const T* x = static_cast<const T*>(a.logits) + (long long)row * a.stride + w0;
  T* y = static_cast<T*>(a.out) + (long long)row * a.out_stride + w0;
  const Row r(a, row, tid == 0 && blockIdx.x == 0, err);
  float v[kGroups][4];
  unsigned bits[kGroups];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const int i = 4 * (tid + g * kThreads);
    bits[g] = mask4(a, row, w0 + i, i < n);
    load4<T, VEC>(x + i, n - i, v[g]);
  }
  load_list(a, row, n_list, s_word, s_bias, tid, kThreads);
  __syncthreads();
  const unsigned mine = count_slice<kThreads>(r, w0, n, s_count, s_word, n_list, tid);
  __syncthreads();
  store_biased<T, kThreads>(a, r, row, w0, s_count, s_word, s_bias, n_list, mine, tid);
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const int i = 4 * (tid + g * kThreads);
    if (i < n) put4<T, VEC, false>(y + i, n - i, v[g], s_count + i, bits[g], r.p);
  }
}

// A large batch: CTA b has slices b `each` + min(b, extra) on of all rows' in a row, `len` words each (at most kBigSlice).
constexpr int kStreamers = 768, kCounters = 256, kBoth = kStreamers + kCounters;  // threads
constexpr int kGroups = 4, kBigSlice = 4 * kGroups * kStreamers;                    // of four words a streaming thread

constexpr int kBarFull = 1, kBarEmpty = 3, kBarCount = 5;  // named barriers: full and empty, one for each set of counters
__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int n) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory"); }

template <class T>
__global__ void __launch_bounds__(kBoth, 1) rows_adjust_stream_kernel(const AdjustArgs a, int slices, int len, int each,
                                                                      int extra, unsigned* __restrict__ err) {
  extern __shared__ __align__(16) unsigned s_count[];  // [2][kBigSlice], then the list: words, biases
  const int n_list = (a.n_bias + 3) & ~3, b = blockIdx.x;
  int* s_word = reinterpret_cast<int*>(s_count + 2 * kBigSlice);
  float* s_bias = reinterpret_cast<float*>(s_word + n_list);
  pdl_trigger();
  for (int i = threadIdx.x; i < 2 * kBigSlice / 4; i += kBoth) reinterpret_cast<uint4*>(s_count)[i] = make_uint4(0u, 0u, 0u, 0u);
  pdl_wait();
  __syncthreads();
  const int first = b * each + min(b, extra), items = each + (b < extra);
  int row = -1;
  Row r;
  if (threadIdx.x >= kStreamers) {
    // ---------------- counting ----------------
    const int tid = threadIdx.x - kStreamers;
    for (int k = 0; k < items; ++k) {
      const int item = first + k, w0 = item % slices * len, n = min(len, a.n - w0);
      unsigned* count = s_count + (k & 1) * kBigSlice;
      if (item / slices != row) {
        row = item / slices;
        r = Row(a, row, tid == 0 && w0 == 0, err);
        bar_sync(kBarCount, kCounters);  // the last row's list is no longer read
        load_list(a, row, n_list, s_word, s_bias, tid, kCounters);
        bar_sync(kBarCount, kCounters);
      }
      if (k >= 2) bar_sync(kBarEmpty + (k & 1), kBoth);  // streamed, and zero again
      const unsigned mine = count_slice<kCounters>(r, w0, n, count, s_word, n_list, tid);
      if (n_list) {
        bar_sync(kBarCount, kCounters);
        store_biased<T, kCounters>(a, r, row, w0, count, s_word, s_bias, n_list, mine, tid);
      }
      bar_arrive(kBarFull + (k & 1), kBoth);
    }
    return;
  }
  // ---------------- streaming ----------------
  // A slice's logits and mask are asked for a slice ahead and left as they come: a conversion right behind a load would
  // wait for it.
  const int tid = threadIdx.x;
  struct Ahead {
    Raw4<T> x[kGroups];
    unsigned mask[kGroups];
  };
  auto ask = [&](int k, Ahead& z) {
    const int item = first + k, row = item / slices, w0 = item % slices * len, n = min(len, a.n - w0);
    const T* x = static_cast<const T*>(a.logits) + (long long)row * a.stride + w0;
    const int32_t* mask = a.allowed + (long long)row * a.allowed_stride;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int i = 4 * (tid + g * kStreamers);
      z.mask[g] = a.allowed && i < n ? (unsigned)__ldcg(mask + ((w0 + i) >> 5)) : 0xFFFFFFFFu;
      if (i + 4 <= n) z.x[g] = __ldcg(reinterpret_cast<const Raw4<T>*>(x + i));
    }
  };
  auto step = [&](int k, Ahead& z, Ahead& next) {
    const int item = first + k, w0 = item % slices * len, n = min(len, a.n - w0);
    unsigned* count = s_count + (k & 1) * kBigSlice;
    if (k + 1 < items) ask(k + 1, next);
    if (item / slices != row) {
      row = item / slices;
      r = Row(a, row, false, err);
    }
    bar_sync(kBarFull + (k & 1), kBoth);
    const T* x = static_cast<const T*>(a.logits) + (long long)row * a.stride + w0;
    T* y = static_cast<T*>(a.out) + (long long)row * a.out_stride + w0;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int i = 4 * (tid + g * kStreamers);
      if (i >= n) continue;
      float v[4];
      if (i + 4 <= n) unpack4<T>(z.x[g], v);
      else load4<T, false>(x + i, n - i, v);
      put4<T, true, true>(y + i, n - i, v, count + i, z.mask[g] >> ((w0 + i) & 31), r.p);
    }
    if (k + 2 < items) bar_arrive(kBarEmpty + (k & 1), kBoth);
  };
  Ahead z[2];
  if (items > 0) ask(0, z[0]);
  for (int k = 0; k < items; k += 2) {
    step(k, z[0], z[1]);
    if (k + 1 < items) step(k + 1, z[1], z[0]);
  }
}

// Words of a batch from which on the second kernel is the faster one, where its rows are aligned (both, the first one
// first; fp32 and bf16, us).  1024 tokens a row: 0.5 M words 4.1 and 4.7, 4.2 and 4.1; 1 M 6.2 and 6.2, 6.2 and 5.8 (32 rows),
// 5.3 and 5.7, 5.4 and 5.3 (8); 2 M 7.9 and 8.0, 8.0 and 7.3; 3.9 M 12.3 and 10.9, 12.3 and 9.7.  8192 tokens: 0.5 M 5.3 and
// 6.2, 5.4 and 5.9; 1 M 7.1 and 7.4, 7.2 and 6.4 (8 rows); 2 M 10.8 and 10.5, 10.9 and 10.3.
constexpr long long kSmallBatch = 1 << 20;

template <class... Args>
cudaError_t launch(void (*kernel)(Args...), dim3 grid, int threads, int smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_opt_pdl.load() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <class T>
cudaError_t launch_type(const AdjustArgs& a, cudaStream_t stream, unsigned* err) {
  const auto aligned = [&](const void* p, long long stride) {
    return (uintptr_t)p % (4 * sizeof(T)) == 0 && (a.rows == 1 || stride % 4 == 0);
  };
  const bool vec = aligned(a.logits, a.stride) && aligned(a.out, a.out_stride);
  if ((long long)a.rows * a.n < kSmallBatch || !vec) {
    return launch(vec ? rows_adjust_slice_kernel<T, true> : rows_adjust_slice_kernel<T, false>,
                  dim3((unsigned)((a.n + kSmallSlice - 1) / kSmallSlice), (unsigned)a.rows), 256, 0, stream, a, err);
  }
  auto kernel = rows_adjust_stream_kernel<T>;
  static std::atomic<unsigned long long> done{0};
  int sms = 0;
  const cudaError_t e = kernel_setup(reinterpret_cast<const void*>(kernel), (2 * kBigSlice + 2 * kAdjustMaxBias) * 4, done, &sms);
  if (e != cudaSuccess) return e;
  const int slices = (a.n + kBigSlice - 1) / kBigSlice, len = ((a.n + slices - 1) / slices + 31) & ~31;
  const int items = a.rows * slices, ctas = items < sms ? items : sms;
  return launch(kernel, dim3((unsigned)ctas), kBoth, (2 * kBigSlice + 2 * ((a.n_bias + 3) & ~3)) * 4, stream, a, slices, len,
                items / ctas, items % ctas, err);
}

}  // namespace

cudaError_t launch_rows_adjust(const AdjustArgs& a, cudaStream_t stream) {
  unsigned* err = device_error_word();
  if (!err) return cudaErrorUnknown;
  return a.dtype == kDtF32 ? launch_type<float>(a, stream, err)
                           : a.dtype == kDtF16 ? launch_type<__half>(a, stream, err)
                                               : launch_type<__nv_bfloat16>(a, stream, err);
}

}  // namespace asmllm
