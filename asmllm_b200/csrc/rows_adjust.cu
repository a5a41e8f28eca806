// asmllm_b200/csrc/rows_adjust.cu -- what is done to logits before a word is
// chosen: penalties for words that have come already, biases of some words,
// and a mask of the allowed ones.
//
// For word w of a row, seen `all` times among the row's tokens and c times
// among those behind its prompt, in fp32, each step rounded:
//   1. all > 0:  x = x > 0 ? x / repetition : x * repetition
//   2. c > 0:    x = (x - frequency * c) - presence
//   3. x = x + the sum of the word's biases (added up in 64 bits in their order)
//   4. not allowed: -inf
// and one rounding to the logits' type; other words are copied.
//
// Bound by HBM: logits are read and written once.  A CTA has a slice of a
// row's words and a counter for each in shared memory.  It asks for its logits
// first, counts the row's tokens that fall into the slice while they are on
// their way (integer atomics: their order does not matter), then changes and
// stores.  The few biased words are taken out of the stream: their logits are
// read before anything is stored, so that `out` may be the logits themselves,
// and stored last.
#include "matvec.cuh"
#include "serving_q8.cuh"

namespace asmllm {

namespace {

constexpr unsigned kSeen = 0x80000000u;  // in the prompt; the other bits count the tokens behind it

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
  float repetition, frequency, presence;
  __device__ __forceinline__ float operator()(float x, unsigned n) const {
    if (n == 0) return x;
    x = x > 0.0f ? __fdiv_rn(x, repetition) : __fmul_rn(x, repetition);
    const unsigned c = n & ~kSeen;
    return c ? __fsub_rn(__fsub_rn(x, __fmul_rn(frequency, (float)c)), presence) : x;
  }
};

// THREADS threads, PER groups of 4 words each.  VEC: rows whose groups are aligned.
template <class T, int THREADS, int PER, bool VEC>
__global__ void __launch_bounds__(THREADS) rows_adjust_kernel(const AdjustArgs a, unsigned* __restrict__ err) {
  constexpr int kSlice = THREADS * PER * 4;
  extern __shared__ __align__(16) unsigned s_count[];  // [kSlice], then the biased words [n_bias]
  int* s_word = reinterpret_cast<int*>(s_count + kSlice);
  pdl_trigger();
  const int tid = threadIdx.x, row = blockIdx.y, w0 = blockIdx.x * kSlice, n = min(kSlice, a.n - w0);
  for (int i = tid; i < kSlice / 4; i += THREADS) reinterpret_cast<uint4*>(s_count)[i] = make_uint4(0u, 0u, 0u, 0u);
  pdl_wait();
  const T* x = static_cast<const T*>(a.logits) + (long long)row * a.stride + w0;
  T* y = static_cast<T*>(a.out) + (long long)row * a.out_stride + w0;

  // this thread's words, group g: 4 (tid + g THREADS) ..
  float v[PER][4];
#pragma unroll
  for (int g = 0; g < PER; ++g) {
    const int i = 4 * (tid + g * THREADS);
    if (VEC && i + 4 <= n) {
      if constexpr (sizeof(T) == 4) {
        const float4 f = __ldcg(reinterpret_cast<const float4*>(x + i));
        v[g][0] = f.x; v[g][1] = f.y; v[g][2] = f.z; v[g][3] = f.w;
      } else {
        const uint2 f = __ldcg(reinterpret_cast<const uint2*>(x + i));
        const float2 lo = unpack16<T>(f.x), hi = unpack16<T>(f.y);
        v[g][0] = lo.x; v[g][1] = lo.y; v[g][2] = hi.x; v[g][3] = hi.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[g][e] = i + e < n ? load1(x + i + e) : 0.0f;
    }
  }
  Penalty p;
  p.repetition = a.repetition ? __ldcg(a.repetition + row) : 1.0f;
  p.frequency = a.frequency ? __ldcg(a.frequency + row) : 0.0f;
  p.presence = a.presence ? __ldcg(a.presence + row) : 0.0f;
  int held = 0, prompt = 0;
  if (a.tokens) {
    held = a.n_tokens ? __ldcg(a.n_tokens + row) : a.held;
    if (held < 0 || held > a.held) {
      if (tid == 0 && blockIdx.x == 0) atomicOr(err, kErrDecodeRange);
      held = held < 0 ? 0 : a.held;
    }
    prompt = a.n_prompt ? __ldcg(a.n_prompt + row) : 0;
  }
  for (int i = tid; i < a.n_bias; i += THREADS) s_word[i] = __ldcg(a.bias_tokens + (long long)row * a.n_bias + i) - w0;
  __syncthreads();  // counters are zero, the biased words are there
  const int32_t* tokens = a.tokens + (long long)row * a.token_stride;
  auto count = [&](int i, int token) {
    const unsigned w = (unsigned)token - (unsigned)w0;
    if (w < (unsigned)n) {
      if (i < prompt) atomicOr(s_count + w, kSeen);
      else atomicAdd(s_count + w, 1u);
    }
  };
  const bool wide = (reinterpret_cast<uintptr_t>(tokens) & 15u) == 0;
  const int first = wide ? held & ~3 : 0;
  for (int i = 4 * tid; i < first; i += 4 * THREADS) {
    const int4 t = __ldcg(reinterpret_cast<const int4*>(tokens + i));
    count(i, t.x);
    count(i + 1, t.y);
    count(i + 2, t.z);
    count(i + 3, t.w);
  }
  for (int i = first + tid; i < held; i += THREADS) count(i, __ldcg(tokens + i));
  __syncthreads();

  const int32_t* allowed = a.allowed + (long long)row * a.allowed_stride;
  auto is_allowed = [&](int w) -> bool {
    return !a.allowed || (__ldcg(allowed + ((w0 + w) >> 5)) >> ((w0 + w) & 31) & 1);
  };
  // biased words: the first of a word's entries finds its new logit
  constexpr int kOwn = (kAdjustMaxBias + THREADS - 1) / THREADS;
  float biased[kOwn];
  unsigned mine = 0u;
#pragma unroll
  for (int k = 0; k < kOwn; ++k) {
    const int i = tid + k * THREADS;
    if (i >= a.n_bias) break;
    const int w = s_word[i];
    if ((unsigned)w >= (unsigned)n) continue;
    bool before = false;
    for (int j = 0; j < i; ++j) before |= s_word[j] == w;
    if (before) continue;
    double sum = 0.0;
    for (int j = i; j < a.n_bias; ++j)
      if (s_word[j] == w) sum += (double)__ldcg(a.bias + (long long)row * a.n_bias + j);
    biased[k] = is_allowed(w) ? __fadd_rn(p(load1(x + w), s_count[w]), (float)sum) : -INFINITY;
    mine |= 1u << k;
  }
  if (a.n_bias) __syncthreads();  // every biased word's logit has been read

#pragma unroll
  for (int g = 0; g < PER; ++g) {
    const int i = 4 * (tid + g * THREADS);
    if (i >= n) break;
    const uint4 c = *reinterpret_cast<const uint4*>(s_count + i);
    v[g][0] = p(v[g][0], c.x);
    v[g][1] = p(v[g][1], c.y);
    v[g][2] = p(v[g][2], c.z);
    v[g][3] = p(v[g][3], c.w);
    if (a.allowed) {  // four words from a multiple of 4 on: bits of one word of the mask
      const unsigned m = (unsigned)__ldcg(allowed + ((w0 + i) >> 5)) >> ((w0 + i) & 31);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!(m >> e & 1u)) v[g][e] = -INFINITY;
    }
    if (VEC && i + 4 <= n) {
      if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(y + i) = make_float4(v[g][0], v[g][1], v[g][2], v[g][3]);
      else *reinterpret_cast<uint2*>(y + i) = make_uint2(pack16<T>(v[g][0], v[g][1]), pack16<T>(v[g][2], v[g][3]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < n) store1(y + i + e, v[g][e]);
    }
  }
  if (a.n_bias) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kOwn; ++k)
      if (mine >> k & 1u) store1(y + s_word[tid + k * THREADS], biased[k]);
  }
}

template <class T, int THREADS, int PER, bool VEC>
cudaError_t launch_typed(const AdjustArgs& a, cudaStream_t stream, unsigned* err) {
  constexpr int kSlice = THREADS * PER * 4;
  constexpr int kSmem = (kSlice + kAdjustMaxBias) * 4;
  auto kernel = rows_adjust_kernel<T, THREADS, PER, VEC>;
  static std::atomic<unsigned long long> done{0};
  int sms = 0;
  const cudaError_t e = kernel_setup(reinterpret_cast<const void*>(kernel), kSmem, done, &sms);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.n + kSlice - 1) / kSlice), (unsigned)a.rows);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = (size_t)(kSlice + a.n_bias) * 4;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_opt_pdl.load() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, a, err);
}

template <class T>
cudaError_t launch_type(const AdjustArgs& a, cudaStream_t stream, unsigned* err) {
  const auto aligned = [&](const void* p, long long stride) {
    return (uintptr_t)p % (4 * sizeof(T)) == 0 && (a.rows == 1 || stride % 4 == 0);
  };
  const bool vec = aligned(a.logits, a.stride) && aligned(a.out, a.out_stride);
  // Slices of 16384 words (every CTA of a row counts all its tokens) where they fill the GPU, else of 2048.
  const bool large = (long long)a.rows * ((a.n + 16383) / 16384) >= 296;
  if (large)
    return vec ? launch_typed<T, 512, 8, true>(a, stream, err) : launch_typed<T, 512, 8, false>(a, stream, err);
  return vec ? launch_typed<T, 256, 2, true>(a, stream, err) : launch_typed<T, 256, 2, false>(a, stream, err);
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
