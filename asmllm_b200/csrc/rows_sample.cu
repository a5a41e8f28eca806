// asmllm_b200/csrc/rows_sample.cu -- the next token of each row of logits
// from one given random number per row, with temperature, top-k, top-p and
// min-p.
//
// The words of a row are ordered by (logit descending, index ascending); NaN
// comes last and is never chosen.  With m the largest logit and
// w_i = exp((x_i - m) / temperature):
//   1. top_k > 0 keeps the first top_k words of the order;
//   2. of those, top_p keeps each word whose predecessors' mass is below
//      top_p times the mass of the words kept so far (the first word always);
//   3. min_p keeps the words with w_i >= min_p (the first word always);
//   4. the token is the first kept word, in index order, whose cumulative
//      mass exceeds u times the kept mass.
// temperature <= 0 (or NaN) takes the first maximum; a row without a finite
// or +inf logit gives -1.
//
// A border between two words is decided by sums over the whole row, so the
// masses are fixed-point integers: w_i is computed in 64 bits and rounded to
// a multiple of 2^-45 (a row of 2^18 words sums below 2^63).  Integer sums do
// not depend on their order, so atomics and any split of the row give the
// same token.
#include "matvec.cuh"
#include "pipeline.cuh"
#include "serving.cuh"

namespace asmllm {

namespace {

constexpr int kThreads = 1024;
typedef unsigned long long u64;

// Order of logits as unsigned integers; 0 for NaN, so every number is above it.
__device__ __forceinline__ unsigned order_key(float v) {
  const unsigned u = __float_as_uint(v == 0.0f ? 0.0f : v);  // -0 and +0 are one value
  return v == v ? ((u & 0x80000000u) ? ~u : (u | 0x80000000u)) : 0u;
}
__device__ __forceinline__ float key_value(unsigned k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

__device__ __forceinline__ u64 mass(unsigned key, unsigned top, float value_top, double inv_t) {
  if (key == top) return 1ull << 45;
  if (key == 0u) return 0ull;
  const double d = ((double)key_value(key) - (double)value_top) * inv_t;
  if (!(d > -32.0)) return 0ull;  // below half a unit: e^-32 < 2^-46 (and -inf, and NaN from -inf * 0)
  return __double2ull_rn(exp(d) * 35184372088832.0);
}

template <class V>
__device__ __forceinline__ V block_sum(V v, V* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  V r = 0;
  for (int i = 0; i < kThreads / 32; ++i) r += red[i];
  return r;
}

// The cut of the order at a total: the largest key t such that the words
// above t weigh less than `want` (weight 1 or mass), and their weight.
template <bool MASS, class L>
__device__ unsigned cut_key(L key_at, int n, unsigned top, float vtop, double inv_t, u64 want, u64* hist, u64* above) {
  unsigned prefix = 0;
  u64 over = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) hist[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const unsigned k = key_at(i);
      if (shift < 24 && (k >> (shift + 8)) != prefix) continue;
      const u64 w = MASS ? mass(k, top, vtop, inv_t) : 1ull;
      if (w) atomicAdd(hist + ((k >> shift) & 255u), w);
    }
    __syncthreads();
    int b = 255;
    u64 sum = over;
    for (; b > 0 && sum + hist[b] < want; --b) sum += hist[b];
    over = sum;
    prefix = (prefix << 8) | (unsigned)b;
  }
  *above = over;
  return prefix;
}

template <class T>
__global__ void __launch_bounds__(kThreads) rows_sample_kernel(const SampleArgs a) {
  __shared__ u64 hist[256];
  __shared__ u64 red[kThreads / 32];
  __shared__ u64 s_best;
  pdl_trigger();
  pdl_wait();
  const int r = blockIdx.x, tid = threadIdx.x, n = a.n;
  const T* row = static_cast<const T*>(a.logits) + (long long)r * a.stride;
  auto key_at = [&](int i) { return order_key(to_f32(row[i])); };
  const float temp = a.temperature ? __ldcg(a.temperature + r) : 1.0f;
  const int k = a.top_k ? __ldcg(a.top_k + r) : 0;
  const float tp = a.top_p ? __ldcg(a.top_p + r) : 1.0f, mp = a.min_p ? __ldcg(a.min_p + r) : 0.0f;
  const float u = __ldcg(a.u + r);

  if (tid == 0) s_best = 0;
  __syncthreads();
  u64 best = 0;
  for (int i = tid; i < n; i += kThreads) {
    const unsigned key = key_at(i);
    const u64 b = ((u64)key << 32) | (0xFFFFFFFFu - (unsigned)i);
    if (key) best = b > best ? b : best;
  }
  atomicMax(&s_best, best);
  __syncthreads();
  best = s_best;
  const unsigned top = (unsigned)(best >> 32);
  const float vtop = key_value(top);
  if (best == 0 || vtop == -INFINITY || !(temp > 0.0f)) {
    if (tid == 0) a.tokens[r] = best == 0 || vtop == -INFINITY ? -1 : (int)(0xFFFFFFFFu - (unsigned)best);
    return;
  }
  const double inv_t = 1.0 / (double)temp;

  // the cut: keys above `cut` are kept, and the first `ties` words that equal it
  unsigned cut = 0;
  u64 ties = 0, above = 0;
  bool limited = false;
  if (k > 0 && k < n) {
    cut = cut_key<false>(key_at, n, top, vtop, inv_t, (u64)k, hist, &above);
    ties = (u64)k - above;
    limited = true;
  }
  if (tp < 1.0f) {
    u64 w = 0;  // mass of the words kept so far
    for (int i = tid; i < n; i += kThreads) {
      const unsigned key = key_at(i);
      if (!limited || key > cut) w += mass(key, top, vtop, inv_t);
    }
    w = block_sum(w, red);
    if (limited) w += ties * mass(cut, top, vtop, inv_t);
    double lim = (double)tp * (double)w;  // predecessors weigh less than this
    if (!(lim > 0.0)) lim = 0.0;
    const u64 want = max(1ull, (u64)ceil(lim));
    u64 wa;
    const unsigned c = cut_key<true>(key_at, n, top, vtop, inv_t, want, hist, &wa);
    const u64 one = mass(c, top, vtop, inv_t);
    const u64 t = (want - wa + one - 1) / max(1ull, one);  // words equal to c whose predecessors weigh < want
    if (!limited || c > cut) {
      cut = c;
      ties = max(1ull, t);
    } else if (c == cut) {
      ties = min(ties, max(1ull, t));
    }
    limited = true;
  }
  const double least = (double)mp;
  // kept mass per thread's contiguous share of the row, then the crossing
  const int per = (n + kThreads - 1) / kThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
  u64 eq = 0;
  for (int i = i0; i < i1; ++i) eq += key_at(i) == cut;
  // exclusive count of ties before this thread
  __shared__ u64 scan[kThreads];
  scan[tid] = eq;
  __syncthreads();
  for (int o = 1; o < kThreads; o <<= 1) {
    const u64 v = tid >= o ? scan[tid - o] : 0;
    __syncthreads();
    scan[tid] += v;
    __syncthreads();
  }
  const u64 eq0 = scan[tid] - eq;
  auto kept = [&](unsigned key, u64& e) -> u64 {
    if (limited) {
      if (key < cut) return 0;
      if (key == cut && e++ >= ties) return 0;
    }
    const u64 w = mass(key, top, vtop, inv_t);
    return key == top || !(least > 0.0) || (key && exp(((double)key_value(key) - (double)vtop) * inv_t) >= least) ? w : 0;
  };
  u64 e = eq0, w = 0;
  for (int i = i0; i < i1; ++i) w += kept(key_at(i), e);
  __syncthreads();
  scan[tid] = w;
  __syncthreads();
  for (int o = 1; o < kThreads; o <<= 1) {
    const u64 v = tid >= o ? scan[tid - o] : 0;
    __syncthreads();
    scan[tid] += v;
    __syncthreads();
  }
  const u64 total = scan[kThreads - 1];
  double x = (double)u * (double)total;
  u64 target = x > 0.0 ? (u64)x : 0ull;  // cumulative > u total  <=>  cumulative > floor(u total)
  if (target >= total) target = total - 1;
  u64 cum = scan[tid] - w;
  if (cum <= target && target < cum + w) {
    e = eq0;
    for (int i = i0; i < i1; ++i) {
      cum += kept(key_at(i), e);
      if (cum > target) {
        a.tokens[r] = i;
        break;
      }
    }
  }
}

}  // namespace

cudaError_t launch_rows_sample(const SampleArgs& a, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_opt_pdl.load() ? 1 : 0;
  if (a.dtype == kDtF32) return cudaLaunchKernelEx(&cfg, rows_sample_kernel<float>, a);
  if (a.dtype == kDtF16) return cudaLaunchKernelEx(&cfg, rows_sample_kernel<__half>, a);
  return cudaLaunchKernelEx(&cfg, rows_sample_kernel<__nv_bfloat16>, a);
}

}  // namespace asmllm
