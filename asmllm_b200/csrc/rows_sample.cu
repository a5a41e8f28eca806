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
// same token.  Words more than about e^-32 below the largest weigh nothing.
//
// A row is read once, into the shared memory of a cluster of up to 8 CTAs (a
// slice each); everything after is a few passes over shared memory, so what
// bounds a small batch is the chain of cluster barriers, and a large one the
// 64-bit exponentials.  No sort: words fall into bins of equal width in
// (m - x) / temperature, a scan over the bins finds the one that holds the
// border, and only that bin's words are put in order.  A small top_k takes
// the short way: the bins down to the border hold little more than top_k
// words, which one CTA finishes alone (three barriers in all).
#include <cooperative_groups.h>

#include "matvec.cuh"
#include "pipeline.cuh"
#include "serving.cuh"

namespace asmllm {

namespace {

namespace cg = cooperative_groups;

typedef unsigned long long u64;
constexpr int kThreads = 512;
constexpr int kBins = 2048;   // bins of (m - x) / temperature, 1/64 wide; the last: weighs nothing
constexpr float kBinsPerUnit = 64.0f;
constexpr int kList = 1024;   // words that are put in order by comparing each with each
constexpr int kIndexBits = 18;
static_assert(kSampleMaxN <= 1 << kIndexBits, "the index fits the order word");

__constant__ double kPow2[64] = {  // 2^(j / 64)
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951,
};

// Order of logits as unsigned integers; 0 for NaN, so every number is above it.
__device__ __forceinline__ unsigned order_key(float v) {
  const unsigned u = __float_as_uint(v == 0.0f ? 0.0f : v);  // -0 and +0 are one value
  return v == v ? ((u & 0x80000000u) ? ~u : (u | 0x80000000u)) : 0u;
}
__device__ __forceinline__ float key_value(unsigned k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}
// (key, index) as one word, larger = earlier in the order.
__device__ __forceinline__ u64 order_word(unsigned key, int index) {
  return ((u64)key << kIndexBits) | (u64)((1 << kIndexBits) - 1 - index);
}

struct Shared {
  u64 hist[2][kBins];
  u64 list[kList], mass[kList];
  u64 scan[kThreads / 32];
  u64 out[2], sum;
  double pow2[64];
  u64 best;      // this CTA's first word
  u64 cut;       // the border found by rank 0
  int count[3];  // words in the list of each selection (at most three in a call)
};

struct Row {
  unsigned top;      // key of the largest logit
  float vtop;
  float bin_scale;   // kBinsPerUnit / temperature
  double exp_scale;  // log2(e) / temperature
  const double* pow2;

  __device__ __forceinline__ int bin(unsigned key) const {
    if (key == top) return 0;
    const float t = (vtop - key_value(key)) * bin_scale;
    return key && t < (float)(kBins - 1) ? (int)t : kBins - 1;
  }
  // w = exp((x - m) / temperature) and its fixed-point mass, for a word that is not in the last bin.
  // Table-driven (Tang 1989): x = (64 k + j) / 64 + r in powers of two, |r| <= 1/128, 2^(j/64) from the
  // table and 2^r from its Taylor polynomial; the remainder r^6 ln(2)^6 / 720 is below 2^-54.
  __device__ __forceinline__ double weight(unsigned key) const {
    if (key == top) return 1.0;
    const double y = ((double)key_value(key) - (double)vtop) * exp_scale;
    const double big = y + 105553116266496.0;  // 1.5 * 2^46: rounds to a multiple of 1/64
    const int n = __double2loint(big);
    const double z = (y - (big - 105553116266496.0)) * 0.6931471805599453;
    double p = fma(z, 1.0 / 120.0, 1.0 / 24.0);
    p = fma(z, p, 1.0 / 6.0);
    p = fma(z, p, 0.5);
    p = fma(z, p, 1.0);
    p = fma(z, p, 1.0);
    const double t = pow2[n & 63];
    return __hiloint2double(__double2hiint(t) + (n >> 6) * 1048576, __double2loint(t)) * p;
  }
  __device__ __forceinline__ static u64 fixed(double w) { return __double2ull_rn(w * 35184372088832.0); }  // 2^45
  __device__ __forceinline__ u64 mass(unsigned key) const { return bin(key) == kBins - 1 ? 0ull : fixed(weight(key)); }
};

// Inclusive scan over the CTA; every thread also gets the total.
__device__ __forceinline__ u64 block_scan(u64 v, Shared& sh, u64* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(kFull, v, o);
    if (lane >= o) v += t;
  }
  __syncthreads();
  if (lane == 31) sh.scan[warp] = v;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) {
    const u64 t = sh.scan[i];
    if (i < warp) before += t;
    all += t;
  }
  *total = all;
  return v + before;
}

// One row's slice in a CTA of the cluster and the selections over the whole row.
struct Slice {
  Shared& sh;
  const unsigned* keys;
  int n, first;  // words first .. first + n - 1 of the row
  cg::cluster_group cluster;
  int ranks, rank;
  Row row;
  int levels = 0;  // histograms used so far (two buffers in turn)
  int lists = 0;

  __device__ __forceinline__ u64* clear(int bins) {
    // the other CTAs read this buffer two levels ago and have met at a cluster barrier since
    u64* h = sh.hist[levels & 1];
    for (int i = threadIdx.x; i < bins; i += kThreads) h[i] = 0;
    __syncthreads();
    return h;
  }

  // Adds the cluster's histograms and finds the first bin at which the running sum reaches `want`;
  // bins means "none".  *before: the sum up to that bin; *total: of all bins.
  template <int BINS>
  __device__ int find(u64 want, u64* before, u64* total) {
    constexpr int E = BINS / kThreads;
    cluster.sync();
    u64* h = sh.hist[levels & 1];
    ++levels;
    u64 v[E] = {};
    for (int r = 0; r < ranks; ++r) {
      const u64* p = cluster.map_shared_rank(h, r) + threadIdx.x * E;
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] += p[e];
    }
    u64 mine = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) mine += v[e];
    if (threadIdx.x == 0) sh.out[0] = (u64)BINS;
    u64 run = block_scan(mine, sh, total) - mine;
    if (run < want && run + mine >= want) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (run < want && run + v[e] >= want) {
          sh.out[0] = (u64)(threadIdx.x * E + e);
          sh.out[1] = run;
        }
        run += v[e];
      }
    }
    __syncthreads();
    const int b = (int)sh.out[0];
    *before = sh.out[1];
    __syncthreads();
    return b;
  }

  // Appends a word to rank 0's list (words past its end are only counted).
  __device__ __forceinline__ void append(u64 w) {
    Shared* s0 = cluster.map_shared_rank(&sh, 0);
    const int i = atomicAdd(&s0->count[lists], 1);
    if (i < kList) s0->list[i] = w;
  }

  // The border of the order at `want`: the earliest word such that it and the words before it (of those
  // at or above `from`) weigh at least `want`, each 1 or its mass.  0 if all together weigh less.
  template <bool MASS>
  __device__ u64 border(u64 from, u64 want, u64* total) {
    u64* h = clear(kBins);
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const unsigned key = keys[i];
      const int b = row.bin(key);
      if (b < kBins - 1 && order_word(key, first + i) >= from)
        atomicAdd(h + b, MASS ? Row::fixed(row.weight(key)) : 1ull);
    }
    return border_in(from, want, total, MASS);
  }

  __device__ u64 border_in(u64 from, u64 want, u64* total, bool by_mass) {
    u64 before;
    const int b = find<kBins>(want, &before, total);
    if (b == kBins) return 0;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const unsigned key = keys[i];
      const u64 w = order_word(key, first + i);
      if (row.bin(key) == b && w >= from) append(w);
    }
    cluster.sync();
    const int c = cluster.map_shared_rank(&sh, 0)->count[lists];
    ++lists;
    if (c <= kList) {
      if (rank == 0) {
        for (int i = threadIdx.x; i < c; i += kThreads)
          sh.mass[i] = by_mass ? row.mass((unsigned)(sh.list[i] >> kIndexBits)) : 1ull;
        __syncthreads();
        for (int i = threadIdx.x; i < c; i += kThreads) {
          const u64 w = sh.list[i];
          u64 s = before;
          for (int j = 0; j < c; ++j)
            if (sh.list[j] > w) s += sh.mass[j];
          if (s < want && s + sh.mass[i] >= want) sh.cut = w;
        }
      }
      cluster.sync();
      return cluster.map_shared_rank(&sh, 0)->cut;
    }
    // too many words in one bin (equal logits): digit by digit of the order word, from the top
    u64 prefix = 0;
    for (int shift = 32 + kIndexBits - 10; shift >= 0; shift -= 10) {
      u64* h = clear(1024);
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const unsigned key = keys[i];
        const u64 w = order_word(key, first + i);
        if (row.bin(key) == b && w >= from && (w >> (shift + 10)) == prefix)
          atomicAdd(h + (1023 - (int)((w >> shift) & 1023u)), by_mass ? Row::fixed(row.weight(key)) : 1ull);
      }
      u64 over, sum;
      const int d = find<1024>(want - before, &over, &sum);
      before += over;
      prefix = (prefix << 10) | (u64)(1023 - d);
    }
    return prefix;
  }
};

template <class T>
__global__ void __launch_bounds__(kThreads, 2) rows_sample_kernel(const SampleArgs a, int per) {
  extern __shared__ __align__(16) unsigned char s_raw[];
  Shared& sh = *reinterpret_cast<Shared*>(s_raw);
  unsigned* s_keys = reinterpret_cast<unsigned*>(s_raw + sizeof(Shared));
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int r = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31;
  const int first = min(a.n, rank * per), n = min(a.n, first + per) - first;
  if (tid < 64) sh.pow2[tid] = kPow2[tid];
  if (tid == 0) {
    sh.best = 0;
    sh.cut = 0;
    sh.count[0] = sh.count[1] = sh.count[2] = 0;
  }
  __syncthreads();
  pdl_trigger();
  pdl_wait();
  const float temp = a.temperature ? __ldcg(a.temperature + r) : 1.0f;
  const int k = a.top_k ? __ldcg(a.top_k + r) : 0;
  const float tp = a.top_p ? __ldcg(a.top_p + r) : 1.0f, mp = a.min_p ? __ldcg(a.min_p + r) : 0.0f;
  const float u = __ldcg(a.u + r);

  // the slice, as order keys, and its first word
  const T* row = static_cast<const T*>(a.logits) + (long long)r * a.stride + first;
  u64 best = 0;
  auto put = [&](int i, float v) {
    const unsigned key = order_key(v);
    s_keys[i] = key;
    const u64 w = key ? order_word(key, first + i) : 0ull;
    best = w > best ? w : best;
  };
  int done = 0;
  if ((uintptr_t)row % 16 == 0) {
    done = n & ~7;
#pragma unroll 4
    for (int i = tid * 8; i < done; i += kThreads * 8) {
      float v[8];
      load8(row + i, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) put(i + e, v[e]);
    }
  }
#pragma unroll 4
  for (int i = done + tid; i < n; i += kThreads) {
    float v;
    if constexpr (sizeof(T) == 4) v = __ldcg(reinterpret_cast<const float*>(row) + i);
    else {
      const unsigned short h = __ldcg(reinterpret_cast<const unsigned short*>(row) + i);
      v = to_f32(*reinterpret_cast<const T*>(&h));
    }
    put(i, v);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 t = __shfl_xor_sync(kFull, best, o);
    best = t > best ? t : best;
  }
  if (lane == 0) sh.scan[tid >> 5] = best;
  __syncthreads();
  if (tid < 32) {
    best = tid < kThreads / 32 ? sh.scan[tid] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 t = __shfl_xor_sync(kFull, best, o);
      best = t > best ? t : best;
    }
    if (tid == 0) sh.best = best;
  }
  cluster.sync();
  best = 0;
  for (int q = 0; q < ranks; ++q) {
    const u64 t = cluster.map_shared_rank(&sh, q)->best;
    best = t > best ? t : best;
  }
  const unsigned top = (unsigned)(best >> kIndexBits);
  const float vtop = key_value(top);
  const bool none = best == 0 || vtop == -INFINITY;
  if (none || !(temp > 0.0f)) {
    if (rank == 0 && tid == 0)
      a.tokens[r] = none ? -1 : (1 << kIndexBits) - 1 - (int)(best & ((1u << kIndexBits) - 1));
    cluster.sync();  // nobody leaves while its shared memory may be read
    return;
  }
  Slice s{sh, s_keys, n, first, cluster, ranks, rank,
          Row{top, vtop, kBinsPerUnit / temp, 1.4426950408889634 / (double)temp, sh.pow2}};
  const double least = (double)mp;
  const bool by_k = k > 0 && k < a.n;
  u64 from = 0, total;

  if (by_k) {
    u64* h = s.clear(kBins);
    for (int i = tid; i < n; i += kThreads) {
      const int b = s.row.bin(s_keys[i]);
      if (b < kBins - 1) atomicAdd(h + b, 1ull);
    }
    if (k <= kList / 2) {
      // the short way: every word down to the border's bin, if they fit the list
      u64 before;
      int b = s.find<kBins>((u64)k, &before, &total);
      if (b == kBins) b = kBins - 2;  // fewer than top_k words weigh anything
      for (int i = tid; i < n; i += kThreads)
        if (s.row.bin(s_keys[i]) <= b) s.append(order_word(s_keys[i], first + i));
      cluster.sync();
      const int c = cluster.map_shared_rank(&sh, 0)->count[0];
      ++s.lists;
      if (c <= kList) {
        cluster.sync();
        if (rank != 0) return;
        u64 sum = 0;
        u64* rest = sh.hist[0];  // mass of the words before each (the histograms are no longer needed)
        for (int i = tid; i < c; i += kThreads) sh.mass[i] = s.row.mass((unsigned)(sh.list[i] >> kIndexBits));
        __syncthreads();
        for (int i = tid; i < c; i += kThreads) {
          const u64 w = sh.list[i];
          int pos = 0;
          u64 m = 0;
          for (int j = 0; j < c; ++j)
            if (sh.list[j] > w) {
              ++pos;
              m += sh.mass[j];
            }
          rest[i] = pos < k ? m : ~0ull;
          if (pos < k) sum += sh.mass[i];
        }
        block_scan(sum, sh, &total);
        // predecessors below top_p of the mass
        const double lim = tp < 1.0f ? fmax((double)tp * (double)total, 0.0) : 2e19;
        u64 kept = 0;
        for (int i = tid; i < c; i += kThreads) {
          const bool keep = rest[i] != ~0ull && (rest[i] == 0 || ((double)rest[i] < lim &&
                            (!(least > 0.0) || s.row.weight((unsigned)(sh.list[i] >> kIndexBits)) >= least)));
          if (!keep) sh.mass[i] = 0;
          kept += sh.mass[i];
        }
        block_scan(kept, sh, &total);  // (its barriers also publish the masses)
        const double x = (double)u * (double)total;
        u64 target = x > 0.0 ? (u64)x : 0ull;
        if (target >= total) target = total - 1;
        for (int i = tid; i < c; i += kThreads) {
          if (sh.mass[i] == 0) continue;
          const u64 index = sh.list[i] & ((1u << kIndexBits) - 1);  // larger = lower index
          u64 cum = 0;
          for (int j = 0; j < c; ++j)
            if ((sh.list[j] & ((1u << kIndexBits) - 1)) >= index) cum += sh.mass[j];
          if (cum > target && cum - sh.mass[i] <= target) a.tokens[r] = (1 << kIndexBits) - 1 - (int)index;
        }
        return;
      }
      // they do not fit: order the border's bin alone, over a new histogram
      h = s.clear(kBins);
      for (int i = tid; i < n; i += kThreads) {
        const int q = s.row.bin(s_keys[i]);
        if (q < kBins - 1) atomicAdd(h + q, 1ull);
      }
    }
    from = s.border_in(0ull, (u64)k, &total, false);
  }
  if (tp < 1.0f) {
    // the mass of the words kept so far comes with the histogram, so it is found first with no border
    u64* h = s.clear(kBins);
    for (int i = tid; i < n; i += kThreads) {
      const unsigned key = s_keys[i];
      const int b = s.row.bin(key);
      if (b < kBins - 1 && order_word(key, first + i) >= from) atomicAdd(h + b, Row::fixed(s.row.weight(key)));
    }
    u64 part = 0;
    __syncthreads();
    for (int i = tid; i < kBins; i += kThreads) part += h[i];
    block_scan(part, sh, &part);
    if (tid == 0) sh.sum = part;
    cluster.sync();
    total = 0;
    for (int q = 0; q < ranks; ++q) total += cluster.map_shared_rank(&sh, q)->sum;
    const double lim = fmax((double)tp * (double)total, 0.0);
    const u64 want = max(1ull, (u64)ceil(lim));  // the first word whose predecessors and itself reach it is the last
    const u64 c = s.border_in(from, want, &total, true);
    from = c > from ? c : from;
  }

  // mass of the kept words, in index order: a contiguous share per thread (an odd number of words, so
  // that the shares begin in different banks)
  const int share = ((n + kThreads - 1) / kThreads) | 1, i0 = min(n, tid * share), i1 = min(n, i0 + share);
  auto kept = [&](int i) -> u64 {
    const unsigned key = s_keys[i];
    if (s.row.bin(key) == kBins - 1 || order_word(key, first + i) < from) return 0ull;
    const double w = s.row.weight(key);
    return key == top || !(least > 0.0) || w >= least ? Row::fixed(w) : 0ull;
  };
  u64 mine = 0;
  for (int i = i0; i < i1; ++i) mine += kept(i);
  u64 cta;
  const u64 upto = block_scan(mine, sh, &cta);
  if (tid == 0) sh.best = cta;
  cluster.sync();
  u64 before = 0;
  total = 0;
  for (int q = 0; q < ranks; ++q) {
    const u64 t = cluster.map_shared_rank(&sh, q)->best;
    if (q < rank) before += t;
    total += t;
  }
  const double x = (double)u * (double)total;
  u64 target = x > 0.0 ? (u64)x : 0ull;  // cumulative > u total  <=>  cumulative > floor(u total)
  if (target >= total) target = total - 1;
  u64 cum = before + upto - mine;
  if (cum <= target && target < cum + mine) {
    for (int i = i0; i < i1; ++i) {
      cum += kept(i);
      if (cum > target) {
        a.tokens[r] = first + i;
        break;
      }
    }
  }
  cluster.sync();  // nobody leaves while its shared memory may be read
}

template <class T>
cudaError_t launch_typed(const SampleArgs& a, cudaStream_t stream) {
  auto kernel = rows_sample_kernel<T>;
  // CTAs of a row: at least about 2048 words each
  const int ranks = a.n <= 4096 ? 1 : a.n <= 8192 ? 2 : a.n <= 16384 ? 4 : 8;
  const int per = ((a.n + ranks - 1) / ranks + 7) & ~7;
  const size_t smem = sizeof(Shared) + (size_t)per * sizeof(unsigned);
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)sizeof(Shared) + kSampleMaxN / 8 * (int)sizeof(unsigned));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows * (unsigned)ranks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_opt_pdl.load() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a, per);
}

}  // namespace

cudaError_t launch_rows_sample(const SampleArgs& a, cudaStream_t stream) {
  if (a.dtype == kDtF32) return launch_typed<float>(a, stream);
  if (a.dtype == kDtF16) return launch_typed<__half>(a, stream);
  return launch_typed<__nv_bfloat16>(a, stream);
}

}  // namespace asmllm
