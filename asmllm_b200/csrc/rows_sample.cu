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
// bounds a small batch is the chain of cluster barriers.  A large one too, as
// far as the counters show: a third of the waiting warps wait at a barrier
// (one CTA of the cluster puts a border's words in order while the others
// hold their shared memory), instructions issue in 49 % of the cycles, and
// neither the 64-bit pipe (10 %) nor the shared-memory atomics (8 %) are
// busy.  No sort: words fall into bins of equal width in
// (m - x) / temperature, a scan over the bins finds the one that holds the
// border, and only that bin's words are put in order.  A small top_k takes
// the short way: the bins down to the border hold little more than top_k
// words, which one CTA finishes alone (four barriers in all).
//
// Measured on one B200: one row of 32000 words, top_k 40 and top_p 0.95, 9.1
// us; 128 rows of 128256 words with mixed settings 111 us (the read alone
// would take 10).  Radix selection straight from global memory, a CTA a row:
// 835 and 3231 us.  64-bit histogram atomics in place of three 32-bit ones
// and all CTAs reading all histograms: 39 and 374.
#include <cooperative_groups.h>

#include "matvec.cuh"
#include "pipeline.cuh"
#include "serving.cuh"

namespace asmllm {

namespace {

namespace cg = cooperative_groups;

typedef unsigned long long u64;
constexpr int kThreads = 512;
constexpr int kBins = 1024;   // bins of (m - x) / temperature, 1/32 wide; the last: weighs nothing
constexpr float kBinsPerUnit = 32.0f;
constexpr int kList = 1024;   // words that are put in order by comparing each with each
constexpr int kIndexBits = 18;
constexpr int kPart = 15;     // masses are added up in three parts of 15 bits (45 and the top word's one)
static_assert(kSampleMaxN <= 1 << kIndexBits, "the index fits the order word");
static_assert(kSampleMaxN / 8 <= 1 << 15, "a slice's sum of 16-bit parts fits 32 bits");

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

// (value, index) as one word, larger = earlier in the order.  Values are never NaN or -0 here.
__device__ __forceinline__ u64 order_word(float v, int index) {
  const unsigned u = __float_as_uint(v);
  return ((u64)((u & 0x80000000u) ? ~u : (u | 0x80000000u)) << kIndexBits) | (u64)((1 << kIndexBits) - 1 - index);
}
__device__ __forceinline__ float word_value(u64 w) {
  const unsigned k = (unsigned)(w >> kIndexBits);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}
__device__ __forceinline__ int word_index(u64 w) { return (1 << kIndexBits) - 1 - (int)(w & ((1u << kIndexBits) - 1)); }

struct Shared {
  unsigned hist[2][3][kBins];  // two in turn; counts use the first part alone
  u64 coarse[2][32];           // sums of 32 bins each
  u64 list[kList], mass[kList];
  u64 scan[kThreads / 32];
  u64 found[3];
  double pow2[64];
  u64 best;      // this CTA's first word
  u64 sum;       // this CTA's kept mass
  u64 cut;       // the border found by rank 0
  int count[3];  // words in the list of each selection (at most three in a call)
};

struct Row {
  float vtop;        // the largest logit
  float bin_scale;   // kBinsPerUnit / temperature
  double exp_scale;  // log2(e) / temperature
  const double* pow2;

  // Each step below is rounded as written.  The same word's bin, part of a bin and mass are computed at several
  // places, and a multiplication fused with an addition at one of them alone would give a sum that no word reaches.
  __device__ __forceinline__ float distance(float v) const { return __fmul_rn(__fsub_rn(vtop, v), bin_scale); }
  __device__ __forceinline__ int bin(float v) const {
    const float t = distance(v);
    return v == vtop ? 0 : t < (float)(kBins - 1) ? (int)t : kBins - 1;
  }
  // Which of kThreads parts of bin b.
  __device__ __forceinline__ int part(float v, int b) const {
    const float t = __fsub_rn(distance(v), (float)b);
    return v == vtop ? 0 : min(kThreads - 1, max(0, (int)__fmul_rn(t, (float)kThreads)));
  }
  // w = exp((x - m) / temperature) for a word that is not in the last bin.
  // Table-driven (Tang 1989): x = (64 k + j) / 64 + r in powers of two, |r| <= 1/128, 2^(j/64) from the
  // table and 2^r from its Taylor polynomial; the remainder r^6 ln(2)^6 / 720 is below 2^-54.
  __device__ __forceinline__ double weight(float v) const {
    if (v == vtop) return 1.0;
    const double y = __dmul_rn(__dsub_rn((double)v, (double)vtop), exp_scale);
    const double big = __dadd_rn(y, 105553116266496.0);  // 1.5 * 2^46: rounds to a multiple of 1/64
    const int n = __double2loint(big);
    const double z = __dmul_rn(__dsub_rn(y, __dsub_rn(big, 105553116266496.0)), 0.6931471805599453);
    double p = fma(z, 1.0 / 120.0, 1.0 / 24.0);
    p = fma(z, p, 1.0 / 6.0);
    p = fma(z, p, 0.5);
    p = fma(z, p, 1.0);
    p = fma(z, p, 1.0);
    const double t = pow2[n & 63];
    return __dmul_rn(__hiloint2double(__double2hiint(t) + (n >> 6) * 1048576, __double2loint(t)), p);
  }
  // w <= 1 as a multiple of 2^-45: adding 2^7 leaves 45 bits behind the point, rounded to nearest even
  __device__ __forceinline__ static u64 fixed(double w) {
    return (u64)__double_as_longlong(__dadd_rn(w, 128.0)) - 0x4060000000000000ull;
  }
  __device__ __forceinline__ u64 mass(float v) const { return bin(v) == kBins - 1 ? 0ull : fixed(weight(v)); }
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
  const float* val;
  int n, first;  // words first .. first + n - 1 of the row
  cg::cluster_group cluster;
  int ranks;
  Row row;
  float cut_v = -INFINITY;  // the words at or before (cut_v, cut_i) of the order are kept
  int cut_i = 1 << kIndexBits;
  int levels = 0;           // histograms used so far (two buffers in turn)
  int lists = 0;

  __device__ __forceinline__ bool keep(float v, int i) const { return v > cut_v || (v == cut_v && first + i <= cut_i); }

  // Empties the next histogram.  The other CTAs read this buffer two histograms ago and have met at a
  // cluster barrier since.
  template <bool MASS>
  __device__ __forceinline__ void clear() {
    unsigned* h = &sh.hist[levels & 1][0][0];
    for (int i = threadIdx.x; i < (MASS ? 3 : 1) * kBins; i += kThreads) h[i] = 0;
    __syncthreads();
  }
  template <bool MASS>
  __device__ __forceinline__ void add(int bin, float v) {
    unsigned* h = &sh.hist[levels & 1][0][bin];
    if (MASS) {
      const u64 m = Row::fixed(row.weight(v));
      atomicAdd(h, (unsigned)m & ((1u << kPart) - 1));
      atomicAdd(h + kBins, (unsigned)(m >> kPart) & ((1u << kPart) - 1));
      atomicAdd(h + 2 * kBins, (unsigned)(m >> (2 * kPart)));
    } else {
      atomicAdd(h, 1u);
    }
  }
  template <bool MASS>
  __device__ __forceinline__ static u64 read(const unsigned* h) {
    return MASS ? (u64)h[0] + ((u64)h[kBins] << kPart) + ((u64)h[2 * kBins] << (2 * kPart)) : (u64)h[0];
  }

  // Sums the histogram by 32 bins and meets the other CTAs.  Returns the total of the row.
  template <bool MASS>
  __device__ u64 publish() {
    __syncthreads();
    const unsigned* h = &sh.hist[levels & 1][0][0];
    u64 v = read<MASS>(h + 2 * threadIdx.x) + read<MASS>(h + 2 * threadIdx.x + 1);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    if ((threadIdx.x & 15) == 0) sh.coarse[levels & 1][threadIdx.x >> 4] = v;
    cluster.sync();
    if (threadIdx.x < 32) {
      u64 t = 0;
      for (int r = 0; r < ranks; ++r) t += cluster.map_shared_rank(&sh, r)->coarse[levels & 1][threadIdx.x];
      u64 x = t;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(kFull, x, o);
        if (threadIdx.x >= o) x += y;
      }
      sh.mass[threadIdx.x] = x;  // running sums over the row, for find (the list is idle)
    }
    __syncthreads();
    return sh.mass[31];
  }

  // The first bin at which the row's running sum reaches `want` (kBins: none) and the sum before it.
  template <bool MASS>
  __device__ int find(u64 want, u64* before) {
    static_assert(kBins == 1024, "32 sums of 32 bins");
    if (threadIdx.x < 32) {
      const unsigned lane = threadIdx.x;
      const unsigned hit = __ballot_sync(kFull, sh.mass[lane] >= want);
      int b = kBins;
      u64 run = 0;
      if (hit) {
        const int c = __ffs(hit) - 1;
        if (c) run = sh.mass[c - 1];
        u64 t = 0;
        for (int r = 0; r < ranks; ++r)
          t += read<MASS>(&cluster.map_shared_rank(&sh, r)->hist[levels & 1][0][32 * c + lane]);
        u64 x = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 y = __shfl_up_sync(kFull, x, o);
          if (lane >= o) x += y;
        }
        const int e = __ffs(__ballot_sync(kFull, run + x >= want)) - 1;
        b = 32 * c + e;
        run += __shfl_sync(kFull, x - t, e);
      }
      if (lane == 0) {
        sh.found[0] = (u64)b;
        sh.found[1] = run;
      }
    }
    ++levels;
    __syncthreads();
    const int b = (int)sh.found[0];
    *before = sh.found[1];
    return b;
  }

  // Appends a word to rank 0's list (words past its end are only counted).
  __device__ __forceinline__ void append(u64 w) {
    Shared* s0 = cluster.map_shared_rank(&sh, 0);
    const int i = atomicAdd(&s0->count[lists], 1);
    if (i < kList) s0->list[i] = w;
  }

  // Moves the border to the earliest word such that it and the kept words before it weigh at least
  // `want` (each 1, or its mass); the histogram of the kept words' bins is published.  No change if all
  // weigh less.
  template <bool MASS>
  __device__ void border(u64 want) {
    u64 before;
    const int b = find<MASS>(want, &before);
    if (b == kBins) return;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float v = val[i];
      if (row.bin(v) == b && keep(v, i)) append(order_word(v, first + i));
    }
    cluster.sync();
    const int c = cluster.map_shared_rank(&sh, 0)->count[lists];
    ++lists;
    u64 w = 0;
    if (c <= kList) {
      if (cluster.block_rank() == 0) {
        // The bin once more in kThreads parts (comparing each of its words with each took 10 thousand cycles
        // for 400 words); the words of the part that holds the border are then compared.
        u64* part = reinterpret_cast<u64*>(sh.hist);  // all CTAs are past the histograms
        u64* word = part + kThreads;                   // the words of the one part, and their masses
        u64* weighs = word + kList;
        static_assert((kThreads + 2 * kList) * sizeof(u64) <= sizeof(sh.hist), "room");
        part[threadIdx.x] = 0;
        if (threadIdx.x == 0) sh.found[2] = 0;
        __syncthreads();
        auto part_of = [&](u64 x) { return row.part(word_value(x), b); };
        for (int i = threadIdx.x; i < c; i += kThreads) {
          const u64 m = MASS ? row.mass(word_value(sh.list[i])) : 1ull;
          sh.mass[i] = m;
          atomicAdd(part + part_of(sh.list[i]), m);
        }
        __syncthreads();
        u64 all;
        const u64 mine = part[threadIdx.x], run = before + block_scan(mine, sh, &all) - mine;
        if (run < want && run + mine >= want) {
          sh.found[0] = threadIdx.x;
          sh.found[1] = run;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < c; i += kThreads)
          if (part_of(sh.list[i]) == (int)sh.found[0]) {
            const int at = (int)atomicAdd(&sh.found[2], 1ull);
            word[at] = sh.list[i];
            weighs[at] = sh.mass[i];
          }
        __syncthreads();
        const int few = (int)sh.found[2];
        for (int i = threadIdx.x; i < few; i += kThreads) {
          u64 s = sh.found[1];
          for (int j = 0; j < few; ++j)
            if (word[j] > word[i]) s += weighs[j];
          if (s < want && s + weighs[i] >= want) sh.cut = word[i];
        }
      }
      cluster.sync();
      w = cluster.map_shared_rank(&sh, 0)->cut;
    } else {  // too many words in one bin (equal logits): digit by digit of the order word, from the top
      for (int shift = 32 + kIndexBits - 10; shift >= 0; shift -= 10) {
        clear<MASS>();
        for (int i = threadIdx.x; i < n; i += kThreads) {
          const float v = val[i];
          if (row.bin(v) != b || !keep(v, i)) continue;
          const u64 x = order_word(v, first + i);
          if ((x >> (shift + 10)) == w) add<MASS>(1023 - (int)((x >> shift) & 1023u), v);
        }
        u64 over;
        publish<MASS>();
        const int d = find<MASS>(want - before, &over);
        before += over;
        w = (w << 10) | (u64)(1023 - d);
      }
    }
    cut_v = word_value(w);
    cut_i = word_index(w);
  }
};

template <class T>
__global__ void __launch_bounds__(kThreads, 2) rows_sample_kernel(const SampleArgs a, int per) {
  extern __shared__ __align__(16) unsigned char s_raw[];
  Shared& sh = *reinterpret_cast<Shared*>(s_raw);
  float* s_val = reinterpret_cast<float*>(s_raw + sizeof(Shared));
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int r = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31;
  const int first = min(a.n, rank * per), n = min(a.n, first + per) - first;
  if (tid < 64) sh.pow2[tid] = kPow2[tid];
  if (tid < 3) sh.count[tid] = 0;
  pdl_trigger();
  pdl_wait();
  const float temp = a.temperature ? __ldcg(a.temperature + r) : 1.0f;
  const int k = a.top_k ? __ldcg(a.top_k + r) : 0;
  const float tp = a.top_p ? __ldcg(a.top_p + r) : 1.0f, mp = a.min_p ? __ldcg(a.min_p + r) : 0.0f;
  const float u = __ldcg(a.u + r);

  // The slice (NaN as -inf: neither weighs anything; -0 as +0) and its first word.
  const T* row = static_cast<const T*>(a.logits) + (long long)r * a.stride + first;
  float bv = -INFINITY;
  int bi = 0;
  auto put = [&](int i, float v) -> float {  // a thread's indices rise, so > keeps its lowest one
    v = v == v ? v + 0.0f : -INFINITY;
    if (v > bv) {
      bv = v;
      bi = i;
    }
    return v;
  };
  int done = 0;
  if ((uintptr_t)row % 16 == 0) {
    constexpr int E = 16 / sizeof(T);
    done = n & ~(E - 1);
#pragma unroll 4
    for (int i = tid * E; i < done; i += kThreads * E) {
      const uint4 w = __ldcg(reinterpret_cast<const uint4*>(row + i));
      const T* p = reinterpret_cast<const T*>(&w);
      float v[E];
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = put(i + e, to_f32(p[e]));
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *reinterpret_cast<float4*>(s_val + i + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
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
    s_val[i] = put(i, v);
  }
  u64 best = bv > -INFINITY ? order_word(bv, first + bi) : 0ull;
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
    for (int o = 8; o > 0; o >>= 1) {
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
  if (best == 0 || !(temp > 0.0f)) {
    if (rank == 0 && tid == 0) a.tokens[r] = best == 0 ? -1 : word_index(best);
    cluster.sync();  // nobody leaves while its shared memory may be read
    return;
  }
  const float vtop = word_value(best);
  const int top = word_index(best);  // the first word, which always stays
  Slice s{sh, s_val, n, first, cluster, ranks, Row{vtop, kBinsPerUnit / temp, 1.4426950408889634 / (double)temp, sh.pow2}};
  const double least = (double)mp;
  u64 total;

  if (k > 0 && k < a.n) {
    auto counts = [&]() {
      s.template clear<false>();
#pragma unroll 4
      for (int i = tid; i < n; i += kThreads) {
        const int b = s.row.bin(s_val[i]);
        if (b < kBins - 1) s.template add<false>(b, 0.0f);
      }
      s.template publish<false>();
    };
    counts();
    if (k <= kList / 2) {
      // the short way: every word down to the border's bin, if they fit the list
      u64 before;
      int b = s.template find<false>((u64)k, &before);
      if (b == kBins) b = kBins - 2;  // fewer than top_k words weigh anything
#pragma unroll 4
      for (int i = tid; i < n; i += kThreads)
        if (s.row.bin(s_val[i]) <= b) s.append(order_word(s_val[i], first + i));
      cluster.sync();
      const int c = cluster.map_shared_rank(&sh, 0)->count[0];
      ++s.lists;
      if (c <= kList) {
        cluster.sync();
        if (rank != 0) return;
        u64 sum = 0;
        u64* rest = reinterpret_cast<u64*>(sh.hist);  // mass before each word (the histograms are done with)
        static_assert(sizeof(sh.hist) >= kList * sizeof(u64), "room");
        for (int i = tid; i < c; i += kThreads) sh.mass[i] = s.row.mass(word_value(sh.list[i]));
        __syncthreads();
        for (int i = tid; i < c; i += kThreads) {
          const u64 w = sh.list[i];
          int pos = 0;
          u64 m = 0;
#pragma unroll 4
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
                            (!(least > 0.0) || s.row.weight(word_value(sh.list[i])) >= least)));
          if (!keep) sh.mass[i] = 0;
          kept += sh.mass[i];
        }
        block_scan(kept, sh, &total);  // (its barriers also publish the masses)
        const double x = (double)u * (double)total;
        u64 target = x > 0.0 ? (u64)x : 0ull;
        if (target >= total) target = total - 1;
        for (int i = tid; i < c; i += kThreads) {
          if (sh.mass[i] == 0) continue;
          const int index = word_index(sh.list[i]);
          u64 cum = 0;
#pragma unroll 4
          for (int j = 0; j < c; ++j)
            if (word_index(sh.list[j]) <= index) cum += sh.mass[j];
          if (cum > target && cum - sh.mass[i] <= target) a.tokens[r] = index;
        }
        return;
      }
      counts();  // they do not fit: put the border's bin alone in order
    }
    s.template border<false>((u64)k);
  }
  if (tp < 1.0f) {
    s.template clear<true>();
#pragma unroll 2
    for (int i = tid; i < n; i += kThreads) {
      const float v = s_val[i];
      const int b = s.row.bin(v);
      if (b < kBins - 1 && s.keep(v, i)) s.template add<true>(b, v);
    }
    total = s.template publish<true>();
    const double lim = fmax((double)tp * (double)total, 0.0);
    s.template border<true>(max(1ull, (u64)ceil(lim)));  // the word that brings the sum to top_p is the last
  }

  // Mass of the kept words, in index order: a contiguous share per thread (an odd number of words, so
  // that the shares begin in different banks).
  const int share = ((n + kThreads - 1) / kThreads) | 1, i0 = min(n, tid * share), i1 = min(n, i0 + share);
  auto kept = [&](int i) -> u64 {
    const float v = s_val[i];
    if (!s.keep(v, i) || s.row.bin(v) == kBins - 1) return 0ull;
    const double w = s.row.weight(v);
    return first + i == top || !(least > 0.0) || w >= least ? Row::fixed(w) : 0ull;
  };
  u64 mine = 0;
#pragma unroll 2
  for (int i = i0; i < i1; ++i) mine += kept(i);
  u64 cta;
  const u64 upto = block_scan(mine, sh, &cta);
  if (tid == 0) sh.sum = cta;
  cluster.sync();
  u64 before = 0;
  total = 0;
  for (int q = 0; q < ranks; ++q) {
    const u64 t = cluster.map_shared_rank(&sh, q)->sum;
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
  static std::atomic<unsigned long long> done{0};
  int sms = 0;
  cudaError_t e = kernel_setup(reinterpret_cast<const void*>(kernel),
                               (int)(sizeof(Shared) + kSampleMaxN / 8 * sizeof(unsigned)), done, &sms);
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
