// asmllm_b200/csrc/attention_prompt.cu -- causal attention of whole prompts:
// packed query rows of sequences of different lengths, grouped heads, keys
// and values packed the same way or in the pages of a cache.
//
// Row t of sequence s sits at position p = n_s - (cu_q[s+1] - cu_q[s]) +
// (t - cu_q[s]), n_s the sequence's key count, and
//   out[t][h] = sum_{j <= p} softmax_j(scale q[t][h] . k[j][h / g]) v[j][h / g];
// p < 0: zeros.
//
// 4 head_dim flops per row, head and key: bound by the tensor cores, and next
// to them by the one exponential per row, head and key.  A work item is two
// 128-row query tiles that read the same keys: the same rows of two heads of
// a group (even groups), or 256 rows of one head.  Per 128 keys and query
// tile the tensor core computes S = Q K^T into tensor memory, one thread per
// row takes maximum, exponentials and sum, writes the weights P over S, and
// the tensor core adds P V to the output, which stays in tensor memory.  P is
// rounded once to 16 bits where the output is: it adds an error of about the
// output's own rounding.  For fp32 outputs it is two 16-bit parts (2^-22 of a
// weight in fp16, 2^-16 in bf16), which fill the columns of S, and the second
// product is done for both.  While one tile's weights are computed the tensor
// core works on the other's.  The output is rescaled only when a row's
// maximum has risen by more than 2^kLazy since it was last set (the weights
// then still fit 16 bits and the division by the sum cancels the factor).
//
// CTA (one per SM, persistent), 12 warps:
//   0-3, 4-7  softmax, rescale and output of query tile 0 and 1
//   8         tcgen05.mma issue, by one elected thread (behind lane == 0 each
//             product went through a loop over lanes: 400 cycles, not 100)
//   9         tensor copies: Q (2 tiles), then K and V tiles into one ring
//   10        scheduler: the work items in order of falling key count
//   11        zeroes the values behind a sequence's end
// Every wait is bounded: a role that gives up sets the device error word and
// an abort flag, all roles leave, and tensor memory is released.
//
// Measured on one B200: 8192 tokens on 32 heads of 128 values, bf16, 460 us =
// 1.19 PFLOP/s, 0.71 of the cuBLAS rate; 610 with an fp32 output (465 with
// weights of one rounding there too).  head_dim 64: 379 us and 444 with fp32.
// A step (128 keys, both query tiles) takes 3400 to 3500 cycles; the tensor core's
// part of it, alone, 2049, the exponentials' 2048 (both pipes are busy 60 % of
// the time).  The rest is one tile's chain -- scores, 1900 cycles of softmax,
// products -- which two tiles in turn do not cover.  Columns 64 to 127 of S
// are free from the softmax's read on with 16-bit outputs: the next scores of
// 64 keys could start there.  Not done.
#include <type_traits>

#include "matvec.cuh"
#include "mma16.cuh"
#include "pipeline.cuh"
#include "serving.cuh"
#include "tensor_map.cuh"
#include "tmem.cuh"

namespace asmllm {

namespace {

constexpr int kRows = 128;  // rows of a query tile, positions of a key tile
constexpr float kLazy = 6.0f;
constexpr float kPShift = 8.0f;  // weights are 2^kPShift exp(s - m): fp16 keeps those down to 2^-32 of the largest
constexpr int kThreads = 384;
// Items are dealt out by key tiles (and joined) where there may be fewer of them than SMs and one may have 16
// key tiles or more.  Lengths are on the device, so the rule goes by what the page table (or the packed rows) could
// hold.  Measured, one packed sequence, bf16, 128 values a head (us, by items / by key tiles; the rule's choice *):
//   keys   1 head        4            8            16           24           32           40
//   512    *14.9/17.4   *15.2/18.7   *15.2/19.3   *15.5/19.9   *15.7/20.5   *15.9/22.3   *16.2/22.3
//   1024   *21.5/21.2   *21.9/23.2   *22.3/25.5   *22.4/25.8   *23.3/28.0   *23.4/30.2   *23.7/35.0
//   2048   34.5/*31.0   34.9/*27.4   35.4/*29.1   36.9/*39.3   *37.4/51.3   *39.7/62.6   *51.0/74.4
//   4096   60.6/*36.3   61.4/*38.0   63.3/*55.6   *63.0/97.4   *98/139      *126/178     *159/225
//   8192   112/*41.7    116/*87.3    *116/156     *228/296     *342/456     *463/636     *585/795
// It loses at 2048 keys on 16 heads (2.4 us), and where a wide table holds short sequences: a table for 16384
// positions costs prompts of 1 to 128 rows 3.4 us on 8/1 and 32/32 heads (8.2 -> 11.6 at 33 rows of 32 heads), 512
// rows 3.2 and 6.4, and up to 40 MB of scratch.
constexpr int kSplitTiles = 16;

// A row whose output is not finite, computed again in fp32 key by key by one
// warp: in a matrix product a later position's infinite or NaN value meets
// the row's zero weight and turns its output to NaN, although the row does
// not attend to that position; so does an infinity that it attends to with a
// weight below the 16-bit type's smallest.  Lane l holds values l, l + 32, ...; those from
// 32 e0 to 32 e1 are written.
template <class T, class O, int HD>
__device__ __forceinline__ void attend_row(const PromptArgs& a, const KvArgs& kv, int t, int h, int s, int last, int lane,
                                           int e0, int e1) {
  constexpr int E = HD / 32;
  const T* q = static_cast<const T*>(a.q) + (long long)t * a.q_row_stride + (long long)h * a.q_head_stride;
  const long long ho = (long long)(h / (a.n_heads / kv.n_kv)) * kv.head_stride;
  float o[E] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll 1
  for (int j0 = 0; j0 <= last; j0 += 32) {  // a key per lane, then its value with all lanes
    const int j = j0 + lane;
    const long long off = j <= last ? kv_offset(kv, s, j) : -1;
    float x = 0.0f;
    if (off >= 0) {
#pragma unroll 2
      for (int c = 0; c < HD; c += 8) {
        float kk[8], qq[8];
        load8(static_cast<const T*>(kv.k) + off + ho + c, kk);
        load8(q + c, qq);
#pragma unroll
        for (int e = 0; e < 8; ++e) x = fmaf(qq[e], kk[e], x);
      }
    }
    x = j <= last ? x * (a.scale * 1.4426950408889634f) : -INFINITY;
    float mn = x;
#pragma unroll
    for (int e = 16; e > 0; e >>= 1) mn = fmaxf(mn, __shfl_xor_sync(kFull, mn, e));
    mn = fmaxf(mn, m);
    const float mz = mn == -INFINITY ? 0.0f : mn, f = ex2(m - mz), p = ex2(x - mz);
    m = mn;
    l = l * f + p;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= f;
#pragma unroll 4
    for (int i = 0; i < 32; ++i) {
      const float w = __shfl_sync(kFull, p, i);
      const long long at = __shfl_sync(kFull, off, i);
      if (at < 0) continue;
#pragma unroll
      for (int e = 0; e < E; ++e)
        o[e] = fmaf(w, to_f32(static_cast<const T*>(kv.v)[at + ho + lane + 32 * e]), o[e]);
    }
  }
  l = warp_sum(l);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  O* out = static_cast<O*>(a.out) + ((long long)t * a.n_heads + h) * HD;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (e < e0 || e >= e1) continue;
    const float v = o[e] * inv;
    if constexpr (sizeof(O) == 4) out[lane + 32 * e] = v;
    else {
      const uint32_t w = pack16<O>(v, 0.0f);
      reinterpret_cast<unsigned short*>(out)[lane + 32 * e] = (unsigned short)(w & 0xFFFFu);
    }
  }
}


// Transposes the 4 x 4 matrix of 16-byte pieces that four consecutive lanes hold (lane = row, w = columns).
__device__ __forceinline__ uint4 shfl_xor4(uint4 v, int mask) {
  return make_uint4(__shfl_xor_sync(kFull, v.x, mask), __shfl_xor_sync(kFull, v.y, mask),
                    __shfl_xor_sync(kFull, v.z, mask), __shfl_xor_sync(kFull, v.w, mask));
}
__device__ __forceinline__ void transpose4(uint4 (&w)[4], int lane) {
  const bool odd = lane & 1, high = lane & 2;
#pragma unroll
  for (int q = 0; q < 4; q += 2) {  // 2 x 2 blocks of neighbours
    const uint4 t = shfl_xor4(odd ? w[q] : w[q + 1], 1);
    if (odd) w[q] = t; else w[q + 1] = t;
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {  // and of pairs
    const uint4 t = shfl_xor4(high ? w[q] : w[q + 2], 2);
    if (high) w[q] = t; else w[q + 2] = t;
  }
}

// One work item, written by the scheduler.
struct Item {
  int s;       // sequence; -1: no more
  int t0;      // first query row
  int rows;    // query rows from t0 (at most 128 with two heads, 256 with one)
  int base;    // position of row t0
  int n;       // keys of the sequence
  int head;    // first query head
  int key0;    // packed: first key row of the sequence
  int tiles[2];  // key tiles of each query tile in this item, from key tile j0 on
  int j0;
  int slot;      // -1: the whole of it; else where this part of it goes
};

// The item that begins in a CTA's share and ends in a later one's, for the join.
struct Split {
  Item it;  // whole: j0 = 0, all key tiles; slot: of the first part (CTA c + p, p > 0, has slot 2 (c + p))
  int parts;  // 0: none
  int pad[3];
};
// A part: unnormalised outputs [2 query tiles][HD / 4][128 rows][4], then (maximum, sum) [2][128].
template <int HD>
__host__ __device__ constexpr size_t part_floats() {
  return (size_t)2 * kRows * HD + 4 * kRows;
}
__device__ __forceinline__ int cta_of(long long x, long long total, int ctas) {  // whose share holds x
  return (int)(((x + 1) * ctas - 1) / total);
}

// Whether values [32 e0, 32 e1) of positions [p, stop) hold an infinity, or (NAN_TOO) a NaN.  A position per lane.
template <class T, bool NAN_TOO>
__device__ __forceinline__ bool any_nonfinite(const KvArgs& kv, int s, long long ho, int p, int stop, int lane, int e0,
                                              int e1) {
#pragma unroll 1
  for (; p < stop; p += 32) {
    const long long off = p + lane < stop ? kv_offset(kv, s, p + lane) : -1;
    bool found = false;
    if (off >= 0) {
#pragma unroll 4
      for (int c = 32 * e0; c < 32 * e1; c += 8) {
        float v[8];
        load8(static_cast<const T*>(kv.v) + off + ho + c, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) found |= NAN_TOO ? !(fabsf(v[e]) < INFINITY) : fabsf(v[e]) == INFINITY;
      }
    }
    if (__any_sync(kFull, found)) return true;
  }
  return false;
}

// Rows `todo` of a warp's 32 (lane by lane) are not finite although their weights are: computed again if that may be
// the doing of a later position's value, or of an infinity whose weight a rounding made zero (NaN in place of it).
template <class T, class O, int HD>
__device__ __forceinline__ void mend_rows(const PromptArgs& a, const KvArgs& kv, const Item& it, int i, int pair, int tiles,
                                       int lrow, unsigned todo, int lane, int e0, int e1) {
  const int row = lrow + (pair ? 0 : i * kRows), head = it.head + (pair ? i : 0);
  const int first = max(0, __shfl_sync(kFull, it.base + row, __ffs(todo) - 1) + 1), last = min(it.n, tiles * kRows);
  const long long ho = (long long)(head / (a.n_heads / kv.n_kv)) * kv.head_stride;
  const bool later = any_nonfinite<T, true>(kv, it.s, ho, first, last, lane, e0, e1);
  if (!later && !any_nonfinite<T, false>(kv, it.s, ho, 0, min(first, it.n), lane, e0, e1)) return;
  __syncwarp();  // the rows' first stores come before the second ones
  while (todo) {
    const int rr = __shfl_sync(kFull, row, __ffs(todo) - 1);
    todo &= todo - 1;
    if (!later) {  // an infinity that came through is right
      const O* out = static_cast<const O*>(a.out) + ((long long)(it.t0 + rr) * a.n_heads + head) * HD + lane;
      bool nan = false;
      for (int e = e0; e < e1; ++e) {
        const float v = to_f32(out[32 * e]);
        nan |= v != v;
      }
      if (!__any_sync(kFull, nan)) continue;
    }
    attend_row<T, O, HD>(a, kv, it.t0 + rr, head, it.s, min(it.base + rr, it.n - 1), lane, e0, e1);
  }
}

template <int HD>
struct Cfg {
  static constexpr int kTile = kRows * HD * 2;  // bytes of a Q, K or V tile
  static constexpr int kStages = HD == 128 ? 5 : 8;
  static constexpr int kRing = 2 * kTile;
  static constexpr int kBars = kRing + kStages * kTile;
  static constexpr int kNBars = 2 * kStages + 4 + 10 + 4 + 3;
  static constexpr int kItems = kBars + kNBars * 8 + 24;
  static constexpr int kSmem = kItems + 2 * (int)sizeof(Item) + 16 + 1024;
  static constexpr uint32_t kO = 2 * kRows;  // tensor memory: S0, S1, then the two outputs
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

// Operand descriptors, 128-byte swizzle: the low word is the address and the
// leading offset, the high word the rest.  Q and K: rows of 128 bytes (64
// values along the product's K), eight rows 1024 bytes apart.  V: the product
// runs over its rows, eight of them 1024 bytes apart; 64 values are
// contiguous, the next 64 a half tile away (the leading offset).
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);
constexpr uint32_t kLeading = ((kRows * 128) >> 4) << 16;
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr) { return ((addr >> 4) & 0x3FFFu) | kLeading; }
__device__ __forceinline__ uint64_t desc64(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}

// Tiles of sequence (base, q rows, R rows a tile) with at least w key tiles.
__device__ __forceinline__ int tiles_at_least(int base, int q, int R, int w) {
  const int n = (q + R - 1) / R;
  if (w <= 0) return n;
  const int x = kRows * (w - 1) - base;  // a tile counts when its last row + 1 is above x
  if (q <= x) return 0;
  return n - (x < 0 ? 0 : min(x / R, n - 1));
}

// SPLIT: few items, dealt out by key tiles (an instantiation of its own keeps the code small).
template <class T, class O, int HD, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
attention_prompt_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                        const __grid_constant__ CUtensorMap vmap, const PromptArgs a, const KvArgs kv, int pair,
                        int box_rows, float* __restrict__ parts, Split* __restrict__ splits,
                        unsigned* __restrict__ err) {
  using C = Cfg<HD>;
  constexpr int kHalves = HD / 64, S = C::kStages;
  constexpr bool kTwo = sizeof(O) == 4;  // weights in two 16-bit parts: columns 0-63 and 64-127 of the scores
  constexpr uint32_t kFmt = std::is_same<T, __half>::value ? 0u : 1u;
  constexpr uint32_t kIdescS = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((kRows >> 3) << 17) | ((kRows >> 4) << 24);
  constexpr uint32_t kIdescO =
      (1u << 4) | (kFmt << 7) | (kFmt << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((kRows >> 4) << 24);
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBars);
  uint64_t* kv_full = bars;
  uint64_t* kv_empty = kv_full + S;
  uint64_t* q_full = kv_empty + S;  // [2]
  uint64_t* q_empty = q_full + 2;   // [2]
  uint64_t* s_full = q_empty + 2;   // [2] scores of a tile are in tensor memory
  uint64_t* p_full = s_full + 2;    // [2][2] the weights of its first and second 64 keys are
  uint64_t* o_full = p_full + 4;    // [2] the item's output is complete
  uint64_t* o_empty = o_full + 2;   // [2] and has been read
  uint64_t* i_full = o_empty + 2;   // [2] work items
  uint64_t* i_empty = i_full + 2;
  uint64_t* v_clean = i_empty + 2;  // an item's last value tile is zero behind the sequence's end
  uint64_t* v_dirty = v_clean + 1;  // the tile that needs it has landed
  uint64_t* drain = v_dirty + 1;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(drain + 1);
  volatile uint32_t* s_abort = s_tmem + 1;
  uint32_t* s_mending = s_tmem + 2;  // warps that compute rows again: the others' waits go on meanwhile
  Item* items = reinterpret_cast<Item*>(smem + C::kItems);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    prefetch_map(&qmap);
    prefetch_map(&kmap);
    prefetch_map(&vmap);
    for (int i = 0; i < S; ++i) {
      mbar_init(smem_u32(kv_full + i), 1);
      mbar_init(smem_u32(kv_empty + i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(q_full + i), 1);
      mbar_init(smem_u32(q_empty + i), 1);
      mbar_init(smem_u32(s_full + i), 1);
      mbar_init(smem_u32(p_full + 2 * i), 4);
      mbar_init(smem_u32(p_full + 2 * i + 1), 4);
      mbar_init(smem_u32(o_full + i), 1);
      mbar_init(smem_u32(o_empty + i), 4);
      mbar_init(smem_u32(i_full + i), 1);
      mbar_init(smem_u32(i_empty + i), 11);  // 8 softmax warps, the issuer, the loader, the cleaner
    }
    mbar_init(smem_u32(v_clean), 1);
    mbar_init(smem_u32(v_dirty), 1);
    mbar_init(smem_u32(drain), 1);
    *s_abort = 0u;
    *s_mending = 0u;
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  pdl_trigger();
  pdl_wait();

  auto fail = [&]() {
    *s_abort = 1u;
    atomicOr(err, kErrRingTimeout);
  };
  // Rows computed again for a non-finite later value may keep a role for longer than the bound.
  auto patient = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (mbar_try_wait(smem_u32(bar), parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try_wait(smem_u32(bar), parity)) {
      const long long t = clock64() - t0;
      if (t > kWaitCycles && (*static_cast<volatile uint32_t*>(s_mending) == 0u || t > 60 * kWaitCycles)) return false;
    }
    return true;
  };
  // Warp-wide wait; false (in every lane) when the role has to leave.
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (__all_sync(kFull, mbar_try_wait(smem_u32(bar), parity))) return true;
    const bool ok = patient(bar, parity);
    if (!ok) fail();
    return !__any_sync(kFull, !ok || *s_abort);
  };
  // Work item k; false when there is none left.
  auto take_item = [&](int k, Item* it) -> bool {
    if (!wait(i_full + (k & 1), (k >> 1) & 1)) return false;
    *it = items[k & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(i_empty + (k & 1)));
    return it->s >= 0;
  };
  const int R = pair ? kRows : 2 * kRows, units = pair ? a.n_heads / 2 : a.n_heads;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 10) {
      // ---------------- scheduler ----------------
      // Many items: numbered by falling key-tile count, heads fastest; CTA b takes numbers b, 2G-1-b, 2G+b, ...
      // Few items: the key tiles of all of them in a row are cut into equal shares, one a CTA, and an item that
      // lies in several shares is joined afterwards.
      constexpr int kHeld = 4;  // sequences per lane kept in registers
      int hq[kHeld], hb[kHeld], hr[kHeld];
      bool any_clipped = false;
      auto load = [&](int s, int* q, int* b) -> int {  // query rows, position of the first, its row
        int qb, qe;
        bool clipped;
        any_clipped |= !q_range(a.cu_q, s, a.rows, &qb, &qe);
        const int n = kv_length(kv, s, &clipped);
        any_clipped |= clipped;
        *q = qe - qb;
        *b = n - (qe - qb);
        return qb;
      };
#pragma unroll
      for (int e = 0; e < kHeld; ++e) {
        hq[e] = hb[e] = hr[e] = 0;
        if (!SPLIT && lane + 32 * e < kv.batch) hr[e] = load(lane + 32 * e, hq + e, hb + e);
      }
      // sum over the sequences of f(q rows, base)
      auto total = [&](auto f) -> int {
        int x = 0;
#pragma unroll
        for (int e = 0; e < kHeld; ++e) x += f(hq[e], hb[e]);
#pragma unroll 1
        for (int s = lane + 32 * kHeld; s < kv.batch; s += 32) {
          int q, b;
          load(s, &q, &b);
          x += f(q, b);
        }
        return __reduce_add_sync(kFull, x);
      };
      // key tiles of the item of query rows [tile R, ...) of a sequence; the first i's own; at least 1 counted
      auto tiles_in = [&](int base, int rows, int i) -> int {
        const int r = pair ? rows : min(kRows, rows - i * kRows);
        const int stop = r <= 0 ? 0 : base + (pair ? 0 : i * kRows) + r;
        return stop <= 0 ? 0 : (stop + kRows - 1) / kRows;
      };
      if constexpr (SPLIT) {
        auto weight = [&](int q, int b, int tile) -> int {
          return max(1, (b + min((tile + 1) * R, q) + kRows - 1) / kRows);
        };
        auto weights = [&](int s) -> long long {  // of a sequence, all heads
          if (s >= kv.batch) return 0;
          int q, b;
          load(s, &q, &b);
          long long x = 0;
#pragma unroll 1
          for (int t = 0; t * R < q; ++t) x += weight(q, b, t);
          return x * units;
        };
        long long sum = 0;
#pragma unroll 1
        for (int s0 = 0; s0 < kv.batch; s0 += 32) {
          long long x = weights(s0 + lane);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(kFull, x, o);
          sum += x;
        }
        if (any_clipped && blockIdx.x == 0) atomicOr(err, kErrDecodeRange);
        const int cta = blockIdx.x, ctas = (int)min((long long)gridDim.x, sum);
        long long at = cta < ctas ? sum * cta / ctas : 0;
        const long long begin = at, end = cta < ctas ? sum * (cta + 1) / ctas : 0;
        int s = 0, q = 0, b = 0, tile = 0, unit = 0, t = 0;
        if (at < end) {
          long long before = 0;
#pragma unroll 1
          for (int s0 = 0;; s0 += 32) {  // the sequence that holds `begin`
            const long long w = weights(s0 + lane);
            long long x = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const long long y = __shfl_up_sync(kFull, x, o);
              if (lane >= o) x += y;
            }
            const unsigned hit = __ballot_sync(kFull, begin < before + x);
            if (hit) {
              s = s0 + __ffs(hit) - 1;
              before += __shfl_sync(kFull, x - w, __ffs(hit) - 1);
              break;
            }
            before += __shfl_sync(kFull, x, 31);
          }
          load(s, &q, &b);
          long long left = begin - before;
          for (; left >= (long long)weight(q, b, tile) * units; ++tile) left -= (long long)weight(q, b, tile) * units;
          unit = (int)(left / weight(q, b, tile));
          t = (int)(left % weight(q, b, tile));
        }
        Split mine;
        mine.parts = 0;
        for (int k = 0;; ++k) {
          if (k >= 2 && !wait(i_empty + (k & 1), ((k >> 1) - 1) & 1)) break;
          Item it;
          it.s = -1;
          if (at < end) {
            const int w = weight(q, b, tile), t1 = (int)min((long long)w, t + (end - at));
            int qb, qe;
            q_range(a.cu_q, s, a.rows, &qb, &qe);
            it.s = s;
            it.t0 = qb + tile * R;
            it.rows = min(R, q - tile * R);
            it.base = b + tile * R;
            it.n = q + b;
            it.head = pair ? 2 * unit : unit;
            it.key0 = kv.table ? 0 : __ldcg(kv.cu + s);
            const int f0 = tiles_in(it.base, it.rows, 0), f1 = tiles_in(it.base, it.rows, 1);
            it.j0 = t;
            it.slot = t == 0 && t1 == w ? -1 : 2 * cta + (at == begin ? 0 : 1);
            it.tiles[0] = max(0, min(f0, t1) - t);
            it.tiles[1] = max(0, min(f1, t1) - t);
            if (t == 0 && t1 < w) {
              mine.it = it;
              mine.it.tiles[0] = f0;
              mine.it.tiles[1] = f1;
              mine.parts = cta_of(at + w - 1, sum, ctas) - cta + 1;
            }
            at += t1 - t;
            t = 0;
            if (++unit == units) {
              unit = 0;
              if (++tile * R >= q && at < end) {
                tile = 0;
                do load(++s, &q, &b); while (q == 0);
              }
            }
          }
          if (lane == 0) {
            items[k & 1] = it;
            mbar_arrive(smem_u32(i_full + (k & 1)));
          }
          __syncwarp();
          if (it.s < 0) break;
        }
        if (lane == 0) splits[cta] = mine;
      } else {
      int top = 0;
#pragma unroll
      for (int e = 0; e < kHeld; ++e) top = max(top, hq[e] > 0 ? hq[e] + hb[e] : 0);
#pragma unroll 1
      for (int s = lane + 32 * kHeld; s < kv.batch; s += 32) {
        int q, b;
        load(s, &q, &b);
        top = max(top, q > 0 ? q + b : 0);
      }
      top = (__reduce_max_sync(kFull, top) + kRows - 1) / kRows;  // most key tiles of any item
      if (any_clipped && blockIdx.x == 0) atomicOr(err, kErrDecodeRange);
      const int tiles = total([&](int q, int) { return (q + R - 1) / R; });
      const long long count = (long long)tiles * units;
      // A CTA's ranks rise, so it goes on where its last item was: among tiles with `level` key tiles, the first of
      // sequences `next` .. has rank `from`, and rank `upto` has fewer key tiles.  (From the start again for every
      // item, a call's time grew with the square of the number of sequences: 1024 prompts of up to 100 tokens on
      // 32 heads took 4957 us, now 570; 32768 of them take 18 ms.)
      int level = top + 1, upto = 0, from = 0, next = 0;
      for (int k = 0;; ++k) {
        const long long G = gridDim.x, at = k * G + ((k & 1) ? G - 1 - blockIdx.x : blockIdx.x);
        if (k >= 2 && !wait(i_empty + (k & 1), ((k >> 1) - 1) & 1)) break;
        Item it;
        it.s = -1;
        if (at < count) {
          const int rank = (int)(at / units), unit = (int)(at % units);
          if (rank >= upto) {  // the largest w with more than `rank` tiles of at least w key tiles
            int lo = 0, hi = level - 1, most = tiles;  // tiles of at least lo key tiles; `upto`: of more than hi
            for (int step = 1; lo < hi; step *= 2) {   // from the top: most often the next level
              const int w = max((lo + hi + 1) >> 1, hi + 1 - step), x = total([&](int q, int b) { return tiles_at_least(b, q, R, w); });
              if (x > rank) {
                lo = w;
                most = x;
              } else {
                hi = w - 1;
                upto = x;
              }
            }
            level = lo;
            from = upto;
            upto = most;
            next = 0;
          }
          // which of the tiles with exactly `level` key tiles: true in every lane once it is among these sequences
          auto pick = [&](int s0, int q, int b, int r) -> bool {
            const int c1 = tiles_at_least(b, q, R, level), c = c1 - tiles_at_least(b, q, R, level + 1);
            int x = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const int y = __shfl_up_sync(kFull, x, o);
              if (lane >= o) x += y;
            }
            const int left = rank - from;
            const unsigned hit = __ballot_sync(kFull, left < x);
            if (!hit) {
              from += __shfl_sync(kFull, x, 31);
              next = s0 + 32;
              return false;
            }
            const int src = __ffs(hit) - 1, tile = (q + R - 1) / R - c1 + (left - (x - c));
            it.s = s0 + src;
            it.rows = __shfl_sync(kFull, min(R, q - tile * R), src);
            it.base = __shfl_sync(kFull, b + tile * R, src);
            it.n = __shfl_sync(kFull, q + b, src);
            it.t0 = __shfl_sync(kFull, r + tile * R, src);
            return true;
          };
          bool found = false;
#pragma unroll
          for (int e = 0; e < kHeld; ++e)
            if (!found && 32 * e >= next && 32 * e < kv.batch) found = pick(32 * e, hq[e], hb[e], hr[e]);
#pragma unroll 1
          for (int s0 = max(next, 32 * kHeld); !found && s0 < kv.batch; s0 += 32) {
            int q = 0, b = 0, r = 0;
            if (s0 + lane < kv.batch) r = load(s0 + lane, &q, &b);
            found = pick(s0, q, b, r);
          }
          it.head = pair ? 2 * unit : unit;
          it.key0 = kv.table || !found ? 0 : __ldcg(kv.cu + it.s);
          it.j0 = 0;
          it.slot = -1;
          it.tiles[0] = tiles_in(it.base, it.rows, 0);
          it.tiles[1] = tiles_in(it.base, it.rows, 1);
        }
        if (lane == 0) {
          items[k & 1] = it;
          mbar_arrive(smem_u32(i_full + (k & 1)));
        }
        __syncwarp();
        if (it.s < 0) break;
      }
      }
    } else if (warp == 9) {
      // ---------------- loader ----------------
      const int pages = kv.table ? kRows / box_rows : 1;
      const int my_page = lane / kHalves, half = lane % kHalves;
      const uint32_t box_bytes = (uint32_t)box_rows * 128u;
      const int g = a.n_heads / kv.n_kv;
      int c = 0, nq[2] = {0, 0};
      Item it;
      bool ok = true;
      for (int k = 0; ok && take_item(k, &it); ++k) {
        const int nm = max(it.tiles[0], it.tiles[1]);
        if (nm == 0) continue;
        for (int i = 0; i < 2 && ok; ++i) {
          if (it.tiles[i] == 0) continue;
          if (nq[i] > 0 && !(ok = wait(q_empty + i, (nq[i] - 1) & 1))) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(smem_u32(q_full + i), C::kTile);
            for (int h = 0; h < kHalves; ++h)
              tma_load_4d(smem_u32(smem) + i * C::kTile + h * (kRows * 128), &qmap, h * 64,
                          it.t0 + (pair ? 0 : i * kRows), it.head + (pair ? i : 0), 0, smem_u32(q_full + i));
          }
          __syncwarp();
          ++nq[i];
        }
        const int head = it.head / g;
        // page of this lane's box in key tile j: -1 nothing to read, n_pages reads as zeros
        auto lookup = [&](int j) -> int {
          const int p = (it.j0 + j) * kRows + my_page * box_rows;
          if (my_page >= pages) return -1;
          if (!kv.table) return 0;
          if (j >= nm || p >= it.n) return -1;
          const int page = __ldcg(kv.table + (long long)it.s * kv.table_stride + (p >> kv.page_shift));
          if ((unsigned)page < (unsigned)kv.n_pages) return page;
          atomicOr(err, kErrDecodeRange);
          return kv.n_pages;
        };
        int page = lookup(0);
        for (int j = 0; j < nm && ok; ++j) {
          const int cur = page;
          page = j + 1 < nm ? lookup(j + 1) : -1;
          const unsigned live = __ballot_sync(kFull, cur >= 0);
          const int p = (it.j0 + j) * kRows + my_page * box_rows;
          const int row = kv.table ? p & (kv.page_size - 1) : it.key0 + p;
          for (int v = 0; v < 2; ++v, ++c) {
            const int st = c % S;
            if (c >= S && !(ok = wait(kv_empty + st, ((c / S) - 1) & 1))) break;
            const uint32_t bar = smem_u32(kv_full + st);
            if (lane == 0) mbar_arrive_expect_tx(bar, box_bytes * __popc(live));
            __syncwarp();
            if (cur >= 0)
              tma_load_4d(smem_u32(smem) + C::kRing + st * C::kTile + half * (kRows * 128) + my_page * box_bytes,
                          v ? &vmap : &kmap, half * 64, row, head, cur, bar);
          }
        }
      }
      // what was issued lands before the CTA may end (bounded)
      for (int i = 0; i < 2; ++i)
        if (nq[i] > 0) mbar_wait_bounded(smem_u32(q_full + i), (nq[i] - 1) & 1);
      for (int j = c - S < 0 ? 0 : c - S; j < c; ++j) mbar_wait_bounded(smem_u32(kv_full + j % S), (j / S) & 1);
    } else if (warp == 11) {
      // ---------------- cleaner: zeroes the values behind a sequence's end ----------------
      // (zero weights meet zeros there, whatever the page or the next sequence holds)
      int c = 0, nd = 0;
      Item it;
      for (int k = 0; take_item(k, &it); ++k) {
        const int nm = max(it.tiles[0], it.tiles[1]), valid = it.n - (it.j0 + nm - 1) * kRows;
        c += 2 * nm;
        if (nm == 0 || valid >= kRows) continue;
        const int sv = (c - 1) % S;  // the item's last value tile
        if (!wait(v_dirty, nd & 1)) break;  // the issuer has seen the tile land
        ++nd;
        for (int h = 0; h < kHalves; ++h)
          for (int b = valid * 128 + lane * 16; b < kRows * 128; b += 512)
            *reinterpret_cast<uint4*>(smem + C::kRing + sv * C::kTile + h * (kRows * 128) + b) =
                make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(v_clean));
      }
    } else if (elect_one()) {
      // ---------------- matrix products (one thread) ----------------
      const uint32_t q_lo = desc_lo(smem_u32(smem)), ring_lo = desc_lo(smem_u32(smem) + C::kRing);
      constexpr uint32_t kTileLo = C::kTile >> 4;
      int st = 0, nc = 0, k = 0;
      uint32_t nq = 0, np = 0, no = 3;  // parities, one bit a tile (nobody has to empty the first outputs)
      uint32_t ph = 0;  // ring stage and its parity
      bool ok = true, issued = false;
      auto get = [&](uint64_t* bar, uint32_t parity) { return ok = ok && patient(bar, parity); };
      bool ended = false;
      // The next item with keys; false when there is none.  While products of the last item are outstanding
      // (`ahead`) also where the very next item has no keys: the softmax warps come to that one, and make room for
      // those behind it, only once they have these products.
      auto next_item = [&](Item* it, bool ahead) -> bool {
        for (;;) {
          if (!get(i_full + (k & 1), (k >> 1) & 1)) return false;
          *it = items[k & 1];
          mbar_arrive(smem_u32(i_empty + (k & 1)));
          ++k;
          if (it->s < 0) {
            ended = true;
            return false;
          }
          if (max(it->tiles[0], it->tiles[1]) > 0) return true;
          if (ahead) return false;
        }
      };
      // S_i = Q_i K^T for key tile j of an item, its keys in ring stage st
      auto scores = [&](int i, const Item& it, int j) {
        const int tiles = i ? it.tiles[1] : it.tiles[0];
        if (j >= tiles) return;
        if (j == 0) {
          if (!get(q_full + i, nq >> i & 1)) return;
          nq ^= 1u << i;
        }
        if (!get(kv_full + st, ph)) return;
        const uint32_t ql = q_lo + i * kTileLo, kl = ring_lo + st * kTileLo;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          const uint32_t off = (ks >> 2) * ((kRows * 128) >> 4) + (ks & 3) * 2;
          umma_ss(tmem + i * kRows, desc64(ql + off, kDescHi), desc64(kl + off, kDescHi), kIdescS, ks > 0);
        }
        umma_commit(smem_u32(s_full + i));
        if (j == tiles - 1) umma_commit(smem_u32(q_empty + i));
        issued = true;
      };
      auto release = [&]() {
        umma_commit(smem_u32(kv_empty + st));
        if (++st == S) {
          st = 0;
          ph ^= 1;
        }
      };
      Item it, nx;
      bool live = next_item(&it, false);
      nx = it;
      // Step j of an item: values of its key tile j into the outputs, then the scores of the next key tile,
      // of this item or the next.  Step -1 has no values: the first item's first scores.
      for (int j = -1; live && ok;) {
        const int nm = max(it.tiles[0], it.tiles[1]), sv = st;
        const bool last = j == nm - 1;
        const uint32_t vl = ring_lo + sv * kTileLo;
        if (j >= 0) {  // this step's values are in stage st, the next step's keys behind them
          if (!get(kv_full + sv, ph)) break;
          if (last && it.n < (it.j0 + nm) * kRows) {
            mbar_arrive(smem_u32(v_dirty));
            if (!get(v_clean, nc++ & 1)) break;
          }
          if (++st == S) {
            st = 0;
            ph ^= 1;
          }
        }
        if (last) live = next_item(&nx, true);
        int jn = last ? 0 : j + 1;
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          if (j >= 0 && j < (i ? it.tiles[1] : it.tiles[0])) {
            if (j == 0) {  // the last item's output has been read (the first time: there is none)
              if (!get(o_empty + i, no >> i & 1)) break;
              no ^= 1u << i;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // the first 64 keys while the weights of the others are computed
              if (!get(p_full + 2 * i + h, np >> i & 1)) break;
              tc_fence_after();
#pragma unroll
              for (int ks = 4 * h; ks < 4 * h + 4; ++ks) {
                umma_ts(tmem + C::kO + i * HD, tmem + i * kRows + ks * 8, desc64(vl + ks * (2048 >> 4), kDescHi),
                        kIdescO, ks > 0 || j > 0);
                if constexpr (kTwo)
                  umma_ts(tmem + C::kO + i * HD, tmem + i * kRows + kRows / 2 + ks * 8,
                          desc64(vl + ks * (2048 >> 4), kDescHi), kIdescO, true);
              }
            }
            if (!ok) break;
            np ^= 1u << i;
            if (j == (i ? it.tiles[1] : it.tiles[0]) - 1) umma_commit(smem_u32(o_full + i));
          }
          if (j >= 0 && i == 1) umma_commit(smem_u32(kv_empty + sv));
          if (live) scores(i, nx, jn);
        }
        if (!ok) break;
        if (live) release();
        else if (!ended) {  // an item without keys was next: on from here, nothing outstanding
          live = next_item(&nx, false);
          jn = -1;
        }
        it = nx;
        j = jn;
      }
      if (!ok) fail();
      if (issued) {  // the tensor core is done before tensor memory is released
        umma_commit(smem_u32(drain));
        if (!mbar_wait_bounded(smem_u32(drain), 0)) fail();
      }
    }
  } else {
    // ---------------- softmax ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int i = warp >> 2, lrow = 32 * (warp & 3) + lane;
    const uint32_t ts = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + i * kRows;
    const uint32_t to = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + C::kO + i * HD;
    const float sl2 = a.scale * 1.4426950408889634f;
    int ns = 0, no = 0;
    Item it;
    for (int k = 0; take_item(k, &it); ++k) {
      const int row = lrow + (pair ? 0 : i * kRows), head = it.head + (pair ? i : 0), tiles = it.tiles[i];
      // A row of the tile that is not the item's is masked like the last one that is (its query is another sequence's,
      // or what lies behind them), and has no say in when the warp's rows are rescaled.
      const bool mine = row < it.rows;
      const int pos = it.base + min(row, it.rows - 1);
      float m = -INFINITY, l = 0.0f;
      bool ok = true;
      for (int j = 0; j < tiles; ++j) {
        if (!(ok = wait(s_full + i, ns & 1))) break;
        ++ns;
        tc_fence_after();
        uint32_t x[kRows];
#pragma unroll
        for (int b = 0; b < kRows; b += 32) tmem_ld<32>(ts + b, *reinterpret_cast<uint32_t(*)[32]>(x + b));
        tmem_wait_ld();
        const int limit = pos - (it.j0 + j) * kRows + 1;  // columns below it are attended to
        if (!__all_sync(kFull, limit >= kRows)) {
#pragma unroll
          for (int e = 0; e < kRows; ++e)
            if (e >= limit) x[e] = 0xFF800000u;
        }
        float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < kRows; e += 8)
#pragma unroll
          for (int q = 0; q < 4; ++q) t[q] = max3(t[q], __uint_as_float(x[e + 2 * q]), __uint_as_float(x[e + 2 * q + 1]));
        const float mt = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
        if (j == 0) {
          m = mt;
        } else if (__any_sync(kFull, mine && (mt - m) * sl2 > kLazy)) {  // false for a row that has no key yet
          const float mn = fmaxf(m, mt), f = m == -INFINITY ? 0.0f : ex2((m - mn) * sl2);
          m = mn;
          l *= f;
          const unsigned long long f2 = pack2(f, f);
#pragma unroll 1
          for (int b = 0; b < HD; b += 32) {
            uint32_t y[32];
            tmem_ld<32>(to + b, y);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float y0, y1;
              unpack2(mul2(pack2(__uint_as_float(y[e]), __uint_as_float(y[e + 1])), f2), y0, y1);
              y[e] = __float_as_uint(y0);
              y[e + 1] = __float_as_uint(y1);
            }
            tmem_st32(to + b, y);
          }
        }
        const float off = kPShift - (m == -INFINITY ? 0.0f : m * sl2);
        const unsigned long long sl22 = pack2(sl2, sl2), off2 = pack2(off, off);
        unsigned long long sum[2] = {0ull, 0ull};
#pragma unroll
        for (int b = 0; b < kRows; b += 64) {
          uint32_t w[32], w2[32];
#pragma unroll
          for (int e = 0; e < 64; e += 2) {
            float x0, x1;
            unpack2(fma2(pack2(__uint_as_float(x[b + e]), __uint_as_float(x[b + e + 1])), sl22, off2), x0, x1);
            x0 = ex2(x0);
            x1 = ex2(x1);
            sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], pack2(x0, x1));
            w[e >> 1] = pack16<T>(x0, x1);
            if constexpr (kTwo) {
              const float2 y = unpack16<T>(w[e >> 1]);
              w2[e >> 1] = pack16<T>(x0 - y.x, x1 - y.y);
            }
          }
          tmem_st32(ts + (b >> 1), w);
          if constexpr (kTwo) tmem_st32(ts + kRows / 2 + (b >> 1), w2);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(p_full + 2 * i + (b >> 6)));
        }
        float s0, s1;
        unpack2(add2(sum[0], sum[1]), s0, s1);
        l += s0 + s1;
      }
      if (!ok) break;
      if (SPLIT && it.slot >= 0) {  // a part of an item: as it is, for the join
        float* part = parts + (size_t)it.slot * part_floats<HD>();
        __stcg(reinterpret_cast<float2*>(part + (size_t)2 * kRows * HD) + i * kRows + lrow, make_float2(m, l));
        if (tiles == 0) continue;
        if (!wait(o_full + i, no & 1)) break;
        ++no;
        tc_fence_after();
        float4* o4 = reinterpret_cast<float4*>(part) + (size_t)i * kRows * (HD / 4) + lrow;
#pragma unroll 1
        for (int b = 0; b < HD; b += 32) {
          uint32_t y[32];
          tmem_ld<32>(to + b, y);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            __stcg(o4 + (size_t)((b + e) >> 2) * kRows, make_float4(__uint_as_float(y[e]), __uint_as_float(y[e + 1]),
                                                                   __uint_as_float(y[e + 2]), __uint_as_float(y[e + 3])));
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(o_empty + i));
        continue;
      }
      if (tiles == 0) {  // no key for any row of the tile
        if (mine) {
          O* out = static_cast<O*>(a.out) + ((long long)(it.t0 + row) * a.n_heads + head) * HD;
          const float z[8] = {};
#pragma unroll 1
          for (int b = 0; b < HD; b += 8) store8(out + b, z);
        }
        continue;
      }
      if (!wait(o_full + i, no & 1)) break;
      ++no;
      tc_fence_after();
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      bool bad = false;
      // A thread holds a row; its 16-byte pieces are exchanged within four lanes, so that a store writes 64
      // bytes of a row at a time (16 bytes a row kept the load-store unit busy for 5000 cycles an item).
      constexpr int kPer = 16 / sizeof(O);  // values of a piece
      O* out4 = static_cast<O*>(a.out) + ((long long)(it.t0 + (row & ~3)) * a.n_heads + head) * HD + (lane & 3) * kPer;
      const int rows4 = it.rows - (row & ~3);  // rows of the four lanes that exist
#pragma unroll 1
      for (int b = 0; b < HD; b += 32) {
        uint32_t y[32];
        tmem_ld<32>(to + b, y);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 4 * kPer) {
          uint4 w[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float v[kPer];
#pragma unroll
            for (int z = 0; z < kPer; ++z) {
              v[z] = __uint_as_float(y[e + q * kPer + z]) * inv;
              bad |= !(fabsf(v[z]) < INFINITY);
            }
            if constexpr (sizeof(O) == 4)
              w[q] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
            else
              w[q] = make_uint4(pack16<O>(v[0], v[1]), pack16<O>(v[2], v[3]), pack16<O>(v[4], v[5]), pack16<O>(v[6], v[7]));
          }
          transpose4(w, lane);  // now w[q] is piece lane % 4 of the four lanes' row q
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (q < rows4) *reinterpret_cast<uint4*>(out4 + (long long)q * a.n_heads * HD + b + e) = w[q];
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(o_empty + i));
      // Rows that are not finite: because of the values? (a NaN among the scores shows in the sum)
      const unsigned todo = __ballot_sync(kFull, bad && mine && l == l);
      if (todo) {
        if (lane == 0) atomicAdd(s_mending, 1u);
        mend_rows<T, O, HD>(a, kv, it, i, pair, tiles, lrow, todo, lane, 0, HD / 32);
        __syncwarp();
        if (lane == 0) atomicSub(s_mending, 1u);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// Joins the parts of the item that began in CTA blockIdx.x: query tile blockIdx.y, values 32 blockIdx.z ..,
// in part order.  Thread: a row and 16 of the values.
template <class T, class O, int HD>
__global__ void __launch_bounds__(256) attention_prompt_join_kernel(const PromptArgs a, const KvArgs kv, int pair,
                                                                    const float* __restrict__ parts,
                                                                    const Split* __restrict__ splits) {
  pdl_trigger();
  pdl_wait();
  const int c = blockIdx.x, i = blockIdx.y, z = blockIdx.z, lrow = threadIdx.x & (kRows - 1), half = threadIdx.x >> 7;
  const int n = __ldcg(&splits[c].parts);
  if (n == 0) return;
  const Item it = splits[c].it;
  const int row = lrow + (pair ? 0 : i * kRows), tiles = i ? it.tiles[1] : it.tiles[0];
  const float sl2 = a.scale * 1.4426950408889634f;
  float m = -INFINITY, l = 0.0f, o[16] = {};
  for (int p = 0; p < n; ++p) {
    const float* part = parts + (size_t)(p ? 2 * (c + p) : it.slot) * part_floats<HD>();
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(part + (size_t)2 * kRows * HD) + i * kRows + lrow);
    if (ml.x == -INFINITY && ml.y == 0.0f) continue;  // no key of this part for the row: there may be no output either
    const float mn = fmaxf(m, ml.x), f0 = m == -INFINITY ? 0.0f : ex2((m - mn) * sl2), f1 = ex2((ml.x - mn) * sl2);
    m = mn;
    l = l * f0 + ml.y * f1;
    const float4* o4 = reinterpret_cast<const float4*>(part) + (size_t)i * kRows * (HD / 4) + lrow;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 v = __ldcg(o4 + (size_t)(z * 8 + half * 4 + e) * kRows);
      o[4 * e] = o[4 * e] * f0 + v.x * f1;
      o[4 * e + 1] = o[4 * e + 1] * f0 + v.y * f1;
      o[4 * e + 2] = o[4 * e + 2] * f0 + v.z * f1;
      o[4 * e + 3] = o[4 * e + 3] * f0 + v.w * f1;
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const bool mine = row < it.rows;
  bool bad = false;
  O* out = static_cast<O*>(a.out) + ((long long)(it.t0 + row) * a.n_heads + it.head + (pair ? i : 0)) * HD + z * 32 + half * 16;
#pragma unroll
  for (int e = 0; e < 16; e += 8) {
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      v[q] = o[e + q] * inv;
      bad |= !(fabsf(v[q]) < INFINITY);
    }
    if (mine) store8(out + e, v);
  }
  // a row that is bad in either half is mended by the first (32 values from 32 z on)
  __shared__ unsigned s_bad[8];
  const unsigned vote = __ballot_sync(kFull, bad && mine && l == l);
  if ((threadIdx.x & 31) == 0) s_bad[threadIdx.x >> 5] = vote;
  __syncthreads();
  const int warp = threadIdx.x >> 5;
  const unsigned todo = warp < 4 ? s_bad[warp] | s_bad[warp + 4] : 0u;
  if (todo) mend_rows<T, O, HD>(a, kv, it, i, pair, tiles, lrow, todo, threadIdx.x & 31, z, z + 1);
}

template <class T, class O, int HD>
cudaError_t launch_typed(const PromptArgs& a, const KvArgs& kv, cudaStream_t stream, unsigned* err) {
  using C = Cfg<HD>;
  CUtensorMap qmap, kmap, vmap;
  const int box_rows = kv.table && kv.page_size < kRows ? kv.page_size : kRows;
  if (!encode_4d(&qmap, kv.dtype, a.q, HD, (uint64_t)a.rows, (uint64_t)a.n_heads, 1, (uint64_t)a.q_row_stride,
                 (uint64_t)a.q_head_stride, (uint64_t)a.q_row_stride, kRows) ||
      !encode_kv_map(&kmap, kv, kv.k, box_rows) || !encode_kv_map(&vmap, kv, kv.v, box_rows))
    return cudaErrorInvalidValue;
  static std::atomic<unsigned long long> done[2] = {};
  int sms = 0;
  cudaError_t e = kernel_setup(reinterpret_cast<const void*>(attention_prompt_kernel<T, O, HD, false>), C::kSmem, done[0], &sms);
  if (e == cudaSuccess)
    e = kernel_setup(reinterpret_cast<const void*>(attention_prompt_kernel<T, O, HD, true>), C::kSmem, done[1], &sms);
  if (e != cudaSuccess) return e;
  const int pair = (a.n_heads / kv.n_kv) % 2 == 0, R = pair ? kRows : 2 * kRows;
  const long long items = ((long long)a.rows / R + kv.batch) * (pair ? a.n_heads / 2 : a.n_heads);
  // Lengths are on the device; what is known here bounds the items and an item's key tiles.
  const long long most = ((kv.table ? (long long)kv.width * kv.page_size : kv.page_size) + kRows - 1) / kRows;
  const bool split = items < sms && most >= kSplitTiles;
  float* parts = nullptr;
  Split* splits = nullptr;
  if (split) {
    const size_t floats = (size_t)sms * 2 * part_floats<HD>();
    void* p = nullptr;
    if ((e = scratch_alloc_async(&p, floats * sizeof(float) + (size_t)sms * sizeof(Split), stream)) != cudaSuccess) return e;
    parts = static_cast<float*>(p);
    splits = reinterpret_cast<Split*>(parts + floats);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(split || items >= sms ? sms : items));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_opt_pdl.load() ? 1 : 0;
  if (!split) return cudaLaunchKernelEx(&cfg, attention_prompt_kernel<T, O, HD, false>, qmap, kmap, vmap, a, kv, pair,
                                        box_rows, parts, splits, err);
  e = cudaLaunchKernelEx(&cfg, attention_prompt_kernel<T, O, HD, true>, qmap, kmap, vmap, a, kv, pair, box_rows, parts,
                         splits, err);
  if (e == cudaSuccess) {
    cfg.gridDim = dim3((unsigned)sms, 2, HD / 32);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, attention_prompt_join_kernel<T, O, HD>, a, kv, pair, parts, splits);
  }
  const cudaError_t f = scratch_free_async(parts, stream);
  return e != cudaSuccess ? e : f;
}

template <class T>
cudaError_t launch_type(const PromptArgs& a, const KvArgs& kv, cudaStream_t stream, unsigned* err) {
  const bool f32 = a.out_dtype == kDtF32;
  if (kv.head_dim == 128)
    return f32 ? launch_typed<T, float, 128>(a, kv, stream, err) : launch_typed<T, T, 128>(a, kv, stream, err);
  return f32 ? launch_typed<T, float, 64>(a, kv, stream, err) : launch_typed<T, T, 64>(a, kv, stream, err);
}

}  // namespace

cudaError_t launch_attention_prompt(const PromptArgs& a, const KvArgs& kv, cudaStream_t stream) {
  unsigned* err = device_error_word();
  if (!err) return cudaErrorUnknown;
  return kv.dtype == kDtF16 ? launch_type<__half>(a, kv, stream, err)
                            : launch_type<__nv_bfloat16>(a, kv, stream, err);
}

}  // namespace asmllm
