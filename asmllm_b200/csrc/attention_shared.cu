// asmllm_b200/csrc/attention_shared.cu -- attention of one new token per
// sequence over a paged cache in which groups of sequences begin with the same
// pages, read once for the whole group.
//
// The result is that of attention_paged.cu: softmax is split at the end of
// the shared positions, and the two sides are joined by their maxima and sums.
//   1. Shared pass (here): a group's query rows, (sequences x heads of a KV
//      head), against its shared positions: a matrix product of up to 256 rows
//      a key tile on the 5th-generation tensor cores.
//   2. Own pass (attention_own.cu): every sequence's positions behind those.
//      It does not wait for the first, and runs on the SMs that has left.
//   3. Join: a row's parts, in order.
//
// Shared pass.  A unit is (group, KV head, 256 rows); its positions are tiles,
// and the tiles of all units in a row are cut into one equal range per CTA,
// one CTA an SM.  Two streams of four warps take maximum, exponentials and
// sum, one thread a row: with more than 128 rows the streams have 128 rows
// each and the same keys, with fewer the same rows and every other key tile.
//   16-bit output: tiles of 128 positions.  Weights are rounded once to 16
//     bits and written over the scores; the output adds up in tensor memory and
//     is rescaled only when a row's maximum has risen by more than 2^kLazy.
//   fp32 output: tiles of 64.  Weights are two 16-bit parts (2^-22 of a weight
//     in fp16, 2^-16 in bf16), in columns of their own, so that the next tile's
//     scores are computed as soon as this one's have been read; the output adds
//     up in registers.  (In tensor memory, which truncates its sums, 16384
//     positions came out 1e-5 too small; added up in memory after every 16
//     tiles of 128, 5e-6 and a third slower.)
//
// CTA, 12 warps: 0-3 and 4-7 the streams (they also bring their queries into
// shared memory), 8 tcgen05.mma issue by one elected thread (for an fp32 output
// 8 and 10, a stream each), 9 tensor copies of K and V tiles into a ring (a page
// behind the shared ones reads as zeros).  One thread that issues for both
// streams in turn keeps them half a tile apart: with a thread each they ran in
// step, waiting for the exponentials and for the tensor core at the same time.
// Every wait is bounded, as in attention_prompt.cu.
//
// Measured on one B200, 256 sequences of 64 query and 8 KV heads of 128 values
// in bf16 that share 32768 positions and have up to 1023 of their own: 350 us
// (410 under the power cap), of which this pass takes 257 (1.07 PFLOP/s; matrix
// products alone would take 165, exponentials 119), the own pass 105 and the
// join 16.  With fp32 outputs 600 to 650: twice the products of the weights,
// and every 64 positions the 128 sums of a row are added up in registers, which
// do not hold them beside 64 scores and 64 weights (690 bytes are spilled, 300
// for 16-bit outputs).  The shared
// pass took 276 with two issuing threads and 296 with tiles of 64 positions.
// Three groups of 48 sequences, 32 heads, fp32 outputs: 71 us.  8 sequences of
// 8 heads that share 1024 positions: 12 us.  Giving this pass fewer SMs, so
// that the own pass runs beside it, gained 5 % in the first of these and lost
// up to 25 % elsewhere: a few SMs do not read the own positions fast enough.
#include <type_traits>

#include "matvec.cuh"
#include "mma16.cuh"
#include "pipeline.cuh"
#include "shared_prefix.cuh"
#include "serving_q8.cuh"
#include "tensor_map.cuh"
#include "tmem.cuh"

namespace asmllm {

namespace {

constexpr int kRows = 128;        // rows of a stream
constexpr int kUnit = 2 * kRows;  // rows of a unit
constexpr float kLazy = 6.0f;
constexpr float kPShift = 8.0f;  // weights are 2^kPShift exp(s - m)
constexpr int kThreads = 384;
constexpr int kMaxCtas = 160;

// Where the shared pass leaves its results, unnormalised: whole units by row, twice (the streams of a unit of up to
// 128 rows have a result each), parts in slots of kUnit rows.
struct SharedParts {
  float* o;       // [2][batch][n_heads][head_dim]
  float2* ml;     // [2][batch][n_heads]: (maximum in units of log2, sum); o 2^maximum is the sum of exp(s) v
  float* slots;   // [kMaxCtas][2] of kUnit x head_dim, then kUnit (maximum, sum)
  Found* found;   // [n_kv][found_stride]: unit_index()
  int found_stride;
};
template <int HD>
__host__ __device__ constexpr size_t part_floats() { return (size_t)kUnit * HD + 2 * kUnit; }
// Units of a KV head are numbered so that no two groups meet: rows before them / kUnit + groups before them.
__device__ __forceinline__ int unit_index(int first_row, int group, int blk) { return first_row / kUnit + group + blk; }

template <bool TWO, int HD>
struct Cfg {
  static constexpr int kKeys = TWO ? 64 : 128;  // positions of a key tile
  static constexpr int kQBytes = kRows * HD * 2;
  static constexpr int kTileBytes = kKeys * HD * 2;
  static constexpr int kStages = (HD == 128 ? 160 : 128) * 1024 / kTileBytes;
  static constexpr int kRing = 2 * kQBytes;
  static constexpr int kBars = kRing + kStages * kTileBytes;
  static constexpr int kNBars = 2 * kStages + 7 * 2;
  static constexpr int kSum = kBars + kNBars * 8 + 16;
  static constexpr int kSmem = kSum + 64 + 1024;
  // tensor memory: the streams' scores, weights (over the scores where the output has 16 bits), outputs
  static constexpr uint32_t kP = TWO ? 128 : 0, kO = 256;
  // Operand descriptors, 128-byte swizzle (as in attention_prompt.cu): V's leading offset, a half tile.
  static constexpr uint32_t kLeading = ((kKeys * 128) >> 4) << 16;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t leading) { return ((addr >> 4) & 0x3FFFu) | leading; }
__device__ __forceinline__ uint64_t desc64(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}

// Exchange of 16-byte pieces within four lanes (lane = row, w = columns of a 4 x 4 matrix): its transpose.
__device__ __forceinline__ float4 shfl_xor4(float4 v, int mask) {
  return make_float4(__shfl_xor_sync(kFull, v.x, mask), __shfl_xor_sync(kFull, v.y, mask),
                     __shfl_xor_sync(kFull, v.z, mask), __shfl_xor_sync(kFull, v.w, mask));
}
__device__ __forceinline__ void transpose4(float4 (&w)[4], int lane) {
  const bool odd = lane & 1, high = lane & 2;
#pragma unroll
  for (int q = 0; q < 4; q += 2) {
    const float4 t = shfl_xor4(odd ? w[q] : w[q + 1], 1);
    if (odd) w[q] = t; else w[q + 1] = t;
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const float4 t = shfl_xor4(high ? w[q] : w[q + 2], 2);
    if (high) w[q] = t; else w[q + 2] = t;
  }
}

// A CTA's walk: group, unit (KV head, block of rows), key tile.
struct Tour {
  int grp, b, rows, shared;  // the group, its first sequence, its query rows of a KV head, its positions
  int nb, nt, u, t;          // blocks a KV head, key tiles, unit of the group, tile of the unit
  long long first, at, end;  // number of the unit's first tile; tiles [at, end) are left
};

struct Segment {
  int head, blk, t0, n, rows;  // KV head, block, first tile, tiles, rows of the block
  bool two, whole;             // streams of different rows; nothing of the unit is in another CTA
};
__device__ __forceinline__ Segment segment_of(const Tour& w) {
  Segment x;
  x.head = w.u / w.nb;
  x.blk = w.u % w.nb;
  x.t0 = w.t;
  x.n = (int)min((long long)(w.nt - w.t), w.end - w.at);
  x.rows = min(kUnit, w.rows - x.blk * kUnit);
  x.two = x.rows > kRows;
  x.whole = x.t0 == 0 && x.n == w.nt;
  return x;
}

template <class T, bool TWO, int HD>
__global__ void __launch_bounds__(kThreads, 1)
attention_shared_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                        const PagedArgs a, const KvArgs kv, const SharedView v, const SharedParts parts, int box_rows,
                        unsigned* __restrict__ err) {
  using C = Cfg<TWO, HD>;
  constexpr int kHalves = HD / 64, S = C::kStages, kKeys = C::kKeys;
  constexpr uint32_t kFmt = std::is_same<T, __half>::value ? 0u : 1u;
  constexpr uint32_t kIdescS = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((kKeys >> 3) << 17) | ((kRows >> 4) << 24);
  constexpr uint32_t kIdescO =
      (1u << 4) | (kFmt << 7) | (kFmt << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((kRows >> 4) << 24);
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBars);
  uint64_t* kv_full = bars;
  uint64_t* kv_empty = kv_full + S;
  uint64_t* q_full = kv_empty + S;  // [2] a stream's queries are in shared memory
  uint64_t* s_full = q_full + 2;    // [2] scores of a tile are in tensor memory
  uint64_t* s_free = s_full + 2;    // [2] and have been read (TWO)
  uint64_t* p_full = s_free + 2;    // [2][2] its weights are there, of the first and second half of the keys (TWO: all)
  uint64_t* o_full = p_full + 4;    // [2] the tile's (TWO) or the segment's output is there
  uint64_t* drain = o_full + 2;     // [2]
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(drain + 2);
  volatile uint32_t* s_abort = s_tmem + 1;
  long long* s_sum = reinterpret_cast<long long*>(smem);  // per-warp sums, before the queries come
  long long* s_total = reinterpret_cast<long long*>(smem + C::kSum);
  long long* s_first = s_total + 1;
  int* s_group = reinterpret_cast<int*>(s_total + 2);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = a.n_heads / kv.n_kv;
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    prefetch_map(&kmap);
    prefetch_map(&vmap);
    for (int i = 0; i < S; ++i) {
      mbar_init(smem_u32(kv_full + i), 1);
      mbar_init(smem_u32(kv_empty + i), TWO ? 2 : 1);  // who issues the products that read it
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(q_full + i), 4);
      mbar_init(smem_u32(s_full + i), 1);
      mbar_init(smem_u32(s_free + i), 4);
      mbar_init(smem_u32(p_full + 2 * i), 4);
      mbar_init(smem_u32(p_full + 2 * i + 1), 4);
      mbar_init(smem_u32(o_full + i), 1);
      mbar_init(smem_u32(drain + i), 1);
    }
    *s_abort = 0u;
    fence_mbar_init();
  }
  // The next launch, the own pass, does not wait for this one: it may begin once everything before this one is over.
  pdl_wait();
  pdl_trigger();

  // ---- this CTA's range: the groups' tiles, a contiguous share of the groups per thread ----
  auto load = [&](int grp, Tour* x, bool report) -> long long {
    int b, e;
    const bool ok = group_of(v, kv, grp, &b, &e, &x->shared);
    if (!ok && report) atomicOr(err, kErrDecodeRange);
    x->grp = grp;
    x->b = b;
    x->rows = (e - b) * g;
    x->nb = (x->rows + kUnit - 1) / kUnit;
    x->nt = (x->shared + kKeys - 1) / kKeys;
    return (long long)x->nb * x->nt * kv.n_kv;
  };
  Tour w;
  {
    const int per = (v.groups + kThreads - 1) / kThreads, q0 = min(v.groups, tid * per), q1 = min(v.groups, q0 + per);
    long long mine = 0;
    for (int x = q0; x < q1; ++x) mine += load(x, &w, blockIdx.x == 0);
    long long x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long z = __shfl_up_sync(kFull, x, o);
      if (lane >= o) x += z;
    }
    if (lane == 31) s_sum[warp] = x;  // the warps' sums
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    long long before = x - mine, total = 0;  // tiles of the groups before this thread's; of all
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) {
      const long long y = s_sum[i];
      before += i < warp ? y : 0;
      total += y;
    }
    if (tid == 0) *s_total = total;
    const int ctas = (int)min((long long)gridDim.x, total);
    const Deal deal(total, max(1, ctas));
    w.at = (int)blockIdx.x < ctas ? deal.start(blockIdx.x) : 0;
    w.end = (int)blockIdx.x < ctas ? deal.start(blockIdx.x + 1) : 0;
    const long long at = w.at, end = w.end;
    if (at < end && before <= at && at < before + mine) {
      x = before;
      for (int y = q0; y < q1; ++y) {
        const long long z = load(y, &w, false);
        if (at < x + z) {
          *s_group = y;
          *s_first = x;
          break;
        }
        x += z;
      }
    }
    __syncthreads();
    if (at < end) {
      load(*s_group, &w, false);
      w.u = (int)((at - *s_first) / w.nt);
      w.first = *s_first + (long long)w.u * w.nt;
      w.t = (int)(at - w.first);
    }
    w.at = at;
    w.end = end;
  }
  const uint32_t tmem = *s_tmem;
  // behind the segment of n tiles: the next unit, of this group or the next one that shares something
  auto advance = [&](int n) {
    w.at += n;
    if (w.at >= w.end) return;
    w.t = 0;
    w.first += w.nt;
    if (++w.u == w.nb * kv.n_kv) {
      w.u = 0;
      do {
      } while (load(w.grp + 1, &w, false) == 0);
    }
  };
  auto fail = [&]() {
    *s_abort = 1u;
    atomicOr(err, kErrRingTimeout);
  };
  // Warp-wide wait; false (in every lane) when the role has to leave.
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (__all_sync(kFull, mbar_try_wait(smem_u32(bar), parity))) return true;
    const bool ok = mbar_wait_bounded(smem_u32(bar), parity);
    if (!ok) fail();
    return !__any_sync(kFull, !ok || *s_abort);
  };

  if (warp >= 8) {
    if constexpr (TWO) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");  // 8 x 216 + 4 x 72 = 12 x 168
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");                // 8 x 224 + 4 x 56
    if (warp == 9) {
      // ---------------- loader ----------------
      const int pages = kKeys / box_rows, my_page = lane / kHalves, half = lane % kHalves;
      const uint32_t box_bytes = (uint32_t)box_rows * 128u;
      int c = 0, grp = -1, from = -1;  // from: the sequence whose table is read, -1: none of the group has the positions
      bool ok = true;
      while (ok && w.at < w.end) {
        const Segment x = segment_of(w);
        // page of this lane's box in tile j of the segment: as sequence s has it, and for the copy (n_pages: zeros)
        auto number = [&](int j, int s) -> int {
          const int p = (x.t0 + j) * kKeys + my_page * box_rows;
          if (my_page >= pages || j >= x.n || p >= w.shared || s < 0) return 0;
          return __ldcg(kv.table + (long long)s * kv.table_stride + (p >> kv.page_shift));
        };
        auto box = [&](int j, int page) -> int {
          const int p = (x.t0 + j) * kKeys + my_page * box_rows;
          if (my_page >= pages || j >= x.n) return -1;
          if (p >= w.shared || from < 0) return kv.n_pages;
          if ((unsigned)page < (unsigned)kv.n_pages) return page;
          atomicOr(err, kErrDecodeRange);
          return kv.n_pages;
        };
        int page;
        if (w.grp == grp) {
          page = number(0, from);
        } else {  // the group's first sequence that is as long, most often its first
          grp = w.grp;
          page = number(0, w.b);
          const int members = w.rows / g;
          from = -1;
          for (int i = 0; i < members && from < 0; i += 32) {
            const unsigned hit = __ballot_sync(kFull, i + lane < members && __ldcg(kv.len + w.b + i + lane) >= w.shared);
            if (hit) from = w.b + i + __ffs(hit) - 1;
          }
          if (from != w.b) page = number(0, from);
        }
        for (int j = 0; j < x.n && ok; ++j) {
          const int cur = box(j, page);
          page = number(j + 1, from);
          const int row = ((x.t0 + j) * kKeys + my_page * box_rows) & (kv.page_size - 1);
          for (int y = 0; y < 2; ++y, ++c) {
            const int st = c % S;
            if (c >= S && !(ok = wait(kv_empty + st, ((c / S) - 1) & 1))) break;
            const uint32_t bar = smem_u32(kv_full + st);
            if (lane == 0) mbar_arrive_expect_tx(bar, C::kTileBytes);
            __syncwarp();
            if (cur >= 0)
              tma_load_4d(smem_u32(smem) + C::kRing + st * C::kTileBytes + half * (kKeys * 128) + my_page * box_bytes,
                          y ? &vmap : &kmap, half * 64, row, x.head, cur, bar);
          }
        }
        advance(x.n);
      }
      // what was issued lands before the CTA may end (bounded)
      for (int j = c - S < 0 ? 0 : c - S; j < c; ++j) mbar_wait_bounded(smem_u32(kv_full + j % S), (j / S) & 1);
    } else if ((warp == 8 || (TWO && warp == 10)) && elect_one()) {
      // ---------------- matrix products (one thread; TWO: one for each stream) ----------------
      const uint32_t q_lo = desc_lo(smem_u32(smem), C::kLeading);
      const uint32_t ring_lo = desc_lo(smem_u32(smem) + C::kRing, C::kLeading);
      constexpr uint32_t kTileLo = C::kTileBytes >> 4, kQLo = C::kQBytes >> 4;
      const int mine = warp == 8 ? 0 : 1;
      uint32_t nq = 0, np = 0, nf = 0;  // parities, one bit a stream
      int c = 0;                        // ring entries before this segment
      bool ok = true, issued = false;
      auto get = [&](uint64_t* bar, uint32_t parity) { return ok = ok && mbar_wait_bounded(smem_u32(bar), parity); };
      auto get_tile = [&](int e) { return get(kv_full + e % S, (e / S) & 1); };
      auto release = [&](int e) {
        if (ok) umma_commit(smem_u32(kv_empty + e % S));
      };
      // scores of stream i against the keys in ring entry e
      auto scores = [&](int i, int e, bool first) {
        if (first) {
          if (!get(q_full + i, nq >> i & 1)) return;
          nq ^= 1u << i;
        } else if (TWO) {  // the last ones have been read
          if (!get(s_free + i, nf)) return;
          nf ^= 1u;
        }
        if (!get_tile(e)) return;
        tc_fence_after();
        const uint32_t ql = q_lo + i * kQLo, kl = ring_lo + (e % S) * kTileLo;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          const uint32_t in = (ks & 3) * 2;
          umma_ss(tmem + i * kKeys, desc64(ql + (ks >> 2) * ((kRows * 128) >> 4) + in, kDescHi),
                  desc64(kl + (ks >> 2) * ((kKeys * 128) >> 4) + in, kDescHi), kIdescS, ks > 0);
        }
        umma_commit(smem_u32(s_full + i));
        issued = true;
      };
      // stream i's weights times the values in ring entry e
      auto values = [&](int i, int e, bool first, bool last) {
        if (!get_tile(e)) return;
        const uint32_t vl = ring_lo + (e % S) * kTileLo, tp = tmem + C::kP + i * kKeys, to = tmem + C::kO + i * HD;
        constexpr int kParts = TWO ? 1 : 2, kSteps = kKeys / 16 / kParts;
#pragma unroll
        for (int h = 0; h < kParts; ++h) {  // the first keys while the weights of the others are computed
          if (!get(p_full + 2 * i + h, np >> i & 1)) return;
          tc_fence_after();
#pragma unroll
          for (int ks = h * kSteps; ks < (h + 1) * kSteps; ++ks) {
            umma_ts(to, tp + ks * 8, desc64(vl + ks * (2048 >> 4), kDescHi), kIdescO, ks > 0 || !(TWO || first));
            if constexpr (TWO) umma_ts(to, tp + kKeys / 2 + ks * 8, desc64(vl + ks * (2048 >> 4), kDescHi), kIdescO, true);
          }
        }
        np ^= 1u << i;
        if (TWO || last) umma_commit(smem_u32(o_full + i));
      };
      while (ok && w.at < w.end) {
        const Segment x = segment_of(w);
        if constexpr (TWO) {
          int passed = 0;  // tiles before this one are done with, as far as this stream goes
          auto pass = [&](int tile) {  // those of the other stream: once they are there, this one does not need them
            for (; ok && passed < tile; ++passed)
              for (int y = 0; y < 2; ++y)
                if (get_tile(c + 2 * passed + y)) mbar_arrive(smem_u32(kv_empty + (c + 2 * passed + y) % S));
            ++passed;
          };
          const int step = x.two ? 1 : 2, begin = x.two ? 0 : mine;
          for (int j = begin - step; ok && j < x.n; j += step) {
            const int next = j + step;
            if (next < x.n) {
              pass(next);
              if (ok) scores(mine, c + 2 * next, next == begin);
              release(c + 2 * next);
            }
            if (ok && j >= begin) {
              values(mine, c + 2 * j + 1, false, false);
              release(c + 2 * j + 1);
            }
          }
          if (ok && begin < x.n && get(s_free + mine, nf)) nf ^= 1u;
          pass(x.n);
        } else if (x.two) {  // both streams have all tiles
          for (int j = 0; j <= x.n && ok; ++j) {
#pragma unroll 1
            for (int i = 0; i < 2 && ok; ++i) {
              if (j > 0) values(i, c + 2 * j - 1, j == 1, j == x.n);
              if (j > 0 && i == 1) release(c + 2 * j - 1);
              if (ok && j < x.n) scores(i, c + 2 * j, j == 0);
              if (j < x.n && i == 1) release(c + 2 * j);
            }
          }
        } else {  // every other one
          for (int j = 0; j < x.n + 2 && ok; ++j) {
            if (j >= 2) {
              values(j & 1, c + 2 * j - 3, j < 4, j >= x.n);
              release(c + 2 * j - 3);
            }
            if (ok && j < x.n) {
              scores(j & 1, c + 2 * j, j < 2);
              release(c + 2 * j);
            }
          }
        }
        c += 2 * x.n;
        advance(x.n);
      }
      if (!ok) fail();
      if (issued) {  // the tensor core is done before tensor memory is released
        umma_commit(smem_u32(drain + mine));
        if (!mbar_wait_bounded(smem_u32(drain + mine), 0)) fail();
      }
    }
  } else {
    // ---------------- softmax ----------------
    if constexpr (TWO) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int i = warp >> 2, lrow = 32 * (warp & 3) + lane;
    const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const uint32_t ts = lanes + i * kKeys, tp = lanes + C::kP + i * kKeys, to = lanes + C::kO + i * HD;
    const float sl2 = a.scale * 1.4426950408889634f;
    const long long begin = w.at;
    uint32_t ns = 0, no = 0;  // parities
    bool ok = true;
    auto leave = [&](const Segment& x, int n, int slot) {  // where the unit's results are
      __stcg(reinterpret_cast<int4*>(parts.found + (long long)x.head * parts.found_stride + unit_index(w.b * g, w.grp, x.blk)),
             make_int4(n, (int)blockIdx.x, slot, 0));
    };
    while (ok && w.at < w.end) {
      const Segment x = segment_of(w);
      const int row = lrow + (x.two ? i * kRows : 0), tiles = x.two ? x.n : (x.n + 1 - i) >> 1;
      const bool mine = row < x.rows, idle = row - lane >= x.rows;  // idle: the warp has no row
      const int rr = x.blk * kUnit + row, seq = w.b + rr / g, head = x.head * g + rr % g;
      const int slot = 2 * blockIdx.x + (w.at == begin ? 0 : 1);
      if (x.t0 == 0 && tid == 0) {
        int n = 1;
        if (!x.whole) {
          const int ctas = (int)min((long long)gridDim.x, *s_total);
          n = Deal(*s_total, ctas).range_of(w.first + w.nt - 1) - (int)blockIdx.x + 1;
        }
        leave(x, n, slot);
      }
      if (tiles > 0) {
        // Queries: this warp's 32 rows, a row's pieces in consecutive lanes.  What was read from the buffer before has
        // been: the last segment's last scores were waited for.
        constexpr int P = HD / 8, N = 32 / P;  // pieces of a row, rows at a time
        const long long mine_at = mine ? (long long)seq * a.q_row_stride + (long long)head * a.q_head_stride : -1;
        unsigned char* sq = smem + i * C::kQBytes;
        uint4 y[32 / N];
#pragma unroll
        for (int k = 0; k < 32 / N; ++k) {
          const int rw = k * N + lane / P;
          const long long at = __shfl_sync(kFull, mine_at, rw);
          y[k] = make_uint4(0u, 0u, 0u, 0u);
          if (at >= 0) y[k] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + at) + lane % P);
        }
#pragma unroll
        for (int k = 0; k < 32 / N; ++k) {
          const int rw = 32 * (warp & 3) + k * N + lane / P, ch = lane % P;
          *reinterpret_cast<uint4*>(sq + (ch >> 3) * (kRows * 128) + rw * 128 + (((ch & 7) ^ (rw & 7)) << 4)) = y[k];
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(q_full + i));
      }
      float m = -INFINITY, l = 0.0f;
      float o[TWO ? HD : 1];  // fp32 outputs: the sums over the tiles
#pragma unroll
      for (int e = 0; e < (TWO ? HD : 1); ++e) o[e] = 0.0f;
      // the last tile's output on top of the sums, then times f if the row's maximum has risen
      auto add_output = [&](bool rises, float f) {
#pragma unroll
        for (int b = 0; b < HD; b += 32) {
          uint32_t z[32];
          tmem_ld<32>(to + b, z);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if constexpr (TWO) o[b + e] += __uint_as_float(z[e]);
        }
        if (rises) {
#pragma unroll
          for (int e = 0; e < (TWO ? HD : 1); ++e) o[e] *= f;
        }
      };
      // What a warp does between having scores y of the stream's tile j and having to give their weights: the maximum, and
      // whether the output so far is to be multiplied by *f.
      auto mask = [&](uint32_t(&y)[kKeys], int j) {
        const int limit = w.shared - (x.t0 + (x.two ? j : 2 * j + i)) * kKeys;  // columns below it exist
        if (limit < kKeys) {
#pragma unroll
          for (int e = 0; e < kKeys; ++e)
            if (e >= limit) y[e] = 0xFF800000u;
        }
      };
      auto raise = [&](const uint32_t(&y)[kKeys], int j, float* f) -> bool {
        float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < kKeys; e += 8)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            t[q] = max3(t[q], __uint_as_float(y[e + 2 * q]), __uint_as_float(y[e + 2 * q + 1]));
        const float mt = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
        if (j == 0) {
          m = mt;
          return false;
        }
        if (!__any_sync(kFull, mine && (mt - m) * sl2 > kLazy)) return false;
        const float mn = fmaxf(m, mt);
        *f = m == -INFINITY ? 0.0f : ex2((m - mn) * sl2);
        m = mn;
        l *= *f;
        return true;
      };
      // Weights of keys from .. from + 63 in place of their scores, and their sum.  First the exponentials, then what needs
      // them: with the sum beside each, a warp by itself waits for each in turn.
      auto exponentials = [&](uint32_t(&y)[kKeys], int from) {
        const float off = kPShift - (m == -INFINITY ? 0.0f : m * sl2);
        const unsigned long long sl22 = pack2(sl2, sl2), off2 = pack2(off, off);
#pragma unroll
        for (int e = from; e < from + 64; e += 2) {
          float x0, x1;
          unpack2(fma2(pack2(__uint_as_float(y[e]), __uint_as_float(y[e + 1])), sl22, off2), x0, x1);
          y[e] = __float_as_uint(ex2(x0));
          y[e + 1] = __float_as_uint(ex2(x1));
        }
        unsigned long long sum[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
        for (int e = from; e < from + 64; e += 2)
          sum[(e >> 1) & 3] = add2(sum[(e >> 1) & 3], pack2(__uint_as_float(y[e]), __uint_as_float(y[e + 1])));
        float s0, s1;
        unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), s0, s1);
        l += s0 + s1;
      };
      for (int j = 0; j < tiles; ++j) {
        if (!(ok = wait(s_full + i, ns))) break;
        ns ^= 1u;
        if (idle) {
          if (TWO) {
            if (lane == 0) mbar_arrive(smem_u32(s_free + i));
            if (j > 0) {
              if (!(ok = wait(o_full + i, no))) break;
              no ^= 1u;
            }
          }
          if (lane == 0) {
            mbar_arrive(smem_u32(p_full + 2 * i));
            if (!TWO) mbar_arrive(smem_u32(p_full + 2 * i + 1));
          }
          continue;
        }
        tc_fence_after();
        uint32_t y[kKeys];
#pragma unroll
        for (int b = 0; b < kKeys; b += 32) tmem_ld<32>(ts + b, *reinterpret_cast<uint32_t(*)[32]>(y + b));
        tmem_wait_ld();
        float f = 1.0f;
        if constexpr (TWO) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(s_free + i));
          mask(y, j);
          const bool rises = raise(y, j, &f);
          exponentials(y, 0);
          uint32_t p[32], p2[32];
#pragma unroll
          for (int e = 0; e < 64; e += 2) {
            const float x0 = __uint_as_float(y[e]), x1 = __uint_as_float(y[e + 1]);
            p[e >> 1] = pack16<T>(x0, x1);
            const float2 q = unpack16<T>(p[e >> 1]);
            p2[e >> 1] = pack16<T>(x0 - q.x, x1 - q.y);
          }
          if (j > 0) {  // the last tile's weights have been read and its values added
            if (!(ok = wait(o_full + i, no))) break;
            no ^= 1u;
            tc_fence_after();
          }
          tmem_st32(tp, p);
          tmem_st32(tp + kKeys / 2, p2);
          if (j > 0) add_output(rises, f);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(p_full + 2 * i));
        } else {
          mask(y, j);
          if (raise(y, j, &f)) {  // the last tile's values have been added: its products came before these scores
            const unsigned long long f2 = pack2(f, f);
#pragma unroll 1
            for (int b = 0; b < HD; b += 32) {
              uint32_t z[32];
              tmem_ld<32>(to + b, z);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                float z0, z1;
                unpack2(mul2(pack2(__uint_as_float(z[e]), __uint_as_float(z[e + 1])), f2), z0, z1);
                z[e] = __float_as_uint(z0);
                z[e + 1] = __float_as_uint(z1);
              }
              tmem_st32(to + b, z);
            }
          }
#pragma unroll
          for (int b = 0; b < kKeys; b += 64) {
            exponentials(y, b);
            uint32_t p[32];
#pragma unroll
            for (int e = 0; e < 64; e += 2) p[e >> 1] = pack16<T>(__uint_as_float(y[b + e]), __uint_as_float(y[b + e + 1]));
            tmem_st32(tp + (b >> 1), p);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(p_full + 2 * i + (b >> 6)));
          }
        }
      }
      if (!ok) break;
      // Results: o 2^ml.x is the sum of exp(s) v, l 2^ml.x of exp(s).  A thread holds a row; pieces of 16 bytes are
      // exchanged within four lanes, so that a store writes 64 bytes of a row.
      const long long at = ((long long)seq + (x.two ? 0 : (long long)i * kv.batch)) * a.n_heads + head;
      float* slot_o = parts.slots + (size_t)slot * part_floats<HD>();
      if (mine) {
        const float2 ml = make_float2(m == -INFINITY ? -INFINITY : m * sl2 - kPShift, l);
        if (x.whole) __stcg(parts.ml + at, ml);
        else __stcg(reinterpret_cast<float2*>(slot_o + (size_t)kUnit * HD) + i * kRows + lrow, ml);
      }
      if (tiles > 0) {
        if (!(ok = wait(o_full + i, no))) break;
        no ^= 1u;
        tc_fence_after();
      }
      if (tiles > 0 && !idle) {
        float* base = x.whole ? parts.o + at * HD : slot_o + (size_t)(i * kRows + lrow) * HD;
        float* to4[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          to4[q] = reinterpret_cast<float*>(__shfl_sync(kFull, mine ? reinterpret_cast<unsigned long long>(base) : 0ull,
                                                        (lane & ~3) + q));
#pragma unroll
        for (int b = 0; b < HD; b += 32) {
          uint32_t z[32];
          tmem_ld<32>(to + b, z);
          tmem_wait_ld();
          if constexpr (TWO) {
#pragma unroll
            for (int e = 0; e < 32; ++e) z[e] = __float_as_uint(__uint_as_float(z[e]) + o[b + e]);
          }
#pragma unroll
          for (int e = 0; e < 32; e += 16) {
            float4 p[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
              p[q] = make_float4(__uint_as_float(z[e + 4 * q]), __uint_as_float(z[e + 4 * q + 1]),
                                 __uint_as_float(z[e + 4 * q + 2]), __uint_as_float(z[e + 4 * q + 3]));
            transpose4(p, lane);  // p[q]: piece lane % 4 of the four lanes' row q
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (to4[q]) __stcg(reinterpret_cast<float4*>(to4[q] + b + e) + (lane & 3), p[q]);
          }
        }
        tc_fence_before();
      }
      advance(x.n);
    }
    if (!ok && tid == 0) abandon(w, [&]() { leave(segment_of(w), 0, 0); }, advance);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// Joins a row's parts: those of its own positions, then of the shared ones.  The own pass has left what leads to them (its
// parts, the group), so that three loads follow one another: that, the shared pass's parts, and all parts' outputs, maxima
// and sums at once.  ROWS rows a CTA: 1, by all warps, or 8, by a warp each, or one after the other by all where one of them
// has more than kFew parts.
constexpr int kFew = 64;
template <class O, int HD, int ROWS>
__global__ void __launch_bounds__(256, ROWS == 8 ? 4 : 3)
attention_shared_join_kernel(const PagedArgs a, const KvArgs kv, const SharedView v, const SharedParts parts, int zs) {
  constexpr int E = HD / 32, W = 8, U = ROWS == 8 ? 4 : 8;  // values of a lane, warps, parts at a time
  __shared__ float s_o[W][HD];
  __shared__ float2 s_ml[W];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = a.n_heads / kv.n_kv, R = g <= 8 ? 8 : 16;
  const long long rows = (long long)kv.batch * a.n_heads, row0 = (long long)blockIdx.x * ROWS;
  struct Way {  // to a row's parts
    int4 own, shared;  // parts, range, slot
    int in, local, streams, total;
    long long row;
  };
  auto way = [&](long long row) -> Way {
    Way x = {};
    x.row = row;
    if (row >= rows) return x;
    const int s = (int)(row / a.n_heads), h = (int)(row % a.n_heads), j = h / g;
    x.in = h % g;
    const int4* at_own = reinterpret_cast<const int4*>(v.own_found + ((long long)s * kv.n_kv + j) * zs + x.in / 16);
    x.own = __ldcg(at_own);
    const int4 grp = __ldcg(at_own + 1);  // group (-1: none), its sequences
    x.own.x = parts_of({x.own.x, x.own.y, x.own.z, 0}, kOwnRanges);
    x.streams = 1;
    if (in_group(grp.x, grp.y, grp.z, s, v.groups, kv.batch)) {
      const int rr = (s - grp.y) * g + x.in, blk = rr / kUnit;
      x.local = rr % kUnit;
      x.streams = min(kUnit, (grp.z - grp.y) * g - blk * kUnit) > kRows ? 1 : 2;
      x.shared = __ldcg(reinterpret_cast<const int4*>(parts.found + (long long)j * parts.found_stride +
                                                      unit_index(grp.y * g, grp.x, blk)));
      x.shared.x = parts_of({x.shared.x, x.shared.y, x.shared.z, 0}, kMaxCtas);
    }
    x.total = x.own.x + x.shared.x * x.streams;
    return x;
  };
  // where part p's output row is, and its (maximum, sum)
  auto find = [&](const Way& x, int p, const float** o) -> const float2* {
    if (p < x.own.x) {
      if (x.own.x == 1) {
        *o = v.own_o + x.row * HD;
        return v.own_ml + x.row;
      }
      const float* slot = v.own_slots + (size_t)(p ? 2 * (x.own.y + p) : x.own.z) * (size_t)slot_floats(R, HD);
      *o = slot + (x.in % 16) * HD;
      return reinterpret_cast<const float2*>(slot + R * HD) + x.in % 16;
    }
    p -= x.own.x;
    const int i = x.streams == 2 ? p & 1 : 0, k = x.streams == 2 ? p >> 1 : p;
    if (x.shared.x == 1) {
      const long long at = x.row + (long long)i * kv.batch * a.n_heads;
      *o = parts.o + at * HD;
      return parts.ml + at;
    }
    const float* slot = parts.slots + (size_t)(k ? 2 * (x.shared.y + k) : x.shared.z) * part_floats<HD>();
    *o = slot + (size_t)(x.local + i * kRows) * HD;
    return reinterpret_cast<const float2*>(slot + (size_t)kUnit * HD) + x.local + i * kRows;
  };
  float m, l, o[E];
  auto join = [&](const Way& w, int first, int warps) {  // every `warps`-th part
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int z = 0; z < E; ++z) o[z] = 0.0f;
    for (int p0 = first; p0 < w.total; p0 += U * warps) {
      float x[U][E];
      float2 ml[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int p = p0 + u * warps;
        ml[u] = make_float2(-INFINITY, 0.0f);
        if (p < w.total) {
          const float* src;
          ml[u] = __ldcg(find(w, p, &src));
#pragma unroll
          for (int z = 0; z < E; z += 2) {
            const float2 y = __ldcg(reinterpret_cast<const float2*>(src + lane * E + z));
            x[u][z] = y.x;
            x[u][z + 1] = y.y;
          }
        }
      }
      float mn = m;
#pragma unroll
      for (int u = 0; u < U; ++u) mn = fmaxf(mn, ml[u].x);
      const float mz = mn == -INFINITY ? 0.0f : mn, f0 = ex2(m - mz);
      m = mn;
      l *= f0;
#pragma unroll
      for (int z = 0; z < E; ++z) o[z] *= f0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (ml[u].x == -INFINITY && ml[u].y == 0.0f) continue;  // nothing in it: there may be no output either
        const float by = ex2(ml[u].x - mz);
        l = fmaf(by, ml[u].y, l);
#pragma unroll
        for (int z = 0; z < E; ++z) o[z] = fmaf(by, x[u][z], o[z]);
      }
    }
  };
  auto put = [&](long long row) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    O* out = static_cast<O*>(a.out) + row * HD + lane * E;
#pragma unroll
    for (int z = 0; z < E; z += 2) {
      if constexpr (sizeof(O) == 4) *reinterpret_cast<float2*>(out + z) = make_float2(o[z] * inv, o[z + 1] * inv);
      else *reinterpret_cast<uint32_t*>(out + z) = pack16<O>(o[z] * inv, o[z + 1] * inv);
    }
  };
  if constexpr (ROWS == 8) {
    const Way w = way(row0 + warp);
    if (!__syncthreads_or(w.total > kFew)) {
      if (w.row >= rows) return;
      join(w, 0, 1);
      put(w.row);
      return;
    }
  }
  for (int i = 0; i < ROWS; ++i) {
    if (row0 + i >= rows) return;
    join(way(row0 + i), warp, W);
#pragma unroll
    for (int q = 0; q < E; ++q) s_o[warp][lane * E + q] = o[q];
    if (lane == 0) s_ml[warp] = make_float2(m, l);
    __syncthreads();
    if (warp == 0) {
      m = -INFINITY;
#pragma unroll
      for (int x = 0; x < W; ++x) m = fmaxf(m, s_ml[x].x);
      const float mz = m == -INFINITY ? 0.0f : m;
      l = 0.0f;
#pragma unroll
      for (int q = 0; q < E; ++q) o[q] = 0.0f;
#pragma unroll
      for (int x = 0; x < W; ++x) {
        const float fx = ex2(s_ml[x].x - mz);
        l = fmaf(fx, s_ml[x].y, l);
#pragma unroll
        for (int q = 0; q < E; ++q) o[q] = fmaf(fx, s_o[x][lane * E + q], o[q]);
      }
      put(row0 + i);
    }
    __syncthreads();
  }
}

// Workspace: all parts, 16-byte aligned.
struct Space {
  size_t slots, o, ml, found, own_slots, own_o, own_ml, own_found, bytes;
  int found_stride, zs;
};
Space space_of(int batch, int groups, int n_heads, int n_kv, int head_dim) {
  Space x;
  const size_t rows = (size_t)batch * n_heads;
  const int g = n_heads / n_kv;
  x.zs = (g + 15) / 16;
  x.found_stride = (int)((long long)batch * g / kUnit) + groups + 1;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t was = at;
    at += (bytes + 15) / 16 * 16;
    return was;
  };
  x.slots = take((size_t)kMaxCtas * 2 * (head_dim == 128 ? part_floats<128>() : part_floats<64>()) * 4);
  x.o = take(2 * rows * head_dim * 4);
  x.ml = take(2 * rows * 8);
  x.found = take((size_t)n_kv * x.found_stride * sizeof(Found));
  x.own_slots = take(own_slots_floats(n_heads, n_kv, head_dim) * 4);
  x.own_o = take(rows * head_dim * 4);
  x.own_ml = take(rows * 8);
  x.own_found = take((size_t)batch * n_kv * x.zs * sizeof(OwnFound));
  x.bytes = at;
  return x;
}

template <class T, class O, int HD>
cudaError_t launch_typed(const SharedArgs& sa, const KvArgs& kv, cudaStream_t stream, unsigned* err) {
  using C = Cfg<sizeof(O) == 4, HD>;
  constexpr int kKeys = C::kKeys;
  const PagedArgs& a = sa.paged;
  auto kernel = attention_shared_kernel<T, sizeof(O) == 4, HD>;
  const Space sp = space_of(kv.batch, sa.groups, a.n_heads, kv.n_kv, HD);
  unsigned char* ws = static_cast<unsigned char*>(a.workspace);
  SharedView v;
  v.cu_group = sa.cu_group;
  v.shared_len = sa.shared_len;
  v.groups = sa.groups;
  v.own_o = reinterpret_cast<float*>(ws + sp.own_o);
  v.own_ml = reinterpret_cast<float2*>(ws + sp.own_ml);
  v.own_found = reinterpret_cast<OwnFound*>(ws + sp.own_found);
  v.own_slots = reinterpret_cast<float*>(ws + sp.own_slots);
  SharedParts parts;
  parts.o = reinterpret_cast<float*>(ws + sp.o);
  parts.ml = reinterpret_cast<float2*>(ws + sp.ml);
  parts.slots = reinterpret_cast<float*>(ws + sp.slots);
  parts.found = reinterpret_cast<Found*>(ws + sp.found);
  parts.found_stride = sp.found_stride;
  CUtensorMap kmap, vmap;
  const int box_rows = kv.page_size < kKeys ? kv.page_size : kKeys;
  if (!encode_kv_map(&kmap, kv, kv.k, box_rows) || !encode_kv_map(&vmap, kv, kv.v, box_rows))
    return cudaErrorInvalidValue;
  static std::atomic<unsigned long long> done{0};
  int sms = 0;
  cudaError_t e = kernel_setup(reinterpret_cast<const void*>(kernel), C::kSmem, done, &sms);
  if (e != cudaSuccess) return e;
  // What is known here bounds the tiles: units of all groups, key tiles by what the page table can hold.
  const long long units = ((long long)kv.batch * (a.n_heads / kv.n_kv) / kUnit + sa.groups) * kv.n_kv;
  const long long most = units * (((long long)kv.width * kv.page_size + kKeys - 1) / kKeys);
  long long ctas = sms < kMaxCtas ? sms : kMaxCtas;
  if (ctas > most) ctas = most < 1 ? 1 : most;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_opt_pdl.load() ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, kernel, kmap, vmap, a, kv, v, parts, box_rows, err);
  if (e != cudaSuccess || (e = launch_attention_own(a, kv, v, stream)) != cudaSuccess) return e;
  // Few rows may have many parts each.  (1536 rows: a block a row makes the call 74 us, not 71; 800 rows of 46 parts: eight
  // rows a block 38, not 31.)
  const long long rows = (long long)kv.batch * a.n_heads;
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  if (rows <= 1184) {
    cfg.gridDim = dim3((unsigned)rows);
    return cudaLaunchKernelEx(&cfg, attention_shared_join_kernel<O, HD, 1>, a, kv, v, parts, sp.zs);
  }
  cfg.gridDim = dim3((unsigned)((rows + 7) / 8));
  return cudaLaunchKernelEx(&cfg, attention_shared_join_kernel<O, HD, 8>, a, kv, v, parts, sp.zs);
}

template <class T>
cudaError_t launch_type(const SharedArgs& a, const KvArgs& kv, cudaStream_t stream, unsigned* err) {
  const bool f32 = a.paged.out_dtype == kDtF32;
  if (kv.head_dim == 128)
    return f32 ? launch_typed<T, float, 128>(a, kv, stream, err) : launch_typed<T, T, 128>(a, kv, stream, err);
  return f32 ? launch_typed<T, float, 64>(a, kv, stream, err) : launch_typed<T, T, 64>(a, kv, stream, err);
}

}  // namespace

size_t attention_shared_workspace(int batch, int groups, int n_heads, int n_kv, int head_dim) {
  return batch == 0 ? 0 : space_of(batch, groups, n_heads, n_kv, head_dim).bytes;
}

cudaError_t launch_attention_shared(const SharedArgs& a, const KvArgs& kv, cudaStream_t stream) {
  unsigned* err = device_error_word();
  if (!err) return cudaErrorUnknown;
  return kv.dtype == kDtF16 ? launch_type<__half>(a, kv, stream, err)
                            : launch_type<__nv_bfloat16>(a, kv, stream, err);
}

}  // namespace asmllm
