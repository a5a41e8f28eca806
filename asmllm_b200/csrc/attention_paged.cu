// asmllm_b200/csrc/attention_paged.cu -- attention of one new token per
// sequence over a paged key-value cache.
//
//   out[s][h] = sum_{p < n_s} softmax_p(scale q[s][h] . k[p][h / g]) v[p][h / g]
// with n_s = len[s]; no position: zeros.
//
// The keys and values are read once (4 head_dim bytes a position and KV head)
// and everything else is small, so the work is dealt out by bytes: a unit is
// one (sequence, KV head, up to 16 of its query heads), a unit's positions
// are tiles of 64, and the tiles of all units in a row are cut into one equal
// range per CTA (two CTAs an SM), whatever the lengths are.  Lengths live on
// the device; each CTA sums them itself.  A range covers whole units and at
// most two parts of units: whole units are written out, parts go to the
// workspace as (maximum, sum, unnormalised output) and a second, small kernel
// (a programmatic dependent launch) joins each split unit's parts in order.
// No atomics and no counters: the result has the same bits every time, and
// the workspace needs no initial content.
//
// CTA: one producer warp brings tiles into a three-stage ring (tensor copies
// with the 128-byte swizzle, one box per page and 64 values); four consumer
// warps take 16 positions of each tile with a running maximum, sum and output
// of their own and meet only at the end of a unit.  Products are m16n8k16
// with the query heads as rows.  The weights enter the second product as
// hi + lo 16-bit parts, which leaves 2^-22 of a weight in fp16 (down to 2^-39
// of the row's largest) and 2^-16 in bf16; a group of up to 8 heads fills rows
// 0-7 with hi and rows 8-15 with lo, and the product costs nothing extra.
// Infinite values take another way (add_values): lo may be negative or zero,
// and then its product with an infinity makes NaN of the sum.  Looking for
// them costs 1 us of the 29 below, nothing of the 355.
//
// Measured on one B200: 64 sequences of up to 16384 positions, 64 query on 8
// KV heads of 128 values (2.26 GB), 355 us = 6.4 TB/s, 0.99 of the copy rate;
// 32 sequences of up to 1024 (74 MB) 28.9 us, where the copy would take 11.4:
// a CTA has about eight tiles in two or three segments, and the counters show
// no busy unit (instructions issued in 29 % of the cycles in which an SM is
// active, matrix products in 13 %, DRAM at 32 %).  What the code pays a
// segment and does not hide: the query rows' load between two barriers, and
// the join of the four warps, four barriers for each 8 rows; the ring holds
// three tiles meanwhile.  With one CTA per unit (no split) one sequence of
// 131071 positions on one KV head took 14 ms; now 30 us (25 in some runs).
#include <type_traits>

#include "matvec.cuh"
#include "mma16.cuh"
#include "pipeline.cuh"
#include "serving.cuh"
#include "tensor_map.cuh"

namespace asmllm {

namespace {

constexpr int kTile = 64;   // positions per tile, 16 per consumer warp
constexpr int kWarps = 4;   // consumer warps
constexpr int kStages = 3;
constexpr int kMaxCtas = 320;
constexpr int kThreads = (kWarps + 1) * 32;

// Parts of split units: [kMaxCtas][2] slots of ROWS x (HD outputs, maximum,
// sum), then one Split per CTA: the split unit that begins in its range.
struct Split {
  int unit;   // -1: none
  int parts;  // CTAs c .. c + parts - 1 hold one each
  int slot;   // slot of the first part (the others are in slot 2 c)
  int pad;
};

__host__ __device__ constexpr size_t slot_floats(int rows, int hd) { return (size_t)rows * hd + 2 * rows; }

template <int ROWS, int HD>
struct Layout {
  static constexpr int kTileBytes = kTile * HD * 2;        // keys or values of a tile
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kJoinRow = HD + 4;                  // floats: a row of the join buffer and its padding
  static constexpr int kJoinOff = kStages * kStageBytes;   // two warps' 8 rows
  static constexpr int kMlOff = kJoinOff + 2 * 8 * kJoinRow * 4;
  static constexpr int kBarOff = kMlOff + 2 * 8 * 8;
  static constexpr int kSmem = kBarOff + 2 * kStages * 8 + 64 + 1024;
  // A unit's query rows pass through the join buffer: padded by 16 bytes for ldmatrix.
  static constexpr int kQRow = HD * 2 + 16;
  static_assert(16 * kQRow <= 2 * 8 * kJoinRow * 4, "the query rows fit the join buffer");
};

__device__ __forceinline__ int tiles_of(int n) { return (n + kTile - 1) / kTile; }

// `total` tiles over `ctas` ranges: the first `extra` have one more than the others.
struct Deal {
  long long each;
  int extra;
  __device__ __forceinline__ Deal(long long total, int ctas) {
    if (total < (1ll << 32)) {  // a 64-bit division costs hundreds of cycles
      each = (unsigned)total / (unsigned)ctas;
      extra = (int)((unsigned)total % (unsigned)ctas);
    } else {
      each = total / ctas;
      extra = (int)(total % ctas);
    }
  }
  __device__ __forceinline__ long long start(int c) const { return c * each + min(c, extra); }
  __device__ __forceinline__ int cta_of(long long x) const {  // whose range holds tile x
    const long long big = (each + 1) * extra;
    return x < big ? (int)(x / (each + 1)) : extra + (int)((x - big) / each);
  }
};

// o += p v in fp32 for D times 8 values from 8 d0 on and the first n of a warp's 16 positions of a tile (values at sv,
// from row r0).  Weights that fp32 rounds to zero count as zero: times infinity that is NaN.  Lane: row
// lane / 4 (and 8 more), values 2 (lane % 4) and the next of each eight; its weights are those of positions
// 2 (lane % 4), the next, and both of these plus 8.
template <class T, int HD, int R, int D>
__device__ __forceinline__ void add_values(float (&o)[HD / 8][4], int d0, const float (&p)[R][4], uint32_t sv,
                                           int r0, int n, int lane) {
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    float w[R];
#pragma unroll
    for (int e = 0; e < R; ++e) {
      const float odd = j < 8 ? p[e][1] : p[e][3], even = j < 8 ? p[e][0] : p[e][2];
      w[e] = __shfl_sync(kFull, j & 1 ? odd : even, (lane & 28) | ((j & 7) >> 1));
    }
#pragma unroll
    for (int d = d0; d < d0 + D; ++d) {
      uint32_t x;
      asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(sv + tile_chunk<kTile>(r0 + j, d) + (lane & 3) * 4));
      const float2 v = unpack16<T>(x);
#pragma unroll
      for (int e = 0; e < R; ++e) {
        o[d][2 * e] = fmaf(w[e], v.x, o[d][2 * e]);
        o[d][2 * e + 1] = fmaf(w[e], v.y, o[d][2 * e + 1]);
      }
    }
  }
}

// A CTA's walk over its tiles: sequence, unit of the sequence, tile.
struct Walk {
  int s, u, t, n, nt;      // n positions, nt tiles of sequence s
  long long first;         // number of the unit's first tile
  long long at, end;       // tiles [at, end) are left
};

template <class T, class O, int HD, int ROWS>
__global__ void __launch_bounds__(kThreads, 2)
attention_paged_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                       const PagedArgs a, const KvArgs kv, int zs, int box_rows, unsigned* __restrict__ err) {
  using L = Layout<ROWS, HD>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* empty = full + kStages;
  volatile int* s_abort = reinterpret_cast<int*>(empty + kStages);
  int* s_start = reinterpret_cast<int*>(empty + kStages + 1);  // [0] sequence of the range's first tile, [1] its positions
  long long* s_first = reinterpret_cast<long long*>(empty + kStages + 2);  // [0] the sequence's first tile, [1] total
  long long* s_part = reinterpret_cast<long long*>(smem + L::kJoinOff);    // per-thread sums (before the join uses it)

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x, units = kv.n_kv * zs, g = a.n_heads / kv.n_kv;
  if (tid == 0) {
    prefetch_map(&kmap);
    prefetch_map(&vmap);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(full + i), 1);
      mbar_init(smem_u32(empty + i), kWarps);
    }
    *s_abort = 0;
    fence_mbar_init();
  }
  pdl_trigger();
  pdl_wait();

  // Sum of all tiles and the sequence this range begins in: a contiguous share of the sequences per thread.
  const int per = (kv.batch + kThreads - 1) / kThreads, q0 = min(kv.batch, tid * per), q1 = min(kv.batch, q0 + per);
  long long mine = 0;
  int held = 0;  // positions of the thread's first sequence
  for (int s = q0; s < q1; ++s) {
    bool clipped;
    const int n = kv_length(kv, s, &clipped);
    if (s == q0) held = n;
    if (clipped && cta == 0) atomicOr(err, kErrDecodeRange);
    mine += tiles_of(n);
    // a sequence without positions: zeros, written by one CTA
    if (n == 0 && s % gridDim.x == cta) {
      O* out = static_cast<O*>(a.out) + (long long)s * a.n_heads * HD;
      const float z[8] = {};
      for (int i = 0; i < a.n_heads * HD; i += 8) store8(out + i, z);
    }
  }
  mine *= units;
  s_part[tid] = mine;
  __syncthreads();
  if (warp == 0) {
    long long run = 0;
    for (int b = 0; b < kThreads; b += 32) {
      const long long v = s_part[b + lane];
      long long x = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(kFull, x, o);
        if (lane >= o) x += y;
      }
      s_part[b + lane] = run + x - v;  // exclusive
      run += __shfl_sync(kFull, x, 31);
    }
    if (lane == 0) s_first[1] = run;
  }
  __syncthreads();
  const long long total = s_first[1];
  const int ctas = (int)min((long long)gridDim.x, total);  // every range in use holds a tile; the other CTAs have none
  const Deal deal(total, max(1, ctas));
  const long long begin = cta < ctas ? deal.start(cta) : 0, end = cta < ctas ? deal.start(cta + 1) : 0;
  if (begin < end && s_part[tid] <= begin && begin < s_part[tid] + mine) {
    long long x = s_part[tid];
    for (int s = q0; s < q1; ++s) {
      bool clipped;
      const int n = s == q0 ? held : kv_length(kv, s, &clipped);
      const long long w = (long long)tiles_of(n) * units;
      if (begin < x + w) {
        s_start[0] = s;
        s_start[1] = n;
        s_first[0] = x;
        break;
      }
      x += w;
    }
  }
  __syncthreads();

  float* slots = static_cast<float*>(a.workspace);
  Split* splits = reinterpret_cast<Split*>(slots + (size_t)kMaxCtas * 2 * slot_floats(ROWS, HD));
  if (begin >= end) {
    if (tid == 0) splits[cta].unit = -1;
    return;
  }
  Walk w;
  w.s = s_start[0];
  bool clipped;
  w.n = s_start[1];
  w.nt = tiles_of(w.n);
  const long long into = begin - s_first[0];
  w.u = into < (1ll << 32) ? (int)((unsigned)into / (unsigned)w.nt) : (int)(into / w.nt);
  w.first = s_first[0] + (long long)w.u * w.nt;
  w.t = (int)(begin - w.first);
  w.at = begin;
  w.end = end;
  // the next unit, of this sequence or the next one that holds positions
  auto next_unit = [&](Walk& x) {
    x.first += x.nt;
    x.t = 0;
    if (++x.u == units) {
      x.u = 0;
      do {
        ++x.s;
        x.n = kv_length(kv, x.s, &clipped);
      } while (x.n == 0);
      x.nt = tiles_of(x.n);
    }
  };

  if (warp == kWarps) {
    // ---------------- producer ----------------
    // Lane i of a tile: page i / (2 halves), of it keys or values, 64 values each.
    constexpr int kHalves = HD / 64;
    const int boxes_page = 2 * kHalves, pages_tile = kTile / box_rows;
    const int my_page = lane / boxes_page, my_box = lane % boxes_page;
    const bool worker = my_page < pages_tile;
    const uint32_t box_bytes = (uint32_t)box_rows * 128u;
    // page number of this lane's box in tile t of sequence s; n_pages (filled with zeros) for a bad one
    auto lookup = [&](const Walk& x) -> int {
      const int p = x.t * kTile + my_page * box_rows;
      if (!worker || p >= x.n) return -1;
      const int page = __ldcg(kv.table + (long long)x.s * kv.table_stride + (p >> kv.page_shift));
      if ((unsigned)page < (unsigned)kv.n_pages) return page;
      atomicOr(err, kErrDecodeRange);
      return kv.n_pages;
    };
    bool ok = true;
    int i = 0, page = lookup(w);
    for (; w.at < w.end && ok; ++i) {
      const int st = i % kStages;
      const Walk cur = w;
      const int cur_page = page;
      if (++w.at < w.end) {  // the next tile's page number is on its way while this one waits for its stage
        if (++w.t == w.nt) next_unit(w);
        page = lookup(w);
      }
      if (i >= kStages) ok = mbar_wait_bounded(smem_u32(empty + st), ((i / kStages) - 1) & 1);
      ok = !__any_sync(kFull, !ok || *s_abort);
      if (!ok) break;
      const uint32_t bar = smem_u32(full + st), dst = smem_u32(smem + st * L::kStageBytes);
      const unsigned live = __ballot_sync(kFull, cur_page >= 0);
      if (lane == 0) mbar_arrive_expect_tx(bar, box_bytes * __popc(live));
      __syncwarp();
      if (cur_page >= 0) {
        const int p = cur.t * kTile + my_page * box_rows, half = my_box % kHalves, is_v = my_box / kHalves;
        tma_load_4d(dst + is_v * L::kTileBytes + half * (kTile * 128) + my_page * box_bytes, is_v ? &vmap : &kmap,
                    half * 64, p & (kv.page_size - 1), cur.u / zs, cur_page, bar);
      }
    }
    if (!ok && lane == 0) {
      *s_abort = 1;
      atomicOr(err, kErrRingTimeout);
    }
    // every issued copy lands before the CTA may end (bounded)
    for (int j = i - kStages < 0 ? 0 : i - kStages; j < i; ++j)
      mbar_wait_bounded(smem_u32(full + j % kStages), (j / kStages) & 1);
    return;
  }

  // ---------------- consumers ----------------
  const uint32_t ring = smem_u32(smem);
  const float sl2 = a.scale * 1.4426950408889634f;
  const int r = lane >> 2, c2 = (lane & 3) * 2;
  float* jbuf = reinterpret_cast<float*>(smem + L::kJoinOff);
  float2* jml = reinterpret_cast<float2*>(smem + L::kMlOff);
  bool ok = true;
  int i = 0, split_unit = -1, split_parts = 0, split_slot = 0;
  bool next = true;
  while (next) {
    // one segment: tiles w.t .. of unit (w.s, w.u)
    const int j = w.u / zs, h0 = (w.u % zs) * 16, nh = min(16, g - h0);
    const int t0 = w.t, t1 = (int)min((long long)w.nt, w.t + (w.end - w.at));
    // The unit's query rows, read once by the CTA (each warp for itself made the same lines of a long
    // sequence's one unit a bottleneck of 5 to 14 thousand cycles), then as fragments.
    uint32_t qf[HD / 16][ROWS / 4];
    {
      const T* qb = static_cast<const T*>(a.q) + w.s * a.q_row_stride + (long long)(j * g + h0) * a.q_head_stride;
      unsigned char* sq = smem + L::kJoinOff;
      for (int e = tid; e < ROWS * (HD / 8); e += kWarps * 32) {
        const int row = e / (HD / 8), c = e % (HD / 8);
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (row < nh) v = __ldcg(reinterpret_cast<const uint4*>(qb + row * a.q_head_stride) + c);
        *reinterpret_cast<uint4*>(sq + row * L::kQRow + c * 16) = v;
      }
      consumer_bar_sync(kWarps * 32);
      // matrices of 8 rows x 8 values: [0..1] rows 0-7, [2..3] rows 8-15; each pair the 16 values of a step
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        if constexpr (ROWS == 16) {
          uint32_t f[4];
          ldsm4(f, smem_u32(sq) + ((lane & 7) + 8 * (lane >> 4)) * L::kQRow + (2 * ks + ((lane >> 3) & 1)) * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) qf[ks][e] = f[e];
        } else if ((ks & 1) == 0) {  // two steps at once
          uint32_t f[4];
          ldsm4(f, smem_u32(sq) + (lane & 7) * L::kQRow + (2 * ks + (lane >> 3)) * 16);
          qf[ks][0] = f[0];
          qf[ks][1] = f[1];
          qf[ks + 1][0] = f[2];
          qf[ks + 1][1] = f[3];
        }
      }
      consumer_bar_sync(kWarps * 32);  // the buffer is the join's again
    }
    // with ROWS == 8, rows 8-15 repeat rows 0-7: their scores are the same numbers
    constexpr int Q1 = ROWS == 16 ? 2 : 0, Q3 = ROWS == 16 ? 3 : 1, R = ROWS / 8;
    float o[HD / 8][4], m[R], l[R];
#pragma unroll
    for (int e = 0; e < R; ++e) {
      m[e] = -INFINITY;
      l[e] = 0.0f;
    }
#pragma unroll
    for (int e = 0; e < HD / 8; ++e) o[e][0] = o[e][1] = o[e][2] = o[e][3] = 0.0f;

    for (int t = t0; t < t1; ++t, ++i) {
      const int st = i % kStages;
      if (ok) ok = mbar_wait_bounded(smem_u32(full + st), (i / kStages) & 1) && !*s_abort;
      ok = __all_sync(kFull, ok);
      if (!ok) {  // give up: keep in step with the other warps, but touch no more tiles
        if (lane == 0) {
          *s_abort = 1;
          atomicOr(err, kErrRingTimeout);
        }
        continue;
      }
      const uint32_t sk = ring + st * L::kStageBytes, sv = sk + L::kTileBytes;
      const int r0 = warp * 16, left = w.n - t * kTile - r0;  // positions of this warp's 16 that exist
      if (left > 0) {
        float sc[2][4] = {};
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          uint32_t b[4];
          ldsm4(b, key_frag<kTile>(sk, r0, ks, lane));
          mma16816<T>(sc[0], qf[ks][0], qf[ks][Q1], qf[ks][1], qf[ks][Q3], b[0], b[1]);
          mma16816<T>(sc[1], qf[ks][0], qf[ks][Q1], qf[ks][1], qf[ks][Q3], b[2], b[3]);
        }
        uint32_t hi[4], lo[4];
        float p[R][4];
#pragma unroll
        for (int e = 0; e < R; ++e) {
          float x[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            x[k] = sc[k >> 1][2 * e + (k & 1)] * sl2;
            if (left < 16 && (k >> 1) * 8 + c2 + (k & 1) >= left) x[k] = -INFINITY;
          }
          float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
          mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 2));
          if (__any_sync(kFull, mx > m[e])) {
            const float mn = fmaxf(m[e], mx), f = mn == -INFINITY ? 1.0f : ex2(m[e] - mn);
            m[e] = mn;
            l[e] *= f;
#pragma unroll
            for (int d = 0; d < HD / 8; ++d) {
              o[d][2 * e] *= f;
              o[d][2 * e + 1] *= f;
              if constexpr (ROWS == 8) {
                o[d][2] *= f;
                o[d][3] *= f;
              }
            }
          }
          const float base = (m[e] == -INFINITY ? 0.0f : m[e]) - kShift;
#pragma unroll
          for (int k = 0; k < 4; ++k) p[e][k] = ex2(x[k] - base);
          l[e] += (p[e][0] + p[e][1]) + (p[e][2] + p[e][3]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            hi[2 * k + e] = pack16<T>(p[e][2 * k], p[e][2 * k + 1]);
            const float2 q = unpack16<T>(hi[2 * k + e]);
            lo[2 * k + e] = pack16<T>(p[e][2 * k] - q.x, p[e][2 * k + 1] - q.y);
          }
        }
        // the values of positions that do not exist are whatever the page or the ring holds: zeros instead
        uint32_t keep[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
        if (left < 16) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
            keep[k] = (k * 8 + c2 < left ? 0xFFFFu : 0u) | (k * 8 + c2 + 1 < left ? 0xFFFF0000u : 0u);
        }
        // The second part of a weight may be negative or zero, so an infinite value would come out as NaN:
        // 16 N values of each position among which there is one (or a NaN) are summed weight by weight.
        constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
        constexpr int N = ROWS == 8 ? HD / 16 : 2;  // registers: with 16 rows all at once spill
#pragma unroll
        for (int n0 = 0; n0 < HD / 16; n0 += N) {
          uint32_t b[N][4], big = 0u;
#pragma unroll
          for (int nt = 0; nt < N; ++nt) {
            ldsm4_t(b[nt], value_frag<kTile>(sv, r0, n0 + nt, lane));
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              b[nt][k] &= keep[k & 1];
              big = __vmaxu2(big, b[nt][k] & 0x7FFF7FFFu);
            }
          }
          if (__any_sync(kFull, (big & 0xFFFFu) >= kInf || (big >> 16) >= kInf)) {
            add_values<T, HD, R, 2 * N>(o, 2 * n0, p, sv, r0, min(left, 16), lane);
            continue;
          }
#pragma unroll
          for (int nt = 0; nt < N; ++nt) {
            float(&o0)[4] = o[2 * (n0 + nt)], (&o1)[4] = o[2 * (n0 + nt) + 1];
            if constexpr (ROWS == 8) {
              mma16816<T>(o0, hi[0], lo[0], hi[2], lo[2], b[nt][0], b[nt][1]);
              mma16816<T>(o1, hi[0], lo[0], hi[2], lo[2], b[nt][2], b[nt][3]);
            } else {
              mma16816<T>(o0, hi[0], hi[1], hi[2], hi[3], b[nt][0], b[nt][1]);
              mma16816<T>(o0, lo[0], lo[1], lo[2], lo[3], b[nt][0], b[nt][1]);
              mma16816<T>(o1, hi[0], hi[1], hi[2], hi[3], b[nt][2], b[nt][3]);
              mma16816<T>(o1, lo[0], lo[1], lo[2], lo[3], b[nt][2], b[nt][3]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(empty + st));
    }

    // Join the four warps, 8 rows at a time: 2 -> 0 and 3 -> 1, then 1 -> 0.
    const bool whole = t0 == 0 && t1 == w.nt;
    const int slot = 2 * cta + (w.at == begin ? 0 : 1);
#pragma unroll
    for (int e = 0; e < R; ++e) {
      float v[HD / 8][2];
#pragma unroll
      for (int d = 0; d < HD / 8; ++d) {
        v[d][0] = ROWS == 8 ? o[d][0] + o[d][2] : o[d][2 * e];
        v[d][1] = ROWS == 8 ? o[d][1] + o[d][3] : o[d][2 * e + 1];
      }
      float mm = m[e], ll = l[e];
      ll += __shfl_xor_sync(kFull, ll, 1);
      ll += __shfl_xor_sync(kFull, ll, 2);
      auto give = [&](int at) {
        float* b = jbuf + (at * 8 + r) * L::kJoinRow;
#pragma unroll
        for (int d = 0; d < HD / 8; ++d) *reinterpret_cast<float2*>(b + d * 8 + c2) = make_float2(v[d][0], v[d][1]);
        if ((lane & 3) == 0) jml[at * 8 + r] = make_float2(mm, ll);
      };
      auto take = [&](int at) {
        const float* b = jbuf + (at * 8 + r) * L::kJoinRow;
        const float2 x = jml[at * 8 + r];
        const float mn = fmaxf(mm, x.x), mz = mn == -INFINITY ? 0.0f : mn, f0 = ex2(mm - mz), f1 = ex2(x.x - mz);
        mm = mn;
        ll = ll * f0 + x.y * f1;
#pragma unroll
        for (int d = 0; d < HD / 8; ++d) {
          const float2 y = *reinterpret_cast<const float2*>(b + d * 8 + c2);
          v[d][0] = v[d][0] * f0 + y.x * f1;
          v[d][1] = v[d][1] * f0 + y.y * f1;
        }
      };
      if (warp >= 2) give(warp - 2);
      consumer_bar_sync(kWarps * 32);
      if (warp < 2) take(warp);
      consumer_bar_sync(kWarps * 32);
      if (warp == 1) give(0);
      consumer_bar_sync(kWarps * 32);
      if (warp == 0) {
        take(0);
        const int row = 8 * e + r;
        if (whole) {
          const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
          if (row < nh) {
            O* out = static_cast<O*>(a.out) + ((long long)w.s * a.n_heads + j * g + h0 + row) * HD;
#pragma unroll
            for (int d = 0; d < HD / 8; ++d) {
              if constexpr (sizeof(O) == 4)
                *reinterpret_cast<float2*>(out + d * 8 + c2) = make_float2(v[d][0] * inv, v[d][1] * inv);
              else
                *reinterpret_cast<uint32_t*>(out + d * 8 + c2) = pack16<O>(v[d][0] * inv, v[d][1] * inv);
            }
          }
        } else {
          float* b = slots + (size_t)slot * slot_floats(ROWS, HD);
#pragma unroll
          for (int d = 0; d < HD / 8; ++d)
            __stcg(reinterpret_cast<float2*>(b + row * HD + d * 8 + c2), make_float2(v[d][0], v[d][1]));
          if ((lane & 3) == 0) {
            __stcg(b + ROWS * HD + row, mm);
            __stcg(b + ROWS * HD + ROWS + row, ll);
          }
        }
      }
      consumer_bar_sync(kWarps * 32);
    }
    if (t0 == 0 && !whole) {  // a split unit begins here (it is the range's last segment)
      split_unit = w.s * units + w.u;
      split_slot = slot;
      split_parts = deal.cta_of(w.first + w.nt - 1) - cta + 1;
    }
    w.at += t1 - t0;
    next = w.at < w.end;
    if (next) next_unit(w);
  }
  if (tid == 0) {
    Split x;
    x.unit = split_unit;
    x.parts = split_parts;
    x.slot = split_slot;
    x.pad = 0;
    __stcg(reinterpret_cast<int4*>(splits + cta), *reinterpret_cast<int4*>(&x));
  }
}

// Joins the parts of the split unit that began in CTA blockIdx.x.  Up to four parts (ordinary batches have two
// or three): block y = 0 takes all rows, a warp each.  More (a few long sequences): block y takes row y, its
// warps every eighth part, all maxima and sums first so that the outputs are independent loads.
template <class O, int HD, int ROWS>
__global__ void __launch_bounds__(256) attention_paged_join_kernel(const PagedArgs a, int n_kv, int zs) {
  constexpr int E = HD / 32;
  __shared__ float s_o[8][HD], s_f[kMaxCtas], s_red[8], s_sum[8];
  pdl_trigger();
  pdl_wait();
  const float* slots = static_cast<const float*>(a.workspace);
  const Split* splits = reinterpret_cast<const Split*>(slots + (size_t)kMaxCtas * 2 * slot_floats(ROWS, HD));
  const int c = blockIdx.x, row = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 raw = __ldcg(reinterpret_cast<const int4*>(splits + c));
  if (raw.x < 0) return;
  const int g = a.n_heads / n_kv, units = n_kv * zs, s = raw.x / units, u = raw.x % units, n = raw.y;
  const int h0 = (u % zs) * 16;
  auto part = [&](int p) { return slots + (size_t)(p ? 2 * (c + p) : raw.z) * slot_floats(ROWS, HD); };
  if (n <= 4) {
    if (blockIdx.y) return;
    for (int r = warp; r < min(16, g - h0); r += 8) {
      const float pm = lane < n ? __ldcg(part(lane) + ROWS * HD + r) : -INFINITY;
      const float pl = lane < n ? __ldcg(part(lane) + ROWS * HD + ROWS + r) : 0.0f;
      float m = pm;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
      const float f = ex2(pm - (m == -INFINITY ? 0.0f : m)), sum = warp_sum(f * pl);
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      float o[E] = {};
#pragma unroll 4
      for (int p = 0; p < n; ++p) {
        const float w = __shfl_sync(kFull, f, p);
        const float* b = part(p) + r * HD + lane * E;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(b + e));
          o[e] = fmaf(w, v.x, o[e]);
          o[e + 1] = fmaf(w, v.y, o[e + 1]);
        }
      }
      O* out = static_cast<O*>(a.out) + ((long long)s * a.n_heads + (u / zs) * g + h0 + r) * HD + lane * E;
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        if constexpr (sizeof(O) == 4) *reinterpret_cast<float2*>(out + e) = make_float2(o[e] * inv, o[e + 1] * inv);
        else *reinterpret_cast<uint32_t*>(out + e) = pack16<O>(o[e] * inv, o[e + 1] * inv);
      }
    }
    return;
  }
  if (row >= g - h0) return;
  // weights 2^(m_p - max) of the parts (at most two a thread) and the weighted sum
  float pm[2] = {-INFINITY, -INFINITY}, pl[2] = {0.0f, 0.0f};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int p = threadIdx.x + 256 * e;
    if (p < n) {
      pm[e] = __ldcg(part(p) + ROWS * HD + row);
      pl[e] = __ldcg(part(p) + ROWS * HD + ROWS + row);
    }
  }
  float m = fmaxf(pm[0], pm[1]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
  if (lane == 0) s_red[warp] = m;
  __syncthreads();
  m = s_red[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, s_red[i]);
  const float mz = m == -INFINITY ? 0.0f : m;
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int p = threadIdx.x + 256 * e;
    if (p < n) {
      const float f = ex2(pm[e] - mz);
      s_f[p] = f;
      sum += f * pl[e];
    }
  }
  sum = warp_sum(sum);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  float o[E] = {};
#pragma unroll 8
  for (int p = warp; p < n; p += 8) {
    const float* b = part(p) + row * HD + lane;
    const float f = s_f[p];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(f, __ldcg(b + 32 * e), o[e]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[warp][lane + 32 * e] = o[e];
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= HD) return;
  float v = 0.0f;
  sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v += s_o[i][d];
    sum += s_sum[i];
  }
  v *= sum == 0.0f ? 0.0f : 1.0f / sum;
  O* out = static_cast<O*>(a.out) + ((long long)s * a.n_heads + (u / zs) * g + h0 + row) * HD;
  if constexpr (sizeof(O) == 4) out[d] = v;
  else reinterpret_cast<unsigned short*>(out)[d] = (unsigned short)pack16<O>(v, 0.0f);
}

template <class T, class O, int HD, int ROWS>
cudaError_t launch_typed(const PagedArgs& a, const KvArgs& kv, cudaStream_t stream, unsigned* err) {
  using L = Layout<ROWS, HD>;
  auto kernel = attention_paged_kernel<T, O, HD, ROWS>;
  CUtensorMap kmap, vmap;
  const int box_rows = kv.page_size < kTile ? kv.page_size : kTile;
  if (!encode_kv_map(&kmap, kv, kv.k, box_rows) || !encode_kv_map(&vmap, kv, kv.v, box_rows))
    return cudaErrorInvalidValue;
  static std::atomic<unsigned long long> done{0};
  int sms = 0;
  cudaError_t e = kernel_setup(reinterpret_cast<const void*>(kernel), L::kSmem, done, &sms);
  if (e != cudaSuccess) return e;
  const int g = a.n_heads / kv.n_kv, zs = (g + 15) / 16;
  const int ctas = 2 * sms < kMaxCtas ? 2 * sms : kMaxCtas;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = L::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_opt_pdl.load() ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, kernel, kmap, vmap, a, kv, zs, box_rows, err);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3((unsigned)ctas, (unsigned)(g < 16 ? g : 16));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, attention_paged_join_kernel<O, HD, ROWS>, a, kv.n_kv, zs);
}

template <class T, class O, int HD>
cudaError_t launch_rows(const PagedArgs& a, const KvArgs& kv, cudaStream_t stream, unsigned* err) {
  return a.n_heads / kv.n_kv <= 8 ? launch_typed<T, O, HD, 8>(a, kv, stream, err)
                                  : launch_typed<T, O, HD, 16>(a, kv, stream, err);
}

template <class T>
cudaError_t launch_type(const PagedArgs& a, const KvArgs& kv, cudaStream_t stream, unsigned* err) {
  const bool f32 = a.out_dtype == kDtF32;
  if (kv.head_dim == 128)
    return f32 ? launch_rows<T, float, 128>(a, kv, stream, err) : launch_rows<T, T, 128>(a, kv, stream, err);
  return f32 ? launch_rows<T, float, 64>(a, kv, stream, err) : launch_rows<T, T, 64>(a, kv, stream, err);
}

}  // namespace

size_t attention_paged_workspace(int batch, int n_heads, int n_kv, int head_dim) {
  if (batch == 0) return 0;
  const int rows = n_heads / n_kv <= 8 ? 8 : 16;
  return (size_t)kMaxCtas * 2 * slot_floats(rows, head_dim) * sizeof(float) + kMaxCtas * sizeof(Split);
}

cudaError_t launch_attention_paged(const PagedArgs& a, const KvArgs& kv, cudaStream_t stream) {
  unsigned* err = device_error_word();
  if (!err) return cudaErrorUnknown;
  return kv.dtype == kDtF16 ? launch_type<__half>(a, kv, stream, err)
                            : launch_type<__nv_bfloat16>(a, kv, stream, err);
}

}  // namespace asmllm
