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
#include "paged_deal.cuh"
#include "pipeline.cuh"
#include "serving.cuh"
#include "tensor_map.cuh"

namespace asmllm {

namespace {

constexpr int kWarps = 4;   // consumer warps
constexpr int kStages = 3;
constexpr int kMaxCtas = 320;
constexpr int kThreads = (kWarps + 1) * 32;

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

  auto len = [&](int s, bool report) -> int {
    bool clipped;
    const int n = kv_length(kv, s, &clipped);
    if (clipped && report) atomicOr(err, kErrDecodeRange);
    return n;
  };
  auto none = [&](int s) {  // a sequence without positions: zeros, written by one CTA
    O* out = static_cast<O*>(a.out) + (long long)s * a.n_heads * HD;
    const float z[8] = {};
    for (int i = 0; i < a.n_heads * HD; i += 8) store8(out + i, z);
  };
  Walk w;
  Deal deal(0, 1);
  const bool any = deal_range<kThreads>(kv.batch, units, s_part, s_first, s_start, len, none, &w, &deal);

  float* slots = static_cast<float*>(a.workspace);
  Split* splits = reinterpret_cast<Split*>(slots + (size_t)kMaxCtas * 2 * slot_floats(ROWS, HD));
  if (!any) {
    if (tid == 0) splits[cta].unit = -1;
    return;
  }
  const long long begin = w.at;

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
        if (++w.t == w.nt) next_unit(w, units, len);
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
    if (next) next_unit(w, units, len);
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
  return cudaLaunchKernelEx(&cfg, attention_paged_join_kernel<O, HD, ROWS, kMaxCtas>, a, kv.n_kv, zs);
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
