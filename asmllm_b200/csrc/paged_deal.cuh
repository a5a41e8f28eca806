// asmllm_b200/csrc/paged_deal.cuh -- how the decode attentions over pages
// deal out their work, and the join of units that lie in several CTAs.
//
// A unit is one (sequence, KV head, up to 16 of its query heads); its
// positions are tiles.  The tiles of all units in a row are cut into one equal
// range per CTA (attention_paged.cu, tiles of kTile) or per warp; a range
// covers whole units and at most two parts of units.  Lengths live on the
// device, so each CTA sums them itself.
#pragma once

#include "matvec.cuh"
#include "mma16.cuh"
#include "serving.cuh"

namespace asmllm {

constexpr int kTile = 64;  // positions per tile, 16 per consumer warp

// Parts of split units: [ctas][2] slots of ROWS x (HD outputs, maximum, sum),
// then one Split per CTA: the split unit that begins in its range.
struct Split {
  int unit;   // -1: none
  int parts;  // CTAs c .. c + parts - 1 hold one each
  int slot;   // slot of the first part (the others are in slot 2 c)
  int pad;
};

__host__ __device__ constexpr size_t slot_floats(int rows, int hd) { return (size_t)rows * hd + 2 * rows; }

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

// The transpose of an 8 x 8 matrix of 16-bit values (lane: row lane / 4, columns 2 (lane % 4) and the next).
__device__ __forceinline__ uint32_t transposed8(uint32_t w) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
  return r;
}

// A CTA's walk over its tiles: sequence, unit of the sequence, tile.
struct Walk {
  int s, u, t, n, nt;      // n positions, nt tiles of sequence s
  long long first;         // number of the unit's first tile
  long long at, end;       // tiles [at, end) are left
};

// The range of this warp where every warp of the grid has its own (W: a walk; its n and nt are load's).  load(s, w, report)
// gives a sequence's tiles, empty(w) is called in one thread of one CTA for a sequence without any.  Neighbouring ranges
// lie in different CTAs, so that few units spread over all SMs; a range has `least` tiles, but for the shortest, and there
// are at most kMostParts for each unit, whose parts the join reads (one unit of 131071 positions: 33 us, 58 with one for
// each of 2368 warps).
// s_part: THREADS + 1 values in shared memory.  Gives the range's number, or -1 where the warp has none.
constexpr int kMostParts = 1024;
template <int THREADS, class W, class Load, class Empty>
__device__ __forceinline__ int deal_warps(int batch, int units, int least, long long* s_part, Load load, Empty empty, W* w,
                                          Deal* deal) {
  constexpr int kWarps = THREADS / 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = (batch + THREADS - 1) / THREADS, q0 = min(batch, tid * per), q1 = min(batch, q0 + per);
  long long mine = 0;
  for (int s = q0; s < q1; ++s) {
    const int nt = load(s, w, blockIdx.x == 0);
    mine += nt;
    if (nt == 0 && s % gridDim.x == blockIdx.x) empty(*w);
  }
  mine *= units;
  long long x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(kFull, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) s_part[warp] = x;  // the warps' sums, then every thread's first tile
  __syncthreads();
  long long before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    const long long y = s_part[i];
    before += i < warp ? y : 0;
    total += y;
  }
  __syncthreads();
  s_part[tid] = before + x - mine;
  __syncthreads();
  const int count = (int)min(min((long long)gridDim.x * kWarps, (long long)batch * units * kMostParts), (total + least - 1) / least);
  const int index = warp * gridDim.x + blockIdx.x;
  *deal = Deal(total, max(1, count));
  const long long begin = index < count ? deal->start(index) : 0, end = index < count ? deal->start(index + 1) : 0;
  if (begin >= end) return -1;
  // the last thread whose sequences begin at or before the range (those behind it with the same number have none)
  int lo = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    const unsigned hit = __ballot_sync(kFull, s_part[32 * i + lane] <= begin);
    if (hit) lo = 32 * i + 31 - __clz(hit);
  }
  x = s_part[lo];
  for (int s = lo * per;; ++s) {
    const long long t = (long long)load(s, w, false) * units;
    if (begin < x + t) break;
    x += t;
  }
  const long long into = begin - x;
  w->u = (int)(into / w->nt);
  w->first = x + (long long)w->u * w->nt;
  w->t = (int)(begin - w->first);
  w->at = begin;
  w->end = end;
  return index;
}

// The range of this CTA (of THREADS threads): false when it has none.  len(s, report) is a sequence's positions
// (report: bad lengths are to be reported), empty(s) is called in one thread of one CTA for a sequence without any.
// s_part: THREADS values, s_first: 2, s_start: 2, in shared memory; s_part is free again after the next barrier.
template <int THREADS, class Len, class Empty>
__device__ __forceinline__ bool deal_range(int batch, int units, long long* s_part, long long* s_first, int* s_start,
                                           Len len, Empty empty, Walk* w, Deal* deal) {
  // Sum of all tiles and the sequence this range begins in: a contiguous share of the sequences per thread.
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
  const int per = (batch + THREADS - 1) / THREADS, q0 = min(batch, tid * per), q1 = min(batch, q0 + per);
  long long mine = 0;
  int held = 0;  // positions of the thread's first sequence
  for (int s = q0; s < q1; ++s) {
    const int n = len(s, cta == 0);
    if (s == q0) held = n;
    mine += tiles_of(n);
    if (n == 0 && s % gridDim.x == cta) empty(s);
  }
  mine *= units;
  s_part[tid] = mine;
  __syncthreads();
  if (warp == 0) {
    long long run = 0;
    for (int b = 0; b < THREADS; b += 32) {
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
  *deal = Deal(total, max(1, ctas));
  const long long begin = cta < ctas ? deal->start(cta) : 0, end = cta < ctas ? deal->start(cta + 1) : 0;
  if (begin < end && s_part[tid] <= begin && begin < s_part[tid] + mine) {
    long long x = s_part[tid];
    for (int s = q0; s < q1; ++s) {
      const int n = s == q0 ? held : len(s, false);
      const long long t = (long long)tiles_of(n) * units;
      if (begin < x + t) {
        s_start[0] = s;
        s_start[1] = n;
        s_first[0] = x;
        break;
      }
      x += t;
    }
  }
  __syncthreads();
  if (begin >= end) return false;
  w->s = s_start[0];
  w->n = s_start[1];
  w->nt = tiles_of(w->n);
  const long long into = begin - s_first[0];
  w->u = into < (1ll << 32) ? (int)((unsigned)into / (unsigned)w->nt) : (int)(into / w->nt);
  w->first = s_first[0] + (long long)w->u * w->nt;
  w->t = (int)(begin - w->first);
  w->at = begin;
  w->end = end;
  return true;
}

// The next unit, of this sequence or the next one that holds positions.
template <class Len>
__device__ __forceinline__ void next_unit(Walk& x, int units, Len len) {
  x.first += x.nt;
  x.t = 0;
  if (++x.u == units) {
    x.u = 0;
    do {
      ++x.s;
      x.n = len(x.s, false);
    } while (x.n == 0);
    x.nt = tiles_of(x.n);
  }
}

// Joins the parts of the split unit that began in CTA blockIdx.x.  Up to four parts (ordinary batches have two
// or three): block y = 0 takes all rows, a warp each.  More (a few long sequences): block y takes row y, its
// warps every eighth part, all maxima and sums first so that the outputs are independent loads.
template <class O, int HD, int ROWS, int CTAS>
__global__ void __launch_bounds__(256) attention_paged_join_kernel(const PagedArgs a, int n_kv, int zs) {
  constexpr int E = HD / 32;
  static_assert(CTAS <= 512, "at most two parts a thread");
  __shared__ float s_o[8][HD], s_f[CTAS], s_red[8], s_sum[8];
  pdl_trigger();
  pdl_wait();
  const float* slots = static_cast<const float*>(a.workspace);
  const Split* splits = reinterpret_cast<const Split*>(slots + (size_t)CTAS * 2 * slot_floats(ROWS, HD));
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

}  // namespace asmllm
