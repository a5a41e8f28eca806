// asmllm_b200/csrc/paged_deal.cuh -- how the decode attentions whose warps work
// alone (attention_paged_q8.cu, attention_own.cu) deal out their work.
//
// A unit is one (sequence, KV head, up to 16 of its query heads); its
// positions are tiles.  The tiles of all units in a row are cut into one equal
// range per warp; a range covers whole units and at most two parts of units.
// Lengths live on the device, so each CTA sums them itself.
#pragma once

#include "matvec.cuh"
#include "mma16.cuh"
#include "serving.cuh"

namespace asmllm {

// Floats of a part: ROWS x (HD outputs, maximum, sum).
__host__ __device__ constexpr size_t slot_floats(int rows, int hd) { return (size_t)rows * hd + 2 * rows; }

// `total` tiles over `ranges`: the first `extra` have one more than the others.
struct Deal {
  long long each;
  int extra;
  __device__ __forceinline__ Deal(long long total, int ranges) {
    if (total < (1ll << 32)) {  // a 64-bit division costs hundreds of cycles
      each = (unsigned)total / (unsigned)ranges;
      extra = (int)((unsigned)total % (unsigned)ranges);
    } else {
      each = total / ranges;
      extra = (int)(total % ranges);
    }
  }
  __device__ __forceinline__ long long start(int c) const { return c * each + min(c, extra); }
  __device__ __forceinline__ int range_of(long long x) const {  // which holds tile x
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

// The range of this warp (W: a walk, whose sequence, positions and tiles load fills in).  load(s, w, report)
// gives a sequence's tiles, empty(w) is called in one thread of one CTA for a sequence without any.  Neighbouring ranges
// lie in different CTAs, so that few units spread over all SMs; a range has `least` tiles, but for the shortest, and as many
// more as it takes to cut no unit into more than about kMostParts, which its join reads one after the other (one unit of
// 131071 positions: 33 us, 58 with a part for each of 2368 warps; with one more sequence of a single position 33, 45 with
// twice the parts).
// s_part: THREADS values in shared memory.  Gives the range's number, or -1 where the warp has none.
constexpr int kMostParts = 1024;
template <int THREADS, class W, class Load, class Empty>
__device__ __forceinline__ int deal_warps(int batch, int units, int least, long long* s_part, Load load, Empty empty, W* w,
                                          Deal* deal) {
  constexpr int kWarps = THREADS / 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = (batch + THREADS - 1) / THREADS, q0 = min(batch, tid * per), q1 = min(batch, q0 + per);
  long long mine = 0;
  int longest = 0;
  for (int s = q0; s < q1; ++s) {
    const int nt = load(s, w, blockIdx.x == 0);
    mine += nt;
    longest = max(longest, nt);
    if (nt == 0 && s % gridDim.x == blockIdx.x) empty(*w);
  }
  mine *= units;
  long long x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(kFull, x, o);
    if (lane >= o) x += y;
  }
  longest = __reduce_max_sync(kFull, longest);
  if (lane == 31) {  // the warps' sums, then every thread's first tile
    s_part[warp] = x;
    s_part[kWarps + warp] = longest;
  }
  __syncthreads();
  long long before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    const long long y = s_part[i];
    before += i < warp ? y : 0;
    total += y;
    longest = max(longest, (int)s_part[kWarps + i]);
  }
  __syncthreads();
  s_part[tid] = before + x - mine;
  __syncthreads();
  long long count = (total + least - 1) / least;
  if (longest > kMostParts * least) {
    const int n = (longest + kMostParts - 1) / kMostParts;
    count = total < (1ll << 31) ? (long long)((unsigned)(total + n - 1) / (unsigned)n) : (total + n - 1) / n;
  }
  count = min((long long)gridDim.x * kWarps, count);
  const int index = warp * gridDim.x + blockIdx.x;
  *deal = Deal(total, (int)max(1ll, count));
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

}  // namespace asmllm
