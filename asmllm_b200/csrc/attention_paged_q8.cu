// asmllm_b200/csrc/attention_paged_q8.cu -- attention of one new token per
// sequence over a paged key-value cache in Q8_0.
//
//   out[s][h] = sum_p softmax_p(scale q[s][h] . (dk ck)[p][h / g]) (dv cv)[p][h / g]
// with codes c and a scale d for each block of 32 values; no position: zeros.
//
// The codes go into the matrix products as they are (an int8 is exact in
// fp16) and the scales stay outside: a score is the sum over the blocks of d
// times the block's product in fp32, and a block of values is added with the
// weights p d.  So nothing of the cache is rounded on the way.  The weights p
// d enter as hi + lo 16-bit parts (2^-22 of a weight, down to 2^-39 of the
// largest weight times the largest scale): d is held relative to a power of
// two, the largest d a warp has met, and the output is rescaled when that
// rises, as it is when the maximum does.  bf16 queries are scaled by a power
// of two per row into fp16's range, where their 8 bits are exact (those below
// 2^-31 of the row's largest round).
//
// 2 head_dim (1 + 1/16) bytes a position and KV head, read once.  The work is
// dealt out and joined as in attention_paged.cu.  A tile of 64 positions: codes
// by tensor copies, their scales (side by side in a page) by bulk copies.
// Fragments come from ldmatrix on pairs of codes: a word holds four values of
// one position (keys), or two values of two positions (values, transposed),
// and is split into its even and odd bytes.  The order of the values within a
// product is free as long as the query's is the same.
#include "matvec.cuh"
#include "mma16.cuh"
#include "paged_deal.cuh"
#include "pipeline.cuh"
#include "serving_q8.cuh"
#include "tensor_map.cuh"

namespace asmllm {

namespace {

constexpr int kWarps = 4;  // consumer warps
constexpr int kStages = 3;
constexpr int kMaxCtas = 448;
constexpr int kThreads = (kWarps + 1) * 32;

template <int ROWS, int HD>
struct LayoutQ8 {
  static constexpr int kCtasPerSm = ROWS == 8 ? 3 : 2;
  static constexpr int kCodes = kTile * HD;             // bytes of keys or values of a tile
  static constexpr int kScales = kTile * (HD / 32) * 2;
  static constexpr int kStageBytes = 2 * kCodes + 1024; // scales of keys and of values behind the codes
  static_assert(2 * kScales <= 1024 && kStageBytes % 1024 == 0, "stages are aligned for the swizzle");
  static constexpr int kJoinRow = HD + 4;               // floats: a row of the join buffer and its padding
  static constexpr int kJoinOff = kStages * kStageBytes;
  static constexpr int kMlOff = kJoinOff + 2 * 8 * kJoinRow * 4;
  static constexpr int kScaleOff = kMlOff + 2 * 8 * 8;  // 16 rows' factors
  static constexpr int kBarOff = kScaleOff + 64;
  static constexpr int kSmem = kBarOff + 2 * kStages * 8 + 64 + 1024;
  static constexpr int kQRow = HD * 2 + 16;
  static_assert(16 * kQRow <= 2 * 8 * kJoinRow * 4, "the query rows fit the join buffer");
};

// Byte offset of 16-byte chunk c of position r in a tile of HD-byte rows, as a tensor copy swizzles it.
template <int HD>
__device__ __forceinline__ uint32_t code_chunk(int r, int c) {
  return (uint32_t)(r * HD + ((HD == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4));
}

// Bytes 0 and 2 (odd: 1 and 3) of w, signed, as two fp16 values: 0x6400 + u is 1024 + u.
__device__ __forceinline__ uint32_t codes_even(uint32_t w) {
  const uint32_t x = (w & 0x00FF00FFu) ^ 0x64806480u;
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ uint32_t codes_odd(uint32_t w) { return codes_even(w >> 8); }

template <class T, class O, int HD, int ROWS>
__global__ void __launch_bounds__(kThreads, LayoutQ8<ROWS, HD>::kCtasPerSm)
attention_paged_q8_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                          const PagedArgs a, const KvQ8Args c, int zs, int box_rows, unsigned* __restrict__ err) {
  using L = LayoutQ8<ROWS, HD>;
  constexpr int B = HD / 32;  // blocks of a position
  const KvArgs& kv = c.kv;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* empty = full + kStages;
  volatile int* s_abort = reinterpret_cast<int*>(empty + kStages);
  int* s_start = reinterpret_cast<int*>(empty + kStages + 1);
  long long* s_first = reinterpret_cast<long long*>(empty + kStages + 2);
  long long* s_part = reinterpret_cast<long long*>(smem + L::kJoinOff);  // before the join uses it
  float* s_row = reinterpret_cast<float*>(smem + L::kScaleOff);

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
  auto none = [&](int s) {  // a sequence without positions: zeros
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
    // Lane i of a tile: page i / 4; of it keys' or values' codes, keys' or values' scales.
    const int pages_tile = kTile / box_rows, my_page = lane >> 2, what = lane & 3;
    const bool worker = my_page < pages_tile;
    const uint32_t code_bytes = (uint32_t)box_rows * HD, scale_bytes = (uint32_t)box_rows * (B * 2);
    auto lookup = [&](const Walk& x) -> int {  // n_pages for a bad one: zeros
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
      const uint32_t at_scales = 2 * L::kCodes + (what & 1) * L::kScales + my_page * scale_bytes;
      const bool codes = cur_page >= 0 && what < 2, scales = cur_page >= 0 && what >= 2 && cur_page < kv.n_pages;
      if (cur_page == kv.n_pages && what >= 2)  // no page: the copy of the codes gives zeros, the scales have to be set
        for (uint32_t b = 0; b < scale_bytes; b += 16)
          *reinterpret_cast<uint4*>(smem + st * L::kStageBytes + at_scales + b) = make_uint4(0u, 0u, 0u, 0u);
      const unsigned nc = __popc(__ballot_sync(kFull, codes)), ns = __popc(__ballot_sync(kFull, scales));
      if (lane == 0) mbar_arrive_expect_tx(bar, code_bytes * nc + scale_bytes * ns);
      __syncwarp();
      const int p = cur.t * kTile + my_page * box_rows, in = p & (kv.page_size - 1), head = cur.u / zs;
      if (codes) {
        tma_load_4d(dst + what * L::kCodes + my_page * code_bytes, what ? &vmap : &kmap, 0, in, head, cur_page, bar);
      } else if (scales) {
        const __half* src = (what & 1 ? c.vs : c.ks) + (long long)cur_page * c.scale_page_stride +
                            (long long)head * c.scale_head_stride + in * B;
        bulk_g2s(dst + at_scales, src, scale_bytes, bar);
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
  const int r = lane >> 2, t4 = lane & 3, c2 = t4 * 2;
  float* jbuf = reinterpret_cast<float*>(smem + L::kJoinOff);
  float2* jml = reinterpret_cast<float2*>(smem + L::kMlOff);
  bool ok = true;
  int i = 0, split_unit = -1, split_parts = 0, split_slot = 0;
  bool next = true;
  while (next) {
    // one segment: tiles w.t .. of unit (w.s, w.u)
    const int j = w.u / zs, h0 = (w.u % zs) * 16, nh = min(16, g - h0);
    const int t0 = w.t, t1 = (int)min((long long)w.nt, w.t + (w.end - w.at));
    constexpr int R = ROWS / 8;
    // The unit's query rows in fp16, read once by the CTA, then as fragments.  Thread: 8 values of a row.
    uint32_t qf[2 * B][2 * R];  // step 2 b + s: values 32 b + 16 s ..; [2 e]: 4 t4 and 4 t4 + 2 of row r + 8 e, [2 e + 1]: the next ones
    float rs[R];                // a score is this times its row's product
    {
      const T* qb = static_cast<const T*>(a.q) + w.s * a.q_row_stride + (long long)(j * g + h0) * a.q_head_stride;
      unsigned char* sq = smem + L::kJoinOff;
      for (int e = tid; e < ROWS * (HD / 8); e += kWarps * 32) {
        const int row = e / (HD / 8), x = e % (HD / 8);
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (row < nh) v = __ldcg(reinterpret_cast<const uint4*>(qb + row * a.q_head_stride) + x);
        if constexpr (!std::is_same<T, __half>::value) {
          const uint32_t wd[4] = {v.x, v.y, v.z, v.w};
          float f[8], top = 0.0f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 y = unpack16<T>(wd[k]);
            f[2 * k] = y.x;
            f[2 * k + 1] = y.y;
            top = fmaxf(top, fmaxf(fabsf(y.x), fabsf(y.y)));
          }
#pragma unroll
          for (int o = HD / 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
          // 2^n times the row with the largest value in [2^14, 2^15); an infinity leaves the row as it is
          const int ex = (int)(__float_as_uint(top) >> 23) - 127, n = ex > 127 || top == 0.0f ? 0 : min(14 - ex, 100);
          const float up = __uint_as_float((unsigned)(127 + n) << 23);
          if (x == 0) s_row[row] = sl2 * __uint_as_float((unsigned)(127 - n) << 23);
          v.x = pack16<__half>(f[0] * up, f[1] * up);
          v.y = pack16<__half>(f[2] * up, f[3] * up);
          v.z = pack16<__half>(f[4] * up, f[5] * up);
          v.w = pack16<__half>(f[6] * up, f[7] * up);
        }
        *reinterpret_cast<uint4*>(sq + row * L::kQRow + x * 16) = v;
      }
      consumer_bar_sync(kWarps * 32);
#pragma unroll
      for (int e = 0; e < R; ++e) {
        rs[e] = std::is_same<T, __half>::value ? sl2 : s_row[r + 8 * e];
#pragma unroll
        for (int k = 0; k < 2 * B; ++k) {
          const uint2 x = *reinterpret_cast<const uint2*>(sq + (r + 8 * e) * L::kQRow + k * 32 + t4 * 8);
          qf[k][2 * e] = __byte_perm(x.x, x.y, 0x5410);
          qf[k][2 * e + 1] = __byte_perm(x.x, x.y, 0x7632);
        }
      }
      consumer_bar_sync(kWarps * 32);  // the buffer is the join's again
    }
    // with ROWS == 8, rows 8-15 repeat rows 0-7: their scores are the same numbers
    constexpr int Q1 = ROWS == 16 ? 2 : 0, Q3 = ROWS == 16 ? 3 : 1;
    // o[x]: values 16 x + 4 t4 .. + 3 of rows r and r + 8: [0] and [2] the even ones of row r, [1] the odd ones'
    float o[HD / 16][2][4], m[R], l[R];
    unsigned top = 0x0400u;  // exponent of the largest scale met, as an fp16 power of two
    float inv = 16384.0f;    // 1 / it
#pragma unroll
    for (int e = 0; e < R; ++e) {
      m[e] = -INFINITY;
      l[e] = 0.0f;
    }
#pragma unroll
    for (int e = 0; e < HD / 16; ++e)
#pragma unroll
      for (int k = 0; k < 2; ++k) o[e][k][0] = o[e][k][1] = o[e][k][2] = o[e][k][3] = 0.0f;

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
      const uint32_t sk = ring + st * L::kStageBytes, sv = sk + L::kCodes;
      const unsigned char* sc = smem + st * L::kStageBytes + 2 * L::kCodes;
      const int r0 = warp * 16, left = w.n - t * kTile - r0;  // positions of this warp's 16 that exist
      if (left > 0) {
        // scales of positions c2, c2 + 1, c2 + 8, c2 + 9: B halves each
        uint32_t ks[4][B / 2], vs[4][B / 2];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int p = r0 + c2 + (k & 1) + 8 * (k >> 1);
          if constexpr (B == 4) {
            const uint2 x = *reinterpret_cast<const uint2*>(sc + p * 8);
            const uint2 y = *reinterpret_cast<const uint2*>(sc + L::kScales + p * 8);
            ks[k][0] = x.x; ks[k][1] = x.y;
            vs[k][0] = y.x; vs[k][1] = y.y;
          } else {
            ks[k][0] = *reinterpret_cast<const uint32_t*>(sc + p * 4);
            vs[k][0] = *reinterpret_cast<const uint32_t*>(sc + L::kScales + p * 4);
          }
          if (left < 16 && c2 + (k & 1) + 8 * (k >> 1) >= left) {  // whatever the page or the ring holds
#pragma unroll
            for (int b = 0; b < B / 2; ++b) vs[k][b] = 0u;
          }
        }
        float s[R][4] = {};
#pragma unroll
        for (int b = 0; b < B; ++b) {
          uint32_t f[4];  // chunk 2 b of positions 0-7, chunk 2 b + 1; the same of positions 8-15
          ldsm4(f, sk + code_chunk<HD>(r0 + (lane >> 4) * 8 + (lane & 7), 2 * b + ((lane >> 3) & 1)));
          float x[2][4] = {};
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t(&q)[2 * R] = qf[2 * b + u];
            mma16816<__half>(x[0], q[0], q[Q1], q[1], q[Q3], codes_even(f[u]), codes_odd(f[u]));
            mma16816<__half>(x[1], q[0], q[Q1], q[1], q[Q3], codes_even(f[2 + u]), codes_odd(f[2 + u]));
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 d2 = unpack16<__half>(ks[k][b >> 1]);
            const float d = b & 1 ? d2.y : d2.x;
#pragma unroll
            for (int e = 0; e < R; ++e) s[e][k] = fmaf(x[k >> 1][2 * e + (k & 1)], d, s[e][k]);
          }
        }
        // the largest finite scale so far: o is held in units of a power of two no larger than it
        auto largest = [&](bool finite) -> unsigned {
          unsigned x = 0u;
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int b = 0; b < B / 2; ++b) {
              unsigned y = vs[k][b] & 0x7FFF7FFFu;
              if (finite) y &= ~__vcmpgeu2(y, 0x7C007C00u);
              x = __vmaxu2(x, y);
            }
          x = max(x & 0xFFFFu, x >> 16);
          x = max(x, __shfl_xor_sync(kFull, x, 1));
          return max(x, __shfl_xor_sync(kFull, x, 2));
        };
        unsigned big = largest(false);
        if (big >= 0x7C00u) big = largest(true);
        big &= 0x7C00u;
        if (big > top) {  // the same in every lane
          const float f = __uint_as_float((127u << 23) - ((big - top) << 13));
          top = big;
          inv *= f;
#pragma unroll
          for (int e = 0; e < HD / 16; ++e)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int z = 0; z < 4; ++z) o[e][k][z] *= f;
        }
        float p[R][4];
#pragma unroll
        for (int e = 0; e < R; ++e) {
          float x[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            x[k] = s[e][k] * rs[e];
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
            for (int d = 0; d < HD / 16; ++d)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                o[d][k][2 * e] *= f;
                o[d][k][2 * e + 1] *= f;
                if constexpr (ROWS == 8) {
                  o[d][k][2] *= f;
                  o[d][k][3] *= f;
                }
              }
          }
          const float base = (m[e] == -INFINITY ? 0.0f : m[e]) - kShift;
#pragma unroll
          for (int k = 0; k < 4; ++k) p[e][k] = ex2(x[k] - base);
          l[e] += (p[e][0] + p[e][1]) + (p[e][2] + p[e][3]);
#pragma unroll
          for (int k = 0; k < 4; ++k) p[e][k] *= inv;
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
          uint32_t hi[2 * R], lo[2 * R];  // [2 k + e] of rows r + 8 e
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 d0 = unpack16<__half>(vs[2 * k][b >> 1]), d1 = unpack16<__half>(vs[2 * k + 1][b >> 1]);
            const float y0 = b & 1 ? d0.y : d0.x, y1 = b & 1 ? d1.y : d1.x;
#pragma unroll
            for (int e = 0; e < R; ++e) {
              const float w0 = p[e][2 * k] * y0, w1 = p[e][2 * k + 1] * y1;
              hi[R * k + e] = pack16<__half>(w0, w1);
              const float2 q = unpack16<__half>(hi[R * k + e]);
              lo[R * k + e] = pack16<__half>(w0 - q.x, w1 - q.y);
            }
          }
          uint32_t f[4];  // chunk 2 b of positions 0-7 and 8-15, the same of chunk 2 b + 1
          ldsm4_t(f, sv + code_chunk<HD>(r0 + ((lane >> 3) & 1) * 8 + (lane & 7), 2 * b + (lane >> 4)));
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float(&o0)[4] = o[2 * b + x][0], (&o1)[4] = o[2 * b + x][1];
            const uint32_t e0 = codes_even(f[2 * x]), e1 = codes_even(f[2 * x + 1]);
            const uint32_t u0 = codes_odd(f[2 * x]), u1 = codes_odd(f[2 * x + 1]);
            if constexpr (ROWS == 8) {
              mma16816<__half>(o0, hi[0], lo[0], hi[1], lo[1], e0, e1);
              mma16816<__half>(o1, hi[0], lo[0], hi[1], lo[1], u0, u1);
            } else {
              mma16816<__half>(o0, hi[0], hi[1], hi[2], hi[3], e0, e1);
              mma16816<__half>(o0, lo[0], lo[1], lo[2], lo[3], e0, e1);
              mma16816<__half>(o1, hi[0], hi[1], hi[2], hi[3], u0, u1);
              mma16816<__half>(o1, lo[0], lo[1], lo[2], lo[3], u0, u1);
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
    const float unit = 1.0f / inv;
#pragma unroll
    for (int e = 0; e < R; ++e) {
      float v[HD / 16][4];
#pragma unroll
      for (int d = 0; d < HD / 16; ++d)
#pragma unroll
        for (int k = 0; k < 4; ++k)  // value 4 t4 + k
          v[d][k] = unit * (ROWS == 8 ? o[d][k & 1][k >> 1] + o[d][k & 1][2 + (k >> 1)] : o[d][k & 1][2 * e + (k >> 1)]);
      float mm = m[e], ll = l[e];
      ll += __shfl_xor_sync(kFull, ll, 1);
      ll += __shfl_xor_sync(kFull, ll, 2);
      auto give = [&](int at) {
        float* b = jbuf + (at * 8 + r) * L::kJoinRow + 4 * t4;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) *reinterpret_cast<float4*>(b + d * 16) = make_float4(v[d][0], v[d][1], v[d][2], v[d][3]);
        if (t4 == 0) jml[at * 8 + r] = make_float2(mm, ll);
      };
      auto take = [&](int at) {
        const float* b = jbuf + (at * 8 + r) * L::kJoinRow + 4 * t4;
        const float2 x = jml[at * 8 + r];
        const float mn = fmaxf(mm, x.x), mz = mn == -INFINITY ? 0.0f : mn, f0 = ex2(mm - mz), f1 = ex2(x.x - mz);
        mm = mn;
        ll = ll * f0 + x.y * f1;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) {
          const float4 y = *reinterpret_cast<const float4*>(b + d * 16);
          v[d][0] = v[d][0] * f0 + y.x * f1;
          v[d][1] = v[d][1] * f0 + y.y * f1;
          v[d][2] = v[d][2] * f0 + y.z * f1;
          v[d][3] = v[d][3] * f0 + y.w * f1;
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
          const float d = ll == 0.0f ? 0.0f : 1.0f / ll;
          if (row < nh) {
            O* out = static_cast<O*>(a.out) + ((long long)w.s * a.n_heads + j * g + h0 + row) * HD + 4 * t4;
#pragma unroll
            for (int x = 0; x < HD / 16; ++x) {
              if constexpr (sizeof(O) == 4)
                *reinterpret_cast<float4*>(out + x * 16) = make_float4(v[x][0] * d, v[x][1] * d, v[x][2] * d, v[x][3] * d);
              else
                *reinterpret_cast<uint2*>(out + x * 16) = make_uint2(pack16<O>(v[x][0] * d, v[x][1] * d),
                                                                    pack16<O>(v[x][2] * d, v[x][3] * d));
            }
          }
        } else {
          float* b = slots + (size_t)slot * slot_floats(ROWS, HD);
#pragma unroll
          for (int x = 0; x < HD / 16; ++x)
            __stcg(reinterpret_cast<float4*>(b + row * HD + x * 16 + 4 * t4), make_float4(v[x][0], v[x][1], v[x][2], v[x][3]));
          if (t4 == 0) {
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
  if (tid == 0) __stcg(reinterpret_cast<int4*>(splits + cta), make_int4(split_unit, split_parts, split_slot, 0));
}

// Codes of keys or values: (value, offset in page, KV head, page), bytes, a box a page and head.
template <int HD>
bool encode_codes(CUtensorMap* map, const KvArgs& kv, const void* base, int box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 encode = tensor_map_encode_fn();
  if (!encode) return false;
  const cuuint64_t dim[4] = {(cuuint64_t)HD, (cuuint64_t)kv.page_size, (cuuint64_t)kv.n_kv, (cuuint64_t)kv.n_pages};
  const cuuint64_t stride[3] = {(cuuint64_t)kv.token_stride, (cuuint64_t)kv.head_stride, (cuuint64_t)kv.page_stride};
  const cuuint32_t box[4] = {(cuuint32_t)HD, (cuuint32_t)box_rows, 1u, 1u}, step[4] = {1u, 1u, 1u, 1u};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dim, stride, box, step,
                CU_TENSOR_MAP_INTERLEAVE_NONE, HD == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, class O, int HD, int ROWS>
cudaError_t launch_typed(const PagedArgs& a, const KvQ8Args& c, cudaStream_t stream, unsigned* err) {
  using L = LayoutQ8<ROWS, HD>;
  const KvArgs& kv = c.kv;
  auto kernel = attention_paged_q8_kernel<T, O, HD, ROWS>;
  CUtensorMap kmap, vmap;
  const int box_rows = kv.page_size < kTile ? kv.page_size : kTile;
  if (!encode_codes<HD>(&kmap, kv, kv.k, box_rows) || !encode_codes<HD>(&vmap, kv, kv.v, box_rows))
    return cudaErrorInvalidValue;
  static std::atomic<unsigned long long> done{0};
  int sms = 0;
  cudaError_t e = kernel_setup(reinterpret_cast<const void*>(kernel), L::kSmem, done, &sms);
  if (e != cudaSuccess) return e;
  const int g = a.n_heads / kv.n_kv, zs = (g + 15) / 16;
  const int ctas = L::kCtasPerSm * sms < kMaxCtas ? L::kCtasPerSm * sms : kMaxCtas;
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
  e = cudaLaunchKernelEx(&cfg, kernel, kmap, vmap, a, c, zs, box_rows, err);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3((unsigned)ctas, (unsigned)(g < 16 ? g : 16));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, attention_paged_join_kernel<O, HD, ROWS, kMaxCtas>, a, kv.n_kv, zs);
}

template <class T, class O, int HD>
cudaError_t launch_rows(const PagedArgs& a, const KvQ8Args& c, cudaStream_t stream, unsigned* err) {
  return a.n_heads / c.kv.n_kv <= 8 ? launch_typed<T, O, HD, 8>(a, c, stream, err)
                                    : launch_typed<T, O, HD, 16>(a, c, stream, err);
}

template <class T>
cudaError_t launch_type(const PagedArgs& a, const KvQ8Args& c, cudaStream_t stream, unsigned* err) {
  const bool f32 = a.out_dtype == kDtF32;
  if (c.kv.head_dim == 128)
    return f32 ? launch_rows<T, float, 128>(a, c, stream, err) : launch_rows<T, T, 128>(a, c, stream, err);
  return f32 ? launch_rows<T, float, 64>(a, c, stream, err) : launch_rows<T, T, 64>(a, c, stream, err);
}

}  // namespace

size_t attention_paged_q8_workspace(int batch, int n_heads, int n_kv, int head_dim) {
  if (batch == 0) return 0;
  const int rows = n_heads / n_kv <= 8 ? 8 : 16;
  return (size_t)kMaxCtas * 2 * slot_floats(rows, head_dim) * sizeof(float) + kMaxCtas * sizeof(Split);
}

cudaError_t launch_attention_paged_q8(const PagedArgs& a, int q_dtype, const KvQ8Args& c, cudaStream_t stream) {
  unsigned* err = device_error_word();
  if (!err) return cudaErrorUnknown;
  return q_dtype == kDtF16 ? launch_type<__half>(a, c, stream, err) : launch_type<__nv_bfloat16>(a, c, stream, err);
}

}  // namespace asmllm
