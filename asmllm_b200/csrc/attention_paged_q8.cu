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
// and their products with d are hi + lo 16-bit parts (2^-22 of a weight, down
// to 2^-34 of the largest weight times its block's largest scale): d is held
// relative to a power of two, the largest d of its block that a warp has met,
// and the block's output is rescaled when that rises, as it is when the
// maximum does.  bf16 queries are scaled by a power
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
//
// Measured on one B200, 64 sequences of 64 query and 8 KV heads of 128 values
// that hold up to 16384 positions: 235 us (5.1 TB/s; the copy takes 184).  Codes
// to fp16 and the scales are most of its instructions, 505 for 16 positions and
// a warp, which issue in 55 % of the cycles.  355 for the fp16 cache of twice the
// bytes (attention_paged.cu).  With positions as the right side, padded to 8
// rows of heads as the left, 341; with 4 CTAs an SM of 2 stages 273, not 3 of 3.
// 32 sequences of 1 to 1024: 22 us.  One of 32 heads and 512 positions: 10.
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
// The output is rescaled only when a row's maximum has risen by more than 2^kLazy since it was last set; the weights,
// 2^kPShift exp(s - m), stay below 2^15 then.
constexpr float kLazy = 5.0f, kPShift = 9.0f;

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

// The four signed bytes of w as fp16: 0 and 2, and 1 and 3.  With the sign bit turned a byte is u = code + 128, and
// 0x6400 + u is 1024 + u.
__device__ __forceinline__ void codes_of(uint32_t w, uint32_t& even, uint32_t& odd) {
  const uint32_t u = w ^ 0x80808080u, e = __byte_perm(u, 0x64646464u, 0x4240), o = __byte_perm(u, 0x64646464u, 0x4341);
  const __half2 base = __half2half2(__ushort_as_half(0x6480));
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&e), base), y = __hsub2(*reinterpret_cast<const __half2*>(&o), base);
  even = *reinterpret_cast<const uint32_t*>(&x);
  odd = *reinterpret_cast<const uint32_t*>(&y);
}

// c += a b, and c = a b, as mma16816 but free to be moved among the conversions.
__device__ __forceinline__ void product(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void first_product(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ __half2 as_half2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
__device__ __forceinline__ uint32_t as_word(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

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
  constexpr int N = ROWS / 8;  // groups of 8 query heads
  const uint32_t ring = smem_u32(smem);
  const float sl2 = a.scale * 1.4426950408889634f;
  const int r = lane >> 2, t4 = lane & 3, c2 = t4 * 2, r0 = warp * 16;
  float* jbuf = reinterpret_cast<float*>(smem + L::kJoinOff);
  float2* jml = reinterpret_cast<float2*>(smem + L::kMlOff);
  // Fragments' places in a tile: chunk 2 b of keys is at key_at ^ 32 b (positions 0-7, chunk + 1, positions 8-15, chunk
  // + 1), values at value_at ^ 32 b (positions 0-7, 8-15, the same of chunk + 1).
  const uint32_t key_at = code_chunk<HD>(r0 + (lane >> 4) * 8 + (lane & 7), (lane >> 3) & 1);
  const uint32_t value_at = code_chunk<HD>(r0 + ((lane >> 3) & 1) * 8 + (lane & 7), lane >> 4);
  bool ok = true;
  int st = 0, phase = 0, split_unit = -1, split_parts = 0, split_slot = 0;
  bool next = true;
  while (next) {
    // one segment: tiles w.t .. of unit (w.s, w.u)
    const int j = w.u / zs, h0 = (w.u % zs) * 16, nh = min(16, g - h0);
    const int t0 = w.t, t1 = (int)min((long long)w.nt, w.t + (w.end - w.at));
    // The unit's query rows in fp16, read once by the CTA (thread: 8 values of a row), then as fragments: those of head
    // 8 n + r, values 32 b + 16 s + 4 t4 and + 2 in [0] of step 2 b + s, + 1 and + 3 in [1].
    uint32_t qf[N][2 * B][2];
    float rs[N][2];  // a score of head 8 n + c2 + e is this times its product
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
      for (int n = 0; n < N; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) rs[n][e] = std::is_same<T, __half>::value ? sl2 : s_row[8 * n + c2 + e];
#pragma unroll
        for (int k = 0; k < 2 * B; ++k) {
          const uint2 x = *reinterpret_cast<const uint2*>(sq + (8 * n + r) * L::kQRow + k * 32 + t4 * 8);
          qf[n][k][0] = __byte_perm(x.x, x.y, 0x5410);
          qf[n][k][1] = __byte_perm(x.x, x.y, 0x7632);
        }
      }
      consumer_bar_sync(kWarps * 32);  // the buffer is the join's again
    }
    // o[n][x]: values 16 x + 2 r ([0], [1]) and the next ([2], [3]) of heads 8 n + c2 and the next
    float o[N][HD / 16][4], m[N][2], l[N][2];
    // largest scales met, as fp16 powers of two, and one over them: two blocks a word
    unsigned top[B / 2], inv[B / 2];
#pragma unroll
    for (int b = 0; b < B / 2; ++b) {
      top[b] = 0x04000400u;
      inv[b] = 0x74007400u;
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.0f;
#pragma unroll
      for (int e = 0; e < HD / 16; ++e) o[n][e][0] = o[n][e][1] = o[n][e][2] = o[n][e][3] = 0.0f;
    }

    for (int t = t0; t < t1; ++t) {
      if (!__all_sync(kFull, ok && mbar_try_wait(smem_u32(full + st), phase))) {
        if (ok) ok = mbar_wait_bounded(smem_u32(full + st), phase) && !*s_abort;
        ok = __all_sync(kFull, ok);
      }
      if (!ok) {  // give up: keep in step with the other warps, but touch no more tiles
        if (lane == 0) {
          *s_abort = 1;
          atomicOr(err, kErrRingTimeout);
        }
        continue;
      }
      const uint32_t sk = ring + st * L::kStageBytes;
      const unsigned char* sc = smem + st * L::kStageBytes + 2 * L::kCodes;
      const int left = w.n - t * kTile - r0;  // positions of this warp's 16 that exist
      if (left > 0) {
        // scores of positions r ([0], [1]) and r + 8, heads 8 n + c2 and the next
        float s[N][4] = {};
        {
          uint32_t d[2][B / 2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const unsigned char* at = sc + (r0 + r + 8 * k) * (2 * B);
            if constexpr (B == 4) {
              const uint2 x = *reinterpret_cast<const uint2*>(at);
              d[k][0] = x.x;
              d[k][1] = x.y;
            } else {
              d[k][0] = *reinterpret_cast<const uint32_t*>(at);
            }
          }
          const uint32_t at = sk + key_at;
#pragma unroll
          for (int b = 0; b < B; ++b) {
            uint32_t f[4], c[8];
            ldsm4(f, at ^ (32u * b));
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              codes_of(f[k], c[2 * k], c[2 * k + 1]);
            }
            const float2 d0 = unpack16<__half>(d[0][b >> 1]), d1 = unpack16<__half>(d[1][b >> 1]);
            const float y0 = b & 1 ? d0.y : d0.x, y1 = b & 1 ? d1.y : d1.x;
#pragma unroll
            for (int n = 0; n < N; ++n) {
              float x[4];
              first_product(x, c[0], c[4], c[1], c[5], qf[n][2 * b][0], qf[n][2 * b][1]);
              product(x, c[2], c[6], c[3], c[7], qf[n][2 * b + 1][0], qf[n][2 * b + 1][1]);
              s[n][0] = fmaf(x[0], y0, s[n][0]);
              s[n][1] = fmaf(x[1], y0, s[n][1]);
              s[n][2] = fmaf(x[2], y1, s[n][2]);
              s[n][3] = fmaf(x[3], y1, s[n][3]);
            }
          }
        }
        bool rises = false;
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
          for (int k = 0; k < 4; ++k) s[n][k] *= rs[n][k & 1];
          if (left < 16) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (r + 8 * (k >> 1) >= left) s[n][k] = -INFINITY;
          }
          rises |= fmaxf(s[n][0], s[n][2]) > m[n][0] + kLazy || fmaxf(s[n][1], s[n][3]) > m[n][1] + kLazy;
        }
        if (__any_sync(kFull, rises)) {
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = fmaxf(s[n][e], s[n][2 + e]);
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, x));
              const float mn = fmaxf(m[n][e], mx), f = mn == -INFINITY ? 1.0f : ex2(m[n][e] - mn);
              m[n][e] = mn;
              l[n][e] *= f;
#pragma unroll
              for (int x = 0; x < HD / 16; ++x) {
                o[n][x][e] *= f;
                o[n][x][2 + e] *= f;
              }
            }
        }
        // weights as two fp16 parts: [k] of positions c2 + 8 k and the next, head 8 n + r (transposed by exchange)
        uint32_t ph[N][2], pl[N][2];
#pragma unroll
        for (int n = 0; n < N; ++n) {
          float base[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) base[e] = (m[n][e] == -INFINITY ? 0.0f : m[n][e]) - kPShift;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float p0 = ex2(s[n][2 * k] - base[0]), p1 = ex2(s[n][2 * k + 1] - base[1]);
            l[n][0] += p0;
            l[n][1] += p1;
            const uint32_t hi = pack16<__half>(p0, p1);
            const float2 q = unpack16<__half>(hi);
            ph[n][k] = transposed8(hi);
            pl[n][k] = transposed8(pack16<__half>(p0 - q.x, p1 - q.y));
          }
        }
        // scales of the values of positions c2, c2 + 1, c2 + 8, c2 + 9
        uint32_t vs[4][B / 2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const unsigned char* at = sc + L::kScales + (r0 + c2 + 8 * k) * (2 * B);
          if constexpr (B == 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(at);
            vs[2 * k][0] = x.x;
            vs[2 * k][1] = x.y;
            vs[2 * k + 1][0] = x.z;
            vs[2 * k + 1][1] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(at);
            vs[2 * k][0] = x.x;
            vs[2 * k + 1][0] = x.y;
          }
        }
        if (left < 16) {  // whatever the page or the ring holds there
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (c2 + (k & 1) + 8 * (k >> 1) >= left) {
#pragma unroll
              for (int b = 0; b < B / 2; ++b) vs[k][b] = 0u;
            }
        }
        bool risen = false;
#pragma unroll
        for (int b = 0; b < B / 2; ++b) {  // below twice its power of two (a sign, infinities and NaN are above)
          const unsigned big = __vmaxu2(__vmaxu2(vs[0][b], vs[1][b]), __vmaxu2(vs[2][b], vs[3][b]));
          risen |= __vmaxu2(big, top[b] | 0x03FF03FFu) != (top[b] | 0x03FF03FFu);
        }
        if (__any_sync(kFull, risen)) {
#pragma unroll
          for (int b = 0; b < B; ++b) {
            const int sh = 16 * (b & 1);
            unsigned big = 0u;  // the largest finite one
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const unsigned y = vs[k][b >> 1] >> sh & 0x7FFFu;
              big = y < 0x7C00u ? max(big, y) : big;
            }
            big = max(big, __shfl_xor_sync(kFull, big, 1));
            big = max(big, __shfl_xor_sync(kFull, big, 2)) & 0x7C00u;
            const unsigned was = top[b >> 1] >> sh & 0x7C00u;
            if (big <= was) continue;
            const unsigned one_over = big == 0x7800u ? 0x0200u : 0x7800u - big;
            top[b >> 1] = (top[b >> 1] & ~(0xFFFFu << sh)) | big << sh;
            inv[b >> 1] = (inv[b >> 1] & ~(0xFFFFu << sh)) | one_over << sh;
            const float f = __uint_as_float((127u << 23) - ((big - was) << 13));
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
              for (int x = 2 * b; x < 2 * b + 2; ++x)
#pragma unroll
                for (int z = 0; z < 4; ++z) o[n][x][z] *= f;
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int b = 0; b < B / 2; ++b) vs[k][b] = as_word(__hmul2(as_half2(vs[k][b]), as_half2(inv[b])));
        const uint32_t at = sk + L::kCodes + value_at;
#pragma unroll
        for (int b = 0; b < B; ++b) {
          uint32_t f[4], c[8];
          ldsm4_t(f, at ^ (32u * b));
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            codes_of(f[k], c[2 * k], c[2 * k + 1]);
          }
          const __half2 d0 = as_half2(__byte_perm(vs[0][b >> 1], vs[1][b >> 1], b & 1 ? 0x7632 : 0x5410));
          const __half2 d1 = as_half2(__byte_perm(vs[2][b >> 1], vs[3][b >> 1], b & 1 ? 0x7632 : 0x5410));
#pragma unroll
          for (int n = 0; n < N; ++n) {  // p d = hi + lo: the product's rounding is in lo
            const __half2 x0 = as_half2(ph[n][0]), x1 = as_half2(ph[n][1]);
            const __half2 h0 = __hmul2(x0, d0), h1 = __hmul2(x1, d1);
            const __half2 l0 = __hfma2(as_half2(pl[n][0]), d0, __hfma2(x0, d0, __hneg2(h0)));
            const __half2 l1 = __hfma2(as_half2(pl[n][1]), d1, __hfma2(x1, d1, __hneg2(h1)));
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              // The tensor core truncates its sums: 256 tiles in a row come out 5e-6 too small, which an fp32 output shows.
              // There each tile starts from zero and is added with rounding.
              if constexpr (sizeof(O) == 4) {
                float y[4];
                first_product(y, c[4 * x], c[4 * x + 1], c[4 * x + 2], c[4 * x + 3], as_word(h0), as_word(h1));
                product(y, c[4 * x], c[4 * x + 1], c[4 * x + 2], c[4 * x + 3], as_word(l0), as_word(l1));
#pragma unroll
                for (int z = 0; z < 4; ++z) o[n][2 * b + x][z] += y[z];
              } else {
                product(o[n][2 * b + x], c[4 * x], c[4 * x + 1], c[4 * x + 2], c[4 * x + 3], as_word(h0), as_word(h1));
                product(o[n][2 * b + x], c[4 * x], c[4 * x + 1], c[4 * x + 2], c[4 * x + 3], as_word(l0), as_word(l1));
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(empty + st));
      if (++st == kStages) {
        st = 0;
        phase ^= 1;
      }
    }

    // Join the four warps, 8 heads at a time: 2 -> 0 and 3 -> 1, then 1 -> 0.
    const bool whole = t0 == 0 && t1 == w.nt;
    const int slot = 2 * cta + (w.at == begin ? 0 : 1);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float (&v)[HD / 16][4] = o[n];
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) {
        const float unit = __half2float(__ushort_as_half((unsigned short)(top[d >> 2] >> 16 * (d >> 1 & 1))));
#pragma unroll
        for (int k = 0; k < 4; ++k) v[d][k] *= unit;
      }
      float mm[2], ll[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mm[e] = m[n][e];
        ll[e] = l[n][e];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) ll[e] += __shfl_xor_sync(kFull, ll[e], x);
      }
      auto give = [&](int at) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float* b = jbuf + (at * 8 + c2 + e) * L::kJoinRow + 2 * r;
#pragma unroll
          for (int d = 0; d < HD / 16; ++d) *reinterpret_cast<float2*>(b + d * 16) = make_float2(v[d][e], v[d][2 + e]);
          if (r == 0) jml[at * 8 + c2 + e] = make_float2(mm[e], ll[e]);
        }
      };
      auto take = [&](int at) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float* b = jbuf + (at * 8 + c2 + e) * L::kJoinRow + 2 * r;
          const float2 x = jml[at * 8 + c2 + e];
          const float mn = fmaxf(mm[e], x.x), mz = mn == -INFINITY ? 0.0f : mn, f0 = ex2(mm[e] - mz), f1 = ex2(x.x - mz);
          mm[e] = mn;
          ll[e] = ll[e] * f0 + x.y * f1;
#pragma unroll
          for (int d = 0; d < HD / 16; ++d) {
            const float2 y = *reinterpret_cast<const float2*>(b + d * 16);
            v[d][e] = v[d][e] * f0 + y.x * f1;
            v[d][2 + e] = v[d][2 + e] * f0 + y.y * f1;
          }
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
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = 8 * n + c2 + e;
          if (whole) {
            const float d = ll[e] == 0.0f ? 0.0f : 1.0f / ll[e];
            if (row < nh) {
              O* out = static_cast<O*>(a.out) + ((long long)w.s * a.n_heads + j * g + h0 + row) * HD + 2 * r;
#pragma unroll
              for (int x = 0; x < HD / 16; ++x) {
                if constexpr (sizeof(O) == 4)
                  *reinterpret_cast<float2*>(out + x * 16) = make_float2(v[x][e] * d, v[x][2 + e] * d);
                else
                  *reinterpret_cast<uint32_t*>(out + x * 16) = pack16<O>(v[x][e] * d, v[x][2 + e] * d);
              }
            }
          } else {
            float* b = slots + (size_t)slot * slot_floats(ROWS, HD);
#pragma unroll
            for (int x = 0; x < HD / 16; ++x)
              __stcg(reinterpret_cast<float2*>(b + row * HD + x * 16 + 2 * r), make_float2(v[x][e], v[x][2 + e]));
            if (r == 0) {
              __stcg(b + ROWS * HD + row, mm[e]);
              __stcg(b + ROWS * HD + ROWS + row, ll[e]);
            }
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
                HD == 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_64B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
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
