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
// maximum does.  A tile with scales below 2^-14 of that, which would lose bits
// in fp16, is added up by itself, in three passes; the registers of that code
// cost the other tiles 1 to 2 %, a call of 32 short sequences 1 us.  bf16
// queries are scaled by a power of two per row into fp16's range, where their 8
// bits are exact (those below 2^-31 of the row's largest round).
//
// 2 head_dim (1 + 1/16) bytes a position and KV head, read once.  The warps work
// alone, as in attention_own.cu: each has an equal range of all tiles of 16
// positions, copies its own (codes by tensor copies, scales, side by side in a
// page, by bulk copies) and leaves whole units and parts unnormalised for the
// join.  Fragments come from ldmatrix on pairs of codes: a word holds four
// values of one position (keys), or two values of two positions (values,
// transposed), and is split into its even and odd bytes.  The order of the
// values within a product is free as long as the query's is the same.
//
// Measured on one B200, 64 sequences of 64 query and 8 KV heads of 128 values
// in bf16 that hold up to 16384 positions: 239 us (5.0 TB/s; the copy takes
// 184; the 16-bit cache of twice the bytes 356).  Called for a second and more,
// under the power cap, 268 (364).  571 where every tile takes three passes.
// Codes to fp16 and the scales are most of a warp's 600 instructions for 16
// positions, and 63 % of the cycles issue one.  32 sequences of up to 1024: 22
// us; one of 32 heads and 512 positions: 9.5; one of 8 heads and 131071: 33; 32
// of 32 heads, up to 4096, fp32 outputs: 165.  Before there were three passes:
// 236, 21, 9.4, 33 and 161; with a CTA's four warps on one ring of tiles of 64,
// fed by a fifth, and their join: 232, 22, 10.1, 32 and 202; with positions as
// the right side, padded to 8 rows of heads as the left, 341 in the first.
#include "found.cuh"
#include "matvec.cuh"
#include "mma16.cuh"
#include "paged_deal.cuh"
#include "pipeline.cuh"
#include "serving_q8.cuh"
#include "tensor_map.cuh"

namespace asmllm {

namespace {

constexpr int kSmall = 16;  // positions per tile
// Tiles of a warp at least, where there are few: with 4 one sequence of 512 positions takes 11.6 us, not 9.4.
constexpr int kLeast = 2;
constexpr int kRanges = 2400;  // at most, one a warp
// The output is rescaled only when a row's maximum has risen by more than 2^kLazy since it was last set; the weights,
// 2^kPShift exp(s - m), stay below 2^15 then.
constexpr float kLazy = 5.0f, kPShift = 9.0f;

template <int HD, int ROWS>
struct LayoutQ8 {
  static constexpr int kWarps = ROWS == 8 ? 8 : 6;     // two CTAs an SM: what the registers allow
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kCodes = kSmall * HD;           // bytes of keys or values of a tile
  static constexpr int kScales = kSmall * (HD / 32) * 2;
  static constexpr int kStageBytes = 2 * kCodes + 1024;  // scales of keys and of values behind the codes
  static_assert(2 * kScales <= 1024 && kStageBytes % 1024 == 0, "stages are aligned for the swizzle");
  static constexpr int kStages = 2 * 128 / HD;
  static constexpr int kRing = kStages * kStageBytes;  // of a warp
  static constexpr int kBarOff = kWarps * kRing;
  static constexpr int kSmem = kBarOff + kWarps * kStages * 8 + 1024;
};

// Where units' results are, unnormalised: whole ones by row, parts in slots of ROWS rows.
struct Parts {
  float* o;       // [batch][n_heads][head_dim]
  float2* ml;     // [batch][n_heads]: (maximum in units of log2, sum); o 2^maximum is the sum of exp(s) v
  int4* found;    // [batch][units]: a Found
  float* slots;
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

// hi + lo = weights p = h + l of positions c2, c2 + 1 ([0]) and 8 behind times their scales d0, d1: the product's rounding is
// in lo.
__device__ __forceinline__ void weighted(const uint32_t (&h)[2], const uint32_t (&l)[2], __half2 d0, __half2 d1,
                                         uint32_t (&hi)[2], uint32_t (&lo)[2]) {
  const __half2 x0 = as_half2(h[0]), x1 = as_half2(h[1]);
  const __half2 h0 = __hmul2(x0, d0), h1 = __hmul2(x1, d1);
  hi[0] = as_word(h0);
  hi[1] = as_word(h1);
  lo[0] = as_word(__hfma2(as_half2(l[0]), d0, __hfma2(x0, d0, __hneg2(h0))));
  lo[1] = as_word(__hfma2(as_half2(l[1]), d1, __hfma2(x1, d1, __hneg2(h1))));
}

struct Steps {  // a warp's walk over its tiles
  int s, n, nt, u, t;
  long long first, at, end;  // number of the unit's first tile; tiles [at, end) are left
};

// EXACT: fp32 outputs.
template <class T, bool EXACT, int HD, int ROWS>
__global__ void __launch_bounds__(LayoutQ8<HD, ROWS>::kThreads, 2)
attention_paged_q8_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                          const PagedArgs a, const KvQ8Args c, const Parts parts, int zs, unsigned* __restrict__ err) {
  using L = LayoutQ8<HD, ROWS>;
  constexpr int B = HD / 32, S = L::kStages, N = ROWS / 8;  // blocks of a position, tiles under way, groups of 8 heads
  const KvArgs& kv = c.kv;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ long long s_part[L::kThreads];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff) + warp * S;
  unsigned char* ring = smem + warp * L::kRing;
  const int units = kv.n_kv * zs, g = a.n_heads / kv.n_kv;
  if (lane == 0) {
    if (warp == 0) {
      prefetch_map(&kmap);
      prefetch_map(&vmap);
    }
    for (int i = 0; i < S; ++i) mbar_init(smem_u32(full + i), 1);
    fence_mbar_init();
  }
  __syncwarp();
  pdl_trigger();
  pdl_wait();

  auto load = [&](int s, Steps* x, bool report) -> int {
    bool clipped;
    x->n = kv_length(kv, s, &clipped);
    if (clipped && report) atomicOr(err, kErrDecodeRange);
    x->s = s;
    x->nt = (x->n + kSmall - 1) / kSmall;
    return x->nt;
  };
  auto leave = [&](const Steps& x, int u, int n, int index, int slot) {
    __stcg(parts.found + (long long)x.s * units + u, make_int4(n, index, slot, 0));
  };
  Steps w;
  Deal deal(0, 1);
  const int index = deal_warps<L::kThreads>(kv.batch, units, kLeast, s_part, load, [&](const Steps& x) {
    for (int u = 0; u < units; ++u) leave(x, u, 0, 0, 0);
  }, &w, &deal);
  if (index < 0) return;
  const long long begin = w.at;
  auto next_unit = [&](Steps& x) {
    x.first += x.nt;
    x.t = 0;
    if (++x.u == units) {
      x.u = 0;
      while (load(x.s + 1, &x, false) == 0) {
      }
    }
  };
  auto advance = [&](int n) {
    w.at += n;
    if (w.at < w.end) next_unit(w);
  };

  // ---- copies, S tiles ahead, by four lanes: codes of keys and values, their scales; the page number of the next one is on
  // its way ----
  Steps ahead = w;
  int asked = 0, page = 0, head = w.u / zs;
  const int32_t* pages = kv.table + (long long)w.s * kv.table_stride;
  const __half* from = (lane & 1 ? c.vs : c.ks) + (long long)head * c.scale_head_stride;
  auto lookup = [&]() { page = __ldcg(pages + (ahead.t * kSmall >> kv.page_shift)); };
  auto ask = [&]() {
    const int st = asked % S, in = ahead.t * kSmall & (kv.page_size - 1);
    unsigned char* dst = ring + st * L::kStageBytes;
    unsigned char* scales = dst + 2 * L::kCodes + (lane & 1) * L::kScales;
    const bool good = (unsigned)page < (unsigned)kv.n_pages;
    if (!good) {  // no page: the copies of codes give zeros, the scales have to be set
      atomicOr(err, kErrDecodeRange);
      if (lane < 2) {
#pragma unroll
        for (int i = 0; i < L::kScales; i += 16) *reinterpret_cast<uint4*>(scales + i) = make_uint4(0u, 0u, 0u, 0u);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    const uint32_t bar = smem_u32(full + st);
    if (lane == 0) mbar_arrive_expect_tx(bar, 2 * (L::kCodes + (good ? L::kScales : 0)));
    __syncwarp();
    if (lane < 2) {
      tma_load_4d(smem_u32(dst) + lane * L::kCodes, lane ? &vmap : &kmap, 0, in, head, good ? page : kv.n_pages, bar);
    } else if (lane < 4 && good) {
      bulk_g2s(smem_u32(scales), from + (long long)page * c.scale_page_stride + in * B, L::kScales, bar);
    }
    ++asked;
    if (++ahead.at < ahead.end) {
      if (++ahead.t == ahead.nt) {
        next_unit(ahead);
        head = ahead.u / zs;
        pages = kv.table + (long long)ahead.s * kv.table_stride;
        from = (lane & 1 ? c.vs : c.ks) + (long long)head * c.scale_head_stride;
      }
      lookup();
    }
  };
  lookup();
  while (asked < S && ahead.at < ahead.end) ask();

  const float sl2 = a.scale * 1.4426950408889634f;
  const int r = lane >> 2, t4 = lane & 3, c2 = t4 * 2;
  // Fragments' places in a tile: chunk 2 b of keys is at key_at ^ 32 b (positions 0-7, chunk + 1, positions 8-15, chunk
  // + 1), values at value_at ^ 32 b (positions 0-7, 8-15, the same of chunk + 1).
  const uint32_t key_at = code_chunk<HD>((lane >> 4) * 8 + (lane & 7), (lane >> 3) & 1);
  const uint32_t value_at = code_chunk<HD>(((lane >> 3) & 1) * 8 + (lane & 7), lane >> 4);
  int done = 0;
  bool ok = true;
  while (ok && w.at < w.end) {
    // one segment: tiles w.t .. of unit (w.s, w.u)
    const int j = w.u / zs, h0 = (w.u % zs) * 16, nh = min(16, g - h0);
    const int t0 = w.t, t1 = (int)min((long long)w.nt, w.t + (w.end - w.at));
    // The unit's query rows in fp16 as fragments: those of head 8 n + r, values 32 b + 16 s + 4 t4 and + 2 in [0] of step
    // 2 b + s, + 1 and + 3 in [1].
    uint32_t qf[N][2 * B][2];
    float rs[N][2];  // a score of head 8 n + c2 + e is this times its product
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const T* q = static_cast<const T*>(a.q) + w.s * a.q_row_stride + (long long)(j * g + h0 + 8 * n + r) * a.q_head_stride + 4 * t4;
      uint2 v[2 * B];
#pragma unroll
      for (int k = 0; k < 2 * B; ++k) v[k] = 8 * n + r < nh ? __ldcg(reinterpret_cast<const uint2*>(q + 16 * k)) : make_uint2(0u, 0u);
      if constexpr (std::is_same<T, __half>::value) {
        rs[n][0] = rs[n][1] = sl2;
      } else {
        float top = 0.0f;
#pragma unroll
        for (int k = 0; k < 2 * B; ++k) {
          const float2 x = unpack16<T>(v[k].x), y = unpack16<T>(v[k].y);
          top = fmaxf(fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(y.x), fabsf(y.y)));
        }
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
        // 2^n times the row with the largest value in [2^14, 2^15); an infinity leaves the row as it is
        const int ex = (int)(__float_as_uint(top) >> 23) - 127, up = ex > 127 || top == 0.0f ? 0 : min(14 - ex, 100);
        const float by = __uint_as_float((unsigned)(127 + up) << 23), down = sl2 * __uint_as_float((unsigned)(127 - up) << 23);
#pragma unroll
        for (int e = 0; e < 2; ++e) rs[n][e] = __shfl_sync(kFull, down, 4 * (c2 + e));
#pragma unroll
        for (int k = 0; k < 2 * B; ++k) {
          const float2 x = unpack16<T>(v[k].x), y = unpack16<T>(v[k].y);
          v[k] = make_uint2(pack16<__half>(x.x * by, x.y * by), pack16<__half>(y.x * by, y.y * by));
        }
      }
#pragma unroll
      for (int k = 0; k < 2 * B; ++k) {
        qf[n][k][0] = __byte_perm(v[k].x, v[k].y, 0x5410);
        qf[n][k][1] = __byte_perm(v[k].x, v[k].y, 0x7632);
      }
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

    for (int t = t0; t < t1; ++t, ++done) {
      const int st = done % S;
      if (!__all_sync(kFull, mbar_try_wait(smem_u32(full + st), (done / S) & 1)))
        ok = __all_sync(kFull, mbar_wait_bounded(smem_u32(full + st), (done / S) & 1));
      if (!ok) {
        if (lane == 0) atomicOr(err, kErrRingTimeout);
        break;
      }
      const unsigned char* stage = ring + st * L::kStageBytes;
      const uint32_t sk = smem_u32(stage);
      const unsigned char* sc = stage + 2 * L::kCodes;
      const int left = w.n - t * kSmall;  // positions of the tile that exist
      // scores of positions r ([0], [1]) and r + 8, heads 8 n + c2 and the next
      float s[N][4] = {};
      {
        uint32_t d[2][B / 2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const unsigned char* at = sc + (r + 8 * k) * (2 * B);
          if constexpr (B == 4) {
            const uint2 x = *reinterpret_cast<const uint2*>(at);
            d[k][0] = x.x;
            d[k][1] = x.y;
          } else {
            d[k][0] = *reinterpret_cast<const uint32_t*>(at);
          }
          // An infinite scale stands for infinities of both signs and 0 times infinity: NaN, where its product with the
          // block's sum could be a score of minus infinity, which has no weight.
#pragma unroll
          for (int b = 0; b < B / 2; ++b) d[k][b] = as_word(__hfma2(as_half2(d[k][b]), as_half2(0u), as_half2(d[k][b])));
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
        const unsigned char* at = sc + L::kScales + (c2 + 8 * k) * (2 * B);
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
      // One word of the tile's scales a lane: has one risen to twice its block's power of two (infinities and NaN are
      // above it), or is one, other than zero, so far below that fp16 would lose bits of it relative to that?
      bool apart = false;
      {
        const int word = B == 4 ? lane : lane & 15;
        unsigned y = *reinterpret_cast<const uint32_t*>(sc + L::kScales + 4 * word) & 0x7FFF7FFFu;
        y = word / (B / 2) < left ? y : 0u;
        auto unit = [&]() { return B == 4 && (lane & 1) ? top[B / 2 - 1] : top[0]; };
        auto far_below = [&]() {
          const unsigned least = __vmaxu2(unit(), 0x38013801u) - 0x38013801u;
          return __vminu2(__vsub2(y, 0x00010001u), least) != least;
        };
        const unsigned most = unit() | 0x03FF03FFu;
        if (__any_sync(kFull, __vmaxu2(y, most) != most || far_below())) {
#pragma unroll
          for (int b = 0; b < B; ++b) {
            const int sh = 16 * (b & 1);
            unsigned big = 0u;  // the largest finite one
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const unsigned z = vs[k][b >> 1] >> sh & 0x7FFFu;
              big = z < 0x7C00u ? max(big, z) : big;
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
          apart = __any_sync(kFull, far_below());
        }
      }
      const uint32_t at = sk + L::kCodes + value_at;
      if (!apart) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int b = 0; b < B / 2; ++b) vs[k][b] = as_word(__hmul2(as_half2(vs[k][b]), as_half2(inv[b])));
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
          for (int n = 0; n < N; ++n) {
            uint32_t hi[2], lo[2];
            weighted(ph[n], pl[n], d0, d1, hi, lo);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              // The tensor core truncates its sums: 256 tiles in a row come out 5e-6 too small, which an fp32 output shows.
              // There each tile starts from zero and is added with rounding.
              if constexpr (EXACT) {
                float y[4];
                first_product(y, c[4 * x], c[4 * x + 1], c[4 * x + 2], c[4 * x + 3], hi[0], hi[1]);
                product(y, c[4 * x], c[4 * x + 1], c[4 * x + 2], c[4 * x + 3], lo[0], lo[1]);
#pragma unroll
                for (int z = 0; z < 4; ++z) o[n][2 * b + x][z] += y[z];
              } else {
                product(o[n][2 * b + x], c[4 * x], c[4 * x + 1], c[4 * x + 2], c[4 * x + 3], hi[0], hi[1]);
                product(o[n][2 * b + x], c[4 * x], c[4 * x + 1], c[4 * x + 2], c[4 * x + 3], lo[0], lo[1]);
              }
            }
          }
        }
      } else {
        // Scales 2^-14 and more below their block's power of two: three passes, with those from 2^-14 of it on, those from
        // 2^-28 on, 2^14 times as large, and the rest (2^-24 beside 2^15), 2^28 times; the products come back in fp32.
#pragma unroll
        for (int b = 0; b < B; ++b) {
          const int sh = 16 * (b & 1);
          const unsigned unit = top[b >> 1] >> sh & 0x7C00u, over = inv[b >> 1] >> sh & 0xFFFFu;
          uint32_t f[4], c[8];
          ldsm4_t(f, at ^ (32u * b));
#pragma unroll
          for (int k = 0; k < 4; ++k) codes_of(f[k], c[2 * k], c[2 * k + 1]);
#pragma unroll 1
          for (unsigned by = 0u; by < 0xA800u; by += 0x3800u) {
            const float back = __uint_as_float((127u << 23) - (by << 13));
            const unsigned above = by ? max(unit, by) - by : 0x8000u, least = max(unit, by + 0x3800u) - (by + 0x3800u);
            __half d[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int p = c2 + (k & 1) + 8 * (k >> 1);
              const unsigned y = p < left ? *reinterpret_cast<const unsigned short*>(sc + L::kScales + 2 * (p * B + b)) : 0u;
              const unsigned z = y & 0x7FFFu;
              const __half y14 = __hmul(__ushort_as_half((unsigned short)y), __ushort_as_half(by ? 0x7400 : 0x3C00));
              const __half y28 = __hmul(y14, __ushort_as_half(by > 0x3800u ? 0x7400 : 0x3C00));
              d[k] = z >= least && z < above ? __hmul(y28, __ushort_as_half((unsigned short)over)) : __ushort_as_half(0);
            }
#pragma unroll
            for (int n = 0; n < N; ++n) {
              uint32_t hi[2], lo[2];
              weighted(ph[n], pl[n], __halves2half2(d[0], d[1]), __halves2half2(d[2], d[3]), hi, lo);
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                float y[4];
                first_product(y, c[4 * x], c[4 * x + 1], c[4 * x + 2], c[4 * x + 3], hi[0], hi[1]);
                product(y, c[4 * x], c[4 * x + 1], c[4 * x + 2], c[4 * x + 3], lo[0], lo[1]);
#pragma unroll
                for (int z = 0; z < 4; ++z) o[n][2 * b + x][z] = fmaf(y[z], back, o[n][2 * b + x][z]);
              }
            }
          }
        }
      }
      __syncwarp();
      if (ahead.at < ahead.end) ask();  // into the stage that has just been read
    }
    if (!ok) break;

    const bool whole = t0 == 0 && t1 == w.nt;
    const int slot = 2 * index + (w.at == begin ? 0 : 1);
    float* part = parts.slots + (size_t)slot * slot_floats(ROWS, HD);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float (&v)[HD / 16][4] = o[n];
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) {
        const float unit = __half2float(__ushort_as_half((unsigned short)(top[d >> 2] >> 16 * (d >> 1 & 1))));
#pragma unroll
        for (int k = 0; k < 4; ++k) v[d][k] *= unit;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 8 * n + c2 + e;
        float sum = l[n][e];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(kFull, sum, x);
        if (row >= nh) continue;
        const long long at = (long long)w.s * a.n_heads + j * g + h0 + row;
        float* to = (whole ? parts.o + at * HD : part + row * HD) + 2 * r;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) __stcg(reinterpret_cast<float2*>(to + 16 * d), make_float2(v[d][e], v[d][2 + e]));
        if (r == 0)
          __stcg(whole ? parts.ml + at : reinterpret_cast<float2*>(part + ROWS * HD) + row, make_float2(m[n][e] - kPShift, sum));
      }
    }
    if (t0 == 0 && lane == 0) leave(w, w.u, whole ? 1 : deal.range_of(w.first + w.nt - 1) - index + 1, index, slot);
    advance(t1 - t0);
  }
  if (!ok) abandon(w, [&]() { if (lane == 0) leave(w, w.u, 0, 0, 0); }, advance);
  // every issued copy lands before the CTA may end (bounded)
  for (int i = done; i < asked; ++i) mbar_wait_bounded(smem_u32(full + i % S), (i / S) & 1);
}

// A row's parts, by the warp with every `warps`-th from `first` on: (maximum, sum) and the outputs lane E and on.
template <int HD, int U>
__device__ __forceinline__ float2 join_parts(const Parts& parts, int4 f, long long row, int in, int R, int first, int warps,
                                             float (&o)[HD / 32]) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int z = 0; z < E; ++z) o[z] = 0.0f;
  for (int p0 = first; p0 < f.x; p0 += U * warps) {  // U parts at a time
    float x[U][E];
    float2 ml[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int p = p0 + u * warps;
      ml[u] = make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int z = 0; z < E; ++z) x[u][z] = 0.0f;
      if (p < f.x) {
        const float* slot = parts.slots + (size_t)(p ? 2 * (f.y + p) : f.z) * slot_floats(R, HD);
        const float* src = f.x == 1 ? parts.o + row * HD : slot + in * HD;
        ml[u] = __ldcg(f.x == 1 ? parts.ml + row : reinterpret_cast<const float2*>(slot + R * HD) + in);
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
      const float w = ex2(ml[u].x - mz);
      l = fmaf(w, ml[u].y, l);
#pragma unroll
      for (int z = 0; z < E; ++z) o[z] = fmaf(w, x[u][z], o[z]);
    }
  }
  return make_float2(m, l);
}

// ROWS rows a CTA of W warps: 1, by all of them, or 8, by a warp each, or one after the other by all where one of them has more than kFew
// parts.
constexpr int kFew = 64;
template <class O, int HD, int ROWS, int W>
__global__ void __launch_bounds__(W * 32, ROWS == 8 ? 4 : W == 16 ? 1 : 3) attention_paged_q8_join_kernel(const PagedArgs a, const Parts parts, int batch, int n_kv,
                                                                      int zs) {
  constexpr int E = HD / 32;
  __shared__ float s_o[W][HD];
  __shared__ float2 s_ml[W];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = a.n_heads / n_kv, R = g <= 8 ? 8 : 16;
  const long long rows = (long long)batch * a.n_heads, row0 = (long long)blockIdx.x * ROWS;
  auto found = [&](long long row) -> int4 {
    if (row >= rows) return make_int4(0, 0, 0, 0);
    const int s = (int)(row / a.n_heads), h = (int)(row % a.n_heads);
    int4 f = __ldcg(parts.found + ((long long)s * n_kv + h / g) * zs + h % g / 16);
    f.x = parts_of({f.x, f.y, f.z, 0}, kRanges);
    return f;
  };
  auto put = [&](long long row, float l, const float (&o)[E]) {
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    O* out = static_cast<O*>(a.out) + row * HD + lane * E;
#pragma unroll
    for (int z = 0; z < E; z += 2) {
      if constexpr (sizeof(O) == 4) *reinterpret_cast<float2*>(out + z) = make_float2(o[z] * by, o[z + 1] * by);
      else *reinterpret_cast<uint32_t*>(out + z) = pack16<O>(o[z] * by, o[z + 1] * by);
    }
  };
  float o[E];
  if constexpr (ROWS == 8) {
    const int4 f = found(row0 + warp);
    if (!__syncthreads_or(f.x > kFew)) {
      const long long row = row0 + warp;
      if (row >= rows) return;
      const float2 ml = join_parts<HD, 4>(parts, f, row, (int)(row % a.n_heads) % g % 16, R, 0, 1, o);
      put(row, ml.y, o);
      return;
    }
  }
  for (int i = 0; i < ROWS; ++i) {
    const long long row = row0 + i;
    if (row >= rows) return;
    const float2 ml = join_parts<HD, 64 / W / (ROWS == 8 ? 2 : 1)>(parts, found(row), row, (int)(row % a.n_heads) % g % 16, R, warp, W, o);
#pragma unroll
    for (int q = 0; q < E; ++q) s_o[warp][lane * E + q] = o[q];
    if (lane == 0) s_ml[warp] = ml;
    __syncthreads();
    if (warp == 0) {
      float m = -INFINITY, l = 0.0f;
#pragma unroll
      for (int x = 0; x < W; ++x) m = fmaxf(m, s_ml[x].x);
      const float mz = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int q = 0; q < E; ++q) o[q] = 0.0f;
#pragma unroll
      for (int x = 0; x < W; ++x) {
        const float fx = ex2(s_ml[x].x - mz);
        l = fmaf(fx, s_ml[x].y, l);
#pragma unroll
        for (int q = 0; q < E; ++q) o[q] = fmaf(fx, s_o[x][lane * E + q], o[q]);
      }
      put(row, l, o);
    }
    __syncthreads();
  }
}

// Workspace: all parts, 16-byte aligned.
struct Space {
  size_t slots, o, ml, found, bytes;
};
Space space_of(int batch, int n_heads, int n_kv, int head_dim) {
  Space x;
  const size_t rows = (size_t)batch * n_heads;
  const int g = n_heads / n_kv;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t was = at;
    at += (bytes + 15) / 16 * 16;
    return was;
  };
  x.slots = take((size_t)kRanges * 2 * slot_floats(g <= 8 ? 8 : 16, head_dim) * 4);
  x.o = take(rows * head_dim * 4);
  x.ml = take(rows * 8);
  x.found = take((size_t)batch * n_kv * ((g + 15) / 16) * sizeof(int4));
  x.bytes = at;
  return x;
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
  using L = LayoutQ8<HD, ROWS>;
  const KvArgs& kv = c.kv;
  auto kernel = attention_paged_q8_kernel<T, sizeof(O) == 4, HD, ROWS>;
  const Space sp = space_of(kv.batch, a.n_heads, kv.n_kv, HD);
  unsigned char* ws = static_cast<unsigned char*>(a.workspace);
  Parts parts;
  parts.slots = reinterpret_cast<float*>(ws + sp.slots);
  parts.o = reinterpret_cast<float*>(ws + sp.o);
  parts.ml = reinterpret_cast<float2*>(ws + sp.ml);
  parts.found = reinterpret_cast<int4*>(ws + sp.found);
  CUtensorMap kmap, vmap;
  if (!encode_codes<HD>(&kmap, kv, kv.k, kSmall) || !encode_codes<HD>(&vmap, kv, kv.v, kSmall)) return cudaErrorInvalidValue;
  static std::atomic<unsigned long long> done{0};
  int sms = 0;
  cudaError_t e = kernel_setup(reinterpret_cast<const void*>(kernel), L::kSmem, done, &sms);
  if (e != cudaSuccess) return e;
  const int g = a.n_heads / kv.n_kv, zs = (g + 15) / 16;
  const int ctas = 2 * sms * L::kWarps < kRanges ? 2 * sms : kRanges / L::kWarps;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(L::kThreads);
  cfg.dynamicSmemBytes = L::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_opt_pdl.load() ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, kernel, kmap, vmap, a, c, parts, zs, err);
  if (e != cudaSuccess) return e;
  // Few rows may have many parts each.  (2048 rows of 9 parts: a block a row makes the call 24.7 us, not 21; 640 rows of 37
  // parts: eight rows a block 24, not 15; 8 rows of 1024 parts: blocks of 8 warps 39, not 33.)
  const long long rows = (long long)kv.batch * a.n_heads;
  cfg.dynamicSmemBytes = 0;
  if (rows <= sms) {
    cfg.blockDim = dim3(512);
    cfg.gridDim = dim3((unsigned)rows);
    return cudaLaunchKernelEx(&cfg, attention_paged_q8_join_kernel<O, HD, 1, 16>, a, parts, kv.batch, kv.n_kv, zs);
  }
  cfg.blockDim = dim3(256);
  if (rows <= 1184) {
    cfg.gridDim = dim3((unsigned)rows);
    return cudaLaunchKernelEx(&cfg, attention_paged_q8_join_kernel<O, HD, 1, 8>, a, parts, kv.batch, kv.n_kv, zs);
  }
  cfg.gridDim = dim3((unsigned)((rows + 7) / 8));
  return cudaLaunchKernelEx(&cfg, attention_paged_q8_join_kernel<O, HD, 8, 8>, a, parts, kv.batch, kv.n_kv, zs);
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
  return batch == 0 ? 0 : space_of(batch, n_heads, n_kv, head_dim).bytes;
}

cudaError_t launch_attention_paged_q8(const PagedArgs& a, int q_dtype, const KvQ8Args& c, cudaStream_t stream) {
  unsigned* err = device_error_word();
  if (!err) return cudaErrorUnknown;
  return q_dtype == kDtF16 ? launch_type<__half>(a, c, stream, err) : launch_type<__nv_bfloat16>(a, c, stream, err);
}

}  // namespace asmllm
