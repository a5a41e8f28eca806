// asmllm_b200/csrc/attention_own.cu -- the second pass of attention over
// shared prefixes (attention_shared.cu): every sequence's positions behind
// those that its group shares.
//
// They are few (what a sequence has said since the system prompt), so a unit,
// (sequence, KV head, up to 16 of its query heads), is a few tiles of 16
// positions, and what it costs beside them is what counts.  So the warps work
// alone: the tiles of all units in a row are cut into one equal range per warp,
// each warp has a ring of its own, copies its own tiles and keeps its own
// maximum, sum and output, and nothing in a CTA meets before its end.  Whole
// units and parts of units are left unnormalised for the join of both passes.
//
// Keys are the left side of the scores' product (16 positions x 8 heads), and
// values, transposed, of the second (16 values x 8 heads), so that up to 8
// heads fill them; the weights go from the one's layout to the other's by an
// exchange within the warp, and enter as two 16-bit parts (2^-22 of a weight in
// fp16, 2^-16 in bf16).  The output is rescaled only when a maximum has risen
// by more than 2^kLazy.
//
// Measured on one B200: 256 sequences of 8 KV heads with 1 to 1023 positions of
// 128 values each, about 105 us (5.2 TB/s), where a quarter of the cycles issue
// an instruction: a tile is one chain of copy, products, softmax, products.  So
// as many warps as registers allow, with one tile each: 128 sequences of up to
// 8000 positions of their own take 398 us, 444 with half the warps and three
// tiles each, 409 with two.  48 sequences of 32 KV heads with 1 to 299 behind
// three prefixes: 71 us a call, 95 with a CTA's warps on one ring of tiles of 64
// and their join.
#include <type_traits>

#include "matvec.cuh"
#include "mma16.cuh"
#include "pipeline.cuh"
#include "shared_prefix.cuh"
#include "tensor_map.cuh"

namespace asmllm {

namespace {

constexpr int kSmall = 16;  // positions per tile
// Tiles of a warp at least, where there are few: a part costs the join more than the second tile its warp (100 sequences of
// one KV head, 512 positions of their own: 31.7 us, 34.2 with one tile; 8 sequences of 64: 16 us with 4 tiles, 12 with 2).
constexpr int kLeast = 2;
constexpr float kLazy = 5.0f, kPShift = 9.0f;  // weights 2^kPShift exp(s - m) stay below 2^15

template <int HD, int ROWS>
struct LayoutOwn {
  static constexpr int kWarps = ROWS == 8 ? 8 : 6;    // two CTAs an SM: what the registers allow
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kTileBytes = kSmall * HD * 2;  // keys or values of a tile
  static constexpr int kStages = 128 / HD;
  static constexpr int kRing = kStages * 2 * kTileBytes;  // of a warp
  static constexpr int kBarOff = kWarps * kRing;
  static constexpr int kSmem = kBarOff + kWarps * kStages * 8 + 1024;
};

// c += a b, and c = a b, free to be moved.
template <class T>
__device__ __forceinline__ void product(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <class T>
__device__ __forceinline__ void first_product(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  c[0] = c[1] = c[2] = c[3] = 0.0f;
  product<T>(c, a, b0, b1);
}

// A warp's walk over its tiles: sequence, where its own positions begin, how many there are, unit, tile.
struct Steps {
  int s, base, n, nt, u, t;
  int4 group;               // (group, its sequences)
  long long first, at, end;  // number of the unit's first tile; tiles [at, end) are left
};

// EXACT: fp32 outputs: each tile is added with rounding (the tensor core truncates its sums).
template <class T, int HD, int ROWS, bool EXACT>
__global__ void __launch_bounds__(LayoutOwn<HD, ROWS>::kThreads, 2)
attention_own_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                     const PagedArgs a, const KvArgs kv, const SharedView v, int zs, unsigned* __restrict__ err) {
  using L = LayoutOwn<HD, ROWS>;
  constexpr int kThreads = L::kThreads, S = L::kStages, N = ROWS / 8, kHalves = HD / 64;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ long long s_part[kThreads];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff) + warp * S;
  const uint32_t ring = smem_u32(smem) + warp * L::kRing;
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
  // The launch before this one is the shared pass, which nothing here reads; it began behind whatever wrote the queries
  // and the cache.  Its end is waited for at this kernel's, so that the join behind has both.
  pdl_trigger();

  // a sequence's own positions
  auto load = [&](int s, Steps* x, bool report) -> int {
    bool clipped;
    const int n = kv_length(kv, s, &clipped);
    if (clipped && report) atomicOr(err, kErrDecodeRange);
    x->s = s;
    x->base = shared_base(v, kv, s, n, &x->group);
    x->n = n - x->base;
    x->nt = (x->n + kSmall - 1) / kSmall;
    return x->nt;
  };
  // where unit u's result is, and the group it is joined with
  auto leave = [&](const Steps& x, int u, int parts, int index, int slot) {
    int4* at = reinterpret_cast<int4*>(v.own_found + (long long)x.s * units + u);
    __stcg(at, make_int4(parts, index, slot, 0));
    __stcg(at + 1, x.group);
  };

  Steps w;
  Deal deal(0, 1);
  const int index = deal_warps<kThreads>(kv.batch, units, kLeast, s_part, load, [&](const Steps& x) {
    for (int u = 0; u < units; ++u) leave(x, u, 0, 0, 0);
  }, &w, &deal);
  if (index >= 0) {
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
    // ---- copies, S tiles ahead; the page number of the next one is on its way ----
    Steps ahead = w;
    int asked = 0, page = 0;
    auto lookup = [&]() {
      const int p = ahead.base + ahead.t * kSmall;
      page = __ldcg(kv.table + (long long)ahead.s * kv.table_stride + (p >> kv.page_shift));
    };
    auto ask = [&]() {
      const int st = asked % S;
      int pg = page;
      if ((unsigned)pg >= (unsigned)kv.n_pages) {
        atomicOr(err, kErrDecodeRange);
        pg = kv.n_pages;  // reads as zeros
      }
      const uint32_t bar = smem_u32(full + st), dst = ring + st * 2 * L::kTileBytes;
      if (lane == 0) mbar_arrive_expect_tx(bar, 2 * L::kTileBytes);
      __syncwarp();
      if (lane < 2 * kHalves) {
        const int half = lane % kHalves, is_v = lane / kHalves;
        tma_load_4d(dst + is_v * L::kTileBytes + half * (kSmall * 128), is_v ? &vmap : &kmap, half * 64,
                    (ahead.base + ahead.t * kSmall) & (kv.page_size - 1), ahead.u / zs, pg, bar);
      }
      ++asked;
      if (++ahead.at < ahead.end) {
        if (++ahead.t == ahead.nt) next_unit(ahead);
        lookup();
      }
    };
    lookup();
    while (asked < S && ahead.at < ahead.end) ask();

    const float sl2 = a.scale * 1.4426950408889634f;
    const int r = lane >> 2, c2 = (lane & 3) * 2;
    // fragments' places in a tile: keys (positions 0-7, 8-15 of a chunk, the same of the next), values (positions 0-7 of a
    // chunk and the next, positions 8-15)
    const int key_row = ((lane >> 3) & 1) * 8 + (lane & 7), key_chunk = lane >> 4;
    const int value_row = (lane >> 4) * 8 + (lane & 7), value_chunk = (lane >> 3) & 1;
    int done = 0;
    bool ok = true;
    while (ok && w.at < w.end) {
      // one segment: tiles w.t .. of unit (w.s, w.u)
      const int j = w.u / zs, h0 = (w.u % zs) * 16, nh = min(16, g - h0);
      const int t0 = w.t, t1 = (int)min((long long)w.nt, w.t + (w.end - w.at));
      uint32_t qf[N][HD / 16][2];  // head 8 n + r: values 16 k + c2 and the next, and 8 behind
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const T* q = static_cast<const T*>(a.q) + w.s * a.q_row_stride + (long long)(j * g + h0 + 8 * n + r) * a.q_head_stride + c2;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            qf[n][k][e] = 8 * n + r < nh ? __ldcg(reinterpret_cast<const unsigned*>(q + 16 * k + 8 * e)) : 0u;
      }
      // o[n][x]: values 16 x + r ([0], [1]) and 8 behind ([2], [3]) of heads 8 n + c2 and the next
      float o[N][HD / 16][4], m[N][2], l[N][2];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.0f;
#pragma unroll
        for (int x = 0; x < HD / 16; ++x) o[n][x][0] = o[n][x][1] = o[n][x][2] = o[n][x][3] = 0.0f;
      }
      for (int t = t0; t < t1; ++t, ++done) {
        const int st = done % S;
        if (!__all_sync(kFull, mbar_try_wait(smem_u32(full + st), (done / S) & 1)))
          ok = __all_sync(kFull, mbar_wait_bounded(smem_u32(full + st), (done / S) & 1));
        if (!ok) {
          if (lane == 0) atomicOr(err, kErrRingTimeout);
          break;
        }
        const uint32_t sk = ring + st * 2 * L::kTileBytes, sv = sk + L::kTileBytes;
        const int left = w.n - t * kSmall;
        // scores of positions r ([0], [1]) and r + 8, heads 8 n + c2 and the next
        float s[N][4];
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          uint32_t f[4];
          ldsm4(f, sk + tile_chunk<kSmall>(key_row, 2 * k + key_chunk));
#pragma unroll
          for (int n = 0; n < N; ++n) {
            if (k == 0) first_product<T>(s[n], f, qf[n][k][0], qf[n][k][1]);
            else product<T>(s[n], f, qf[n][k][0], qf[n][k][1]);
          }
        }
        bool rises = false;
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
          for (int k = 0; k < 4; ++k) s[n][k] *= sl2;
          if (left < kSmall) {
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
        // weights as two 16-bit parts: [k] of positions c2 + 8 k and the next, head 8 n + r
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
            const uint32_t hi = pack16<T>(p0, p1);
            const float2 q = unpack16<T>(hi);
            ph[n][k] = transposed8(hi);
            pl[n][k] = transposed8(pack16<T>(p0 - q.x, p1 - q.y));
          }
        }
        // the values of positions that do not exist are whatever the page holds: zeros instead
        uint32_t keep[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
        if (left < kSmall) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
            keep[k] = (k * 8 + c2 < left ? 0xFFFFu : 0u) | (k * 8 + c2 + 1 < left ? 0xFFFF0000u : 0u);
        }
#pragma unroll
        for (int x = 0; x < HD / 16; ++x) {
          uint32_t f[4];
          ldsm4_t(f, sv + tile_chunk<kSmall>(value_row, 2 * x + value_chunk));
          if (left < kSmall) {
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] &= keep[e >> 1];
          }
#pragma unroll
          for (int n = 0; n < N; ++n) {
            if constexpr (EXACT) {
              float y[4];
              first_product<T>(y, f, ph[n][0], ph[n][1]);
              product<T>(y, f, pl[n][0], pl[n][1]);
#pragma unroll
              for (int z = 0; z < 4; ++z) o[n][x][z] += y[z];
            } else {
              product<T>(o[n][x], f, ph[n][0], ph[n][1]);
              product<T>(o[n][x], f, pl[n][0], pl[n][1]);
            }
          }
        }
        __syncwarp();
        if (ahead.at < ahead.end) ask();  // into the stage that has just been read
      }
      if (!ok) break;

      const bool whole = t0 == 0 && t1 == w.nt;
      const int slot = 2 * index + (w.at == begin ? 0 : 1);
      float* part = v.own_slots + (size_t)slot * slot_floats(ROWS, HD);
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = 8 * n + c2 + e;
          float sum = l[n][e];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(kFull, sum, x);
          if (row >= nh) continue;
          const long long at = (long long)w.s * a.n_heads + j * g + h0 + row;
          float* to = whole ? v.own_o + at * HD : part + row * HD;
#pragma unroll
          for (int x = 0; x < HD / 16; ++x) {
            __stcg(to + 16 * x + r, o[n][x][e]);
            __stcg(to + 16 * x + 8 + r, o[n][x][2 + e]);
          }
          if (r == 0)
            __stcg(whole ? v.own_ml + at : reinterpret_cast<float2*>(part + ROWS * HD) + row, make_float2(m[n][e] - kPShift, sum));
        }
      if (t0 == 0 && lane == 0) leave(w, w.u, whole ? 1 : deal.range_of(w.first + w.nt - 1) - index + 1, index, slot);
      advance(t1 - t0);
    }
    if (!ok) abandon(w, [&]() { if (lane == 0) leave(w, w.u, 0, 0, 0); }, advance);
    // every issued copy lands before the CTA may end (bounded)
    for (int i = done; i < asked; ++i) mbar_wait_bounded(smem_u32(full + i % S), (i / S) & 1);
  }
  // The join may begin once every CTA here has ended: one that waits for the shared pass is enough, and the others leave
  // their SM to the next ones.
  if (blockIdx.x == gridDim.x - 1) pdl_wait();
}

template <class T, int HD, int ROWS, bool EXACT>
cudaError_t launch_typed(const PagedArgs& a, const KvArgs& kv, const SharedView& v, cudaStream_t stream, unsigned* err) {
  using L = LayoutOwn<HD, ROWS>;
  auto kernel = attention_own_kernel<T, HD, ROWS, EXACT>;
  CUtensorMap kmap, vmap;
  if (!encode_kv_map(&kmap, kv, kv.k, kSmall) || !encode_kv_map(&vmap, kv, kv.v, kSmall)) return cudaErrorInvalidValue;
  static std::atomic<unsigned long long> done{0};
  int sms = 0;
  const cudaError_t e = kernel_setup(reinterpret_cast<const void*>(kernel), L::kSmem, done, &sms);
  if (e != cudaSuccess) return e;
  const int ctas = 2 * sms * L::kWarps < kOwnRanges ? 2 * sms : kOwnRanges / L::kWarps;
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
  const int zs = (a.n_heads / kv.n_kv + 15) / 16;
  return cudaLaunchKernelEx(&cfg, kernel, kmap, vmap, a, kv, v, zs, err);
}

template <class T, int HD>
cudaError_t launch_rows(const PagedArgs& a, const KvArgs& kv, const SharedView& v, cudaStream_t stream, unsigned* err) {
  const bool exact = a.out_dtype == kDtF32;
  if (a.n_heads / kv.n_kv <= 8)
    return exact ? launch_typed<T, HD, 8, true>(a, kv, v, stream, err) : launch_typed<T, HD, 8, false>(a, kv, v, stream, err);
  return exact ? launch_typed<T, HD, 16, true>(a, kv, v, stream, err) : launch_typed<T, HD, 16, false>(a, kv, v, stream, err);
}

}  // namespace

size_t own_slots_floats(int n_heads, int n_kv, int head_dim) {
  return (size_t)kOwnRanges * 2 * slot_floats(n_heads / n_kv <= 8 ? 8 : 16, head_dim);
}

cudaError_t launch_attention_own(const PagedArgs& a, const KvArgs& kv, const SharedView& v, cudaStream_t stream) {
  unsigned* err = device_error_word();
  if (!err) return cudaErrorUnknown;
  if (kv.dtype == kDtF16)
    return kv.head_dim == 128 ? launch_rows<__half, 128>(a, kv, v, stream, err) : launch_rows<__half, 64>(a, kv, v, stream, err);
  return kv.head_dim == 128 ? launch_rows<__nv_bfloat16, 128>(a, kv, v, stream, err)
                            : launch_rows<__nv_bfloat16, 64>(a, kv, v, stream, err);
}

}  // namespace asmllm
