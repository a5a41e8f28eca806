// asmllm_b200/csrc/cache_q8.cu -- a paged key-value cache in Q8_0: rotary
// positions and append (the rows quantised as they are written), and rows read
// back in 16 bits.
//
// Append: the rotary arithmetic of rope_append.cu in fp32 (each product and
// sum rounded), then for each block of 32 values of a key or value head
//   a = max |x|,  code = rne(x (127 / a)),  scale = fp16(a / 127)
// in the fp32 steps of common.cuh, so the codes are those asm_quantize_q8_0
// gives for the rotated row.  A NaN or an infinity makes its block's scale NaN
// or infinity, and so the whole block NaN to every reader.
// Read back: code * scale is exact in fp32 (8 and 11 bits) and rounded once.
//
// Both are bound by HBM: every input is read and every output written once.
// At 8192 rows of 32 heads of 128 values the append of fp32 rows takes 96 us
// (5.7 TB/s) and the read 36 us (5.7 TB/s); for 32 single tokens 3.7 and 3.4.
// 2048 rows of 64 + 2 x 8 heads in 16 bits, half the bytes for the same
// arithmetic, 18.6 (4.3 TB/s: the quantizer's instructions).
#include "matvec.cuh"
#include "serving_q8.cuh"

namespace asmllm {

namespace {

// The sequence that holds packed row t: the last one that begins at or before it (batch: none).
__device__ __forceinline__ int seq_of(const int32_t* cu, int batch, int t) {
  int lo = 0, hi = batch;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldcg(cu + mid + 1) <= t) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// Lengths and offsets out of range are reported whether a row meets them or not.
__device__ __forceinline__ void report_ranges(const KvArgs& kv, const int32_t* cu, int rows, unsigned* err) {
  for (int s = blockDim.x - 1 - threadIdx.x; s < kv.batch; s += blockDim.x) {
    bool clipped;
    int b, e;
    kv_length(kv, s, &clipped);
    if (clipped || !q_range(cu, s, rows, &b, &e)) atomicOr(err, kErrDecodeRange);
  }
}

constexpr int kRows = 32;  // of a CTA, at most

// max |x|, |y| with NaN where either is.
__device__ __forceinline__ float max_abs(float x, float y) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(fabsf(x)), "f"(fabsf(y)));
  return m;
}

// The codes rne(v inv) of 8 values of a block whose largest |v| is a and inv = 127 / a.  |v inv| < 127.5 there, so adding
// 1.5 2^23 rounds to an integer whose low byte is the code.  A block with a NaN or an infinity, or so small that 127 / a
// overflows, takes the conversion instead: NaN to 0, the rest clamped.
__device__ __forceinline__ uint2 codes_of(const float (&v)[8], float a, float inv) {
  uint32_t c[8];
  if (a + inv < INFINITY) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = __float_as_uint(__fadd_rn(__fmul_rn(v[j], inv), 12582912.0f));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float t = __fmul_rn(v[j], inv);
      c[j] = t != t ? 0u : (uint32_t)__float2int_rn(fminf(fmaxf(t, -128.0f), 127.0f));
    }
  }
  return make_uint2(__byte_perm(__byte_perm(c[0], c[1], 0x0040u), __byte_perm(c[2], c[3], 0x0040u), 0x5410u),
                    __byte_perm(__byte_perm(c[4], c[5], 0x0040u), __byte_perm(c[6], c[7], 0x0040u), 0x5410u));
}

// `per_cta` rows a CTA (their sequences and pages are looked up by as many threads), one thread per 8 values: four lanes
// hold a block of 32.  A thread has the same values of every head that it comes to, so its part of the rotary table stays in
// registers.  Two heads go at a time: their loads are under way together, and each of a block's four lanes divides for one of
// them.  8192 rows of 96 fp32 heads 96 us; with four heads at a time (80 registers, 24 warps an SM) 108, with one division
// for each block in every lane and 64-bit addresses made for each head 115.
template <class S, class T, int HD>
__global__ void __launch_bounds__(256, 4) rope_append_q8_kernel(const RopeAppendArgs a, const KvQ8Args c, int per_cta,
                                                                unsigned* __restrict__ err) {
  constexpr int kPer = HD / 8, kStep = 256 / kPer, kHeads = 2;
  __shared__ int s_pos[kRows], s_page[kRows];
  pdl_trigger();
  pdl_wait();
  const KvArgs& kv = c.kv;
  const int t0 = blockIdx.x * per_cta, rows = min(per_cta, a.rows - t0);
  if (threadIdx.x < rows) {
    const int t = t0 + threadIdx.x, seq = a.cu_q ? seq_of(a.cu_q, kv.batch, t) : t;
    int pos = -2, page = -1;  // -2: a row behind the last sequence, left as it is
    if (seq < kv.batch) {
      int b, e;
      q_range(a.cu_q, seq, a.rows, &b, &e);
      if (t >= b && t < e) {
        pos = max(-1, __ldcg(kv.len + seq) - (e - b) + (t - b));
        if (pos >= 0) {  // outside the rotary table, the sequence's pages or the pool: skipped
          if (pos < a.rope_len && pos < ((long long)kv.width << kv.page_shift)) {
            page = __ldcg(kv.table + (long long)seq * kv.table_stride + (pos >> kv.page_shift));
            if ((unsigned)page >= (unsigned)kv.n_pages) page = -1;
          }
          if (page < 0) {
            atomicOr(err, kErrDecodeRange);
            pos = -1;
          }
        }
      }
    }
    s_pos[threadIdx.x] = pos;
    s_page[threadIdx.x] = page;
  }
  if (blockIdx.x == 0) report_ranges(kv, a.cu_q, a.rows, err);
  const int nq = a.n_heads, nk = kv.n_kv, heads = nq + 2 * nk, e = (threadIdx.x % kPer) * 8;
  const S* src = static_cast<const S*>(a.qkv) + (long long)t0 * a.qkv_stride + e;
  float v[kHeads][8];
  auto load = [&](int h0) {
#pragma unroll
    for (int u = 0; u < kHeads; ++u)
      if (h0 + u * kStep < heads) load8(src + (h0 + u * kStep) * HD, v[u]);
  };
  load(threadIdx.x / kPer);  // where the rows go is looked up meanwhile
  __syncthreads();
  const int first = (int)(threadIdx.x & ~31u) / kPer, own = threadIdx.x % 4;  // the warp's first head; the head divided for
  for (int r = 0; r < rows; ++r, src += a.qkv_stride) {
    const int t = t0 + r, pos = s_pos[r], page = s_page[r], in = pos & (kv.page_size - 1);
    if (pos == -2) continue;
    const long long codes = (long long)page * kv.page_stride + (long long)in * kv.token_stride + e;
    const long long scales = (long long)page * c.scale_page_stride + in * (HD / 32) + e / 32;
    float f[8];
    load8(a.rope_cs + (long long)(pos < 0 ? 0 : pos) * HD + e, f);
    for (int base = first; base < heads; base += kHeads * kStep) {  // whole warps
      const int h0 = base + (int)(threadIdx.x % 32) / kPer;
      if (r > 0 || base != first) load(h0);
      float top[kHeads] = {};
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        const int h = h0 + u * kStep;
        if (h < min(heads, nq + nk)) {
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const float x0 = v[u][j], x1 = v[u][j + 1];
            v[u][j] = __fsub_rn(__fmul_rn(x0, f[j]), __fmul_rn(x1, f[j + 1]));
            v[u][j + 1] = __fadd_rn(__fmul_rn(x0, f[j + 1]), __fmul_rn(x1, f[j]));
          }
          if (h < nq) {
            if (pos < 0) {
#pragma unroll
              for (int j = 0; j < 8; ++j) v[u][j] = 0.0f;
            }
            store8(static_cast<T*>(a.q_out) + ((long long)t * nq + h) * HD + e, v[u]);
          }
        }
        if (h >= nq && h < heads)
          top[u] = max_abs(max_abs(max_abs(v[u][0], v[u][1]), max_abs(v[u][2], v[u][3])),
                           max_abs(max_abs(v[u][4], v[u][5]), max_abs(v[u][6], v[u][7])));
      }
      if (page < 0 || base + (kHeads - 1) * kStep + 32 / kPer <= nq) continue;  // queries alone
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        top[u] = max_abs(top[u], __shfl_xor_sync(kFull, top[u], 1));
        top[u] = max_abs(top[u], __shfl_xor_sync(kFull, top[u], 2));
      }
      const float m = own & 1 ? top[1] : top[0];
      const float d = __fdiv_rn(m, 127.0f), inv = m == 0.0f ? 0.0f : __fdiv_rn(127.0f, m);
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        const int h = h0 + u * kStep;
        const float by = __shfl_sync(kFull, inv, u, 4);
        if (h < nq || h >= heads) continue;
        const bool is_k = h < nq + nk;
        const int j = h - (is_k ? nq : nq + nk);
        *reinterpret_cast<uint2*>(static_cast<int8_t*>(is_k ? kv.k : kv.v) + codes + (long long)j * kv.head_stride) =
            codes_of(v[u], top[u], by);
        if (own == u) (is_k ? c.ks : c.vs)[scales + (long long)j * c.scale_head_stride] = __float2half_rn(d);
      }
    }
  }
}

// code * scale of 16 codes, rounded once, in one 32-byte store where the rows start on 32 bytes (the address is on 16).
__device__ __forceinline__ void store32(void* p, const uint32_t (&x)[8]) {
  if (((uintptr_t)p & 31) == 0) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(x[0]), "r"(x[1]), "r"(x[2]),
                 "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7])
                 : "memory");
  } else {
    static_cast<uint4*>(p)[0] = make_uint4(x[0], x[1], x[2], x[3]);
    static_cast<uint4*>(p)[1] = make_uint4(x[4], x[5], x[6], x[7]);
  }
}
__device__ __forceinline__ void store16(__half* p, uint4 w, __half d) {  // 1024 + 128 + code in 16 bits; the product rounds once
  const uint32_t b[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
  const __half2 off = __float2half2_rn(1152.0f), d2 = __half2half2(d);
  uint32_t x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t c = __byte_perm(b[j >> 1], 0x64646464u, j & 1 ? 0x4342u : 0x4140u);
    const __half2 v = __hmul2_rn(__hsub2_rn(*reinterpret_cast<const __half2*>(&c), off), d2);
    x[j] = *reinterpret_cast<const uint32_t*>(&v);
  }
  store32(p, x);
}
__device__ __forceinline__ void store16(__nv_bfloat16* p, uint4 w, __half d) {
  const uint32_t b[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
  const float scale = __half2float(d);
  uint32_t x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t q = b[j >> 1];
    const int k = 2 * (j & 1);
    const __nv_bfloat162 v = __floats2bfloat162_rn(s8_biased_to_f32(q, k) * scale, s8_biased_to_f32(q, k + 1) * scale);
    x[j] = *reinterpret_cast<const uint32_t*>(&v);
  }
  store32(p, x);
}

// `per_cta` rows a CTA (their sequences and pages are looked up by as many threads), one thread per 16 values.
// One piece at a time: two or four under way together cost registers and are slower (39 and 43 us against 36).
template <class T, int HD>
__global__ void __launch_bounds__(256) cache_read_q8_kernel(const CacheReadArgs a, const KvQ8Args c, int per_cta,
                                                            unsigned* __restrict__ err) {
  __shared__ int s_page[kRows];
  __shared__ long long s_codes[kRows], s_scales[kRows];
  pdl_trigger();
  pdl_wait();
  const KvArgs& kv = c.kv;
  const int t0 = blockIdx.x * per_cta, rows = min(per_cta, a.rows - t0);
  if (threadIdx.x < rows) {
    const int t = t0 + threadIdx.x, seq = seq_of(a.cu, kv.batch, t);
    int page = -2, in = 0;  // -2: a row behind the last sequence, left as it is; -1: zeros
    if (seq < kv.batch) {
      int b, e;
      bool clipped;
      q_range(a.cu, seq, a.rows, &b, &e);
      if (t >= b && t < e) {
        const int len = kv_length(kv, seq, &clipped), pos = len - (e - b) + (t - b);
        page = -1;
        if (pos >= 0) {
          page = __ldcg(kv.table + (long long)seq * kv.table_stride + (pos >> kv.page_shift));
          in = pos & (kv.page_size - 1);
          if ((unsigned)page >= (unsigned)kv.n_pages) {
            atomicOr(err, kErrDecodeRange);
            page = -1;
          }
        }
      }
    }
    s_page[threadIdx.x] = page;
    s_codes[threadIdx.x] = (long long)page * kv.page_stride + (long long)in * kv.token_stride;
    s_scales[threadIdx.x] = (long long)page * c.scale_page_stride + in * (HD / 32);
  }
  if (blockIdx.x == 0) report_ranges(kv, a.cu, a.rows, err);
  __syncthreads();
  constexpr int kPer = HD / 16;  // pieces of a head
  const int half = kv.n_kv * kPer, row = 2 * half;
  int r = threadIdx.x / row, x = threadIdx.x % row;  // this thread's next piece: its row, its place there
  const int dr = 256 / row, dx = 256 % row;
  while (r < rows) {
    const int page = s_page[r];
    if (page != -2) {
      const bool is_v = x >= half;
      const int y = x - (is_v ? half : 0), h = y / kPer, e = (y % kPer) * 16;
      uint4 w = make_uint4(0u, 0u, 0u, 0u);
      __half d = __ushort_as_half(0);
      if (page >= 0) {
        w = __ldcg(reinterpret_cast<const uint4*>(static_cast<const int8_t*>(is_v ? kv.v : kv.k) + s_codes[r] +
                                                  (long long)h * kv.head_stride + e));
        d = (is_v ? c.vs : c.ks)[s_scales[r] + (long long)h * c.scale_head_stride + e / 32];
      }
      store16(static_cast<T*>(is_v ? a.v : a.k) + (long long)(t0 + r) * (half * 16) + y * 16, w, d);
    }
    r += dr;
    x += dx;
    if (x >= row) {
      x -= row;
      ++r;
    }
  }
}

template <class... Args>
cudaError_t launch(void (*kernel)(Args...), int grid, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_opt_pdl.load() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace

cudaError_t launch_rope_append_q8(const RopeAppendArgs& a, int q_dtype, const KvQ8Args& c, cudaStream_t stream) {
  unsigned* err = device_error_word();
  if (!err) return cudaErrorUnknown;
  const bool f32 = a.src_dtype == kDtF32, wide = c.kv.head_dim == 128;
  // Four rows a CTA, whose places are looked up once, where that leaves four CTAs an SM or more.
  int per = 4;
  while (per > 1 && (a.rows + per - 1) / per < 4 * 148) per >>= 1;
  auto go = [&](auto* k128, auto* k64) { return launch(wide ? k128 : k64, (a.rows + per - 1) / per, stream, a, c, per, err); };
  if (q_dtype == kDtF16)
    return f32 ? go(rope_append_q8_kernel<float, __half, 128>, rope_append_q8_kernel<float, __half, 64>)
               : go(rope_append_q8_kernel<__half, __half, 128>, rope_append_q8_kernel<__half, __half, 64>);
  return f32 ? go(rope_append_q8_kernel<float, __nv_bfloat16, 128>, rope_append_q8_kernel<float, __nv_bfloat16, 64>)
             : go(rope_append_q8_kernel<__nv_bfloat16, __nv_bfloat16, 128>, rope_append_q8_kernel<__nv_bfloat16, __nv_bfloat16, 64>);
}

cudaError_t launch_cache_read_q8(const CacheReadArgs& a, const KvQ8Args& c, cudaStream_t stream) {
  unsigned* err = device_error_word();
  if (!err) return cudaErrorUnknown;
  // Four pieces a thread (8192 rows of 32 heads: 36 us; eight 36, sixteen 44) where that leaves two CTAs an SM or more,
  // fewer rows a CTA otherwise.
  const int pieces = 2 * c.kv.n_kv * (c.kv.head_dim / 16);
  int per = (1024 + pieces - 1) / pieces;
  per = per > kRows ? kRows : per;
  while (per > 1 && (a.rows + per - 1) / per < 296) per >>= 1;
  const int grid = (a.rows + per - 1) / per;
  auto go = [&](auto* k128, auto* k64) { return launch(c.kv.head_dim == 128 ? k128 : k64, grid, stream, a, c, per, err); };
  return a.dtype == kDtF16 ? go(cache_read_q8_kernel<__half, 128>, cache_read_q8_kernel<__half, 64>)
                           : go(cache_read_q8_kernel<__nv_bfloat16, 128>, cache_read_q8_kernel<__nv_bfloat16, 64>);
}

}  // namespace asmllm
