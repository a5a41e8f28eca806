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

// One CTA per row, one thread per 8 values: four lanes hold a block of 32.
template <class S, class T>
__global__ void __launch_bounds__(256) rope_append_q8_kernel(const RopeAppendArgs a, const KvQ8Args c,
                                                             unsigned* __restrict__ err) {
  __shared__ int s_pos, s_page;
  pdl_trigger();
  pdl_wait();
  const KvArgs& kv = c.kv;
  const int t = blockIdx.x, hd = kv.head_dim;
  if (threadIdx.x == 0) {
    const int seq = a.cu_q ? seq_of(a.cu_q, kv.batch, t) : t;
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
    s_pos = pos;
    s_page = page;
  }
  if (blockIdx.x == 0) report_ranges(kv, a.cu_q, a.rows, err);
  __syncthreads();
  const int pos = s_pos, page = s_page;
  if (pos == -2) return;
  const S* src = static_cast<const S*>(a.qkv) + (long long)t * a.qkv_stride;
  const int per = hd / 8, nq = a.n_heads, nk = kv.n_kv, in = kv.page_size - 1 & pos;
  const float* cs = a.rope_cs + (long long)(pos < 0 ? 0 : pos) * hd;
  const int total = (nq + 2 * nk) * per;
  for (int i0 = threadIdx.x & ~31; i0 < total; i0 += blockDim.x) {  // whole warps: blocks are made with shuffles
    const int i = i0 + (threadIdx.x & 31), h = i / per, e = (i % per) * 8;
    const bool live = i < total;
    float v[8] = {};
    if (live) load8(src + h * hd + e, v);
    if (live && h < nq + nk) {
      const float4 r0 = __ldcg(reinterpret_cast<const float4*>(cs + e));
      const float4 r1 = __ldcg(reinterpret_cast<const float4*>(cs + e) + 1);
      const float f[8] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float x0 = v[j], x1 = v[j + 1];
        v[j] = __fsub_rn(__fmul_rn(x0, f[j]), __fmul_rn(x1, f[j + 1]));
        v[j + 1] = __fadd_rn(__fmul_rn(x0, f[j + 1]), __fmul_rn(x1, f[j]));
      }
    }
    if (live && h < nq) {
      if (pos < 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
      }
      store8(static_cast<T*>(a.q_out) + ((long long)t * nq + h) * hd + e, v);
    }
    if (__all_sync(kFull, !live || h < nq)) continue;
    float d;
    int sum;
    unsigned c0, c1;
    quantize_oct(make_float4(v[0], v[1], v[2], v[3]), make_float4(v[4], v[5], v[6], v[7]), d, sum, c0, c1);
    if (!live || h < nq || page < 0) continue;
    const int j = (h - nq) % nk;
    const bool is_k = h < nq + nk;
    int8_t* codes = static_cast<int8_t*>(is_k ? kv.k : kv.v) + (long long)page * kv.page_stride +
                    (long long)in * kv.token_stride + (long long)j * kv.head_stride + e;
    *reinterpret_cast<uint2*>(codes) = make_uint2(c0, c1);
    if ((e & 31) == 0)
      (is_k ? c.ks : c.vs)[(long long)page * c.scale_page_stride + (long long)j * c.scale_head_stride + in * (hd / 32) +
                           e / 32] = __float2half_rn(d);
  }
}

constexpr int kReadRows = 32;  // at most

// `per_cta` rows a CTA (their sequences and pages are looked up by as many threads), one thread per 16 values.
template <class T>
__global__ void __launch_bounds__(256) cache_read_q8_kernel(const CacheReadArgs a, const KvQ8Args c, int per_cta,
                                                            unsigned* __restrict__ err) {
  __shared__ int s_page[kReadRows], s_in[kReadRows];
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
    s_in[threadIdx.x] = in;
  }
  if (blockIdx.x == 0) report_ranges(kv, a.cu, a.rows, err);
  __syncthreads();
  const int hd = kv.head_dim, per = hd / 16, row = kv.n_kv * per;  // pieces of a head, of a row of keys
  for (int i = threadIdx.x; i < rows * 2 * row; i += blockDim.x) {
    const int r = i / (2 * row), x = i % (2 * row), is_v = x >= row, h = (x - is_v * row) / per, e = (x % per) * 16;
    const int page = s_page[r], in = s_in[r];
    if (page == -2) continue;
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    float d = 0.0f;
    if (page >= 0) {
      const int8_t* codes = static_cast<const int8_t*>(is_v ? kv.v : kv.k) + (long long)page * kv.page_stride +
                            (long long)in * kv.token_stride + (long long)h * kv.head_stride + e;
      w = __ldcg(reinterpret_cast<const uint4*>(codes));
      d = __half2float((is_v ? c.vs : c.ks)[(long long)page * c.scale_page_stride + (long long)h * c.scale_head_stride +
                                            in * (hd / 32) + e / 32]);
    }
    const uint32_t b[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
    T* out = static_cast<T*>(is_v ? a.v : a.k) + ((long long)(t0 + r) * kv.n_kv + h) * hd + e;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = s8_biased_to_f32(b[2 * q + (j >> 2)], j & 3) * d;
      store8(out + 8 * q, v);
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
  const bool f32 = a.src_dtype == kDtF32;
  if (q_dtype == kDtF16)
    return f32 ? launch(rope_append_q8_kernel<float, __half>, a.rows, stream, a, c, err)
               : launch(rope_append_q8_kernel<__half, __half>, a.rows, stream, a, c, err);
  return f32 ? launch(rope_append_q8_kernel<float, __nv_bfloat16>, a.rows, stream, a, c, err)
             : launch(rope_append_q8_kernel<__nv_bfloat16, __nv_bfloat16>, a.rows, stream, a, c, err);
}

cudaError_t launch_cache_read_q8(const CacheReadArgs& a, const KvQ8Args& c, cudaStream_t stream) {
  unsigned* err = device_error_word();
  if (!err) return cudaErrorUnknown;
  // Eight pieces a thread where that leaves two CTAs an SM or more, fewer rows a CTA otherwise.
  const int pieces = 2 * c.kv.n_kv * (c.kv.head_dim / 16);
  int per = (2048 + pieces - 1) / pieces;
  per = per > kReadRows ? kReadRows : per;
  while (per > 1 && (a.rows + per - 1) / per < 296) per >>= 1;
  const int grid = (a.rows + per - 1) / per;
  return a.dtype == kDtF16 ? launch(cache_read_q8_kernel<__half>, grid, stream, a, c, per, err)
                           : launch(cache_read_q8_kernel<__nv_bfloat16>, grid, stream, a, c, per, err);
}

}  // namespace asmllm
