// asmllm_b200/csrc/rope_append.cu -- rotary positions on the query and key
// heads of packed rows, the rotated query rounded to the cache's type, keys
// and values appended to their pages.
//
// The arithmetic is the batch-1 decode kernel's (attention.cuh): interleaved
// pairs (x0 c - x1 s, x0 s + x1 c) with each product and sum rounded to fp32,
// then one rounding to 16 bits (THRISHAL12345/asmllm tests/reference/ops.py:
// 119-141).  Row t of sequence s holds position
//   p = len[s] - (cu_q[s + 1] - cu_q[s]) + (t - cu_q[s]);
// a row at p < 0 (a sequence with more rows than positions) gets a zero query
// and appends nothing; so does one whose position or page is out of range,
// which also sets the device error word.
//
// Bound by HBM: every input is read and every output written once.  8192 rows
// of 32 query and 32 + 32 key and value heads of 128 values, fp32 to fp16,
// take 93 us on one B200 = 6.5 TB/s, the copy rate; 32 rows 3.9 us, a launch.
#include "matvec.cuh"
#include "serving.cuh"

namespace asmllm {

namespace {

// One thread per 8 values (4 pairs): two 16-byte loads of fp32 input, one
// 16-byte store.  One CTA per row: the row's sequence and page are looked up
// once by thread 0.
template <class S, class T>
__global__ void __launch_bounds__(256) rope_append_kernel(const RopeAppendArgs a, const KvArgs kv,
                                                          unsigned* __restrict__ err) {
  __shared__ int s_pos;
  __shared__ long long s_off;
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x, hd = kv.head_dim;
  if (threadIdx.x == 0) {
    int seq = t;
    if (a.cu_q) {  // the last sequence that begins at or before row t
      int lo = 0, hi = kv.batch;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (__ldcg(a.cu_q + mid + 1) <= t) lo = mid + 1; else hi = mid;
      }
      seq = lo;
    }
    int pos = -2;  // a row behind the last sequence: left as it is
    long long off = -1;
    if (seq < kv.batch) {
      int b, e;
      q_range(a.cu_q, seq, a.rows, &b, &e);
      if (t >= b && t < e) {
        pos = max(-1, __ldcg(kv.len + seq) - (e - b) + (t - b));
        if (pos >= 0) {  // outside the rotary table, the sequence's pages or the pool: skipped
          if (pos < a.rope_len && pos < ((long long)kv.width << kv.page_shift)) off = kv_offset(kv, seq, pos);
          if (off < 0) {
            atomicOr(err, kErrDecodeRange);
            pos = -1;
          }
        }
      }
    }
    s_pos = pos;
    s_off = off;
  }
  if (blockIdx.x == 0) {  // lengths and offsets out of range are reported whether a row meets them or not
    for (int s = blockDim.x - 1 - threadIdx.x; s < kv.batch; s += blockDim.x) {
      bool clipped;
      int b, e;
      kv_length(kv, s, &clipped);
      if (clipped || !q_range(a.cu_q, s, a.rows, &b, &e)) atomicOr(err, kErrDecodeRange);
    }
  }
  __syncthreads();
  const int pos = s_pos;
  const long long off = s_off;
  if (pos == -2) return;
  const S* src = static_cast<const S*>(a.qkv) + (long long)t * a.qkv_stride;
  const int per = hd / 8, nq = a.n_heads, nk = kv.n_kv;
  const float* cs = a.rope_cs + (long long)(pos < 0 ? 0 : pos) * hd;
  for (int i = threadIdx.x; i < (nq + 2 * nk) * per; i += blockDim.x) {
    const int h = i / per, c = (i % per) * 8;
    float v[8];
    load8(src + h * hd + c, v);
    if (h < nq + nk) {
      const float4 r0 = __ldcg(reinterpret_cast<const float4*>(cs + c));
      const float4 r1 = __ldcg(reinterpret_cast<const float4*>(cs + c) + 1);
      const float f[8] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float x0 = v[j], x1 = v[j + 1];
        v[j] = __fsub_rn(__fmul_rn(x0, f[j]), __fmul_rn(x1, f[j + 1]));
        v[j + 1] = __fadd_rn(__fmul_rn(x0, f[j + 1]), __fmul_rn(x1, f[j]));
      }
    }
    if (h < nq) {
      if (pos < 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
      }
      store8(static_cast<T*>(a.q_out) + ((long long)t * nq + h) * hd + c, v);
    } else if (off >= 0) {
      T* base = static_cast<T*>(h < nq + nk ? kv.k : kv.v);
      store8(base + off + (long long)((h - nq) % nk) * kv.head_stride + c, v);
    }
  }
}

template <class S, class T>
cudaError_t launch_typed(const RopeAppendArgs& a, const KvArgs& kv, cudaStream_t stream, unsigned* err) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_opt_pdl.load() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, rope_append_kernel<S, T>, a, kv, err);
}

}  // namespace

cudaError_t launch_rope_append(const RopeAppendArgs& a, const KvArgs& kv, cudaStream_t stream) {
  unsigned* err = device_error_word();
  if (!err) return cudaErrorUnknown;
  if (kv.dtype == kDtF16)
    return a.src_dtype == kDtF32 ? launch_typed<float, __half>(a, kv, stream, err)
                                 : launch_typed<__half, __half>(a, kv, stream, err);
  return a.src_dtype == kDtF32 ? launch_typed<float, __nv_bfloat16>(a, kv, stream, err)
                               : launch_typed<__nv_bfloat16, __nv_bfloat16>(a, kv, stream, err);
}

}  // namespace asmllm
