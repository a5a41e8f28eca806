// asmllm_b200/csrc/serving.cuh -- shared by the serving operators: the paged
// (or packed) key-value view, the two 16-bit types, and the launchers that
// capi.cu calls (rope_append.cu, attention_paged.cu, attention_prompt.cu,
// rows_sample.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "common.cuh"

namespace asmllm {

// Element types (ASM_DT_* of the C ABI).
constexpr int kDtF32 = 0, kDtF16 = 1, kDtBf16 = 2;

// Keys and values of a batch of sequences.  Element d of head j at (page,
// offset) is k[page * page_stride + offset * token_stride + j * head_stride + d]
// (strides in elements, the same for v).
//   paged  (table set): position p of sequence s lives at page
//     table[s * table_stride + p / page_size], offset p % page_size; the
//     sequence holds len[s] positions.
//   packed (table null): one page of page_size rows; position p of sequence s
//     is row cu[s] + p, the sequence holds cu[s + 1] - cu[s] positions.
struct KvArgs {
  void* k = nullptr;
  void* v = nullptr;
  long long page_stride = 0, token_stride = 0, head_stride = 0;
  const int32_t* table = nullptr;
  long long table_stride = 0;
  const int32_t* len = nullptr;
  const int32_t* cu = nullptr;
  int batch = 0, n_pages = 0, page_size = 0, page_shift = 0, width = 0;
  int n_kv = 0, head_dim = 0, dtype = kDtF16;
};

struct RopeAppendArgs {
  const void* qkv = nullptr;  // [rows][(n_heads + 2 n_kv) * head_dim]
  int src_dtype = kDtF32;
  long long qkv_stride = 0;
  const float* rope_cs = nullptr;  // [rope_len][head_dim / 2][2]
  int rope_len = 0;
  const int32_t* cu_q = nullptr;  // [batch + 1], or null: row r = sequence r
  int rows = 0, n_heads = 0;
  void* q_out = nullptr;  // [rows][n_heads][head_dim]
};

struct PromptArgs {
  const void* q = nullptr;  // [rows] x q_row_stride, heads q_head_stride apart
  long long q_row_stride = 0, q_head_stride = 0;
  void* out = nullptr;  // [rows][n_heads][head_dim]
  int out_dtype = kDtF16;
  const int32_t* cu_q = nullptr;
  int rows = 0, n_heads = 0;
  float scale = 0.0f;
};

struct PagedArgs {
  const void* q = nullptr;  // [batch] x q_row_stride, heads q_head_stride apart
  long long q_row_stride = 0, q_head_stride = 0;
  void* out = nullptr;  // [batch][n_heads][head_dim]
  int out_dtype = kDtF16;
  int n_heads = 0;
  float scale = 0.0f;
  void* workspace = nullptr;
};

struct SampleArgs {
  const void* logits = nullptr;
  int dtype = kDtF32;
  long long stride = 0;
  int rows = 0, n = 0;
  const float* u = nullptr;
  const float* temperature = nullptr;  // each [rows] or null: 1, off, 1, 0
  const int32_t* top_k = nullptr;
  const float* top_p = nullptr;
  const float* min_p = nullptr;
  int32_t* tokens = nullptr;
};
constexpr int kSampleMaxN = 1 << 18;

cudaError_t launch_rope_append(const RopeAppendArgs& a, const KvArgs& kv, cudaStream_t stream);
cudaError_t launch_attention_prompt(const PromptArgs& a, const KvArgs& kv, cudaStream_t stream);
size_t attention_paged_workspace(int batch, int n_heads, int n_kv, int head_dim);
cudaError_t launch_attention_paged(const PagedArgs& a, const KvArgs& kv, cudaStream_t stream);
cudaError_t launch_rows_sample(const SampleArgs& a, cudaStream_t stream);

// The current device's SM count, and a kernel's shared-memory limit raised
// once per device (`done`: one flag a device, of this kernel alone).
inline cudaError_t kernel_setup(const void* kernel, int smem, std::atomic<unsigned long long>& done, int* sms) {
  static std::atomic<int> count[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!(done.load() >> dev & 1ull)) {
    int n = 0;
    if ((e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
    if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return e;
    count[dev].store(n);
    done.fetch_or(1ull << dev);
  }
  *sms = count[dev].load();
  return cudaSuccess;
}

#ifdef __CUDACC__

// ---- the two 16-bit types ----
template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// Two floats rounded to nearest-even into one 32-bit word, lo in the low half.
template <class T> __device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <> __device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <class T> __device__ __forceinline__ float2 unpack16(uint32_t w);
template <> __device__ __forceinline__ float2 unpack16<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <> __device__ __forceinline__ float2 unpack16<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// Eight consecutive values as floats; T float (two 16-byte loads) or 16-bit (one).
template <class T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = __ldcg(reinterpret_cast<const float4*>(p)), b = __ldcg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 a = __ldcg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack16<T>(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

template <class T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack16<T>(v[0], v[1]), pack16<T>(v[2], v[3]), pack16<T>(v[4], v[5]),
                                              pack16<T>(v[6], v[7]));
  }
}

// Positions of sequence s that may be read: its length, held inside what the
// table (or the packed rows) can address.  *clipped says that it had to be.
__device__ __forceinline__ int kv_length(const KvArgs& kv, int s, bool* clipped) {
  if (kv.table) {
    const int n = __ldcg(kv.len + s);
    const long long cap = (long long)kv.width << kv.page_shift;
    *clipped = n < 0 || n > cap;
    return n < 0 ? 0 : (int)(n > cap ? cap : n);
  }
  const int b = __ldcg(kv.cu + s), e = __ldcg(kv.cu + s + 1);
  *clipped = b < 0 || e > kv.page_size || e < b;
  return *clipped ? 0 : e - b;
}

// Rows [begin, end) of sequence s in a packed query of `rows` rows; false
// for offsets outside it, which give an empty sequence.
__device__ __forceinline__ bool q_range(const int32_t* cu_q, int s, int rows, int* begin, int* end) {
  if (!cu_q) {
    *begin = s;
    *end = s + 1;
    return true;
  }
  const int b = __ldcg(cu_q + s), e = __ldcg(cu_q + s + 1);
  const bool ok = b >= 0 && e <= rows && b <= e;
  *begin = ok ? b : 0;
  *end = ok ? e : 0;
  return ok;
}

// Element offset of position p of sequence s, head 0; negative when the page
// number is outside the pool.  p must be below kv_length().
__device__ __forceinline__ long long kv_offset(const KvArgs& kv, int s, int p) {
  if (!kv.table) return (long long)(__ldcg(kv.cu + s) + p) * kv.token_stride;
  const int page = __ldcg(kv.table + (long long)s * kv.table_stride + (p >> kv.page_shift));
  if ((unsigned)page >= (unsigned)kv.n_pages) return -1;
  return (long long)page * kv.page_stride + (long long)(p & (kv.page_size - 1)) * kv.token_stride;
}

#endif  // __CUDACC__

}  // namespace asmllm
