// asmllm_b200/csrc/serving_q8.cuh -- the Q8_0 key-value cache, and the
// launchers of the operators around it, of attention over shared prefixes and
// of the changes to logits (cache_q8.cu, attention_paged_q8.cu,
// attention_shared.cu, rows_adjust.cu).
#pragma once

#include "serving.cuh"

namespace asmllm {

// Keys and values in 8 bits: kv.k and kv.v hold the int8 codes (strides in
// bytes, always paged); the fp16 scales of position `offset` of a page and
// head are the head_dim / 32 values from
//   ks + page * scale_page_stride + head * scale_head_stride + offset * head_dim / 32,
// so that a head's scales of a whole page lie side by side.  A value is its
// code times the scale of its block of 32.
struct KvQ8Args {
  KvArgs kv;
  __half* ks = nullptr;
  __half* vs = nullptr;
  long long scale_page_stride = 0, scale_head_stride = 0;
};

struct CacheReadArgs {
  const int32_t* cu = nullptr;  // [batch + 1]: row cu[s] + i holds position len[s] - (cu[s + 1] - cu[s]) + i
  int rows = 0;
  void* k = nullptr;  // [rows][n_kv][head_dim]
  void* v = nullptr;
  int dtype = kDtF16;
};

struct SharedArgs {
  PagedArgs paged;
  const int32_t* cu_group = nullptr;    // [groups + 1]: the sequences of each group
  const int32_t* shared_len = nullptr;  // [groups]
  int groups = 0;
};

struct AdjustArgs {
  const void* logits = nullptr;
  void* out = nullptr;
  int dtype = kDtF32;
  long long stride = 0, out_stride = 0;
  int rows = 0, n = 0;
  const int32_t* tokens = nullptr;  // [rows] x token_stride, held tokens each; null: no penalties
  long long token_stride = 0;
  int held = 0;
  const int32_t* n_tokens = nullptr;  // each [rows] or null: held, 0, 1, 0, 0
  const int32_t* n_prompt = nullptr;
  const float* repetition = nullptr;
  const float* frequency = nullptr;
  const float* presence = nullptr;
  const int32_t* bias_tokens = nullptr;  // [rows][n_bias] or null
  const float* bias = nullptr;
  int n_bias = 0;
  const int32_t* allowed = nullptr;  // [rows] x allowed_stride words of 32 bits, or null
  long long allowed_stride = 0;
};
constexpr int kAdjustMaxBias = 1024, kAdjustMaxN = 1 << 18;

cudaError_t launch_rope_append_q8(const RopeAppendArgs& a, int q_dtype, const KvQ8Args& c, cudaStream_t stream);
cudaError_t launch_cache_read_q8(const CacheReadArgs& a, const KvQ8Args& c, cudaStream_t stream);
size_t attention_paged_q8_workspace(int batch, int n_heads, int n_kv, int head_dim);
cudaError_t launch_attention_paged_q8(const PagedArgs& a, int q_dtype, const KvQ8Args& c, cudaStream_t stream);
size_t attention_shared_workspace(int batch, int groups, int n_heads, int n_kv, int head_dim);
cudaError_t launch_attention_shared(const SharedArgs& a, const KvArgs& kv, cudaStream_t stream);
cudaError_t launch_rows_adjust(const AdjustArgs& a, cudaStream_t stream);

}  // namespace asmllm
