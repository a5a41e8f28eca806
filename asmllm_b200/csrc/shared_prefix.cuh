// asmllm_b200/csrc/shared_prefix.cuh -- groups of sequences that share their
// first positions: what the pass over those (attention_shared.cu) and the pass
// over the rest (attention_own.cu) agree on.
#pragma once

#include "found.cuh"
#include "paged_deal.cuh"

namespace asmllm {

// Of a sequence's own positions, and the group whose result is to be joined with it.
struct OwnFound {
  Found found;
  int group;       // -1: none
  int first, end;  // the group's sequences
  int pad;
};

struct SharedView {
  const int32_t* cu_group = nullptr;
  const int32_t* shared_len = nullptr;
  int groups = 0;
  // results of the positions that are not shared, unnormalised: [batch][n_heads][head_dim], (maximum in units of
  // log2, sum) [batch][n_heads], and where each unit's are
  float* own_o = nullptr;
  float2* own_ml = nullptr;
  OwnFound* own_found = nullptr;  // [batch][n_kv * zs]
  float* own_slots = nullptr;
};

#ifdef __CUDACC__

// Sequences [*b, *e) of group g, and how many positions they share (whole pages); false for offsets out of range.
__device__ __forceinline__ bool group_of(const SharedView& v, const KvArgs& kv, int g, int* b, int* e, int* shared) {
  *b = __ldcg(v.cu_group + g);
  *e = __ldcg(v.cu_group + g + 1);
  const int n = __ldcg(v.shared_len + g);
  const long long cap = (long long)kv.width << kv.page_shift;
  *shared = n < 0 ? 0 : (int)(n > cap ? cap : n) & ~(kv.page_size - 1);
  const bool ok = *b >= 0 && *e <= kv.batch && *b <= *e;
  if (!ok) *b = *e = 0;
  return ok && n >= 0 && n <= cap;
}

// Positions of sequence s, of n, that it shares with its group, and (group, its sequences): none, and -1, for a sequence
// without a group, or with fewer positions than the group shares.
__device__ __forceinline__ int shared_base(const SharedView& v, const KvArgs& kv, int s, int n, int4* group) {
  int lo = 0, hi = v.groups;
  while (lo < hi) {  // the first group that ends behind s
    const int mid = (lo + hi) >> 1;
    if (__ldcg(v.cu_group + mid + 1) <= s) lo = mid + 1; else hi = mid;
  }
  *group = make_int4(-1, 0, 0, 0);
  if (lo >= v.groups) return 0;
  int b, e, shared;
  group_of(v, kv, lo, &b, &e, &shared);
  if (s < b || s >= e || n < shared || shared == 0) return 0;
  *group = make_int4(lo, b, e, 0);
  return shared;
}

#endif  // __CUDACC__

// The pass over the positions that are not shared (attention_own.cu): results into `v`, none joined.
constexpr int kOwnRanges = 2400;  // at most, one a warp
size_t own_slots_floats(int n_heads, int n_kv, int head_dim);
cudaError_t launch_attention_own(const PagedArgs& a, const KvArgs& kv, const SharedView& v, cudaStream_t stream);

}  // namespace asmllm
