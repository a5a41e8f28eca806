// asmllm_b200/csrc/attention_prompt.cu -- causal attention of whole prompts:
// packed query rows of sequences of different lengths, grouped heads, keys
// and values packed the same way or in the pages of a cache.
//
// Row t of sequence s sits at position p = n_s - (cu_q[s+1] - cu_q[s]) +
// (t - cu_q[s]), n_s the sequence's key count, and
//   out[t][h] = sum_{j <= p} softmax_j(scale q[t][h] . k[j][h / g]) v[j][h / g];
// p < 0: zeros.
#include "matvec.cuh"
#include "mma16.cuh"
#include "serving.cuh"

namespace asmllm {

namespace {

constexpr int kTile = 64;   // query rows per CTA (16 per warp) and positions per tile
constexpr int kWarps = 4;

// A row whose output is not finite, computed again key by key by one warp:
// in a matrix product a later position's infinite or NaN value meets the
// row's zero weight and turns its output to NaN, although the row does not
// attend to that position.  Lane l holds values l, l + 32, ...
template <class T, class O, int HD>
__device__ void attend_row(const PromptArgs& a, const KvArgs& kv, int t, int h, int s, int last, int lane) {
  constexpr int E = HD / 32;
  const T* q = static_cast<const T*>(a.q) + (long long)t * a.q_row_stride + (long long)h * a.q_head_stride;
  const long long ho = (long long)(h / (a.n_heads / kv.n_kv)) * kv.head_stride;
  float qv[E], o[E], m = -INFINITY, l = 0.0f;
  for (int e = 0; e < E; ++e) {
    qv[e] = to_f32(q[lane + 32 * e]);
    o[e] = 0.0f;
  }
  for (int j = 0; j <= last; ++j) {
    const long long off = kv_offset(kv, s, j);
    float x = 0.0f;
    if (off >= 0)
      for (int e = 0; e < E; ++e) x = fmaf(qv[e], to_f32(static_cast<const T*>(kv.k)[off + ho + lane + 32 * e]), x);
    x = warp_sum(x) * (a.scale * 1.4426950408889634f);
    const float mn = fmaxf(m, x), mz = mn == -INFINITY ? 0.0f : mn;
    const float f = ex2(m - mz), p = ex2(x - mz);
    m = mn;
    l = l * f + p;
    for (int e = 0; e < E; ++e) {
      const float v = off >= 0 ? to_f32(static_cast<const T*>(kv.v)[off + ho + lane + 32 * e]) : 0.0f;
      o[e] = o[e] * f + p * v;
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  O* out = static_cast<O*>(a.out) + ((long long)t * a.n_heads + h) * HD;
  for (int e = 0; e < E; ++e) {
    const float v = o[e] * inv;
    if constexpr (sizeof(O) == 4) out[lane + 32 * e] = v;
    else {
      const uint32_t w = pack16<O>(v, 0.0f);
      reinterpret_cast<unsigned short*>(out)[lane + 32 * e] = (unsigned short)(w & 0xFFFFu);
    }
  }
}

template <class T, class O, int HD>
__global__ void __launch_bounds__(kWarps * 32) attention_prompt_kernel(const PromptArgs a, const KvArgs kv,
                                                                       unsigned* __restrict__ err) {
  constexpr int kChunks = HD / 8;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sk = smem_u32(smem), sv = sk + kTile * HD * 2;
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int h = blockIdx.x, j = h / (a.n_heads / kv.n_kv);
  // which sequence and tile block blockIdx.y is
  int s = 0, tile = blockIdx.y, qb = 0, qe = 0;
  for (; s < kv.batch; ++s) {
    q_range(a.cu_q, s, a.rows, &qb, &qe);
    const int nt = (qe - qb + kTile - 1) / kTile;
    if (tile < nt) break;
    tile -= nt;
  }
  if (s == kv.batch) return;
  bool clipped;
  const int n = kv_length(kv, s, &clipped);
  if (clipped && tid == 0) atomicOr(err, kErrDecodeRange);
  const int t0 = qb + tile * kTile;               // first query row of the tile
  const int base = n - (qe - qb) + tile * kTile;  // its position
  const int rows = min(kTile, qe - t0);
  const int stop = min(n, base + rows);           // positions the tile attends to
  const float sl2 = a.scale * 1.4426950408889634f;
  const int r = lane >> 2, c2 = (lane & 3) * 2;

  uint32_t qf[HD / 16][4];
  auto ld = [&](int row, int col) -> uint32_t {
    if (row >= rows) return 0u;
    return __ldcg(reinterpret_cast<const unsigned*>(static_cast<const T*>(a.q) + (long long)(t0 + row) * a.q_row_stride +
                                                    (long long)h * a.q_head_stride + col));
  };
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks) {
    qf[ks][0] = ld(warp * 16 + r, ks * 16 + c2);
    qf[ks][1] = ld(warp * 16 + r + 8, ks * 16 + c2);
    qf[ks][2] = ld(warp * 16 + r, ks * 16 + c2 + 8);
    qf[ks][3] = ld(warp * 16 + r + 8, ks * 16 + c2 + 8);
  }
  float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

  for (int p0 = 0; p0 < stop; p0 += kTile) {
    __syncthreads();
    for (int i = tid; i < kTile * kChunks; i += kWarps * 32) {
      const int row = i / kChunks, c = i % kChunks;
      const long long off = p0 + row < stop ? kv_offset(kv, s, p0 + row) : -1;
      uint4 kk = make_uint4(0u, 0u, 0u, 0u), vv = kk;
      if (off >= 0) {
        kk = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(kv.k) + off + j * kv.head_stride) + c);
        vv = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(kv.v) + off + j * kv.head_stride) + c);
      } else if (p0 + row < stop) {
        atomicOr(err, kErrDecodeRange);
      }
      *reinterpret_cast<uint4*>(smem + tile_chunk<kTile>(row, c)) = kk;
      *reinterpret_cast<uint4*>(smem + kTile * HD * 2 + tile_chunk<kTile>(row, c)) = vv;
    }
    __syncthreads();
    float sc[kTile / 8][4] = {};
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
      for (int kt = 0; kt < kTile / 16; ++kt) {
        uint32_t b[4];
        ldsm4(b, key_frag<kTile>(sk, kt * 16, ks, lane));
        mma16816<T>(sc[2 * kt], qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3], b[0], b[1]);
        mma16816<T>(sc[2 * kt + 1], qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3], b[2], b[3]);
      }
    uint32_t pf[kTile / 8][2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int last = base + warp * 16 + r + 8 * q;  // this row's position
      float t = -INFINITY;
#pragma unroll
      for (int i = 0; i < kTile / 8; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int p = p0 + i * 8 + c2 + e;
          float& x = sc[i][2 * q + e];
          x = (p <= last && p < n) ? x * sl2 : -INFINITY;
          t = fmaxf(t, x);
        }
      t = fmaxf(t, __shfl_xor_sync(kFull, t, 1));
      t = fmaxf(t, __shfl_xor_sync(kFull, t, 2));
      const float mn = fmaxf(m[q], t), mz = mn == -INFINITY ? 0.0f : mn;
      const float f = ex2(m[q] - mz);
      m[q] = mn;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kTile / 8; ++i) {
        const float p0f = ex2(sc[i][2 * q] - mz + kShift), p1f = ex2(sc[i][2 * q + 1] - mz + kShift);
        sum += p0f + p1f;
        pf[i][q] = pack16<T>(p0f, p1f);
      }
      l[q] = l[q] * f + sum;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        o[i][2 * q] *= f;
        o[i][2 * q + 1] *= f;
      }
    }
#pragma unroll
    for (int kt = 0; kt < kTile / 16; ++kt)
#pragma unroll
      for (int nt = 0; nt < HD / 16; ++nt) {
        uint32_t b[4];
        ldsm4_t(b, value_frag<kTile>(sv, kt * 16, nt, lane));
        mma16816<T>(o[2 * nt], pf[2 * kt][0], pf[2 * kt][1], pf[2 * kt + 1][0], pf[2 * kt + 1][1], b[0], b[1]);
        mma16816<T>(o[2 * nt + 1], pf[2 * kt][0], pf[2 * kt][1], pf[2 * kt + 1][0], pf[2 * kt + 1][1], b[2], b[3]);
      }
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    l[q] += __shfl_xor_sync(kFull, l[q], 1);
    l[q] += __shfl_xor_sync(kFull, l[q], 2);
    const float inv = l[q] == 0.0f ? 0.0f : 1.0f / l[q];
    const int row = warp * 16 + r + 8 * q;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) {
      const float v0 = o[i][2 * q] * inv, v1 = o[i][2 * q + 1] * inv;
      bad |= !(fabsf(v0) < INFINITY) || !(fabsf(v1) < INFINITY);
      if (row < rows) {
        O* p = static_cast<O*>(a.out) + ((long long)(t0 + row) * a.n_heads + h) * HD + i * 8 + c2;
        if constexpr (sizeof(O) == 4) *reinterpret_cast<float2*>(p) = make_float2(v0, v1);
        else *reinterpret_cast<uint32_t*>(p) = pack16<O>(v0, v1);
      }
    }
    unsigned todo = __ballot_sync(kFull, bad && row < rows);
    while (todo) {  // one row of the warp at a time
      const int rr = (__ffs(todo) - 1) >> 2;
      todo &= ~(0xFu << (4 * rr));
      const int rw = warp * 16 + rr + 8 * q;
      __syncwarp();
      attend_row<T, O, HD>(a, kv, t0 + rw, h, s, min(base + rw, n - 1), lane);
    }
  }
}

template <class T, class O, int HD>
cudaError_t launch_typed(const PromptArgs& a, const KvArgs& kv, cudaStream_t stream, unsigned* err) {
  auto kernel = attention_prompt_kernel<T, O, HD>;
  const size_t smem = 2 * kTile * HD * 2 + 1024;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.n_heads, (unsigned)(a.rows / kTile + kv.batch));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_opt_pdl.load() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, a, kv, err);
}

template <class T>
cudaError_t launch_type(const PromptArgs& a, const KvArgs& kv, cudaStream_t stream, unsigned* err) {
  const bool f32 = a.out_dtype == kDtF32;
  if (kv.head_dim == 128)
    return f32 ? launch_typed<T, float, 128>(a, kv, stream, err) : launch_typed<T, T, 128>(a, kv, stream, err);
  return f32 ? launch_typed<T, float, 64>(a, kv, stream, err) : launch_typed<T, T, 64>(a, kv, stream, err);
}

}  // namespace

cudaError_t launch_attention_prompt(const PromptArgs& a, const KvArgs& kv, cudaStream_t stream) {
  unsigned* err = device_error_word();
  if (!err) return cudaErrorUnknown;
  return kv.dtype == kDtF16 ? launch_type<__half>(a, kv, stream, err)
                            : launch_type<__nv_bfloat16>(a, kv, stream, err);
}

}  // namespace asmllm
