// asmllm_b200/csrc/attention_paged.cu -- attention of one new token per
// sequence over a paged key-value cache.
//
//   out[s][h] = sum_{p < n_s} softmax_p(scale q[s][h] . k[p][h / g]) v[p][h / g]
// with n_s = len[s]; no position: zeros.
//
// One CTA per (sequence, KV head, 16 query heads of its group): four warps,
// each taking 16 of every 64 positions with its own running maximum, sum and
// output; the four are joined in shared memory at the end, in warp order.
#include "matvec.cuh"
#include "mma16.cuh"
#include "serving.cuh"

namespace asmllm {

namespace {

constexpr int kTile = 64;   // positions per tile, 16 per warp
constexpr int kWarps = 4;

template <class T, class O, int HD>
__global__ void __launch_bounds__(kWarps * 32) attention_paged_kernel(const PagedArgs a, const KvArgs kv,
                                                                      unsigned* __restrict__ err) {
  constexpr int kChunks = HD / 8;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sk = smem_u32(smem), sv = sk + kTile * HD * 2;
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = a.n_heads / kv.n_kv, j = blockIdx.x, s = blockIdx.y, h0 = blockIdx.z * 16;
  const int nh = min(16, g - h0);  // query heads of this CTA
  bool clipped;
  const int n = kv_length(kv, s, &clipped);
  if (clipped && tid == 0) atomicOr(err, kErrDecodeRange);
  const float sl2 = a.scale * 1.4426950408889634f;

  uint32_t qf[HD / 16][4];
  {
    const T* qb = static_cast<const T*>(a.q) + s * a.q_row_stride;
    const int r = lane >> 2, c = (lane & 3) * 2;
    auto ld = [&](int row, int col) -> uint32_t {
      if (row >= nh) return 0u;
      return __ldcg(reinterpret_cast<const unsigned*>(qb + (long long)(j * g + h0 + row) * a.q_head_stride + col));
    };
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      qf[ks][0] = ld(r, ks * 16 + c);
      qf[ks][1] = ld(r + 8, ks * 16 + c);
      qf[ks][2] = ld(r, ks * 16 + c + 8);
      qf[ks][3] = ld(r + 8, ks * 16 + c + 8);
    }
  }
  float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

  for (int p0 = 0; p0 < n; p0 += kTile) {
    __syncthreads();
    for (int i = tid; i < kTile * kChunks; i += kWarps * 32) {
      const int r = i / kChunks, c = i % kChunks;
      const long long off = p0 + r < n ? kv_offset(kv, s, p0 + r) : -1;
      uint4 kk = make_uint4(0u, 0u, 0u, 0u), vv = kk;
      if (off >= 0) {
        kk = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(kv.k) + off + j * kv.head_stride) + c);
        vv = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(kv.v) + off + j * kv.head_stride) + c);
      } else if (p0 + r < n) {
        atomicOr(err, kErrDecodeRange);
      }
      *reinterpret_cast<uint4*>(smem + tile_chunk<kTile>(r, c)) = kk;
      *reinterpret_cast<uint4*>(smem + kTile * HD * 2 + tile_chunk<kTile>(r, c)) = vv;
    }
    __syncthreads();
    const int r0 = warp * 16;
    float sc[2][4] = {};
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      uint32_t b[4];
      ldsm4(b, key_frag<kTile>(sk, r0, ks, lane));
      mma16816<T>(sc[0], qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3], b[0], b[1]);
      mma16816<T>(sc[1], qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3], b[2], b[3]);
    }
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = p0 + r0 + (i >> 1) * 8 + (lane & 3) * 2 + (i & 1);
        x[i] = p < n ? sc[i >> 1][2 * r + (i & 1)] * sl2 : -INFINITY;
      }
      float t = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
      t = fmaxf(t, __shfl_xor_sync(kFull, t, 1));
      t = fmaxf(t, __shfl_xor_sync(kFull, t, 2));
      const float mn = fmaxf(m[r], t), mz = mn == -INFINITY ? 0.0f : mn;
      const float f = ex2(m[r] - mz);
      m[r] = mn;
      float p[4], sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = ex2(x[i] - mz + kShift);
        sum += p[i];
      }
      l[r] = l[r] * f + sum;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        o[i][2 * r] *= f;
        o[i][2 * r + 1] *= f;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // p = hi + lo to twice the 16-bit type's digits
        hi[2 * i + r] = pack16<T>(p[2 * i], p[2 * i + 1]);
        const float2 q = unpack16<T>(hi[2 * i + r]);
        lo[2 * i + r] = pack16<T>(p[2 * i] - q.x, p[2 * i + 1] - q.y);
      }
    }
#pragma unroll
    for (int nt = 0; nt < HD / 16; ++nt) {
      uint32_t b[4];
      ldsm4_t(b, value_frag<kTile>(sv, r0, nt, lane));
      mma16816<T>(o[2 * nt], hi[0], hi[1], hi[2], hi[3], b[0], b[1]);
      mma16816<T>(o[2 * nt], lo[0], lo[1], lo[2], lo[3], b[0], b[1]);
      mma16816<T>(o[2 * nt + 1], hi[0], hi[1], hi[2], hi[3], b[2], b[3]);
      mma16816<T>(o[2 * nt + 1], lo[0], lo[1], lo[2], lo[3], b[2], b[3]);
    }
  }
  // join the four warps: [warp][row][HD] outputs, [warp][row] (maximum, sum)
  __syncthreads();
  float* jo = reinterpret_cast<float*>(smem);
  float2* ml = reinterpret_cast<float2*>(smem + kWarps * 16 * HD * 4);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(kFull, l[r], 1);
    l[r] += __shfl_xor_sync(kFull, l[r], 2);
    const int row = (lane >> 2) + 8 * r;
    if ((lane & 3) == 0) ml[warp * 16 + row] = make_float2(m[r], l[r]);
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
      *reinterpret_cast<float2*>(jo + (warp * 16 + row) * HD + i * 8 + (lane & 3) * 2) =
          make_float2(o[i][2 * r], o[i][2 * r + 1]);
  }
  __syncthreads();
  for (int i = tid; i < nh * (HD / 8); i += kWarps * 32) {
    const int row = i / (HD / 8), c = (i % (HD / 8)) * 8;
    float mm = -INFINITY;
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, ml[w * 16 + row].x);
    const float mz = mm == -INFINITY ? 0.0f : mm;
    float ll = 0.0f, v[8] = {};
    for (int w = 0; w < kWarps; ++w) {
      const float2 t = ml[w * 16 + row];
      const float f = ex2(t.x - mz);
      ll += f * t.y;
      for (int e = 0; e < 8; ++e) v[e] += f * jo[(w * 16 + row) * HD + c + e];
    }
    const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;  // no position left: zeros
    for (int e = 0; e < 8; ++e) v[e] *= inv;
    store8(static_cast<O*>(a.out) + ((long long)s * a.n_heads + j * g + h0 + row) * HD + c, v);
  }
}

template <class T, class O, int HD>
cudaError_t launch_typed(const PagedArgs& a, const KvArgs& kv, cudaStream_t stream, unsigned* err) {
  const int g = a.n_heads / kv.n_kv;
  auto kernel = attention_paged_kernel<T, O, HD>;
  const size_t tiles = 2 * kTile * HD * 2, join = kWarps * 16 * (HD + 2) * 4;
  const size_t smem = (tiles > join ? tiles : join) + 1024;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)kv.n_kv, (unsigned)kv.batch, (unsigned)((g + 15) / 16));
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
cudaError_t launch_type(const PagedArgs& a, const KvArgs& kv, cudaStream_t stream, unsigned* err) {
  const bool f32 = a.out_dtype == kDtF32;
  if (kv.head_dim == 128)
    return f32 ? launch_typed<T, float, 128>(a, kv, stream, err) : launch_typed<T, T, 128>(a, kv, stream, err);
  return f32 ? launch_typed<T, float, 64>(a, kv, stream, err) : launch_typed<T, T, 64>(a, kv, stream, err);
}

}  // namespace

size_t attention_paged_workspace(int, int, int, int) { return 0; }

cudaError_t launch_attention_paged(const PagedArgs& a, const KvArgs& kv, cudaStream_t stream) {
  unsigned* err = device_error_word();
  if (!err) return cudaErrorUnknown;
  return kv.dtype == kDtF16 ? launch_type<__half>(a, kv, stream, err)
                            : launch_type<__nv_bfloat16>(a, kv, stream, err);
}

}  // namespace asmllm
