// asmllm_b200/csrc/mma16.cuh -- warp-level 16-bit matrix products with fp32
// accumulators (m16n8k16) and the shared-memory tile layout they read.
//
// A key or value tile holds N positions of HD values as HD/64 halves of
// [N][64] values: 128 bytes a position, 16-byte chunk c of position r stored
// at chunk c ^ (r % 8) (the 128-byte swizzle of a tensor copy into a
// 1024-byte aligned buffer), so eight positions' equal chunks, which one
// ldmatrix reads, lie in eight different bank groups.
#pragma once

#include <stdint.h>

#include "pipeline.cuh"
#include "serving.cuh"

namespace asmllm {

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// c += a b: a 16x16 (rows x k), b 16x8 (k x columns).
template <class T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                 uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ex2(float x) {  // 2^x, relative error below 2^-22; 2^-inf = 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Softmax weights are kept as 2^kShift exp(s - m): fp16 then holds weights down
// to 2^-24-kShift of the largest, and the many small weights of a long row
// are not flushed to zero; the factor cancels in the division by the sum.
constexpr float kShift = 14.0f;

// Byte offset of 16-byte chunk c (of HD/8) of position r in a tile of N positions.
template <int N>
__device__ __forceinline__ uint32_t tile_chunk(int r, int c) {
  return (uint32_t)((c >> 3) * (N * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// Address of the B fragments (k = 16 values from chunk 2 ks, columns = 16
// positions from r0) for ldsm4: r[0..1] positions r0.., r[2..3] positions r0 + 8...
template <int N>
__device__ __forceinline__ uint32_t key_frag(uint32_t tile, int r0, int ks, int lane) {
  const int m = lane >> 3, r = lane & 7;
  return tile + tile_chunk<N>(r0 + (m >> 1) * 8 + r, ks * 2 + (m & 1));
}

// Address of the B fragments (k = 16 positions from r0, columns = 16 values
// from chunk 2 nt) for ldsm4_t: r[0..1] the first eight values, r[2..3] the next.
template <int N>
__device__ __forceinline__ uint32_t value_frag(uint32_t tile, int r0, int nt, int lane) {
  const int m = lane >> 3, r = lane & 7;
  return tile + tile_chunk<N>(r0 + (m & 1) * 8 + r, nt * 2 + (m >> 1));
}

}  // namespace asmllm
