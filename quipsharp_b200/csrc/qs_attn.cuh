// Pieces shared by the attention kernels: 16-bit products through mma.sync, swizzled
// rows in shared memory, asynchronous copies.
#pragma once

#include "qs_common.cuh"
#include "qs_launch.h"
#include "qs_pair.cuh"

namespace qs {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What a partial sum with maximum m weighs beside the joint maximum (1 where both are
// -inf: an empty sum, or one of NaN alone, which has to stay NaN).
__device__ __forceinline__ float weight(float m, float joint) { return m == joint ? 1.f : ex2(m - joint); }

// Byte offset of 16-byte piece `piece` of row `row` in a tile of rows of DP 16-bit
// values: pieces of eight consecutive rows fall on distinct banks.
template <int DP>
__device__ __forceinline__ uint32_t swizzled(int row, int piece) {
  return row * (DP * 2) + ((piece ^ (row & 7)) << 4);
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma_16816(d, a[0], a[1], a[2], a[3], b0, b1);
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x, y rounded to T and packed; returns the rounded values.
template <typename T>
__device__ __forceinline__ float2 split16(float x, float y, uint32_t &packed);
template <>
__device__ __forceinline__ float2 split16<__half>(float x, float y, uint32_t &packed) {
  const __half2 h = __floats2half2_rn(x, y);
  packed = *reinterpret_cast<const uint32_t *>(&h);
  return __half22float2(h);
}
template <>
__device__ __forceinline__ float2 split16<__nv_bfloat16>(float x, float y, uint32_t &packed) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  packed = *reinterpret_cast<const uint32_t *>(&h);
  return __bfloat1622float2(h);
}

__device__ __forceinline__ void store1(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store1(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// 16 bytes global -> shared; zeros (and no read) where `in` is false.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

}  // namespace
}  // namespace qs
