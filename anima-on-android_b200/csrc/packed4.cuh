// packed4.cuh -- the packed 4-bit format and its unpacking in registers.
//
// A packed row holds K values (K a multiple of 128) as 4-bit codes and one fp16 scale per
// 32 values: value = n * s with n in [-8, 7], 4.5 bits a value.  Codes are stored offset by
// 8.  A block of 128 values is 64 bytes, sixteen 32-bit words; word 4 i + g holds values
// 32 g + 8 i + e, e = 0..7 (group g, i = 0..3), value e at nibble (e >> 1) + 4 (e & 1).
//
// The order is chosen for the matrix instructions.  In an m16n8k16 operand fragment the four
// lanes of a quad hold different k of one row; lane i reads words 4 i .. 4 i + 3 of a block,
// one 16-byte load, and has eight consecutive values of every group.  Since both operands
// may list k in any common order, word g then feeds two k-steps that lie wholly in group g,
// and the group's scale can be applied to the fp32 accumulator: the products are of whole
// numbers n, exact in fp16 and bf16.  Within a word, nibbles p and p + 4 are neighbours e =
// 2 p, 2 p + 1, so masking with 0x000f000f leaves a pair in consecutive order.
#pragma once
#include <utility>

#include "common.cuh"
#include "smem_attr.cuh"

namespace anima {
namespace p4 {

constexpr int kGroup = 32;   // values that share a scale
constexpr int kBlock = 128;  // values of one 64-byte code block

// (w & mask) | bits in one instruction.
template <uint32_t kMask, uint32_t kBits>
__device__ __forceinline__ uint32_t mask_or(uint32_t w) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "n"(kMask), "r"(kBits));
  return r;
}

// Eight codes of word w as whole numbers n, four pairs in value order.  In fp16, 0x6400 | c is
// 1024 + c and 0x6400 | 16 c is 1024 + 16 c, so one subtraction, or one fused multiply-add
// with 1/16 for the codes that sit four bits up, leaves n = c - 8 exactly.
__device__ __forceinline__ void numbers_f16(uint32_t w, uint32_t (&n)[4]) {
  const uint32_t w8 = w >> 8;
  const __half2 lo = __half2half2(__ushort_as_half(0x6408));         // 1032
  const __half2 sc = __half2half2(__ushort_as_half(0x2c00));         // 1 / 16
  const __half2 hi = __half2half2(__ushort_as_half(0xd480));         // -72
  const uint32_t t[4] = {mask_or<0x000f000fu, 0x64006400u>(w), mask_or<0x00f000f0u, 0x64006400u>(w),
                         mask_or<0x000f000fu, 0x64006400u>(w8), mask_or<0x00f000f0u, 0x64006400u>(w8)};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __half2 v = *reinterpret_cast<const __half2*>(&t[k]);
    const __half2 r = (k & 1) ? __hfma2(v, sc, hi) : __hsub2(v, lo);
    n[k] = *reinterpret_cast<const uint32_t*>(&r);
  }
}

// The same in bf16: 0x4300 | c is 128 + c (seven mantissa bits hold the four of c).
__device__ __forceinline__ void numbers_bf16(uint32_t w, uint32_t (&n)[4]) {
  const __nv_bfloat162 one = __bfloat162bfloat162(__ushort_as_bfloat16(0x3f80));
  const __nv_bfloat162 off = __bfloat162bfloat162(__ushort_as_bfloat16(0xc308));  // -136
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t t = mask_or<0x000f000fu, 0x43004300u>(w >> (4 * k));
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&t), one, off);
    n[k] = *reinterpret_cast<const uint32_t*>(&r);
  }
}

template <bool kBf16>
__device__ __forceinline__ void numbers(uint32_t w, uint32_t (&n)[4]) {
  if (kBf16)
    numbers_bf16(w, n);
  else
    numbers_f16(w, n);
}

// The four fp16 scales of a 128-value block, as fp32.
__device__ __forceinline__ float4 scales4(uint2 u) {
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}

// Asynchronous copies of 16 and 8 bytes to shared memory; the _if forms write zeros, and read
// nothing, where `take` is false.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16_if(uint32_t dst, const void* src, bool take) {
  const int n = take ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp8_if(uint32_t dst, const void* src, bool take) {
  const int n = take ? 8 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kN>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kN) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ float lds4(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}

// D += A B, m16n8k16 with fp32 accumulation.  Lane 4 j + i holds A rows j (a0, a2) and j + 8
// (a1, a3), B column j, and D rows j (d0, d1) and j + 8 (d2, d3) of columns 2 i, 2 i + 1.
template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  if (kBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// D = A B of the same shapes.
template <bool kBf16>
__device__ __forceinline__ void mma16816_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  if (kBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// D = A B + C, m16n8k32 on whole numbers: A unsigned and B signed bytes.  Lane 4 j + i holds k = 4 i .. + 3 and 16 + 4 i .. + 3 of A rows j (a0, a2) and j + 8 (a1,
// a3) and of B column j; D as in m16n8k16.
__device__ __forceinline__ void mma16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1, const uint4& c) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%12,%13};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c.x), "r"(c.y), "r"(c.z), "r"(c.w));
}

}  // namespace p4

// Launches a kernel as a programmatic dependent of the one before it on the stream, optionally in
// clusters: its blocks may start while that one drains.  Every block of the kernel has to run
// grid_dependency_wait() before it touches global memory.
template <typename... Params, typename... Args>
static int launch_clusters(void (*kern)(Params...), int grid, int cluster, int threads, size_t smem, cudaStream_t st,
                           Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)cluster;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kern, Params(std::forward<Args>(args))...) != cudaSuccess) {
    cudaGetLastError();
    return ANIMA_ERR_CUDA;
  }
  return ANIMA_OK;
}
template <typename... Params, typename... Args>
static int launch_dependent(void (*kern)(Params...), int grid, int threads, size_t smem, cudaStream_t st,
                            Args&&... args) {
  return launch_clusters(kern, grid, 0, threads, smem, st, std::forward<Args>(args)...);
}

}  // namespace anima
