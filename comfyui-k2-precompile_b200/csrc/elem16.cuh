// elem16.cuh -- what the bf16 / fp16 kernels of the conditioning operators
// share: conversions of a pair of 16-bit elements, streaming loads, and the
// warp-level m16n8k16 matrix product.
//
// w4_linear and the few-row attention kernel read far more than they compute (a
// weight or a key is used by up to 16 rows at a time), so the warp-level product
// is enough to keep up with memory.  Attention of many queries runs on tcgen05
// where that takes less time; w4_linear has no such kernel and reads its weight
// again for every 16 rows.
#pragma once
#include <type_traits>

#include "k2b_common.cuh"

namespace k2b {

template <typename T>
struct Elem16;

template <>
struct Elem16<__nv_bfloat16> {
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
  static __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem16<__half> {
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
};

// 16 bytes that this kernel reads once: not kept in L1, and fetched with their
// neighbours into L2 (rows of 64 bytes at a time are what these kernels ask for).
__device__ __forceinline__ uint4 ldg_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// A 16-bit value loaded ahead of its use: volatile, so that the compiler does
// not move the load down to the use to save the register.
__device__ __forceinline__ uint32_t ldg_ahead_u16(const void* p) {
  unsigned short v;
  asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return v;
}

// D += A B for a 16 x 16 A and a 16 x 8 B.  Lane l, with r = l / 4 and
// t = l % 4, holds A rows r (a0, a2) and r + 8 (a1, a3) at the k pairs 2t
// (a0, a1) and 2t + 8 (a2, a3); B column r at the k pairs 2t (b0) and
// 2t + 8 (b1); D rows r (d0, d1) and r + 8 (d2, d3) at columns 2t, 2t + 1.
// The 16 k of a product may be any 16 of the sum as long as A and B agree.
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

// Programmatic dependent launch: everything above the wait may run while the
// kernel before it on the stream still does; what that kernel wrote is
// visible below it.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace k2b
