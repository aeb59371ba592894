// Numbers as two fp16 pieces and powers of two, for products on the tensor cores that keep float32's accuracy; the warp's own products and
// their operands.
#pragma once
#include "device_utils.cuh"

#include <type_traits>

namespace sb {

// 2^n for a biased exponent n + 127 in [1, 254]
__device__ __forceinline__ float pow2_biased(int b) { return __int_as_float(b << 23); }
__device__ __forceinline__ int exponent_of(float x) { return (__float_as_int(x) >> 23) & 255; }
__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// x = hi + lo, both fp16: 22 bits; |x| <= 2^15.  (hi by a conversion and back, not by a mask: a mask takes the pipe that the conversions
// wait for.)
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h), r = fma2(f, make_float2(-1.0f, -1.0f), make_float2(x, y));     // exact (packed sums take no sign)
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = pack_half(r.x, r.y);
}

// Four 8 x 8 matrices of 16-bit values out of shared memory.
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// d += a b, 16 x 8 of depth 16, T values, sums in float32
template <typename T> __device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

}  // namespace sb
