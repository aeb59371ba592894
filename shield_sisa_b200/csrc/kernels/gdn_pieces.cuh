// Numbers as two fp16 pieces and powers of two, for products on the tensor cores that keep float32's accuracy.
#pragma once
#include "device_utils.cuh"

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

}  // namespace sb
