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
// x = hi + lo: hi the upper eleven bits (an fp16 as it is), lo the rest rounded to fp16; |x| <= 2^15
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
    const float xh = __int_as_float(__float_as_int(x) & 0xffffe000), yh = __int_as_float(__float_as_int(y) & 0xffffe000);
    const float2 r = fma2(make_float2(xh, yh), make_float2(-1.0f, -1.0f), make_float2(x, y));     // exact (packed sums take no sign)
    hi = pack_half(xh, yh);
    lo = pack_half(r.x, r.y);
}

}  // namespace sb
