// Rows of 16- and 32-bit values, eight columns at a time, and the blocks of 128 columns that share a scale in 8 bits.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

namespace nep {
namespace rows {

constexpr int kBlock = 128;        // columns that share a scale
constexpr float kLargest = 448.f;  // largest e4m3 value
// A block whose largest value is below this is scaled as if it were this: its values round to zero, and the quotient stays finite.
constexpr float kTiny = 1e-30f;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ void unpack2(uint32_t v, float* f, __nv_bfloat16) {
    const float2 p = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
    f[0] = p.x;
    f[1] = p.y;
}
__device__ __forceinline__ void unpack2(uint32_t v, float* f, __half) {
    const float2 p = __half22float2(*reinterpret_cast<__half2*>(&v));
    f[0] = p.x;
    f[1] = p.y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 p = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
}

// Eight neighbouring values as they lie in memory (16-byte aligned).
template <typename T>
struct Raw8 {
    uint4 v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void clear() { v = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float* f) const {
        unpack2(v.x, f, T());
        unpack2(v.y, f + 2, T());
        unpack2(v.z, f + 4, T());
        unpack2(v.w, f + 6, T());
    }
    __device__ __forceinline__ void set(const float* f) {
        v = make_uint4(pack2(f[0], f[1], T()), pack2(f[2], f[3], T()), pack2(f[4], f[5], T()), pack2(f[6], f[7], T()));
    }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = v; }
};
template <>
struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = reinterpret_cast<const float4*>(p)[0];
        b = reinterpret_cast<const float4*>(p)[1];
    }
    __device__ __forceinline__ void clear() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ void get(float* f) const {
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    }
    __device__ __forceinline__ void set(const float* f) {
        a = make_float4(f[0], f[1], f[2], f[3]);
        b = make_float4(f[4], f[5], f[6], f[7]);
    }
    __device__ __forceinline__ void store(float* p) const {
        reinterpret_cast<float4*>(p)[0] = a;
        reinterpret_cast<float4*>(p)[1] = b;
    }
};

// Larger of two values; a NaN stays one, so that a block that holds one is marked in its scale.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Four quotients rounded to e4m3 (to nearest, ties to even), the first in the lowest byte.
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}
// Values in units of their block's scale: v * 448 / m with m = the block's largest.  Exact ties are common where v is a product of two
// 16-bit values (v * 7 is exact then), and they have to stay ties.  q0 = r * (1 / d), off by 2^-22 at most; its remainder r - q0 * d is exact
// in a fused multiply-add; q0 plus the remainder over d is the quotient to within its rounding.  Where that is a tie, 5 significant bits,
// it is hit; where not, it lies 2^-21 from one at least, since r and d have 19 and 16 bits.  (__fdiv_rn: 51 us instead of 44 for 4096 rows of 7168.)
struct Quotient {
    float d, inverse;
    __device__ __forceinline__ explicit Quotient(float m) {
        d = m * 0x1p-10f;  // 448 = 7 / 16 * 2^10: neither side overflows
        inverse = __frcp_rn(d);
        if (inverse == 0.f) d = 0.f;  // an infinite block: finite values are 0 of it, infinities NaN
    }
    __device__ __forceinline__ float operator()(float v) const {
        const float r = v * 0.4375f, q0 = r * inverse;
        return fmaf(fmaf(-q0, d, r), inverse, q0);
    }
};

template <int kWidth>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int d = kWidth / 2; d > 0; d >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

}  // namespace rows
}  // namespace nep
