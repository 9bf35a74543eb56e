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
// Values in units of their block's scale, v * 448 / m with m = the block's largest, as e4m3: what the exact quotient rounds to.  Exact ties between two
// e4m3 values, 5 significant bits, are common and have to stay ties; quotients next to one have to stay on their side.
//
// With d = m / 2^10 (448 = 7 / 16 * 2^10: neither side overflows), r = v * 7 / 16, q0 = r * (1 / d), off by 2^-22 at most: the remainder r - q0 * d is exact in a
// fused multiply-add, and q0 plus the remainder over d is the quotient to within its rounding.
struct Quotient {
    float d, inverse;
    __device__ __forceinline__ explicit Quotient(float m) {
        d = m * 0x1p-10f;
        inverse = __frcp_rn(d);
        if (inverse == 0.f) d = 0.f;  // an infinite block: finite values are 0 of it, infinities NaN
    }
    // v and m of up to 16 bits: r is exact, a tie is hit, and any other quotient lies 2^-21 from one at least, since r and d have 19 and 16 bits.
    __device__ __forceinline__ float narrow(float v) const {
        const float r = v * 0.4375f, q0 = r * inverse;
        return fmaf(fmaf(-q0, d, r), inverse, q0);
    }
    // Any v and m: what r has lost goes into the remainder.  A quotient within half a 32-bit step of a tie is rounded onto it; the sign of its remainder, exact
    // there, moves it off again.  (A block's largest is at least kTiny: nothing here loses bits below the smallest 32-bit value.)
    __device__ __forceinline__ float wide(float v) const {
        const float r = v * 0.4375f, lost = fmaf(v, 0.4375f, -r), q0 = r * inverse;
        const float q = fmaf(fmaf(-q0, d, r) + lost, inverse, q0), left = fmaf(-q, d, r) + lost;
        int bits = __float_as_int(q);
        if (left != 0.f && (bits & 0x7ffff) == 0) bits += (left > 0.f) == (v > 0.f) ? 1 : -1;
        return __int_as_float(bits);
    }
};
// Products of two bf16 values, and 16-bit values.  (4096 rows of 7168: 44 us, with __fdiv_rn 51.)
struct NarrowBlock {
    Quotient of;
    __device__ __forceinline__ explicit NarrowBlock(float m) : of(m) {}
    __device__ __forceinline__ uint32_t pack(const float* v) const { return pack_e4m3(of.narrow(v[0]), of.narrow(v[1]), of.narrow(v[2]), of.narrow(v[3])); }
};
// 32-bit values.  Products with 448 / m a little smaller and a little larger, 2^-22 where three roundings take 3 * 2^-24, enclose the quotient: where both round to
// the same e4m3 value, so does the quotient.  They do for all but about one value in 2 * 10^5.  (4096 rows of 7168 with a 32-bit weight: 50 us, with Quotient::wide for every
// value 61, with a quotient that may miss a tie 48.)
struct WideBlock {
    float m, low, high;
    __device__ __forceinline__ explicit WideBlock(float largest) : m(largest) {
        const float per = __fdiv_rn(kLargest, m);
        low = per * (1.f - 0x1p-22f);
        high = per * (1.f + 0x1p-22f);
    }
    // Bits of `unsure` are set where the result may be the neighbour of the right one.
    __device__ __forceinline__ uint32_t guess(const float* v, uint32_t& unsure) const {
        const uint32_t a = pack_e4m3(v[0] * low, v[1] * low, v[2] * low, v[3] * low), b = pack_e4m3(v[0] * high, v[1] * high, v[2] * high, v[3] * high);
        unsure |= a ^ b;
        return a;
    }
    __device__ __forceinline__ uint32_t exact(const float* v) const {
        const Quotient of(m);
        return pack_e4m3(of.wide(v[0]), of.wide(v[1]), of.wide(v[2]), of.wide(v[3]));
    }
    __device__ __forceinline__ uint32_t pack(const float* v) const {
        uint32_t unsure = 0;
        const uint32_t q = guess(v, unsure);
        return unsure == 0 ? q : exact(v);
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
