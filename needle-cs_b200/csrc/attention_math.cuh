// Numbers the attention kernels over caller-owned pages share: int8 codes as
// fp16, queries and value scales brought into fp16's range by powers of two,
// and rows of 32- or 16-bit elements.
#pragma once

#include "paged.cuh"

namespace ndl {

#ifdef __CUDACC__
constexpr float kLog2E = 1.44269504088896341f;
// The running maximum follows the true one only where that is this many
// binary orders above it (a probability is then at most 2^7).
constexpr float kLazy = 7.0f;
// The power of two that value scales are divided by is at least 2^-110, so
// that it and 2^8 over it are floats; smaller scales do not move it.
constexpr int kMinExponent = -110;

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^e as a float, -126 <= e <= 127.
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ __half2 as_half2(uint32_t bits) { return *reinterpret_cast<const __half2 *>(&bits); }
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }
// Four int8 codes of a word as two pairs of fp16, exactly: the biased byte in
// the low mantissa bits of 1024, less 1024 + 128.
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t &lo, uint32_t &hi) {
    const uint32_t u = w ^ 0x80808080u;
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
    __half2 a, b;
    *reinterpret_cast<uint32_t *>(&a) = __byte_perm(u, 0x64646464u, 0x4140);
    *reinterpret_cast<uint32_t *>(&b) = __byte_perm(u, 0x64646464u, 0x4342);
    a = __hsub2(a, bias), b = __hsub2(b, bias);
    lo = *reinterpret_cast<uint32_t *>(&a), hi = *reinterpret_cast<uint32_t *>(&b);
}
__device__ __forceinline__ uint32_t half_pair(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// The remainders of a pair behind its fp16 rounding.
__device__ __forceinline__ uint32_t half_rest(float a, float b, uint32_t pair) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&pair));
    return half_pair(a - f.x, b - f.y);
}

// Four int8 codes of a word times a scale as two pairs of fp16, the scale given
// as two fp16 (its rounding and the rest, each twice): two roundings of the
// product.
__device__ __forceinline__ void folded_codes(uint32_t w, uint32_t scale, uint32_t rest, uint32_t &a, uint32_t &b) {
    codes_to_half(w, a, b);
    a = half2_bits(__hfma2(as_half2(a), as_half2(rest), __hmul2(as_half2(a), as_half2(scale))));
    b = half2_bits(__hfma2(as_half2(b), as_half2(rest), __hmul2(as_half2(b), as_half2(scale))));
}

// Four elements of a query row.
template <class T>
__device__ __forceinline__ void load4(const T *p, float (&x)[4]) {
    if constexpr (sizeof(T) == 4) {
        const float4 v = *reinterpret_cast<const float4 *>(p);
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        const T *h = reinterpret_cast<const T *>(&v);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = to_float(h[i]);
    }
}
template <class T>
__device__ __forceinline__ void store16(T *p, const float *x) {  // 16 bytes: 4 or 8 elements
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
        alignas(16) T h[8];
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = from_float<T>(x[i]);
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(h);
    }
}


template <class T>
__device__ __forceinline__ void store2(T *p, float a, float b) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float2 *>(p) = make_float2(a, b);
    } else {
        alignas(4) T h[2] = {from_float<T>(a), from_float<T>(b)};
        *reinterpret_cast<uint32_t *>(p) = *reinterpret_cast<const uint32_t *>(h);
    }
}

// Factors that bring a row whose largest magnitude is `peak` to [2^10, 2^11)
// and back.  (An infinity or NaN stays one; below 2^-100 the row stays
// smaller than that, exact all the same.)
__device__ __forceinline__ void query_norm(float peak, float &up, float &down) {
    int e = (int)((__float_as_uint(peak) >> 23) & 0xFF) - 127;
    e = e == 128 ? 10 : max(e, -100);
    up = pow2(10 - e), down = pow2(e - 10);
}
// Biased exponent of a value scale, 0 for an infinity or NaN (which do not
// move the common power of two): the scale is below 2^(result - 126).
__device__ __forceinline__ int scale_exponent(float s) {
    const int e = (int)((__float_as_uint(s) >> 23) & 0xFF);
    return e == 255 ? 0 : e;
}
#endif

}  // namespace ndl
