// quant.cuh — the 8-bit row codec: how 16-bit cache rows are stored and what they read back as.
//
// A row is quant_elems values followed by plain_elems ones. For each group of 128 of the former,
// with a = max |x| over the group and Q the largest code (448 for e4m3, 127 for int8):
//   a is inf or NaN:  scale = the quiet NaN 0x7FC00000, codes 0: the group reads back as NaN, never as wrong numbers;
//   a < 2^-100:       scale = 0, codes 0 (Q / a would leave the fp32 range);
//   otherwise:        scale = fl32(a / Q), code = round_to_nearest_even(fl32(x * fl32(Q / a))).
// A code stands for fl16(fl32(code * scale)), fl16 rounding to the row's 16-bit type. Every step is
// one IEEE fp32 operation, so the codes and the values are the same wherever they are computed.
// The stored row is the codes, then the fp32 scales padded to 16 bytes, then the plain values:
// 656 bytes for the 512 + 64 values of a 1152-byte row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "kvops_internal.cuh"

namespace kvb {

// Two fp32 products, or sums, in one instruction (each rounded as __fmul_rn and __fadd_rn do).
__device__ __forceinline__ float2 mul2(const float2 &a, const float2 &b)
{
    float2 d;
    asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mul.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z; }"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 add2(const float2 &a, const float2 &b)
{
    float2 d;
    asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; add.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z; }"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// The 16-bit types of rows.
struct Fp16 {
    static constexpr uint32_t kInf = 0x7C00u;  // magnitude bits from which a value is not finite
    __device__ static __forceinline__ float2 unpack(uint32_t v)
    {
        return __half22float2(*reinterpret_cast<const __half2 *>(&v));
    }
    __device__ static __forceinline__ uint32_t pack(float a, float b)
    {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};
struct Bf16 {
    static constexpr uint32_t kInf = 0x7F80u;
    __device__ static __forceinline__ float2 unpack(uint32_t v)
    {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
    }
    __device__ static __forceinline__ uint32_t pack(float a, float b)
    {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};

// The 8-bit codes: four at a time.
struct E4m3 {
    static constexpr float kMax = 448.f;
    __device__ static __forceinline__ uint32_t encode4(float a, float b, float c, float d)
    {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
        return lo | (hi << 16);
    }
    __device__ static __forceinline__ float4 decode4(uint32_t v)
    {
        const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v & 0xFFFFu), __NV_E4M3);
        const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v >> 16), __NV_E4M3);
        const float2 x = __half22float2(__half2(lo)), y = __half22float2(__half2(hi));
        return make_float4(x.x, x.y, y.x, y.y);
    }
};
struct Int8 {
    static constexpr float kMax = 127.f;
    __device__ static __forceinline__ uint32_t encode4(float a, float b, float c, float d)
    {
        // |x * fl(127 / a)| < 127.5, so no code leaves [-127, 127].
        const uint32_t lo = __byte_perm(__float2int_rn(a), __float2int_rn(b), 0x0040);
        const uint32_t hi = __byte_perm(__float2int_rn(c), __float2int_rn(d), 0x0040);
        return __byte_perm(lo, hi, 0x5410);
    }
    // A code c as a float: its byte, offset by 128, in the low mantissa of 2^23, less 2^23 + 128
    // (both exact), which costs a byte permute and an add instead of a conversion.
    __device__ static __forceinline__ float4 decode4(uint32_t v)
    {
        const uint32_t u = v ^ 0x80808080u;
        const float2 k = make_float2(-(8388608.f + 128.f), -(8388608.f + 128.f));
        const float2 x = add2(make_float2(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440)),
                                          __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7441))), k);
        const float2 y = add2(make_float2(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7442)),
                                          __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7443))), k);
        return make_float4(x.x, x.y, y.x, y.y);
    }
};

// Eight groups of 128 values at once, by the 16 lanes of a half-warp: lane l has unit l (16 bytes, eight
// values) of each group in v[0..7], and gets its codes; scale is that of group scale_group(l).
// The eight maxima are reduced together, each step halving what a lane still holds, so that one lane
// (of two) ends up with one group's maximum and the two divisions are done once for eight groups: they
// and 32 shuffles a lane would otherwise cost more than the rest.
__device__ __forceinline__ int scale_group(int lane) { return (lane >> 1) & 7; }
template <typename T, typename Code>
__device__ __forceinline__ void encode_groups(const uint4 (&v)[8], int lane, uint2 (&codes)[8], float *scale)
{
    // The largest magnitudes by their bits, which order like the values and put inf and NaN on top.
    uint32_t m[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const uint32_t p = __vmaxu2(__vmaxu2(v[k].x & 0x7FFF7FFFu, v[k].y & 0x7FFF7FFFu),
                                    __vmaxu2(v[k].z & 0x7FFF7FFFu, v[k].w & 0x7FFF7FFFu));
        m[k] = max(p & 0xFFFFu, p >> 16);
    }
#pragma unroll
    for (int w = 4; w > 0; w /= 2) {  // bit 2 w of the lane takes the upper half of the groups
#pragma unroll
        for (int k = 0; k < w; ++k) {
            const bool up = (lane & (2 * w)) != 0;
            const uint32_t give = up ? m[k] : m[k + w], keep = up ? m[k + w] : m[k];
            m[k] = max(keep, __shfl_xor_sync(0xFFFFFFFFu, give, 2 * w));
        }
    }
    const uint32_t top = max(m[0], __shfl_xor_sync(0xFFFFFFFFu, m[0], 1));
    const float a = T::unpack(top).x;
    float inv = 0.f;
    *scale = 0.f;
    if (top >= T::kInf) {
        *scale = __int_as_float(0x7FC00000);
    } else if (a >= 0x1p-100f) {
        inv = __fdiv_rn(Code::kMax, a);
        *scale = __fdiv_rn(a, Code::kMax);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float f = __shfl_sync(0xFFFFFFFFu, inv, 2 * k, 16);
        const uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 p = mul2(T::unpack(w[i]), make_float2(f, f));
            x[2 * i] = p.x;
            x[2 * i + 1] = p.y;
        }
        codes[k] = make_uint2(Code::encode4(x[0], x[1], x[2], x[3]), Code::encode4(x[4], x[5], x[6], x[7]));
        if (f == 0.f) codes[k] = make_uint2(0u, 0u);  // (no product of 0 and inf or NaN, no negative zeros)
    }
}

// Eight codes -> the eight 16-bit values they stand for.
template <typename T, typename Code>
__device__ __forceinline__ uint4 decode_unit(const uint2 &c, float scale)
{
    const float4 a = Code::decode4(c.x), b = Code::decode4(c.y);
    const float2 f = make_float2(scale, scale);
    const float2 v[4] = {mul2(make_float2(a.x, a.y), f), mul2(make_float2(a.z, a.w), f), mul2(make_float2(b.x, b.y), f),
                         mul2(make_float2(b.z, b.w), f)};
    return make_uint4(T::pack(v[0].x, v[0].y), T::pack(v[1].x, v[1].y), T::pack(v[2].x, v[2].y), T::pack(v[3].x, v[3].y));
}

}  // namespace kvb
