// The 4-bit number format of the key/value cache and of the 4-bit Linear weights: groups of values held
// as c * s + m, c = 0 .. 15, (s, m) an fp16 pair.  Nibbles are stored so that `(word >> 4 p) & 0x000f000f`
// are two neighbouring values: read as fp16 these are the codes times 2^-24 (subnormal numbers, exact), which
// the tensor core multiplies like any other; s, m and the factor 2^24 are applied to fp32 sums.  A code is
// unpacked by one shift and one AND per two values and never rounded.
#pragma once

#include "common.cuh"

namespace et {
namespace q4 {

constexpr uint32_t NIBBLES = 0x000f000fu;  // two codes, 16 bits apart

// (a & b) | c in one instruction, with b and c in registers
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

// The two codes in the lowest nibbles of w's halves, less 8, as fp16 (exact: 1024 + c, less 1032).
__device__ __forceinline__ uint32_t centred(uint32_t w) {
    const uint32_t c = and_or(w, NIBBLES, 0x64006400u), base = 0x64086408u;
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&c), *reinterpret_cast<const __half2*>(&base));
    return *reinterpret_cast<const uint32_t*>(&v);
}

// The codes in the next nibbles, less 8, times 16 (without a shift: 1024 + 16 c, less 1152).
__device__ __forceinline__ uint32_t centred16(uint32_t w) {
    const uint32_t c = and_or(w, NIBBLES << 4, 0x64006400u), base = 0x64806480u;
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&c), *reinterpret_cast<const __half2*>(&base));
    return *reinterpret_cast<const uint32_t*>(&v);
}

// D (16 x 8, fp32) = A (16 x 16) * B (16 x 8) + D.
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with a zero third operand.
__device__ __forceinline__ void mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                     uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ bool finite16(uint32_t h) { return (h & 0x7c00u) != 0x7c00u; }

// Smallest and largest of a group and whether all of it is finite; combined over lanes by the caller.
struct Range {
    float lo, hi;
    bool finite;
};

__device__ __forceinline__ Range range8(const uint4& v) {
    Range r = {INFINITY, -INFINITY, true};
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r.finite = r.finite && finite16(w[i]) && finite16(w[i] >> 16);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        r.lo = fminf(r.lo, fminf(f.x, f.y));
        r.hi = fmaxf(r.hi, fmaxf(f.x, f.y));
    }
    return r;
}

// Combines the ranges of the four lanes of a group (lanes that differ in their two lowest bits).
__device__ __forceinline__ void range_quad(Range& r) {
#pragma unroll
    for (int d = 1; d <= 2; d <<= 1) {
        r.lo = fminf(r.lo, __shfl_xor_sync(0xffffffffu, r.lo, d));
        r.hi = fmaxf(r.hi, __shfl_xor_sync(0xffffffffu, r.hi, d));
        r.finite = __shfl_xor_sync(0xffffffffu, r.finite ? 1 : 0, d) != 0 && r.finite;
    }
}

// (s, m) of a group as fp16 bits, s in the low half.  Every step is one IEEE operation.
__device__ __forceinline__ uint32_t params_of(const Range& r) {
    if (!r.finite) return 0x7fff7fffu;  // NaN, NaN
    const __half s = __float2half_rn(__fdiv_rn(__fsub_rn(r.hi, r.lo), 15.f));
    return static_cast<uint32_t>(__half_as_ushort(s)) |
           (static_cast<uint32_t>(__half_as_ushort(__float2half_rn(r.lo))) << 16);
}

// round_half_even((x - m) / s) limited to 0 .. 15, of the exact quotient: the fp32 estimate is off by less
// than 1e-5, and what lies within 1e-3 of a border between two codes is decided in 64 bits, where x - m and
// (c + 1/2) s are exact (fp16 inputs: 41 and 16 bits).
__device__ __forceinline__ uint32_t code_of(float x, float m, float s, float inv) {
    const float t = (x - m) * inv;
    const float f = floorf(t);
    float c = rintf(t);
    if (fabsf(t - f - 0.5f) < 1e-3f) {
        const double e = (static_cast<double>(x) - m) - (static_cast<double>(f) + 0.5) * s;
        c = e > 0.0 || (e == 0.0 && (static_cast<int>(f) & 1)) ? f + 1.f : f;
    }
    return static_cast<uint32_t>(fminf(fmaxf(c, 0.f), 15.f));
}

// Codes of eight fp16 values, value k in bits 4 k .. 4 k + 3 of the result.
__device__ __forceinline__ uint32_t codes8(const uint4& v, uint32_t sm) {
    const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(sm & 0xffffu)));
    const float m = __half2float(__ushort_as_half(static_cast<unsigned short>(sm >> 16)));
    if (!(s > 0.f)) return 0u;  // a constant group, or one that is not finite
    const float inv = __frcp_rn(s);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        out |= code_of(f.x, m, s, inv) << (8 * i);
        out |= code_of(f.y, m, s, inv) << (8 * i + 4);
    }
    return out;
}

// Natural nibble order (value k in nibble k) -> pair order (value k in nibble (k >> 1) + 4 (k & 1)), and back.
__device__ __forceinline__ uint32_t to_pairs(uint32_t w) {
    uint32_t r = 0;
#pragma unroll
    for (int p = 0; p < 4; ++p) r |= ((w >> (8 * p)) & 0xfu) << (4 * p) | ((w >> (8 * p + 4)) & 0xfu) << (4 * p + 16);
    return r;
}
__device__ __forceinline__ uint32_t from_pairs(uint32_t w) {
    uint32_t r = 0;
#pragma unroll
    for (int p = 0; p < 4; ++p) r |= ((w >> (4 * p)) & 0xfu) << (8 * p) | ((w >> (4 * p + 16)) & 0xfu) << (8 * p + 4);
    return r;
}

// fp16(c s + m), limited to +-65504 (s is rounded, so 15 s + m may pass the type's largest value); NaN stays.
__device__ __forceinline__ float value_of(uint32_t c, float s, float m) {
    const float v = fmaf(static_cast<float>(c), s, m);
    return v > 65504.f ? 65504.f : v;
}

// Eight values of a word in natural nibble order.
__device__ __forceinline__ uint4 values8(uint32_t w, uint32_t sm) {
    const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(sm & 0xffffu)));
    const float m = __half2float(__ushort_as_half(static_cast<unsigned short>(sm >> 16)));
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        o[i] = pack_half2(value_of((w >> (8 * i)) & 0xfu, s, m), value_of((w >> (8 * i + 4)) & 0xfu, s, m));
    return make_uint4(o[0], o[1], o[2], o[3]);
}

}  // namespace q4
}  // namespace et
