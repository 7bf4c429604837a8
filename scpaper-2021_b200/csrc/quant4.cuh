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
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with a zero third operand.
__device__ __forceinline__ void mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                     uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{0f00000000, 0f00000000, 0f00000000, 0f00000000};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ bool finite16(uint32_t h) { return (h & 0x7c00u) != 0x7c00u; }

// Smallest value and the largest's negative of a group, as an fp16 pair; NaN where the group holds one.
constexpr uint32_t EMPTY_RANGE = 0x7c007c00u;  // (inf, inf)

__device__ __forceinline__ uint32_t range_join(uint32_t a, uint32_t b) {
    const __half2 r = __hmin2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t range8(const uint4& v) {
    const uint32_t lo = range_join(range_join(v.x, v.y), range_join(v.z, v.w));
    const uint32_t hi = range_join(range_join(v.x ^ 0x80008000u, v.y ^ 0x80008000u),
                                   range_join(v.z ^ 0x80008000u, v.w ^ 0x80008000u));
    return range_join(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
}
// Joins the ranges of the four lanes of a group of 32 (lanes that differ in their two lowest bits).
__device__ __forceinline__ uint32_t range_quad(uint32_t r) {
    r = range_join(r, __shfl_xor_sync(0xffffffffu, r, 1));
    return range_join(r, __shfl_xor_sync(0xffffffffu, r, 2));
}

// (s, m) of a group as fp16 bits, s in the low half.  Every step is one IEEE operation.
__device__ __forceinline__ uint32_t params_of(uint32_t range) {
    if (!finite16(range) || !finite16(range >> 16)) return 0x7fff7fffu;  // NaN, NaN
    const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&range));
    const __half s = __float2half_rn(__fdiv_rn(__fsub_rn(-r.y, r.x), 15.f));
    return static_cast<uint32_t>(__half_as_ushort(s)) | (range << 16);
}

// What codes8 needs of a group: computed once, by one of the lanes that share the group.
__device__ __forceinline__ float inverse_of(uint32_t sm) {
    const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(sm & 0xffffu)));
    return s > 0.f ? __frcp_rn(s) : 0.f;
}

// Codes of eight fp16 values: round_half_even((x - m) / s) limited to 0 .. 15, of the exact quotient.  The fp32
// estimate (x - m)(1 / s) is off by less than 2e-6; where it lies within 1e-5 of a border between two codes, as its
// remainder tells, the eight are done again in 64 bits, where x - m and (c + 1/2) s are exact (fp16 inputs: 41
// and 16 bits).  So are groups with s below 2^-19, whose rounding (to a grid of 2^-24) can leave quotients above
// 15.5; elsewhere the largest is 15.23.  Value k goes to nibble k, or (PAIRS) to (k >> 1) + 4 (k & 1).
template <bool PAIRS>
__device__ __forceinline__ uint32_t codes8(const uint4& v, uint32_t sm, float inv) {
    const float2 sm32 = __half22float2(*reinterpret_cast<const __half2*>(&sm));
    const float s = sm32.x, m = sm32.y;
    constexpr float MAGIC = 12582912.f;  // 1.5 2^23: sums with it are rounded to whole numbers, in their lowest bits
    constexpr uint32_t MAGIC_BITS = 0x4b400000u;
    const uint64_t inv2 = pack_f32x2(inv, inv), m2 = pack_f32x2(-m, -m), s2 = pack_f32x2(-s, -s);
    const uint64_t magic2 = pack_f32x2(MAGIC, MAGIC), back2 = pack_f32x2(-MAGIC, -MAGIC);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t c[8];
    float worst = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        const uint64_t d = add_f32x2(pack_f32x2(x.x, x.y), m2);
        const uint64_t u = fma_f32x2(d, inv2, magic2);
        float u0, u1, e0, e1;
        unpack_f32x2(u, u0, u1);
        unpack_f32x2(fma_f32x2(add_f32x2(u, back2), s2, d), e0, e1);
        worst = fmaxf(worst, fmaxf(fabsf(e0), fabsf(e1)));
        c[2 * i] = __float_as_uint(u0);
        c[2 * i + 1] = __float_as_uint(u1);
    }
    if (worst > (s < 0x1p-19f ? -1.f : 0.49999f * s) && s > 0.f) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const double d = static_cast<double>(__half2float(__ushort_as_half(
                                 static_cast<unsigned short>(w[k >> 1] >> (16 * (k & 1)))))) - m;
            const double f = floor(d * inv);  // (next to a border that is the number below it)
            const double e = d - (f + 0.5) * s;
            const int n = static_cast<int>(f);
            c[k] = MAGIC_BITS + max(0, min(15, n + (e > 0.0 || (e == 0.0 && (n & 1)))));
        }
    }
    // nibbles from the highest down; what the floats' other bits add up to is a constant
    uint32_t out = 0;
#pragma unroll
    for (int n = 7; n >= 0; --n) out = out * 16 + c[PAIRS ? 2 * (n & 3) + (n >> 2) : n];
    out -= MAGIC_BITS * 0x11111111u;
    return s > 0.f ? out : 0u;  // a constant group, or one that is not finite: 0
}

// Nonzero where c s + m may pass the type's end for some code: |s| 2^11 or more, or |m| 2^15 or more (and for what is
// not finite); below, |15 s + m| < 30720 + 32768.
__device__ __forceinline__ uint32_t may_pass_end(uint32_t sm) {
    return ((sm & 0x7fff7fffu) + 0x08001800u) & 0x80008000u;  // (the exponents carry)
}

// fp16(c s + m), rounded once.
__device__ __forceinline__ uint32_t unlimited2(uint32_t code_pair, __half2 s, __half2 m) {
    const uint32_t c = and_or(code_pair, NIBBLES, 0x64006400u);
    const __half2 base = __floats2half2_rn(1024.f, 1024.f);
    const __half2 v = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&c), base), s, m);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// Two values limited to +-65504; NaN stays.  (s below 0 is nothing that the quantisers write, but arrays may come
// from elsewhere.)
__device__ __forceinline__ uint32_t limited2(uint32_t v) {
    const __half2 most = __floats2half2_rn(65504.f, 65504.f), least = __floats2half2_rn(-65504.f, -65504.f);
    const __half2 y = __hmax2_nan(__hmin2_nan(*reinterpret_cast<const __half2*>(&v), most), least);
    return *reinterpret_cast<const uint32_t*>(&y);
}
// fp16(c s + m), rounded once and limited (s is rounded, so 15 s + m may pass the type's end).
__device__ __forceinline__ uint32_t value2(uint32_t code_pair, __half2 s, __half2 m) {
    return limited2(unlimited2(code_pair, s, m));
}

// Eight values of a word whose value k is in nibble k, or (PAIRS) in (k >> 1) + 4 (k & 1).
template <bool PAIRS>
__device__ __forceinline__ uint4 values8(uint32_t w, uint32_t sm) {
    const __half2 pair = *reinterpret_cast<const __half2*>(&sm);
    const __half2 s = __low2half2(pair), m = __high2half2(pair);
    const uint32_t a = value2(w, s, m), b = value2(w >> 4, s, m), c = value2(w >> 8, s, m), d = value2(w >> 12, s, m);
    if (PAIRS) return make_uint4(a, b, c, d);
    return make_uint4(__byte_perm(a, b, 0x5410), __byte_perm(c, d, 0x5410), __byte_perm(a, b, 0x7632),
                      __byte_perm(c, d, 0x7632));
}

}  // namespace q4
}  // namespace et
