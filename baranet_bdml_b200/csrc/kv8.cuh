// The 8-bit paged cache: what a block holds, and how numbers become 8 bits and back.
//
// A block is one (page, key head), BN_KV8_BLOCK bytes in a row:
//     [   0, 1024)  K  [16 tokens][64]
//     [1024, 2048)  V  [16 tokens][64], the 16-byte piece c of token t in place c ^ (t / 2 % 4)
//     [2048, 2112)  [16 tokens] (K scale, V scale), bf16
// so that a block is one bulk copy into shared memory, keys are read from there 16 bytes a lane without bank conflicts, and eight
// tokens' pieces of V lie in eight different groups of banks for ldmatrix.
//
// A scale belongs to one token and key head.  One for a page would have to grow with a later token of the page, whose older tokens
// would then be rounded a second time, and what a token is read back as would depend on tokens that came after it or were taken
// back; the finer scales cost 64 bytes of 2112.
//   e4m3: the smallest power of two that leaves no magnitude above 448 (a float format gains nothing from other factors, and division
//         by it is exact)
//   int8: the largest magnitude / 127, rounded up to bf16
// both kept within 2^-100 .. 2^122.  A token with an infinity or a NaN has the scale NaN.
#pragma once

#include "common.cuh"
#include "hybrid.cuh"
#include "ptx.cuh"

namespace bn {

constexpr int KV8_D = 64;
constexpr int KV8_V = 1024, KV8_SCALES = 2048;
constexpr uint32_t KV8_LEAST = (127 - 100) << 23, KV8_MOST = (127 + 122) << 23;
static_assert(KV8_SCALES + BN_PAGE_TOKENS * 4 == BN_KV8_BLOCK, "block of the 8-bit cache");

// where byte d of a token's values lies in its row of V
__host__ __device__ __forceinline__ constexpr int kv8_v_place(int token, int d) { return (((d >> 4) ^ ((token >> 1) & 3)) << 4) | (d & 15); }

// the frequencies of the 32 rotation pairs
struct RotationFreqs {
    double f[KV8_D / 2];
};
// (a thread's last ones are at hand: 32 powers cost the host 2 us)
inline const RotationFreqs& rotation_freqs(float theta) {
    static thread_local float known = 0.f;
    static thread_local RotationFreqs r;
    if (theta != known) {
        for (int i = 0; i < KV8_D / 2; ++i) r.f[i] = pow((double)theta, -2.0 * i / KV8_D);
        known = theta;
    }
    return r;
}

// cos and sin of position * frequency, each off by little more than a rounding: the product and its reduction to a turn are taken in fp64,
// the functions (of half turns, which need no reduction of their own) in fp32, and what fp32 leaves of the angle is added to first order
__device__ __forceinline__ void kv8_rotation(int position, double freq, float* c, float* s) {
    const double turns = (double)position * freq * 0.15915494309189535, halves = 2.0 * (turns - rint(turns));
    const float at = (float)halves, rest = (float)(halves - (double)at) * 3.14159265f;
    float c0, s0;
    sincospif(at, &s0, &c0);
    *c = fmaf(-rest, s0, c0);
    *s = fmaf(rest, c0, s0);
}

template <int VALUES> __device__ __forceinline__ float kv8_scale(uint32_t most_bits) {
    if (most_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    uint32_t b;
    if (VALUES == BN_KV8_E4M3) {
        // most = 1.m * 2^e: 2^(e - 8) leaves 1.m * 2^8, too much above 1.75
        const int e = (int)(most_bits >> 23) - 8 + ((most_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
        b = e > 0 ? (uint32_t)e << 23 : 0u;
    } else {
        // the bf16 number at or below the quotient, or the next: 127 times it is exact
        b = __float_as_uint(__uint_as_float(most_bits) * (1.f / 127.f)) & 0xffff0000u;
        if (127.f * __uint_as_float(b) < __uint_as_float(most_bits)) b += 0x10000u;
    }
    return __uint_as_float(min(max(b, KV8_LEAST), KV8_MOST));
}

// four numbers / scale, rounded to nearest (ties to even), as four bytes
template <int VALUES> __device__ __forceinline__ uint32_t kv8_pack(float a, float b, float c, float d, float scale) {
    if (scale != scale) return 0u;
    if (VALUES == BN_KV8_E4M3) {
        const float inv = __uint_as_float((254u << 23) - __float_as_uint(scale));      // exact: a power of two
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b * inv), "f"(a * inv));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d * inv), "f"(c * inv));
        return (uint32_t)lo | (uint32_t)hi << 16;
    }
    // x / scale to the nearest whole number: by the reciprocal, whose product is off by less than 2^-14, and by the division itself where
    // that could put it on the other side of a tie
    const float inv = __fdividef(1.f, scale), x[4] = {a, b, c, d};
    uint32_t bits[4];
    bool near = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = fminf(fmaxf(x[i] * inv, -127.f), 127.f), whole = q + 12582912.f;          // 1.5 * 2^23: the whole number is in the low bits
        near |= fabsf(q - (whole - 12582912.f)) > 0.5f - 6.1035156e-5f;
        bits[i] = __float_as_uint(whole);
    }
    if (near) {
#pragma unroll
        for (int i = 0; i < 4; ++i) bits[i] = __float_as_uint(fminf(fmaxf(__fdiv_rn(x[i], scale), -127.f), 127.f) + 12582912.f);
    }
    return __byte_perm(__byte_perm(bits[0], bits[1], 0x0040), __byte_perm(bits[2], bits[3], 0x0040), 0x5410);
}

// bytes (0, 1) and (2, 3) of a word as two fp16 each
template <int VALUES> __device__ __forceinline__ void kv8_halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if (VALUES == BN_KV8_E4M3) {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
    } else {
        // 0x6400 | u is 1024 + u in fp16; u = value + 128
        const uint32_t u = w ^ 0x80808080u;
        uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(x), "r"(0x64806480u));
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(y), "r"(0x64806480u));
    }
}
// the same of bytes (0, 2) and (1, 3): a word of ldmatrix.trans holds two elements of a token, then those of the next token
template <int VALUES> __device__ __forceinline__ void kv8_token_pairs(uint32_t w, uint32_t& first, uint32_t& second) {
    if (VALUES == BN_KV8_E4M3) {
        kv8_halves<VALUES>(__byte_perm(w, 0u, 0x3120), first, second);
    } else {
        const uint32_t u = w ^ 0x80808080u;
        uint32_t x = __byte_perm(u, 0x64646464u, 0x4240), y = __byte_perm(u, 0x64646464u, 0x4341);
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(first) : "r"(x), "r"(0x64806480u));
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(second) : "r"(y), "r"(0x64806480u));
    }
}
__device__ __forceinline__ float2 halves_to_floats(uint32_t h) {
    float2 f;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(f.x), "=f"(f.y) : "r"(h));
    return f;
}

}  // namespace bn
