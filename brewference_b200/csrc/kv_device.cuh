// kv_device.cuh — device helpers shared by the attention kernels over the
// 4-bit K/V cache: code unpacking, fp16 pair arithmetic, word and scale loads
// of a group.
#pragma once

#include "kv.cuh"

namespace brew {
namespace {

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// x0, x1 as two pairs of fp16: the rounded values and what they leave.
__device__ __forceinline__ void split_half2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = pack_half2(x0 - f.x, x1 - f.y);
}

// The values c - 8 of the codes c in nibbles 0 and 4, 1 and 5, 2 and 6, 3 and
// 7 of w, as fp16 pairs: a nibble below the exponent of 1024 is 1024 + c (one
// place up 1024 + 16 c); one exact operation takes the rest off.  (A nibble
// alone, the subnormal c 2^-24, would save that operation, but mma aligns its
// products by their exponent fields and loses 7 bits of a subnormal's.)
__device__ __forceinline__ uint32_t code_bits(uint32_t w, uint32_t mask, uint32_t base) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "r"(mask), "r"(base));   // w & mask | base
    return d;
}
// `base`: 0x64006400, a launch parameter so that it stays in a register and
// each step is one instruction (as a constant it took two: 64 more of 478 per
// 16 positions, and 6 % of the time).
__device__ __forceinline__ void unpack(uint32_t (&x)[4], uint32_t w, uint32_t base) {
    const uint32_t y = w >> 8;
    const uint32_t e0 = code_bits(w, 0x000F000Fu, base), e1 = code_bits(w, 0x00F000F0u, base);
    const uint32_t e2 = code_bits(y, 0x000F000Fu, base), e3 = code_bits(y, 0x00F000F0u, base);
    asm("sub.f16x2 %0, %1, %2;" : "=r"(x[0]) : "r"(e0), "r"(0x64086408u));                            // - 1032
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(x[1]) : "r"(e1), "r"(0x2C002C00u), "r"(0xD480D480u));   // / 16 - 72
    asm("sub.f16x2 %0, %1, %2;" : "=r"(x[2]) : "r"(e2), "r"(0x64086408u));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(x[3]) : "r"(e3), "r"(0x2C002C00u), "r"(0xD480D480u));
}

// Two fp32 numbers at a time.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\t"
        "mov.b64 {%0, %1}, x;}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// fp16 pairs.
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t fma_h2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t neg_h2(uint32_t a) {
    uint32_t d;
    asm("neg.f16x2 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// The larger magnitude, with some sign.
__device__ __forceinline__ uint32_t maxabs_h2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// The smaller one.
__device__ __forceinline__ uint32_t minabs_h2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("min.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Words (u, 0 .. R - 1, lane) of a group's K or V quants.
template <int R>
__device__ __forceinline__ void load_words(uint32_t (&w)[R], const uint8_t* q, int u, int lane) {
    if constexpr (R % 4 == 0) {
#pragma unroll
        for (int c = 0; c < R / 4; ++c) {
            const uint4 v = *reinterpret_cast<const uint4*>(q + 4 * kv_word(R, u, 4 * c, lane));
            w[4 * c] = v.x; w[4 * c + 1] = v.y; w[4 * c + 2] = v.z; w[4 * c + 3] = v.w;
        }
    } else if constexpr (R == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(q + 4 * kv_word(R, u, 0, lane));
        w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
        for (int b = 0; b < R; ++b) w[b] = *reinterpret_cast<const uint32_t*>(q + 4 * kv_word(R, u, b, lane));
    }
}

// Scales of positions 8 u + 2 i and + 1, blocks 0 .. R - 1 (fp16 pairs).
template <int R>
__device__ __forceinline__ void load_scales(uint32_t (&w)[R], const uint8_t* s, int u, int i) {
    const uint8_t* p = s + 4 * R * (4 * u + i);
    if constexpr (R % 4 == 0) {
#pragma unroll
        for (int c = 0; c < R / 4; ++c) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + 16 * c);
            w[4 * c] = v.x; w[4 * c + 1] = v.y; w[4 * c + 2] = v.z; w[4 * c + 3] = v.w;
        }
    } else if constexpr (R == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
        for (int b = 0; b < R; ++b) w[b] = *reinterpret_cast<const uint32_t*>(p + 4 * b);
    }
}

// K scales of position p of a group, blocks 0 .. R - 1.
template <int R>
__device__ __forceinline__ void load_kscales(__half (&d)[R], const uint8_t* s, int p) {
    const uint8_t* q = s + 2 * R * p;
    if constexpr (R % 4 == 0) {
#pragma unroll
        for (int c = 0; c < R / 4; ++c) {
            const uint2 v = *reinterpret_cast<const uint2*>(q + 8 * c);
            const __half2 a = *reinterpret_cast<const __half2*>(&v.x), b = *reinterpret_cast<const __half2*>(&v.y);
            d[4 * c] = __low2half(a); d[4 * c + 1] = __high2half(a);
            d[4 * c + 2] = __low2half(b); d[4 * c + 3] = __high2half(b);
        }
    } else if constexpr (R == 2) {
        const __half2 a = *reinterpret_cast<const __half2*>(q);
        d[0] = __low2half(a); d[1] = __high2half(a);
    } else {
#pragma unroll
        for (int b = 0; b < R; ++b) d[b] = *reinterpret_cast<const __half*>(q + 2 * b);
    }
}

}  // namespace
}  // namespace brew
