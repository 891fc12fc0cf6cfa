// Blocks of 16 values: loading, quantising and decoding them.  Shared by the streaming kernels (fp4_kernels.cu) and by the
// product of a few rows, which quantises its activations itself (fp4_gemm_sm100.cu).
//
// The arithmetic, and why it is exact.  With g = 2^e every decision of the quantiser compares a value with a number of few bits.
//   Block scale: t = RN(b / 6) for b = amax of the block / g, s = e4m3(t).  A border of the E4M3 grid has 5 bits; if b / 6 is no
//   border, b differs from 6 borders' product by at least an ulp of b, more than half an ulp of the border: RN(b / 6) is on the
//   right side of it, and it is the border exactly where b / 6 is.
//   Code: q = x / (s g), s g exact.  A border of the E2M1 grid times s has at most 7 bits.
//     FP32 values.  The quotient is taken with the reciprocal r = RN(1 / (s g)) and one correction by its remainder (Markstein, IBM J.
//     Res. Dev. 34, 1990): q0 = RN(x r), q = RN(q0 + r (x - q0 s g)).  The remainder is exact (its last bit is worth 2^-35 g or
//     more, never below 2^-145), so q is the quotient with a relative error of 2^-46 before its rounding.  At a border q is the
//     border.  Off it the quotient is off by 2^-23 / 1.875 at least (s has 4 bits, so the quantity whose ulp counts has a
//     significand of at most 1.875), 6% more than the half ulp of the border (2^-24).
//     16-bit values have 11 bits at most: a quotient that is no border is 2^-11 of it away from it, 2^-13 or more.  So q is rounded
//     to multiples of 2^-14 (by adding 1.5 2^9, one instruction with the product, and taking it away again): an error of 2^-20 in the
//     quotient vanishes at a border and moves nothing across one, and an approximate reciprocal will do.
// A conversion packs two codes; sign, zero and saturation are its.
#pragma once

#include <cuda_fp16.h>

#include "../../include/llmini_b200_fp4.h"
#include "common.cuh"

namespace b2 {

namespace {

// Largest |value| as bits of a non-negative float: infinities and NaN (of either sign) come out on top.
__device__ __forceinline__ uint32_t max_bits(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t warp_max_bits(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

// The scale on top for a vector whose largest magnitude has these bits.
__device__ __forceinline__ float top_scale(uint32_t amax_bits) {
    const uint32_t e = amax_bits & 0x7f800000u;
    if (e == 0x7f800000u) return __uint_as_float(0x7fffffffu);
    return __uint_as_float((e < (27u << 23) ? (27u << 23) : e) - (10u << 23));   // 27: exponent of 2^-100
}
// 1 / g, 0 for g = NaN
__device__ __forceinline__ float top_inverse(float g) {
    const uint32_t b = __float_as_uint(g);
    return b == 0x7fffffffu ? 0.0f : __uint_as_float((254u << 23) - b);
}

// Two FP32 operations in one instruction.
struct Pair {
    uint64_t v;
};
__device__ __forceinline__ Pair pair(float lo, float hi) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(lo), "f"(hi));
    return p;
}
__device__ __forceinline__ float2 halves(Pair p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p.v));
    return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair mul2_truncated(Pair a, Pair b) {
    Pair r;
    asm("mul.rz.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

// ---- plain values: blocks of 16 -------------------------------------------------------------------------------------------
// How a thread reaches its block: 32 bytes an instruction (a warp's lanes side by side then move whole lines, where two halves of
// 16 bytes touch every line twice), 16 bytes, or value by value.
enum Access : uint32_t { kByValue = 0, kBy16 = 1, kBy32 = 2 };
__host__ __device__ inline uint32_t access_of(const void *p, uint64_t step_bytes) {
    const uint64_t at = reinterpret_cast<uintptr_t>(p) | step_bytes;
    return at % 32 == 0 ? kBy32 : at % 16 == 0 ? kBy16 : kByValue;
}
__device__ __forceinline__ void load_32(const uint8_t *p, uint32_t *w) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p)
                 : "memory");
}
__device__ __forceinline__ void store_32(uint8_t *p, const uint32_t *w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
template <int TYPE>
struct Raw {
    static constexpr int kWords = TYPE == B2_TYPE_F32 ? 16 : 8;
    static constexpr int kSize = TYPE == B2_TYPE_F32 ? 4 : 2;
    uint32_t w[kWords];

    // `n` values (at most 16) from element `p` on, zeros behind them
    __device__ __forceinline__ void load(const uint8_t *p, int n, uint32_t access) {
        if (n >= 16 && access == kBy32) {
#pragma unroll
            for (int i = 0; i < kWords / 8; ++i) load_32(p + 32 * i, w + 8 * i);
            return;
        }
        if (n >= 16 && access == kBy16) {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const uint4 v = *reinterpret_cast<const uint4 *>(p + 16 * i);
                w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
            }
            return;
        }
        if (TYPE == B2_TYPE_F32) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = i < n ? reinterpret_cast<const uint32_t *>(p)[i] : 0u;
        } else {
            const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
            for (int i = 0; i < kWords; ++i)
                w[i] = (2 * i < n ? (uint32_t)h[2 * i] : 0u) | (2 * i + 1 < n ? (uint32_t)h[2 * i + 1] << 16 : 0u);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0u;
    }
    // values 2 i and 2 i + 1
    __device__ __forceinline__ Pair values(int i) const {
        if (TYPE == B2_TYPE_F32) return pair(__uint_as_float(w[(2 * i) % kWords]), __uint_as_float(w[(2 * i + 1) % kWords]));
        if (TYPE == B2_TYPE_BF16) return pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        return pair(f.x, f.y);
    }
    __device__ __forceinline__ uint32_t amax_bits() const {
        if (TYPE == B2_TYPE_F32) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < kWords; ++i) m = max_bits(m, w[i] & 0x7fffffffu);
            return m;
        }
        uint32_t m = 0;   // 16-bit magnitudes order like their bits too
#pragma unroll
        for (int i = 0; i < kWords; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
        m = max_bits(m & 0xffffu, m >> 16);
        if (TYPE == B2_TYPE_BF16) return m << 16;
        return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
    }
};

// Eight values to eight codes, the first in the low half of the first byte.
__device__ __forceinline__ uint32_t pack_codes(Pair a, Pair b, Pair c, Pair d) {
    const float2 p = halves(a), q = halves(b), r = halves(c), t = halves(d);
    uint32_t v;
    asm("{ .reg .b8 a, b, c, d; cvt.rn.satfinite.e2m1x2.f32 a, %2, %1; cvt.rn.satfinite.e2m1x2.f32 b, %4, %3; "
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5; cvt.rn.satfinite.e2m1x2.f32 d, %8, %7; mov.b32 %0, {a, b, c, d}; }"
        : "=r"(v)
        : "f"(p.x), "f"(p.y), "f"(q.x), "f"(q.y), "f"(r.x), "f"(r.y), "f"(t.x), "f"(t.y));
    return v;
}

// Code bytes and scale of a block; g: the scale on top, inv: 1 / g, 0 for a vector that is not finite.
template <int TYPE>
__device__ __forceinline__ uint32_t encode_block(const Raw<TYPE> &block, uint32_t amax_bits, float g, float inv, uint2 &codes) {
    codes = make_uint2(0u, 0u);
    if (inv == 0.0f) return 0u;
    const float b = __uint_as_float(amax_bits) * inv, t = b * (1.0f / 6.0f);
    const uint32_t s = cvt_e4m3x2(0.0f, fmaf(fmaf(-t, 6.0f, b), 1.0f / 6.0f, t)) & 0xffu;
    if (s == 0u) return 0u;
    const float step = e4m3_value((uint16_t)s) * g;
    Pair q[8];
    if (TYPE == B2_TYPE_F32) {
        const float r = __frcp_rn(step);
        const Pair r2 = pair(r, r), n2 = pair(-step, -step);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const Pair x = block.values(i), q0 = mul2(x, r2);
            q[i] = fma2(fma2(q0, n2, x), r2, q0);
        }
    } else {
        const float r = rcp_approx_ftz(step);
        const Pair r2 = pair(r, r), c = pair(768.0f, 768.0f), nc = pair(-768.0f, -768.0f);
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = add2(fma2(block.values(i), r2, c), nc);
    }
    codes.x = pack_codes(q[0], q[1], q[2], q[3]);
    codes.y = pack_codes(q[4], q[5], q[6], q[7]);
    return s;
}

// ---- reading back ----------------------------------------------------------------------------------------------------------
// Values of a block: code * s is exact in FP16 (6 bits, 2^-10 .. 2688), the product with g is rounded in FP32.
// Values that go on to 16 bits are not to be rounded to nearest before: where FP32 has the middle between two 16-bit values for a
// product that lies beside it, the second rounding goes wrong.
//   kTruncate: the product truncated, and its last bit set where g has 14 bits or more (not counting zeros at its end).  Such a product
//     is no middle, which has 12 bits at most, but may be truncated to one.  With fewer bits of g it has 19 at most and is exact.
// A subnormal g, of whatever bits, takes product_to_odd.
enum Decoding : int { kNearest = 0, kTruncate = 1 };
template <int HOW>
__device__ __forceinline__ void decode_block(uint2 codes, uint32_t s, float g, float (&v)[16]) {
    uint32_t sh;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(sh) : "h"((uint16_t)(s | (s << 8))));
    const __half2 s2 = *reinterpret_cast<const __half2 *>(&sh);
    const Pair g2 = pair(g, g);
    const uint32_t last = HOW == kTruncate && (__float_as_uint(g) & 0x7ffu) != 0 ? 1u : 0u;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        uint32_t h[4];
        asm("{ .reg .b8 a, b, c, d; mov.b32 {a, b, c, d}, %4; cvt.rn.f16x2.e2m1x2 %0, a; cvt.rn.f16x2.e2m1x2 %1, b; "
            "cvt.rn.f16x2.e2m1x2 %2, c; cvt.rn.f16x2.e2m1x2 %3, d; }"
            : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
            : "r"(k ? codes.y : codes.x));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(__hmul2(*reinterpret_cast<const __half2 *>(&h[i]), s2));
            if (HOW == kNearest) {
                const float2 o = halves(mul2(pair(f.x, f.y), g2));
                v[8 * k + 2 * i] = o.x;
                v[8 * k + 2 * i + 1] = o.y;
            } else {
                const float2 o = halves(mul2_truncated(pair(f.x, f.y), g2));
                v[8 * k + 2 * i] = __uint_as_float(__float_as_uint(o.x) | last);
                v[8 * k + 2 * i + 1] = __uint_as_float(__float_as_uint(o.y) | last);
            }
        }
    }
}
// The value of an E2M1 code (its low four bits).
__device__ __forceinline__ float e2m1_value(uint32_t code) {
    const uint32_t e = code >> 1 & 3u, f = code & 1u;
    const float v = e == 0 ? 0.5f * f : 0.5f * (2u + f) * (float)(1u << (e - 1));
    return code & 8u ? -v : v;
}
// Rounded to odd: of the two neighbours of an inexact product the one whose last bit is set, which a second rounding, to two bits less or
// fewer still, takes where it would have taken the product itself (Boldo and Melquiond, IEEE Trans. Comput. 57, 2008).
__device__ __forceinline__ float product_to_odd(float a, float b) {
    const float down = __fmul_rd(a, b), up = __fmul_ru(a, b);
    return __float_as_uint(down) & 1u ? down : up;
}
// `n` values (at most 16) to element `p` on
template <int TYPE>
__device__ __forceinline__ void store_block(uint8_t *p, const float (&v)[16], int n, uint32_t access) {
    constexpr int kWords = Raw<TYPE>::kWords;
    uint32_t w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = TYPE == B2_TYPE_F32 ? __float_as_uint(v[i]) : pack_operands(v[2 * i % 16], v[2 * i % 16 + 1], TYPE == B2_TYPE_F16);
    if (n >= 16 && access == kBy32) {
#pragma unroll
        for (int i = 0; i < kWords / 8; ++i) store_32(p + 32 * i, w + 8 * i);
    } else if (n >= 16 && access == kBy16) {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) reinterpret_cast<uint4 *>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i >= n) continue;
            if (TYPE == B2_TYPE_F32) reinterpret_cast<uint32_t *>(p)[i] = w[i % kWords];
            else reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    }
}

}  // namespace

}  // namespace b2
