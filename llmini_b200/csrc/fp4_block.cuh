// Blocks of 16 values: loading, quantising and decoding them.  Shared by the streaming kernels (fp4_kernels.cu) and by the
// product of a few rows, which quantises its activations itself (fp4_gemm_sm100.cu).
//
// The arithmetic, and why it is exact.  With g = 2^e every decision of the quantiser compares a value with a number of few bits.
//   Block scale: t = RN(b / 6) for b = amax of the block / g, s = e4m3(t).  A border of the E4M3 grid has 5 bits; if b / 6 is no
//   border, b differs from 6 borders' product by at least an ulp of b, more than half an ulp of the border: RN(b / 6) is on the
//   right side of it, and it is the border exactly where b / 6 is.
//   Code: q = x / g / s.  A border of the E2M1 grid times s has at most 7 bits, so the same holds for RN(q).  The quotient by
//   s is taken with the reciprocal r = RN(1 / s) and one correction by its remainder (Markstein, IBM J. Res. Dev. 34, 1990):
//   q0 = RN(x r), q = RN(q0 + r (x - q0 s)); the remainder is exact, so q is the quotient with a relative error of 2^-46 before
//   its rounding.  At a border q is the border.  Off it the quotient is off by 2^-23 / 1.875 at least (s has 4 bits, so the
//   quantity whose ulp counts has a significand of at most 1.875), 6% more than the half ulp of the border (2^-24).
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
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

// ---- plain values: blocks of 16 -------------------------------------------------------------------------------------------
template <int TYPE>
struct Raw {
    static constexpr int kWords = TYPE == B2_TYPE_F32 ? 16 : 8;
    static constexpr int kSize = TYPE == B2_TYPE_F32 ? 4 : 2;
    uint32_t w[kWords];

    // `n` values (at most 16) from element `p` on, zeros behind them; `vec`: p is on a 16-byte boundary
    __device__ __forceinline__ void load(const uint8_t *p, int n, bool vec) {
        if (n >= 16 && vec) {
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

// Code bytes and scale of a block; inv = 1 / g, 0 for a vector that is not finite.
template <typename V>
__device__ __forceinline__ uint32_t encode_block(V values, uint32_t amax_bits, float inv, uint2 &codes) {
    codes = make_uint2(0u, 0u);
    if (inv == 0.0f) return 0u;
    const uint32_t s = cvt_e4m3x2(0.0f, div_uniform(__uint_as_float(amax_bits) * inv, 6.0f, 1.0f / 6.0f)) & 0xffu;
    const float sf = e4m3_value((uint16_t)s);
    const float r = s == 0u ? 0.0f : __frcp_rn(sf);
    const Pair inv2 = pair(inv, inv), r2 = pair(r, r), ns2 = pair(-sf, -sf);
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const Pair x = mul2(values(i), inv2);
        const Pair q = mul2(x, r2);
        const float2 v = halves(fma2(fma2(q, ns2, x), r2, q));
        b[i] = cvt_e2m1x2(v.y, v.x);
    }
    codes.x = b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24);
    codes.y = b[4] | (b[5] << 8) | (b[6] << 16) | (b[7] << 24);
    return s;
}

// ---- reading back ----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ __half2 e2m1_values(uint32_t byte) {
    uint32_t r;
    asm("{ .reg .b8 t; cvt.u8.u16 t, %1; cvt.rn.f16x2.e2m1x2 %0, t; }" : "=r"(r) : "h"((uint16_t)byte));
    return *reinterpret_cast<__half2 *>(&r);
}
// Values of a block: code * s is exact in FP16 (6 bits, 2^-10 .. 2688), the product with g is rounded in FP32.
__device__ __forceinline__ void decode_block(uint2 codes, uint32_t s, float g, float (&v)[16]) {
    uint32_t sh;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(sh) : "h"((uint16_t)(s | (s << 8))));
    const __half2 s2 = *reinterpret_cast<const __half2 *>(&sh);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 f = __half22float2(__hmul2(e2m1_values((i < 4 ? codes.x : codes.y) >> (8 * (i & 3)) & 0xffu), s2));
        v[2 * i] = f.x * g;
        v[2 * i + 1] = f.y * g;
    }
}
// `n` values (at most 16) to element `p` on; `vec`: p is on a 16-byte boundary
template <int TYPE>
__device__ __forceinline__ void store_block(uint8_t *p, const float (&v)[16], int n, bool vec) {
    if (TYPE == B2_TYPE_F32) {
        if (n >= 16 && vec) {
#pragma unroll
            for (int i = 0; i < 4; ++i) reinterpret_cast<float4 *>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i < n) reinterpret_cast<float *>(p)[i] = v[i];
        }
    } else {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = pack_operands(v[2 * i], v[2 * i + 1], TYPE == B2_TYPE_F16);
        if (n >= 16 && vec) {
#pragma unroll
            for (int i = 0; i < 2; ++i) reinterpret_cast<uint4 *>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i < n) reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    }
}

}  // namespace

}  // namespace b2
