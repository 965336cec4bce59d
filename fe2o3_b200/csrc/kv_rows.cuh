// Rows on their way into the key-value cache and out of it: pieces of 16 bytes of a row, quantisation, and what codes stand for.
#pragma once
#include "kv_cache.cuh"

#ifdef __CUDACC__

namespace {

__device__ __forceinline__ void widen2(uint32_t v, float *x) {
    x[0] = __uint_as_float(v << 16);
    x[1] = __uint_as_float(v & 0xffff0000u);
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {   // to nearest even
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// A piece of the caller's row.
template <bool F32, bool WHOLE>
__device__ __forceinline__ uint4 fetch(const uint8_t *at) {
    if constexpr (WHOLE) {
        return __ldcs(reinterpret_cast<const uint4 *>(at));
    } else if constexpr (F32) {
        const uint32_t *const e = reinterpret_cast<const uint32_t *>(at);
        return make_uint4(e[0], e[1], e[2], e[3]);
    } else {
        const uint16_t *const e = reinterpret_cast<const uint16_t *>(at);
        return make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
    }
}
template <bool F32, bool WHOLE>
__device__ __forceinline__ void put(uint8_t *at, const uint4 &v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (WHOLE) {
        __stcs(reinterpret_cast<uint4 *>(at), v);
    } else {
#pragma unroll
        for (int i = 0; i < (F32 ? 4 : 8); ++i) {
            if constexpr (F32) reinterpret_cast<uint32_t *>(at)[i] = w[i];
            else reinterpret_cast<uint16_t *>(at)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    }
}
// The same columns in the cache, whose rows start on 16 bytes.
template <int BYTES>
__device__ __forceinline__ uint4 fetch_cached(const uint8_t *at) {
    if constexpr (BYTES == 16) return __ldcs(reinterpret_cast<const uint4 *>(at));
    if constexpr (BYTES == 8) {
        const uint2 v = __ldcs(reinterpret_cast<const uint2 *>(at));
        return make_uint4(v.x, v.y, 0, 0);
    }
    return make_uint4(__ldcs(reinterpret_cast<const uint32_t *>(at)), 0, 0, 0);
}
template <int BYTES>
__device__ __forceinline__ void put_cached(uint8_t *at, const uint4 &v) {
    if constexpr (BYTES == 16) *reinterpret_cast<uint4 *>(at) = v;
    else if constexpr (BYTES == 8) *reinterpret_cast<uint2 *>(at) = make_uint2(v.x, v.y);
    else if constexpr (BYTES == 4) *reinterpret_cast<uint32_t *>(at) = v.x;
    else *reinterpret_cast<uint16_t *>(at) = (uint16_t)v.x;
}

template <int LANES>
__device__ __forceinline__ uint32_t highest(uint32_t v) {
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) v = max(v, __shfl_xor_sync(~0u, v, o));
    return v;
}

// -x / scale, each as IEEE division rounds it; up to the largest code, which a subnormal scale's few bits let it pass.  (With a
// minus, because the corrections of a quotient of 0 are then zeros of the opposite sign and leave it its own.)
template <uint32_t FORMAT, int N>
__device__ __forceinline__ void minus_quotients(float (&x)[N], float scale) {
    if (scale > 8.7e-19f && scale < 1.1e18f) {   // 2^+-60; |x| <= 448 scale, and what is below 2^-60 scale rounds to no code
        const float y = -__frcp_rn(scale);
        const uint64_t y2 = pack_f32x2(y, y), scale2 = pack_f32x2(scale, scale);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint64_t v = pack_f32x2(x[i], x[i + 1]);
            uint64_t r = mul_f32x2(v, y2);
            r = fma_f32x2(fma_f32x2(scale2, r, v), y2, r);
            r = fma_f32x2(fma_f32x2(scale2, r, v), y2, r);
            unpack_f32x2(r, x[i], x[i + 1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = scale > 0.f ? fminf(fmaxf(-__fdiv_rn(x[i], scale), -kKvTop<FORMAT>), kKvTop<FORMAT>) : -0.f;   // (a NaN scale: codes 0)
    }
}
// top / C, rounded to nearest: the same corrections, with 1 / C known beforehand.
template <uint32_t FORMAT>
__device__ __forceinline__ float scale_of(float top) {
    constexpr float kC = kKvTop<FORMAT>, kY = (float)(1.0 / kC);
    if (top > 8.7e-19f && top < 1.1e18f) {
        float r = top * kY;
        r = fmaf(fmaf(-kC, r, top), kY, r);
        return fmaf(fmaf(-kC, r, top), kY, r);
    }
    return __fdiv_rn(top, kC);
}
template <uint32_t FORMAT>
__device__ __forceinline__ uint32_t codes_of(const float *q) {   // four of them, of -q
    uint32_t w;
    if constexpr (FORMAT == FE2O3_KV_E4M3) {
        asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
            "mov.b32 %0, {lo, hi};\n\t}" : "=r"(w) : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]));
        w ^= 0x80808080u;
    } else {   // 1.5 2^23 - q is rounded to a whole number, which stands in its low bits (|q| < 127.5)
        uint32_t e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = __float_as_uint(12582912.f - q[j]);
        w = __byte_perm(__byte_perm(e[0], e[1], 0x0040), __byte_perm(e[2], e[3], 0x0040), 0x5410);
    }
    return w;
}
template <uint32_t FORMAT>
__device__ __forceinline__ void values_of(uint32_t w, float scale, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (FORMAT == FE2O3_KV_I8) {
            // the code's bits + 128 below 2^23's: the sum with -(2^23 + 128) is the code
            x[i] = __uint_as_float(__byte_perm(w ^ 0x80808080u, 0x4b000000u, 0x7440 | i)) - 8388736.f;
        } else if (!(i & 1)) {
            uint32_t h;
            asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(h) : "r"(w >> (8 * i)));
            asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}" : "=f"(x[i]), "=f"(x[i + 1]) : "r"(h));
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __fmul_rn(x[i], scale);
}

// ---- 4 bits: a scale for 16 columns, and one a row ----
// f32 -> e4m3, to nearest even (v is a block scale: 0 .. 448), and back
__device__ __forceinline__ uint32_t e4m3_of(float v) {
    uint32_t w;
    asm("{\n\t.reg .b16 t;\n\tcvt.rn.satfinite.e4m3x2.f32 t, %2, %1;\n\tcvt.u32.u16 %0, t;\n\t}" : "=r"(w) : "f"(v), "f"(0.f));
    return w;
}
__device__ __forceinline__ float of_e4m3(uint32_t code) {
    float v;
    asm("{\n\t.reg .b32 h;\n\t.reg .b16 t, u;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 h, t;\n\tmov.b32 {t, u}, h;\n\tcvt.f32.f16 %0, t;\n\t}" : "=f"(v) : "r"(code));
    return v;
}
// n / m, rounded to nearest, from y near 1 / m (the corrections of minus_quotients).
__device__ __forceinline__ float corrected(float n, float m, float y) {
    float r = n * y;
    r = fmaf(fmaf(-m, r, n), y, r);
    return fmaf(fmaf(-m, r, n), y, r);
}
// A row's scale and 448 / m of its largest magnitude m (an infinity or a NaN: scale NaN; below 2^-100: both 0, and all codes).
__device__ __forceinline__ void row_scales4(float m, float &scale, float &up) {
    scale = up = 0.f;
    if (m > 8.7e-19f && m < 1.1e18f) {   // 2^+-60: nothing leaves the normal range
        scale = corrected(m, 2688.f, (float)(1.0 / 2688.0));
        up = corrected(448.f, m, __frcp_rn(m));
    } else if (m >= 0x1p-100f && m < INFINITY) {
        scale = __fdiv_rn(m, 2688.f);
        up = __fdiv_rn(448.f, m);
    } else if (!(m < INFINITY)) {
        scale = __uint_as_float(0x7fc00000u);
    }
}
// A block's scale, and the factor that turns its elements into units of the code (0: a block of zeros).
__device__ __forceinline__ uint32_t block_scale4(float m, float scale, float up, float &factor) {
    factor = 0.f;
    if (!(up > 0.f)) return 0;
    const uint32_t code = e4m3_of(m * up);
    if (code) factor = __frcp_rn(of_e4m3(code) * scale);
    return code;
}
// Elements as codes, the first in the lowest bits.  (With a block of zeros nothing keeps a sign.)
__device__ __forceinline__ uint32_t codes4(const float *x, float factor) {
    if (!(factor > 0.f)) return 0;
    uint32_t w;
    asm("{\n\t.reg .b8 a, b, no;\n\tcvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "mov.b32 %0, {a, b, a, b};\n\t}" : "=r"(w) : "f"(x[0] * factor), "f"(x[1] * factor), "f"(x[2] * factor), "f"(x[3] * factor));
    return w & 0xffffu;
}
__device__ __forceinline__ uint32_t codes8(const float *x, float factor) {
    if (!(factor > 0.f)) return 0;
    float y[8];
    const uint64_t by = pack_f32x2(factor, factor);
#pragma unroll
    for (int i = 0; i < 8; i += 2) unpack_f32x2(mul_f32x2(pack_f32x2(x[i], x[i + 1]), by), y[i], y[i + 1]);
    uint32_t w;
    asm("{\n\t.reg .b8 a, b, c, d;\n\tcvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\tmov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(w) : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
    return w;
}
// What eight codes of a block stand for; a code times its block's scale has 6 bits, f16's 11 hold it exactly.
__device__ __forceinline__ void values8(uint32_t w, uint32_t block, float scale, float *x) {
    uint32_t h[4], by;
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}" : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(by) : "r"(block * 0x101u));
    const uint64_t scale2 = pack_f32x2(scale, scale);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float lo, hi;
        asm("{\n\t.reg .b32 p;\n\t.reg .b16 a, b;\n\tmul.rn.f16x2 p, %2, %3;\n\tmov.b32 {a, b}, p;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(lo), "=f"(hi) : "r"(h[i]), "r"(by));
        unpack_f32x2(mul_f32x2(pack_f32x2(lo, hi), scale2), x[2 * i], x[2 * i + 1]);
    }
}

}  // namespace

#endif  // __CUDACC__
