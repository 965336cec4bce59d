// Paged key-value cache: new rows written (rounded or quantised) and rows read back.  The formulas stand at
// fe2o3_kv_cache_append_v1_args and fe2o3_kv_cache_read_v1_args.
//
// HBM-bound: each element is read once and written once.  A row is 2 to 32 lanes of eight columns each, so that a
// row's largest magnitude is a shuffle tree and every access is 8, 16 or 32 bytes a lane; rows that do not start on 16
// bytes are read or written element by element.  A block takes up to kTokens tokens, all their heads, K and V: it finds
// their slots once (one look at the offsets and one at the page table), and each lane has kDeep rows in flight.
// Quantisation needs the quotients as IEEE rounds them.  One division a row gives y, the reciprocal of the scale
// rounded to nearest; q = x y, corrected twice by q + (x - q scale) y, is the correctly rounded quotient (Markstein,
// Computation of elementary functions on the IBM RISC System/6000 processor, 1990) while nothing leaves the normal range:
// scales outside 2^+-60 take the division itself.
#include "kv_cache.cuh"

namespace {

constexpr int kThreads = 256, kTokens = 8, kDeep = 4;

struct KvRows {
    uint8_t *p[2];   // k, v: sources of an append, destinations of a read
    uint32_t token_stride[2], head_stride[2];
    const uint32_t *offsets;
    uint32_t tokens, per_block, lanes_log2, heads_inverse;   // lanes of a row; 2^32 / kv_heads rounded up, or 0
    uint32_t whole;                                          // rows start on 16 bytes
};

// Row numbers of a token's head 0; ~0 where its page lies outside the cache.  false (reported) where the lengths do not allow it.
__device__ __forceinline__ bool slot_of(const KvCache &c, const KvRows &r, uint32_t t, uint32_t &row) {
    uint32_t before = 1, own = 1, b = t;   // new tokens of the sequence: from this one on, and all
    if (r.offsets) {
        uint32_t n = 0;   // offsets at or below t: the sequence is the last of them (sequences without tokens share an offset)
        const uint32_t lane = threadIdx.x & 31;
        for (uint32_t i = 0; i <= c.batch; i += 32) n += __popc(__ballot_sync(~0u, i + lane <= c.batch && r.offsets[i + lane] <= t));
        if (n == 0 || n > c.batch) {
            kstatus_set(c.status, FE2O3_KSTATUS_LENGTH);
            return false;
        }
        b = n - 1;
        before = r.offsets[n] - t;
        own = r.offsets[n] - r.offsets[n - 1];
    }
    const uint32_t length = c.lengths[b];
    if (length < own || !kv_fits(c, length)) {
        kstatus_set(c.status, FE2O3_KSTATUS_LENGTH);
        return false;
    }
    row = kv_row(c, b, 0, length - before);
    return true;
}

__device__ __forceinline__ void widen(const uint4 &v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ uint4 narrow(const float (&x)[8]) {
    return make_uint4(f32_to_bf16_bits(x[0]) | f32_to_bf16_bits(x[1]) << 16, f32_to_bf16_bits(x[2]) | f32_to_bf16_bits(x[3]) << 16,
                      f32_to_bf16_bits(x[4]) | f32_to_bf16_bits(x[5]) << 16, f32_to_bf16_bits(x[6]) | f32_to_bf16_bits(x[7]) << 16);
}
// Eight columns in memory order, as they are: f32 takes both halves.
template <bool F32>
__device__ __forceinline__ void fetch(const uint8_t *at, bool whole, uint4 (&v)[2]) {
    if (whole) {
        v[0] = __ldcs(reinterpret_cast<const uint4 *>(at));
        if constexpr (F32) v[1] = __ldcs(reinterpret_cast<const uint4 *>(at + 16));
    } else if constexpr (F32) {
        const uint32_t *const e = reinterpret_cast<const uint32_t *>(at);
        v[0] = make_uint4(e[0], e[1], e[2], e[3]);
        v[1] = make_uint4(e[4], e[5], e[6], e[7]);
    } else {
        const uint16_t *const e = reinterpret_cast<const uint16_t *>(at);
        v[0] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
    }
}
template <bool F32>
__device__ __forceinline__ void put(uint8_t *at, bool whole, const float (&x)[8]) {
    if constexpr (F32) {
        if (whole) {
            __stcs(reinterpret_cast<float4 *>(at), make_float4(x[0], x[1], x[2], x[3]));
            __stcs(reinterpret_cast<float4 *>(at + 16), make_float4(x[4], x[5], x[6], x[7]));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) reinterpret_cast<float *>(at)[i] = x[i];
        }
    } else {
        const uint4 v = narrow(x);
        if (whole) {
            __stcs(reinterpret_cast<uint4 *>(at), v);
        } else {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) reinterpret_cast<uint16_t *>(at)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    }
}

// x / scale for eight columns, each as IEEE division rounds it.
__device__ __forceinline__ void quotients(const float (&x)[8], float scale, float (&q)[8]) {
    if (scale > 8.7e-19f && scale < 1.1e18f) {   // 2^+-60; |x| <= 448 scale, and what is below 2^-60 scale rounds to no code
        const float y = __fdiv_rn(1.f, scale);
        const uint64_t y2 = pack_f32x2(y, y), minus = pack_f32x2(-scale, -scale);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t v = pack_f32x2(x[2 * i], x[2 * i + 1]);
            uint64_t r = mul_f32x2(v, y2);
            r = fma_f32x2(fma_f32x2(minus, r, v), y2, r);
            r = fma_f32x2(fma_f32x2(minus, r, v), y2, r);
            unpack_f32x2(r, q[2 * i], q[2 * i + 1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = scale > 0.f ? __fdiv_rn(x[i], scale) : 0.f;   // (a NaN scale: codes 0)
    }
}
template <uint32_t FORMAT>
__device__ __forceinline__ uint2 codes_of(const float (&q)[8]) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (FORMAT == FE2O3_KV_E4M3) {
            asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
                "mov.b32 %0, {lo, hi};\n\t}" : "=r"(w[i]) : "f"(q[4 * i]), "f"(q[4 * i + 1]), "f"(q[4 * i + 2]), "f"(q[4 * i + 3]));
        } else {   // 1.5 2^23 + q is rounded to a whole number, which stands in its low bits (|q| < 127.5)
            uint32_t e[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) e[j] = __float_as_uint(q[4 * i + j] + 12582912.f);
            w[i] = __byte_perm(__byte_perm(e[0], e[1], 0x0040), __byte_perm(e[2], e[3], 0x0040), 0x5410);
        }
    }
    return make_uint2(w[0], w[1]);
}
template <uint32_t FORMAT>
__device__ __forceinline__ void values_of(const uint2 &c, float scale, float (&x)[8]) {
    const uint32_t w[2] = {c.x, c.y};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (FORMAT == FE2O3_KV_I8) {
            // the code's bits + 128 below 2^23's: the sum with -(2^23 + 128) is the code
            x[i] = __uint_as_float(__byte_perm(w[i / 4] ^ 0x80808080u, 0x4b000000u, 0x7440 | (i & 3))) - 8388736.f;
        } else if (!(i & 1)) {
            uint32_t h;
            asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(h) : "r"(w[i / 4] >> (8 * (i & 3))));
            asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}" : "=f"(x[i]), "=f"(x[i + 1]) : "r"(h));
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(x[i], scale);
}

template <uint32_t FORMAT, bool F32, bool WRITE>
__global__ void __launch_bounds__(kThreads) kv_rows_kernel(KvCache c, KvRows r) {
    __shared__ uint32_t slots[kTokens];
    __shared__ uint32_t known;   // tokens whose lengths allow a slot, a bit each
    constexpr uint32_t kEb = F32 ? 4 : 2;
    begin_after_previous();
    const uint32_t t0 = blockIdx.x * r.per_block, n = min(r.per_block, r.tokens - t0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) known = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x >> 5; i < n; i += kThreads / 32) {
        uint32_t row = ~0u;
        const bool ok = slot_of(c, r, t0 + i, row);
        if (lane == 0) {
            slots[i] = row;
            if (ok) atomicOr(&known, 1u << i);
        }
    }
    __syncthreads();
    const uint32_t lanes = 1u << r.lanes_log2, at_once = kThreads >> r.lanes_log2, column = (threadIdx.x & (lanes - 1)) * 8;
    const bool inside = column < c.dim;
    const uint32_t rows = n * 2 * c.kv_heads;
    for (uint32_t base = 0; base < rows; base += kDeep * at_once) {
        const uint32_t first = base + (threadIdx.x >> r.lanes_log2);
        uint4 raw[kDeep][2];
        float scales[kDeep];
        uint32_t at[kDeep], side[kDeep];
        uint64_t there[kDeep];
        bool active[kDeep];
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            const uint32_t i = min(first + d * at_once, rows - 1), of_side = r.heads_inverse ? __umulhi(i, r.heads_inverse) : i / c.kv_heads, h = i - of_side * c.kv_heads;   // head fastest, then K or V, then the token
            const uint32_t token = of_side >> 1, slot = slots[token];
            side[d] = of_side & 1;
            at[d] = slot == ~0u ? ~0u : slot + h * c.page_size;
            active[d] = inside && first + d * at_once < rows && (known >> token & 1) && (slot != ~0u || !WRITE);
            there[d] = ((uint64_t)(t0 + token) * r.token_stride[side[d]] + (uint64_t)h * r.head_stride[side[d]] + column) * kEb;
            raw[d][0] = raw[d][1] = make_uint4(0, 0, 0, 0);
            scales[d] = 0.f;
            if (!active[d]) continue;
            if constexpr (WRITE) {
                fetch<F32>(r.p[side[d]] + there[d], r.whole, raw[d]);
            } else if (slot != ~0u) {
                const uint8_t *const from = (side[d] ? c.v : c.k) + ((uint64_t)at[d] * c.dim + column) * kKvBytes<FORMAT>;
                if constexpr (FORMAT == FE2O3_KV_BF16) {
                    raw[d][0] = __ldcs(reinterpret_cast<const uint4 *>(from));
                } else {
                    const uint2 v = __ldcs(reinterpret_cast<const uint2 *>(from));
                    raw[d][0].x = v.x;
                    raw[d][0].y = v.y;
                    scales[d] = (side[d] ? c.v_scales : c.k_scales)[at[d]];
                }
            }
        }
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            float x[8];
            if constexpr (WRITE) {
                uint8_t *const to = (side[d] ? c.v : c.k) + ((uint64_t)at[d] * c.dim + column) * kKvBytes<FORMAT>;
                if constexpr (FORMAT == FE2O3_KV_BF16 && !F32) {
                    if (active[d]) *reinterpret_cast<uint4 *>(to) = raw[d][0];
                } else {
                    if constexpr (F32) {
                        const uint32_t w[8] = {raw[d][0].x, raw[d][0].y, raw[d][0].z, raw[d][0].w, raw[d][1].x, raw[d][1].y, raw[d][1].z, raw[d][1].w};
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
                    } else {
                        widen(raw[d][0], x);
                    }
                    if constexpr (FORMAT == FE2O3_KV_BF16) {
                        if (active[d]) *reinterpret_cast<uint4 *>(to) = narrow(x);
                    } else {
                        // the largest magnitude as bits: an infinity or a NaN is above every number
                        uint32_t top = 0;
#pragma unroll
                        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
                        for (uint32_t o = 1; o < lanes; o <<= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
                        const float scale = top < 0x7f800000u ? __fdiv_rn(__uint_as_float(top), kKvTop<FORMAT>) : __uint_as_float(0x7fc00000u);
                        float q[8];
                        quotients(x, scale, q);
                        if (active[d]) {
                            *reinterpret_cast<uint2 *>(to) = codes_of<FORMAT>(q);
                            if (column == 0) (side[d] ? c.v_scales : c.k_scales)[at[d]] = scale;
                        }
                    }
                }
            } else {
                if constexpr (FORMAT == FE2O3_KV_BF16) widen(raw[d][0], x);
                else values_of<FORMAT>(make_uint2(raw[d][0].x, raw[d][0].y), scales[d], x);
                if (active[d]) put<F32>(r.p[side[d]] + there[d], r.whole, x);
            }
        }
    }
}

using Kernel = void (*)(KvCache, KvRows);

template <typename Args>
int32_t launch_rows(fe2o3_ctx *ctx, cudaStream_t s, const Args *a, uint32_t dtype, fe2o3_geometry *geo, bool plan_only,
                    const Kernel (&kernels)[3][2], const char *what) {
    // tokens of a block: as many as leave every SM two blocks, up to kTokens
    uint32_t per_block = a->tokens / (2 * (ctx->sm_count > 0 ? ctx->sm_count : 1));
    per_block = per_block < 1 ? 1 : per_block > kTokens ? kTokens : per_block;
    const uint32_t grid = ceil_div_u32(a->tokens, per_block);
    if (geo) *geo = fe2o3_geometry{{grid, 1, 1}, {kThreads, 1, 1}, 0, 1};
    if (plan_only || a->tokens == 0) return FE2O3_OK;
    const uint32_t eb = dtype == FE2O3_DTYPE_F32 ? 4 : 2;
    const uint64_t odd = a->k.ptr | a->v.ptr | (uint64_t)a->k_token_stride * eb | (uint64_t)a->v_token_stride * eb | (uint64_t)a->k_head_stride * eb | (uint64_t)a->v_head_stride * eb;
    uint32_t lanes_log2 = 1;
    while ((8u << lanes_log2) < a->dim) ++lanes_log2;
    const KvRows r{{reinterpret_cast<uint8_t *>(a->k.ptr), reinterpret_cast<uint8_t *>(a->v.ptr)},
                   {a->k_token_stride, a->v_token_stride},
                   {a->k_head_stride, a->v_head_stride},
                   reinterpret_cast<const uint32_t *>(a->token_offsets.ptr),
                   a->tokens,
                   per_block,
                   lanes_log2,
                   // exact for the indexes of a block, below 16 kv_heads
                   a->kv_heads == 1 || a->kv_heads > 8192 ? 0 : (uint32_t)((0x100000000ull + a->kv_heads - 1) / a->kv_heads),
                   odd % 16 == 0};
    const cudaError_t e = fe2o3_launch_early(kernels[a->format][dtype == FE2O3_DTYPE_F32], grid, kThreads, 0, s, 1, kv_cache_of(ctx, a), r);
    fe2o3_count_launch(1);
    return fe2o3_cuda_status(e, what);
}

}  // namespace

int32_t launch_kv_cache_append(fe2o3_ctx *ctx, cudaStream_t s, const void *args, fe2o3_geometry *geo, bool plan_only) {
    static const Kernel kernels[3][2] = {{kv_rows_kernel<0, false, true>, kv_rows_kernel<0, true, true>},
                                         {kv_rows_kernel<1, false, true>, kv_rows_kernel<1, true, true>},
                                         {kv_rows_kernel<2, false, true>, kv_rows_kernel<2, true, true>}};
    const fe2o3_kv_cache_append_v1_args *a = static_cast<const fe2o3_kv_cache_append_v1_args *>(args);
    return launch_rows(ctx, s, a, a->input_dtype, geo, plan_only, kernels, "kv_cache_append_v1");
}
int32_t launch_kv_cache_read(fe2o3_ctx *ctx, cudaStream_t s, const void *args, fe2o3_geometry *geo, bool plan_only) {
    static const Kernel kernels[3][2] = {{kv_rows_kernel<0, false, false>, kv_rows_kernel<0, true, false>},
                                         {kv_rows_kernel<1, false, false>, kv_rows_kernel<1, true, false>},
                                         {kv_rows_kernel<2, false, false>, kv_rows_kernel<2, true, false>}};
    const fe2o3_kv_cache_read_v1_args *a = static_cast<const fe2o3_kv_cache_read_v1_args *>(args);
    return launch_rows(ctx, s, a, a->output_dtype, geo, plan_only, kernels, "kv_cache_read_v1");
}

static Fe2o3KernelRegistration reg_append("kv_cache_append_v1", reinterpret_cast<const void *>(kv_rows_kernel<0, false, true>));
static Fe2o3KernelRegistration reg_read("kv_cache_read_v1", reinterpret_cast<const void *>(kv_rows_kernel<0, false, false>));
