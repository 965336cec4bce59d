// Paged key-value cache: new rows written (rounded or quantised) and rows read back.  The formulas stand at
// fe2o3_kv_cache_append_v1_args and fe2o3_kv_cache_read_v1_args.
//
// HBM-bound: each element is read once and written once.  A row is 2 to 32 lanes of eight columns each, so that a
// row's largest magnitude is a shuffle tree and every access is 4 to 16 bytes a lane, without gaps between lanes: of f32 rows a
// lane has four columns in each half (a store of every other 16 bytes costs half as much again).  Rows that do not
// start on 16 bytes are read or written element by element.  A block takes up to kTokens tokens, all their heads, K and V: one
// warp finds their slots (offsets, lengths and page table: three trips to memory a block, not a row), and each
// lane has kDeep rows in flight.  Blocks are as many as fill the SMs a whole number of times.
// 131072 tokens of 8 heads of 128 read from bf16 pages 172 us (6.2 TB/s); 16384 tokens bf16 to e4m3 35 us (2.9 TB/s, 55 % of
// the issue slots: 168 instructions a warp for two rows of K or V) and back to f32 33 us; 256 new tokens 3.0 us, an empty launch's time.
// Quantisation needs the quotients as IEEE rounds them, and is bound by issue slots.  One division a row gives y, the
// reciprocal of the scale rounded to nearest; q = x y, corrected twice by q + (x - q scale) y, is the correctly rounded
// quotient (Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, 1990) while nothing
// leaves the normal range: scales outside 2^+-60 take the division itself.
#include <atomic>

#include "kv_cache.cuh"

namespace {

constexpr int kThreads = 256, kTokens = 32, kDeep = 4;

struct KvRows {
    uint8_t *k, *v;   // sources of an append, destinations of a read
    uint32_t k_token_stride, v_token_stride, k_head_stride, v_head_stride;
    const uint32_t *offsets;
    uint32_t tokens, per_block, lanes_log2, heads_inverse;   // lanes of a row; 2^32 / kv_heads rounded up, or 0
};

// One warp, a lane a token: row number of its head 0, ~0 where its page lies outside the cache.  false (reported) where the
// lengths do not allow the token a slot.
__device__ __forceinline__ bool slot_of(const KvCache &c, const KvRows &r, uint32_t t0, uint32_t n, uint32_t &row) {
    const uint32_t lane = threadIdx.x & 31, t = t0 + lane;
    uint32_t before = 1, own = 1, b = t;   // new tokens of the sequence: from this one on, and all
    bool ok = lane < n;
    if (r.offsets) {
        // offsets at or below a token: its sequence is the last of them (sequences without tokens share an offset)
        uint32_t low = 0, high = 0;
        for (uint32_t i = 0; i <= c.batch; i += 32) {
            const uint32_t offset = i + lane <= c.batch ? r.offsets[i + lane] : ~0u;
            low += __popc(__ballot_sync(~0u, offset <= t0));
            high += __popc(__ballot_sync(~0u, offset <= t0 + n - 1));
        }
        uint32_t at = low;
        while (ok && at < high && r.offsets[at] <= t) ++at;
        ok = ok && at != 0 && at <= c.batch;
        if (ok) {
            b = at - 1;
            before = r.offsets[at] - t;
            own = r.offsets[at] - r.offsets[b];
            ok = r.offsets[b] <= t && t < r.offsets[at];   // (offsets that rise)
        }
    }
    bool report = !ok && lane < n;
    if (ok) {
        const uint32_t length = c.lengths[b];
        ok = length >= own && kv_fits(c, length);
        report = !ok && (r.offsets || length);   // (without offsets a sequence of length 0 has no token)
        if (ok) row = kv_row(c, b, 0, length - before);
    }
    if (report) kstatus_set(c.status, FE2O3_KSTATUS_LENGTH);
    return ok;
}

// A lane's eight columns: those from 8 l on, or for f32 rows four from 4 l and four from 4 (lanes + l) on.
struct Columns {
    uint32_t first, second;   // of the two fours
    bool one, two;            // inside the row
};
__device__ __forceinline__ void widen4(const uint2 &v, float *x) {
    x[0] = __uint_as_float(v.x << 16);
    x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16);
    x[3] = __uint_as_float(v.y & 0xffff0000u);
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {   // to nearest even
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint2 narrow4(const float *x) { return make_uint2(bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3])); }
__device__ __forceinline__ uint4 joined(uint2 a, uint2 b) { return make_uint4(a.x, a.y, b.x, b.y); }

// The caller's rows: f32 bits as two fours, or eight bf16.
template <bool F32, bool WHOLE>
__device__ __forceinline__ void fetch(const uint8_t *row, const Columns &c, uint4 (&v)[2]) {
    if constexpr (F32) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if (!(half ? c.two : c.one)) continue;
            const uint32_t *const e = reinterpret_cast<const uint32_t *>(row) + (half ? c.second : c.first);
            if constexpr (WHOLE) v[half] = __ldcs(reinterpret_cast<const uint4 *>(e));
            else v[half] = make_uint4(e[0], e[1], e[2], e[3]);
        }
    } else if (c.one) {
        const uint16_t *const e = reinterpret_cast<const uint16_t *>(row) + c.first;
        if constexpr (WHOLE) v[0] = __ldcs(reinterpret_cast<const uint4 *>(e));
        else v[0] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
    }
}
template <bool F32, bool WHOLE>
__device__ __forceinline__ void put(uint8_t *row, const Columns &c, const uint4 (&v)[2]) {
    if constexpr (F32) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if (!(half ? c.two : c.one)) continue;
            uint32_t *const e = reinterpret_cast<uint32_t *>(row) + (half ? c.second : c.first);
            if constexpr (WHOLE) __stcs(reinterpret_cast<uint4 *>(e), v[half]);
            else e[0] = v[half].x, e[1] = v[half].y, e[2] = v[half].z, e[3] = v[half].w;
        }
    } else if (c.one) {
        uint16_t *const e = reinterpret_cast<uint16_t *>(row) + c.first;
        const uint32_t w[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
        if constexpr (WHOLE) {
            __stcs(reinterpret_cast<uint4 *>(e), v[0]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    }
}
// The cache's rows, which start on 16 bytes: eight elements' bits.
template <uint32_t FORMAT, bool F32>
__device__ __forceinline__ uint4 fetch_cached(const uint8_t *row, const Columns &c) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if constexpr (FORMAT == FE2O3_KV_BF16) {
        if constexpr (!F32) {
            if (c.one) v = __ldcs(reinterpret_cast<const uint4 *>(row + 2 * c.first));
        } else {
            uint2 a = make_uint2(0, 0), b = a;
            if (c.one) a = __ldcs(reinterpret_cast<const uint2 *>(row + 2 * c.first));
            if (c.two) b = __ldcs(reinterpret_cast<const uint2 *>(row + 2 * c.second));
            v = joined(a, b);
        }
    } else {
        if constexpr (!F32) {
            if (c.one) {
                const uint2 a = __ldcs(reinterpret_cast<const uint2 *>(row + c.first));
                v.x = a.x;
                v.y = a.y;
            }
        } else {
            if (c.one) v.x = __ldcs(reinterpret_cast<const uint32_t *>(row + c.first));
            if (c.two) v.y = __ldcs(reinterpret_cast<const uint32_t *>(row + c.second));
        }
    }
    return v;
}
template <uint32_t FORMAT, bool F32>
__device__ __forceinline__ void put_cached(uint8_t *row, const Columns &c, const uint4 &v) {
    if constexpr (FORMAT == FE2O3_KV_BF16) {
        if constexpr (!F32) {
            if (c.one) *reinterpret_cast<uint4 *>(row + 2 * c.first) = v;
        } else {
            if (c.one) *reinterpret_cast<uint2 *>(row + 2 * c.first) = make_uint2(v.x, v.y);
            if (c.two) *reinterpret_cast<uint2 *>(row + 2 * c.second) = make_uint2(v.z, v.w);
        }
    } else {
        if constexpr (!F32) {
            if (c.one) *reinterpret_cast<uint2 *>(row + c.first) = make_uint2(v.x, v.y);
        } else {
            if (c.one) *reinterpret_cast<uint32_t *>(row + c.first) = v.x;
            if (c.two) *reinterpret_cast<uint32_t *>(row + c.second) = v.y;
        }
    }
}

template <int LANES>
__device__ __forceinline__ uint32_t highest(uint32_t v) {
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) v = max(v, __shfl_xor_sync(~0u, v, o));
    return v;
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

// WHOLE: the caller's rows start on 16 bytes.
template <uint32_t FORMAT, bool F32, bool WRITE, bool WHOLE>
__global__ void __launch_bounds__(kThreads) kv_rows_kernel(KvCache c, KvRows r) {
    __shared__ uint32_t slots[kTokens];
    __shared__ uint32_t known;   // tokens whose lengths allow a slot, a bit each
    constexpr uint32_t kEb = F32 ? 4 : 2;
    begin_after_previous();
    const uint32_t t0 = blockIdx.x * r.per_block, n = min(r.per_block, r.tokens - t0), lane = threadIdx.x & 31;
    if (threadIdx.x < 32) {
        uint32_t row = ~0u;
        const uint32_t ok = __ballot_sync(~0u, slot_of(c, r, t0, n, row));
        slots[lane] = row;
        if (lane == 0) known = ok;
    }
    __syncthreads();
    const uint32_t lanes = 1u << r.lanes_log2, at_once = kThreads >> r.lanes_log2, l = threadIdx.x & (lanes - 1);
    const Columns columns = F32 ? Columns{4 * l, 4 * (lanes + l), 4 * l < c.dim, 4 * (lanes + l) < c.dim} : Columns{8 * l, 0, 8 * l < c.dim, false};
    const uint32_t rows = n * 2 * c.kv_heads;
    for (uint32_t base = 0; base < rows; base += kDeep * at_once) {
        const uint32_t first = base + (threadIdx.x >> r.lanes_log2);
        uint4 raw[kDeep][2];
        float scales[kDeep];
        uint32_t at[kDeep], side[kDeep];
        uint8_t *there[kDeep];
        bool active[kDeep];
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            active[d] = false;
            if (base + d * at_once >= rows) continue;   // (for the whole block)
            // head fastest, then K or V, then the token
            const uint32_t i = min(first + d * at_once, rows - 1), of_side = r.heads_inverse ? __umulhi(i, r.heads_inverse) : i / c.kv_heads;
            const uint32_t h = i - of_side * c.kv_heads, token = of_side >> 1, slot = slots[token];
            side[d] = of_side & 1;
            at[d] = slot == ~0u ? ~0u : slot + h * c.page_size;
            active[d] = first + d * at_once < rows && (known >> token & 1) && (slot != ~0u || !WRITE);
            there[d] = (side[d] ? r.v : r.k) + ((uint64_t)(t0 + token) * (side[d] ? r.v_token_stride : r.k_token_stride) +
                                                (uint64_t)h * (side[d] ? r.v_head_stride : r.k_head_stride)) * kEb;
            raw[d][0] = raw[d][1] = make_uint4(0, 0, 0, 0);
            scales[d] = 0.f;
            if (!active[d]) continue;
            if constexpr (WRITE) {
                fetch<F32, WHOLE>(there[d], columns, raw[d]);
            } else if (slot != ~0u) {
                raw[d][0] = fetch_cached<FORMAT, F32>((side[d] ? c.v : c.k) + (uint64_t)at[d] * c.dim * kKvBytes<FORMAT>, columns);
                if constexpr (FORMAT != FE2O3_KV_BF16) scales[d] = (side[d] ? c.v_scales : c.k_scales)[at[d]];
            }
        }
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            if (base + d * at_once >= rows) break;
            if constexpr (FORMAT == FE2O3_KV_BF16 && !F32) {   // as it is
                if (!active[d]) continue;
                if constexpr (WRITE) put_cached<FORMAT, F32>((side[d] ? c.v : c.k) + (uint64_t)at[d] * c.dim * 2, columns, raw[d][0]);
                else put<F32, WHOLE>(there[d], columns, raw[d]);
                continue;
            }
            float x[8];
            if constexpr (WRITE) {
                uint8_t *const to = (side[d] ? c.v : c.k) + (uint64_t)at[d] * c.dim * kKvBytes<FORMAT>;
                // the largest magnitude as bits: an infinity or a NaN is above every number
                uint32_t top = 0;
                if constexpr (F32) {
                    const uint32_t w[8] = {raw[d][0].x, raw[d][0].y, raw[d][0].z, raw[d][0].w, raw[d][1].x, raw[d][1].y, raw[d][1].z, raw[d][1].w};
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        x[i] = __uint_as_float(w[i]);
                        top = max(top, w[i] & 0x7fffffffu);
                    }
                } else {
                    widen4(make_uint2(raw[d][0].x, raw[d][0].y), x);
                    widen4(make_uint2(raw[d][0].z, raw[d][0].w), x + 4);
                    const uint32_t pairs = __vmaxu2(__vmaxu2(raw[d][0].x & 0x7fff7fffu, raw[d][0].y & 0x7fff7fffu),
                                                    __vmaxu2(raw[d][0].z & 0x7fff7fffu, raw[d][0].w & 0x7fff7fffu));
                    top = max(pairs << 16, pairs & 0xffff0000u);
                }
                if constexpr (FORMAT == FE2O3_KV_BF16) {
                    if (active[d]) put_cached<FORMAT, F32>(to, columns, joined(narrow4(x), narrow4(x + 4)));
                } else {
                    if (lanes == 16) top = highest<16>(top);   // (unrolled for the usual rows)
                    else if (lanes == 8) top = highest<8>(top);
                    else
                        for (uint32_t o = 1; o < lanes; o <<= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
                    const float scale = top < 0x7f800000u ? scale_of<FORMAT>(__uint_as_float(top)) : __uint_as_float(0x7fc00000u);
                    float q[8];
                    quotients(x, scale, q);
                    if (active[d]) {
                        const uint2 w = codes_of<FORMAT>(q);
                        put_cached<FORMAT, F32>(to, columns, make_uint4(w.x, w.y, 0, 0));
                        if (l == 0) (side[d] ? c.v_scales : c.k_scales)[at[d]] = scale;
                    }
                }
            } else {
                if constexpr (FORMAT == FE2O3_KV_BF16) {
                    widen4(make_uint2(raw[d][0].x, raw[d][0].y), x);
                    widen4(make_uint2(raw[d][0].z, raw[d][0].w), x + 4);
                } else {
                    values_of<FORMAT>(make_uint2(raw[d][0].x, raw[d][0].y), scales[d], x);
                }
                uint4 v[2];
                if constexpr (F32) {
                    v[0] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
                    v[1] = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
                } else {
                    v[0] = joined(narrow4(x), narrow4(x + 4));
                }
                if (active[d]) put<F32, WHOLE>(there[d], columns, v);
            }
        }
    }
}

using Kernel = void (*)(KvCache, KvRows);

template <typename Args>
int32_t launch_rows(fe2o3_ctx *ctx, cudaStream_t s, const Args *a, uint32_t dtype, fe2o3_geometry *geo, bool plan_only,
                    const Kernel (&kernels)[3][2][2], const char *what) {
    // tokens of a block: up to a warp's lanes, and blocks that fill the SMs a whole number of times
    const uint32_t eb = dtype == FE2O3_DTYPE_F32 ? 4 : 2;
    const uint64_t odd = a->k.ptr | a->v.ptr | (uint64_t)a->k_token_stride * eb | (uint64_t)a->v_token_stride * eb | (uint64_t)a->k_head_stride * eb | (uint64_t)a->v_head_stride * eb;
    static std::atomic<int> per_sm[3][2][2];   // of each kernel, found once
    const int i = dtype == FE2O3_DTYPE_F32, whole = odd % 16 == 0;
    int fit = per_sm[a->format][i][whole].load(std::memory_order_relaxed);
    if (fit == 0) {
        const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kernels[a->format][i][whole], kThreads, 0);
        if (e != cudaSuccess) return fe2o3_cuda_status(e, what);
        if (fit < 1) fit = 1;
        per_sm[a->format][i][whole].store(fit, std::memory_order_relaxed);
    }
    const uint64_t resident = (uint64_t)fit * (ctx->sm_count > 0 ? ctx->sm_count : 1);
    const uint64_t waves = (a->tokens + resident * kTokens - 1) / (resident * kTokens);
    const uint32_t per_block = a->tokens ? ceil_div_u32(a->tokens, resident * waves) : 1;
    const uint32_t grid = ceil_div_u32(a->tokens, per_block);
    if (geo) *geo = fe2o3_geometry{{grid, 1, 1}, {kThreads, 1, 1}, 0, 1};
    if (plan_only || a->tokens == 0) return FE2O3_OK;
    uint32_t lanes_log2 = 1;
    while ((8u << lanes_log2) < a->dim) ++lanes_log2;
    const KvRows r{reinterpret_cast<uint8_t *>(a->k.ptr), reinterpret_cast<uint8_t *>(a->v.ptr), a->k_token_stride, a->v_token_stride,
                   a->k_head_stride, a->v_head_stride, reinterpret_cast<const uint32_t *>(a->token_offsets.ptr), a->tokens, per_block, lanes_log2,
                   // exact for the indexes of a block, below 64 kv_heads
                   a->kv_heads == 1 || a->kv_heads > 4096 ? 0 : (uint32_t)((0x100000000ull + a->kv_heads - 1) / a->kv_heads)};
    const cudaError_t e = fe2o3_launch_early(kernels[a->format][i][whole], grid, kThreads, 0, s, 1, kv_cache_of(ctx, a), r);
    fe2o3_count_launch(1);
    return fe2o3_cuda_status(e, what);
}

}  // namespace

#define KV_FORMAT(FORMAT, WRITE)                                                                                                     \
    {{kv_rows_kernel<FORMAT, false, WRITE, false>, kv_rows_kernel<FORMAT, false, WRITE, true>},                                      \
     {kv_rows_kernel<FORMAT, true, WRITE, false>, kv_rows_kernel<FORMAT, true, WRITE, true>}}
#define KV_FORMATS(WRITE) {KV_FORMAT(FE2O3_KV_BF16, WRITE), KV_FORMAT(FE2O3_KV_E4M3, WRITE), KV_FORMAT(FE2O3_KV_I8, WRITE)}
int32_t launch_kv_cache_append(fe2o3_ctx *ctx, cudaStream_t s, const void *args, fe2o3_geometry *geo, bool plan_only) {
    static const Kernel kernels[3][2][2] = KV_FORMATS(true);
    const fe2o3_kv_cache_append_v1_args *a = static_cast<const fe2o3_kv_cache_append_v1_args *>(args);
    return launch_rows(ctx, s, a, a->input_dtype, geo, plan_only, kernels, "kv_cache_append_v1");
}
int32_t launch_kv_cache_read(fe2o3_ctx *ctx, cudaStream_t s, const void *args, fe2o3_geometry *geo, bool plan_only) {
    static const Kernel kernels[3][2][2] = KV_FORMATS(false);
    const fe2o3_kv_cache_read_v1_args *a = static_cast<const fe2o3_kv_cache_read_v1_args *>(args);
    return launch_rows(ctx, s, a, a->output_dtype, geo, plan_only, kernels, "kv_cache_read_v1");
}

static Fe2o3KernelRegistration reg_append("kv_cache_append_v1", reinterpret_cast<const void *>(kv_rows_kernel<0, false, true, true>));
static Fe2o3KernelRegistration reg_read("kv_cache_read_v1", reinterpret_cast<const void *>(kv_rows_kernel<0, false, false, true>));
