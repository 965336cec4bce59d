// Paged key-value cache: new rows written (rounded or quantised) and rows read back.  The formulas stand at
// fe2o3_kv_cache_append_v1_args and fe2o3_kv_cache_read_v1_args.
//
// HBM-bound: each element is read once and written once.  A row is pieces of 16 bytes of the caller's, two to each of 2 to 32
// lanes (the second as far on as there are lanes, so that neither leaves gaps between lanes: a store of every other 16 bytes costs
// half as much again); a row's largest magnitude is a shuffle tree.  Two pieces and not one: what a row costs a lane by itself
// (its place, the tree, scale and reciprocal) is shared by 16 bf16 columns and not by 8 (to e4m3 32 -> 24 us, as it is 27 -> 26).
// Rows that do not start on 16 bytes are read or written element by element.  A block takes up to kTokens tokens, all
// their heads, K and V: one warp finds their slots (offsets, lengths and page table: three trips to memory a block, not a
// row), and each lane has kDeep rows in flight.  Blocks are as many as fill the SMs a whole number of times.
// 131072 tokens of 8 heads of 128 read from bf16 pages 168 us (6.4 TB/s); 16384 tokens bf16 to e4m3 24 us (4.2 TB/s; from f32
// 37 us, 4.6 TB/s) and back to f32 34 us (4.9 TB/s); 256 new tokens 3.0 us, an empty launch's time.
// Quantisation needs the quotients as IEEE rounds them; it fills 59 % of the issue slots and 33 % of the DRAM's cycles, and what lies
// between is one wave's beginning (slots, then rows) and a row's chain of maximum, scale and quotients.  One reciprocal a row gives y, that
// of the scale rounded to nearest; q = x y, corrected twice by q + (x - q scale) y (both with a minus), is the correctly rounded
// quotient (Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, 1990) while nothing
// leaves the normal range: scales outside 2^+-60 take the division itself.
#include <atomic>

#include "kv_rows.cuh"

namespace {

constexpr int kThreads = 256, kTokens = 32;

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

// A lane's columns: two pieces of 16 bytes of the caller's row, piece l and piece lanes + l.
struct Columns {
    uint32_t first[2];
    bool inside[2];
};

// WHOLE: the caller's rows start on 16 bytes.
template <uint32_t FORMAT, bool F32, bool WRITE, bool WHOLE>
__global__ void __launch_bounds__(kThreads) kv_rows_kernel(KvCache c, KvRows r) {
    __shared__ uint32_t slots[kTokens];
    __shared__ uint32_t known;   // tokens whose lengths allow a slot, a bit each
    constexpr int kEb = F32 ? 4 : 2, kPiece = 16 / kEb, kCached = kv_bytes<FORMAT>(kPiece);   // a piece: columns, bytes in the cache
    // rows a lane has in flight: two where it quantises (registers: three take 55 us where two take 52, to e4m3 and back), else four
    constexpr int kDeep = WRITE && FORMAT != FE2O3_KV_BF16 ? 2 : 4;
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
    const Columns columns{{kPiece * l, kPiece * (lanes + l)}, {kPiece * l < c.dim, kPiece * (lanes + l) < c.dim}};
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
            const uint8_t *const from = WRITE ? there[d] : (side[d] ? c.v : c.k) + (uint64_t)at[d] * kv_bytes<FORMAT>(c.dim);
            if (!WRITE && slot == ~0u) continue;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (!columns.inside[half]) continue;
                if constexpr (WRITE) raw[d][half] = fetch<F32, WHOLE>(from + columns.first[half] * kEb);
                else raw[d][half] = fetch_cached<kCached>(from + kv_bytes<FORMAT>(columns.first[half]));
            }
            if constexpr (!WRITE && FORMAT != FE2O3_KV_BF16) scales[d] = (side[d] ? c.v_scales : c.k_scales)[at[d]];
        }
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            if (base + d * at_once >= rows) break;
            uint8_t *const to = WRITE ? (side[d] ? c.v : c.k) + (uint64_t)at[d] * kv_bytes<FORMAT>(c.dim) : there[d];
            if constexpr (WRITE && FORMAT != FE2O3_KV_BF16) {
                float x[2 * kPiece];
                uint32_t top = 0;   // the largest magnitude as bits: an infinity or a NaN is above every number
                uint32_t pairs = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint4 &v = raw[d][i / 4];
                    const uint32_t w = i % 4 == 0 ? v.x : i % 4 == 1 ? v.y : i % 4 == 2 ? v.z : v.w;
                    if constexpr (F32) {
                        x[i] = __uint_as_float(w);
                        top = max(top, w & 0x7fffffffu);
                    } else {
                        widen2(w, x + 2 * i);
                        pairs = __vmaxu2(pairs, w & 0x7fff7fffu);
                    }
                }
                if constexpr (!F32) top = max(pairs << 16, pairs & 0xffff0000u);
                if (lanes == 16) top = highest<16>(top);   // (unrolled for the usual rows)
                else if (lanes == 8) top = highest<8>(top);
                else
                    for (uint32_t o = 1; o < lanes; o <<= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
                const float scale = top < 0x7f800000u ? scale_of<FORMAT>(__uint_as_float(top)) : __uint_as_float(0x7fc00000u);
                minus_quotients<FORMAT>(x, scale);
                if (!active[d]) continue;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (!columns.inside[half]) continue;
                    const float *const q = x + half * kPiece;
                    put_cached<kCached>(to + columns.first[half], make_uint4(codes_of<FORMAT>(q), F32 ? 0 : codes_of<FORMAT>(q + kPiece - 4), 0, 0));
                }
                if (l == 0) (side[d] ? c.v_scales : c.k_scales)[at[d]] = scale;
            } else {
                if (!active[d]) continue;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (!columns.inside[half]) continue;
                    uint4 v = raw[d][half];   // (bf16 as it is)
                    if constexpr (FORMAT == FE2O3_KV_BF16 && F32 && WRITE) {
                        v = make_uint4(bf16_pair(__uint_as_float(v.x), __uint_as_float(v.y)), bf16_pair(__uint_as_float(v.z), __uint_as_float(v.w)), 0, 0);
                    } else if constexpr (FORMAT != FE2O3_KV_BF16 || F32) {
                        float x[8];
                        if constexpr (FORMAT == FE2O3_KV_BF16) {
                            widen2(v.x, x);
                            widen2(v.y, x + 2);
                        } else {
                            values_of<FORMAT>(v.x, scales[d], x);
                            if constexpr (!F32) values_of<FORMAT>(v.y, scales[d], x + 4);
                        }
                        if constexpr (F32) v = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
                        else v = make_uint4(bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]), bf16_pair(x[4], x[5]), bf16_pair(x[6], x[7]));
                    }
                    if constexpr (WRITE) put_cached<kCached>(to + kv_bytes<FORMAT>(columns.first[half]), v);
                    else put<F32, WHOLE>(to + columns.first[half] * kEb, v);
                }
            }
        }
    }
}

// ---- 4 bits ----
// Rows of 32 columns a lane (at least two lanes a row): what a row costs a lane by itself is dear beside 16 bytes of codes.  131072 tokens of 8
// heads of 128 are read into bf16 rows in 137 us (148 with the 16 columns of the other formats), of which 537 MB are written: a plain fill of as much
// takes 142.  16384 tokens from bf16 and back to f32 51 us (59 with 16 columns), 37 of it the f32 rows' way out.  A lane that writes takes two
// blocks of 16 columns, l and l + lanes, whose scales it finds by itself.  One that reads takes four words of eight columns, l and every lanes-th
// further: the stores of a row's lanes lie side by side.  (f32 ones, 32 bytes a word, by two neighbours that swap halves of their words first.)
template <bool F32, bool WRITE, bool WHOLE>
__global__ void __launch_bounds__(kThreads) kv_rows4_kernel(KvCache c, KvRows r) {
    __shared__ uint32_t slots[kTokens];
    __shared__ uint32_t known;
    constexpr int kEb = F32 ? 4 : 2, kDeep = WRITE ? (F32 ? 1 : 2) : 4, kPieces = WRITE ? kEb : 1;   // kPieces: 16 bytes each, of a block that is written
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
    const uint32_t rows = n * 2 * c.kv_heads, blocks = c.dim / 16, words = c.dim / 8;
    for (uint32_t base = 0; base < rows; base += kDeep * at_once) {
        const uint32_t first = base + (threadIdx.x >> r.lanes_log2);
        uint4 raw[WRITE ? kDeep : 1][2][kPieces];
        uint32_t code[WRITE ? 1 : kDeep][4], block[WRITE ? 1 : kDeep][4];
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
            if constexpr (WRITE) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t b = l + half * lanes;
#pragma unroll
                    for (int x = 0; x < kPieces; ++x)
                        raw[d][half][x] = active[d] && b < blocks ? fetch<F32, WHOLE>(there[d] + b * 16 * kEb + 16 * x) : make_uint4(0, 0, 0, 0);
                }
            } else {
                const uint8_t *const cache = side[d] ? c.v : c.k;
                const bool held = active[d] && slot != ~0u;
                scales[d] = held ? (side[d] ? c.v_scales : c.k_scales)[at[d]] : 0.f;
                const uint8_t *const codes = cache + (uint64_t)at[d] * (c.dim / 2), *const block_scales = cache + c.blocks + (uint64_t)at[d] * blocks;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint32_t word = l + x * lanes;
                    code[d][x] = block[d][x] = 0;
                    if (!held || word >= words) continue;
                    code[d][x] = __ldcs(reinterpret_cast<const uint32_t *>(codes) + word);
                    block[d][x] = __ldcs(block_scales + word / 2);
                }
            }
        }
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            if (base + d * at_once >= rows) break;
            if constexpr (WRITE) {
                uint32_t tops[2];   // largest magnitudes as bits: an infinity or a NaN is above every number
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t top = 0;
#pragma unroll
                    for (int x = 0; x < kPieces; ++x) {
                        const uint4 &v = raw[d][half][x];
                        if constexpr (F32) top = max(max(top, v.x & 0x7fffffffu), max(max(v.y & 0x7fffffffu, v.z & 0x7fffffffu), v.w & 0x7fffffffu));
                        else top = __vmaxu2(__vmaxu2(top, v.x & 0x7fff7fffu), __vmaxu2(__vmaxu2(v.y & 0x7fff7fffu, v.z & 0x7fff7fffu), v.w & 0x7fff7fffu));
                    }
                    tops[half] = F32 ? top : max(top << 16, top & 0xffff0000u);
                }
                uint32_t top = max(tops[0], tops[1]);
                for (uint32_t o = 1; o < lanes; o <<= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
                if (!active[d]) continue;
                float scale, up;
                row_scales4(__uint_as_float(top), scale, up);
                uint8_t *const cache = side[d] ? c.v : c.k;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t b = l + half * lanes;
                    if (b >= blocks) continue;
                    float factor;
                    const uint32_t code = block_scale4(__uint_as_float(tops[half]), scale, up, factor);
                    uint32_t w[2] = {0, 0};
#pragma unroll
                    for (int x = 0; x < kPieces; ++x) {
                        const uint32_t v[4] = {raw[d][half][x].x, raw[d][half][x].y, raw[d][half][x].z, raw[d][half][x].w};
                        float y[F32 ? 4 : 8];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if constexpr (F32) y[i] = __uint_as_float(v[i]);
                            else widen2(v[i], y + 2 * i);
                        }
                        if constexpr (F32) w[x / 2] |= codes4(y, factor) << (16 * (x & 1));
                        else w[x] = codes8(y, factor);
                    }
                    __stcs(reinterpret_cast<uint2 *>(cache + (uint64_t)at[d] * (c.dim / 2) + 8 * b), make_uint2(w[0], w[1]));
                    cache[c.blocks + (uint64_t)at[d] * blocks + b] = (uint8_t)code;
                }
                if (l == 0) (side[d] ? c.v_scales : c.k_scales)[at[d]] = scale;
            } else {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint32_t word = l + x * lanes;
                    uint32_t w = code[d][x];
                    if constexpr (F32) {   // columns 0 to 3 and 8 to 11 of the two words go to the even lane
                        const uint32_t other = __shfl_xor_sync(~0u, w, 1);
                        w = l & 1 ? __byte_perm(other, w, 0x7632) : __byte_perm(w, other, 0x5410);
                    }
                    if (!active[d] || word >= words) continue;
                    float v[8];
                    values8(w, block[d][x], scales[d], v);
                    if constexpr (F32) {
                        uint8_t *const to = there[d] + (word & ~1u) * 32 + (l & 1) * 16;
                        put<F32, WHOLE>(to, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])));
                        put<F32, WHOLE>(to + 32, make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])));
                    } else {
                        put<F32, WHOLE>(there[d] + word * 16, make_uint4(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7])));
                    }
                }
            }
        }
    }
}

using Kernel = void (*)(KvCache, KvRows);

template <typename Args>
int32_t launch_rows(fe2o3_ctx *ctx, cudaStream_t s, const Args *a, uint32_t dtype, fe2o3_geometry *geo, bool plan_only,
                    const Kernel (&kernels)[4][2][2], const char *what) {
    // tokens of a block: up to a warp's lanes, and blocks that fill the SMs a whole number of times
    const uint32_t eb = dtype == FE2O3_DTYPE_F32 ? 4 : 2;
    const uint64_t odd = a->k.ptr | a->v.ptr | (uint64_t)a->k_token_stride * eb | (uint64_t)a->v_token_stride * eb | (uint64_t)a->k_head_stride * eb | (uint64_t)a->v_head_stride * eb;
    static std::atomic<int> per_sm[4][2][2];   // of each kernel, found once
    const uint32_t format = a->format == FE2O3_KV_E2M1 ? 3 : a->format;   // in the tables
    const int i = dtype == FE2O3_DTYPE_F32, whole = odd % 16 == 0;
    int fit = per_sm[format][i][whole].load(std::memory_order_relaxed);
    if (fit == 0) {
        const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kernels[format][i][whole], kThreads, 0);
        if (e != cudaSuccess) return fe2o3_cuda_status(e, what);
        if (fit < 1) fit = 1;
        per_sm[format][i][whole].store(fit, std::memory_order_relaxed);
    }
    const uint64_t resident = (uint64_t)fit * (ctx->sm_count > 0 ? ctx->sm_count : 1);
    const uint64_t waves = (a->tokens + resident * kTokens - 1) / (resident * kTokens);
    const uint32_t per_block = a->tokens ? ceil_div_u32(a->tokens, resident * waves) : 1;
    const uint32_t grid = ceil_div_u32(a->tokens, per_block);
    if (geo) *geo = fe2o3_geometry{{grid, 1, 1}, {kThreads, 1, 1}, 0, 1};
    if (plan_only || a->tokens == 0) return FE2O3_OK;
    uint32_t lanes_log2 = 1;
    while ((format == 3 ? 32u << lanes_log2 : 32u / eb << lanes_log2) < a->dim) ++lanes_log2;
    const KvRows r{reinterpret_cast<uint8_t *>(a->k.ptr), reinterpret_cast<uint8_t *>(a->v.ptr), a->k_token_stride, a->v_token_stride,
                   a->k_head_stride, a->v_head_stride, reinterpret_cast<const uint32_t *>(a->token_offsets.ptr), a->tokens, per_block, lanes_log2,
                   // exact for the indexes of a block, below 64 kv_heads
                   a->kv_heads == 1 || a->kv_heads > 4096 ? 0 : (uint32_t)((0x100000000ull + a->kv_heads - 1) / a->kv_heads)};
    const cudaError_t e = fe2o3_launch_early(kernels[format][i][whole], grid, kThreads, 0, s, 1, kv_cache_of(ctx, a), r);
    fe2o3_count_launch(1);
    return fe2o3_cuda_status(e, what);
}

}  // namespace

#define KV_FORMAT(FORMAT, WRITE)                                                                                                     \
    {{kv_rows_kernel<FORMAT, false, WRITE, false>, kv_rows_kernel<FORMAT, false, WRITE, true>},                                      \
     {kv_rows_kernel<FORMAT, true, WRITE, false>, kv_rows_kernel<FORMAT, true, WRITE, true>}}
#define KV_FORMATS(WRITE) {KV_FORMAT(FE2O3_KV_BF16, WRITE), KV_FORMAT(FE2O3_KV_E4M3, WRITE), KV_FORMAT(FE2O3_KV_I8, WRITE), {{kv_rows4_kernel<false, WRITE, false>, kv_rows4_kernel<false, WRITE, true>}, {kv_rows4_kernel<true, WRITE, false>, kv_rows4_kernel<true, WRITE, true>}}}
int32_t launch_kv_cache_append(fe2o3_ctx *ctx, cudaStream_t s, const void *args, fe2o3_geometry *geo, bool plan_only) {
    static const Kernel kernels[4][2][2] = KV_FORMATS(true);
    const fe2o3_kv_cache_append_v1_args *a = static_cast<const fe2o3_kv_cache_append_v1_args *>(args);
    return launch_rows(ctx, s, a, a->input_dtype, geo, plan_only, kernels, "kv_cache_append_v1");
}
int32_t launch_kv_cache_read(fe2o3_ctx *ctx, cudaStream_t s, const void *args, fe2o3_geometry *geo, bool plan_only) {
    static const Kernel kernels[4][2][2] = KV_FORMATS(false);
    const fe2o3_kv_cache_read_v1_args *a = static_cast<const fe2o3_kv_cache_read_v1_args *>(args);
    return launch_rows(ctx, s, a, a->output_dtype, geo, plan_only, kernels, "kv_cache_read_v1");
}

static Fe2o3KernelRegistration reg_append("kv_cache_append_v1", reinterpret_cast<const void *>(kv_rows_kernel<0, false, true, true>));
static Fe2o3KernelRegistration reg_read("kv_cache_read_v1", reinterpret_cast<const void *>(kv_rows_kernel<0, false, false, true>));
