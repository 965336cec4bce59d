// Rotary positions: rows of q and k turned pair by pair (rotary_v1), and new tokens turned and written into the key-value cache in one
// pass (kv_cache_rotary_append_v1).  The formulas stand at fe2o3_rotary_v1_args and fe2o3_kv_cache_rotary_append_v1_args.
//
// HBM-bound: each element is read once and written once.  A block takes some tokens, all their rows or a part of them; it first
// works out the tokens' sines and cosines, once for all heads, into shared memory.  A row is pieces of 16 bytes, two to each of up to 32
// lanes: with halves as pairs the two pieces that hold them, so that a lane turns its own columns.  Where half of the turned columns is no
// whole number of pieces, the columns go through shared memory, where a lane takes a pair or two neighbouring ones.  (Partners fetched one by one
// from the first cache instead, and lanes by powers of two: 8191 tokens of 48 rows of 80 columns, 20 of them turned, 73 and 43 us where this
// takes 34; 16384 tokens of 40 rows of 128 with 100 turned, 50 pairs, 110 us with two pairs a lane at once and 142 with one.)  The first
// rows are fetched before the sines are worked out (64 tokens of 40 rows 2.7 us for 3.2).  Into a cache, 16384 tokens of 48 rows of 128: bf16 70 us (6.1 TB/s),
// e4m3, i8 and e2m1 78 (4.7 and 4.6 TB/s: the quantising chain of a row); 64 tokens 2.7 and 3.1.
// 16384 tokens, 40 rows of 128 bf16 columns: 58 us, 5.8 TB/s, 88 % of a copy's rate, neighbours as pairs 61; 1003 tokens of 24 f32 rows of 96 4.4 us.
// Angles: position times frequency has up to 56 bits.  The product p and what rounding took from it, e, are 64-bit numbers that add up
// to it exactly; n whole turns are taken off in two steps (2 pi as two 64-bit numbers), which leaves an angle in [-pi, pi] that is right
// to some 2^-50.  Its sine and cosine are those of its 32-bit rounding, and the rest of it to first order.
#include <atomic>

#include "kv_rows.cuh"

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kPlain = ~0u;   // FORMAT: no cache, q and k go to rows like theirs
constexpr uint32_t kMostTokens = 8;

struct RotaryRows {
    const uint8_t *from[3];            // q, k, v
    uint8_t *to[2];                    // of q and k
    uint32_t token_stride[3], head_stride[3], to_token_stride[2], to_head_stride[2];
    const uint32_t *positions, *slots;
    const float *frequencies;
    uint32_t tokens, heads, rows;      // rows of a token: heads, then kv_heads of k (and of v)
    uint32_t per_block, parts;         // tokens of a block; blocks that share them
    uint32_t dim, kv_heads, pairs, lanes;
    uint32_t groups, token_turns;      // pieces whose pairs lie together (see turn_at); places of a token's sines and cosines
    uint32_t rows_inverse;             // 2^32 / rows rounded up, or 0
    float scale, sign;
};

// Cosine and sine of position * frequency, times scale.
__device__ __forceinline__ float2 turn_of(uint32_t position, float frequency, float scale, float sign) {
    const double x = position, f = frequency, p = x * f, e = fma(x, f, -p);
    const double n = rint(p * 0.15915494309189535);
    const double a = fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586, p)) + e;
    const double h = a * 0.3183098861837907;   // in half turns
    const float near = (float)h, rest = (float)(h - near) * 3.14159274f;
    float s, c;
    sincospif(near, &s, &c);
    return make_float2(fmaf(-rest, s, c) * scale, fmaf(rest, c, s) * scale * sign);
}

__device__ __forceinline__ uint32_t word_of(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// A lane's columns of a row into the cache.  bf16 columns from `turned` on are as they came, bit for bit.
template <uint32_t FORMAT, int kPiece>
__device__ __forceinline__ void store_row(const KvCache &c, float (&x)[2 * kPiece], const uint4 (&raw)[2], uint32_t turned, uint32_t side, uint32_t row, const uint32_t (&first)[2], const bool (&inside)[2],
                                          uint32_t l, uint32_t lanes, bool active) {
    constexpr int kCached = kv_bytes<FORMAT>(kPiece);
    uint8_t *const base = side ? c.v : c.k, *const to = base + (uint64_t)row * kv_bytes<FORMAT>(c.dim);
    float *const scales = side ? c.v_scales : c.k_scales;
    if constexpr (FORMAT == FE2O3_KV_BF16) {
        if (!active) return;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if (!inside[half]) continue;
            const float *const q = x + half * kPiece;
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < kPiece / 2; ++i) w[i] = kPiece == 8 && first[half] + 2 * i >= turned ? word_of(raw[half], i) : bf16_pair(q[2 * i], q[2 * i + 1]);
            put_cached<kCached>(to + 2 * first[half], make_uint4(w[0], w[1], w[2], w[3]));
        }
    } else {
        uint32_t top = 0;   // the largest magnitude as bits: an infinity or a NaN is above every number
#pragma unroll
        for (int i = 0; i < 2 * kPiece; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
        for (uint32_t o = 1; o < lanes; o <<= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
        float scale;
        if constexpr (FORMAT == FE2O3_KV_E2M1) {
            float up;
            row_scales4(__uint_as_float(top), scale, up);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float *const q = x + half * kPiece;
                float m = 0.f;
#pragma unroll
                for (int i = 0; i < kPiece; ++i) m = fmaxf(m, fabsf(q[i]));
#pragma unroll
                for (int o = 1; o < 16 / kPiece; o <<= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
                float factor;
                const uint32_t block = block_scale4(m, scale, up, factor);
                if (!active || !inside[half]) continue;
                put_cached<kCached>(to + first[half] / 2, make_uint4(kPiece == 4 ? codes4(q, factor) : codes8(q, factor), 0, 0, 0));
                if (l % (16 / kPiece) == 0) base[c.blocks + ((uint64_t)row * c.dim + first[half]) / 16] = (uint8_t)block;
            }
        } else {
            scale = top < 0x7f800000u ? scale_of<FORMAT>(__uint_as_float(top)) : __uint_as_float(0x7fc00000u);
            minus_quotients<FORMAT>(x, scale);
            if (!active) return;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (!inside[half]) continue;
                const float *const q = x + half * kPiece;
                put_cached<kCached>(to + first[half], make_uint4(codes_of<FORMAT>(q), kPiece == 4 ? 0 : codes_of<FORMAT>(q + kPiece - 4), 0, 0));
            }
        }
        if (active && l == 0) scales[row] = scale;
    }
}

// How pairs lie: halves whose partners lie in pieces of their own (kPieces) or anywhere (kAnywhere), or neighbours.
enum : int { kPieces, kAnywhere, kNeighbours };

// Where the sine and cosine of pair i lie among those of a token.  A lane takes two at once, its pairs of one piece (PAIRS of them), and the
// lanes of a row take the same two of theirs at the same time: those lie side by side.
template <int MODE, int PAIRS>
__device__ __forceinline__ uint32_t turn_at(uint32_t i, uint32_t groups) {
    if constexpr (MODE == kAnywhere) return i;
    else return (i % PAIRS / 2 * groups + i / PAIRS) * 2 + (i & 1);
}

// WHOLE: the rows start on 16 bytes.
template <uint32_t FORMAT, bool F32, int MODE, bool WHOLE>
__global__ void __launch_bounds__(kThreads, MODE != kAnywhere && (FORMAT == kPlain || FORMAT == FE2O3_KV_BF16) ? 4 : 3) rotary_kernel(KvCache c, RotaryRows r) {
    constexpr int kEb = F32 ? 4 : 2, kPiece = 16 / kEb, kDeep = 2, kPairs = MODE == kNeighbours ? kPiece / 2 : kPiece;
    constexpr bool kCache = FORMAT != kPlain;
    extern __shared__ float4 table[];              // [tokens of the block][pairs]; then the rows in flight, where partners lie anywhere
    __shared__ uint32_t first_rows[kMostTokens];   // in the cache, of head 0; ~0: a token that is left out
    float2 *const turns = reinterpret_cast<float2 *>(table);
    begin_after_previous();
    const uint32_t part = blockIdx.x % r.parts, t0 = blockIdx.x / r.parts * r.per_block, n = min(r.per_block, r.tokens - t0);
    const uint32_t lanes = r.lanes, of_warp = 32 / lanes, at_once = kThreads / 32 * of_warp, in_warp = (threadIdx.x & 31) / lanes, l = (threadIdx.x & 31) - in_warp * lanes;
    const uint32_t mine = (threadIdx.x >> 5) * of_warp + in_warp;   // of the rows at once
    // a lane's columns: two pieces, the partners of one another where pairs allow
    const uint32_t pieces = r.dim / kPiece, paired = MODE == kPieces ? r.groups : 0, rest = (pieces - 2 * paired) / 2;   // rest: half of the other pieces
    const bool pair = l < paired, in = l < pieces / 2 && in_warp < of_warp;   // (lanes left over have none)
    const uint32_t first[2] = {kPiece * (pair ? l : paired + l), kPiece * (pair ? l + paired : paired + l + rest)};
    const bool inside[2] = {in, in};
    float *const scratch = reinterpret_cast<float *>(turns + (uint64_t)r.per_block * r.token_turns) + mine * kDeep * r.dim;
    const uint32_t total = n * r.rows, share = (total + r.parts - 1) / r.parts, end = min(total, (part + 1) * share);
    uint4 raw[kDeep][2];
    uint32_t token[kDeep], head[kDeep], what[kDeep];
    bool there[kDeep];
    auto load = [&](uint32_t base) {
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            const uint32_t i = min(base + mine + d * at_once, end - 1);
            token[d] = r.rows_inverse ? __umulhi(i, r.rows_inverse) : i / r.rows;
            head[d] = i - token[d] * r.rows;
            what[d] = head[d] < r.heads ? 0 : 1;
            if (what[d]) head[d] -= r.heads;
            if (kCache && what[d] && head[d] >= r.kv_heads) {
                what[d] = 2;
                head[d] -= r.kv_heads;
            }
            there[d] = base + mine + d * at_once < end;
            raw[d][0] = raw[d][1] = make_uint4(0, 0, 0, 0);
            if (there[d] && in) {
                const uint32_t ts = what[d] == 0 ? r.token_stride[0] : what[d] == 1 ? r.token_stride[1] : r.token_stride[2];
                const uint32_t hs = what[d] == 0 ? r.head_stride[0] : what[d] == 1 ? r.head_stride[1] : r.head_stride[2];
                const uint8_t *const at = (what[d] == 0 ? r.from[0] : what[d] == 1 ? r.from[1] : r.from[2]) + ((uint64_t)(t0 + token[d]) * ts + (uint64_t)head[d] * hs) * kEb;
#pragma unroll
                for (int half = 0; half < 2; ++half) raw[d][half] = fetch<F32, WHOLE>(at + first[half] * kEb);
            }
        }
    };
    // (the first rows are on their way while the sines are worked out; those of a token that is left out as well, for nothing)
    if (part * share < end) load(part * share);
    if (kCache && threadIdx.x < n) {
        const uint32_t slot = r.slots[t0 + threadIdx.x], page = slot / c.page_size;
        const bool there = page < c.pages;
        if (!there && slot != FE2O3_SLOT_NONE) kstatus_set(c.status, FE2O3_KSTATUS_SLOT_RANGE);
        first_rows[threadIdx.x] = there && slot != FE2O3_SLOT_NONE ? page * c.kv_heads * c.page_size + (slot - page * c.page_size) : ~0u;
    }
    for (uint32_t i = threadIdx.x; i < n * r.pairs; i += kThreads) {
        const uint32_t t = i / r.pairs, pair = i - t * r.pairs;
        turns[t * r.token_turns + turn_at<MODE, kPairs>(pair, r.groups)] = turn_of(r.positions ? r.positions[t0 + t] : t0 + t, r.frequencies[pair], r.scale, r.sign);
    }
    __syncthreads();
    for (uint32_t base = part * share; base < end;) {
        bool active[kDeep];
#pragma unroll
        for (int d = 0; d < kDeep; ++d) active[d] = there[d] && (!kCache || first_rows[token[d]] != ~0u);
        __syncwarp();   // in place: every lane has its columns before one writes
        float x[kDeep][2 * kPiece];
#pragma unroll
        for (int d = 0; d < kDeep; ++d)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t w = word_of(raw[d][i / 4], i % 4);
                if constexpr (F32) x[d][i] = __uint_as_float(w);
                else widen2(w, x[d] + 2 * i);
            }
        if constexpr (MODE == kAnywhere) {   // through shared memory, a pair a lane (a row's lanes are of one warp)
#pragma unroll
            for (int d = 0; d < kDeep; ++d)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    if (what[d] < 2 && in && first[half] < 2 * r.pairs)
#pragma unroll
                        for (int i = 0; i < kPiece; i += 4)
                            *reinterpret_cast<float4 *>(scratch + d * r.dim + first[half] + i) = *reinterpret_cast<const float4 *>(x[d] + half * kPiece + i);
            __syncwarp();
#pragma unroll
            for (int d = 0; d < kDeep; ++d) {
                if (what[d] == 2 || in_warp >= of_warp) continue;
                float *const row = scratch + d * r.dim;
                const float2 *const cs = turns + token[d] * r.token_turns;
                if (r.pairs % 2 == 0) {   // two pairs at once
                    for (uint32_t i = 2 * l; i < r.pairs; i += 2 * lanes) {
                        const float4 t = *reinterpret_cast<const float4 *>(cs + i);
                        float2 &low = *reinterpret_cast<float2 *>(row + i), &high = *reinterpret_cast<float2 *>(row + i + r.pairs);
                        const float2 a = low, b = high;
                        low = make_float2(fmaf(a.x, t.x, -(b.x * t.y)), fmaf(a.y, t.z, -(b.y * t.w)));
                        high = make_float2(fmaf(b.x, t.x, a.x * t.y), fmaf(b.y, t.z, a.y * t.w));
                    }
                    continue;
                }
                for (uint32_t i = l; i < r.pairs; i += lanes) {
                    const float2 t = cs[i];
                    const float a = row[i], b = row[i + r.pairs];
                    row[i] = fmaf(a, t.x, -(b * t.y));
                    row[i + r.pairs] = fmaf(b, t.x, a * t.y);
                }
            }
            __syncwarp();
#pragma unroll
            for (int d = 0; d < kDeep; ++d)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    if (what[d] < 2 && in && first[half] < 2 * r.pairs)
#pragma unroll
                        for (int i = 0; i < kPiece; i += 4)
                            *reinterpret_cast<float4 *>(x[d] + half * kPiece + i) = *reinterpret_cast<const float4 *>(scratch + d * r.dim + first[half] + i);
        }
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            if (base + d * at_once >= end) continue;   // (for the whole block)
            const uint32_t turned = what[d] < 2 ? 2 * r.pairs : 0;
            const float2 *const cs = turns + token[d] * r.token_turns;
            if (MODE == kPieces && turned && pair) {
#pragma unroll
                for (int i = 0; i < kPiece; i += 2) {
                    const float4 t = reinterpret_cast<const float4 *>(cs)[i / 2 * r.groups + l];
                    const float a = x[d][i], b = x[d][kPiece + i], a1 = x[d][i + 1], b1 = x[d][kPiece + i + 1];
                    x[d][i] = fmaf(a, t.x, -(b * t.y));
                    x[d][kPiece + i] = fmaf(b, t.x, a * t.y);
                    x[d][i + 1] = fmaf(a1, t.z, -(b1 * t.w));
                    x[d][kPiece + i + 1] = fmaf(b1, t.z, a1 * t.w);
                }
            }
            if (MODE == kNeighbours && in) {
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int i = 0; i < kPiece; i += 4) {
                        if (first[half] + i >= turned) continue;   // (turned columns end with a pair, the second of two or the first)
                        const float4 t = reinterpret_cast<const float4 *>(cs)[i / 4 * r.groups + first[half] / kPiece];
                        float *const y = x[d] + half * kPiece + i;
                        const float a = y[0], b = y[1], a1 = y[2], b1 = y[3];
                        y[0] = fmaf(a, t.x, -(b * t.y));
                        y[1] = fmaf(b, t.x, a * t.y);
                        if (first[half] + i + 2 >= turned) continue;
                        y[2] = fmaf(a1, t.z, -(b1 * t.w));
                        y[3] = fmaf(b1, t.z, a1 * t.w);
                    }
            }
            const bool cached = kCache && what[d];
            if (!cached && active[d] && in) {
                const uint32_t ts = !kCache && what[d] ? r.to_token_stride[1] : r.to_token_stride[0], hs = !kCache && what[d] ? r.to_head_stride[1] : r.to_head_stride[0];
                uint8_t *const to = (!kCache && what[d] ? r.to[1] : r.to[0]) + ((uint64_t)(t0 + token[d]) * ts + (uint64_t)head[d] * hs) * kEb;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float *const q = x[d] + half * kPiece;
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (F32) w[i] = __float_as_uint(q[i]);
                        else w[i] = first[half] + 2 * i >= turned ? word_of(raw[d][half], i) : bf16_pair(q[2 * i], q[2 * i + 1]);
                    }
                    put<F32, WHOLE>(to + first[half] * kEb, make_uint4(w[0], w[1], w[2], w[3]));
                }
            }
            if constexpr (kCache) {
                // (a row's largest magnitudes go round the whole warp, whose other rows may be queries: all lanes go along, or none)
                if (FORMAT == FE2O3_KV_BF16 ? cached : __any_sync(~0u, cached)) {
                    const uint32_t row = first_rows[token[d]] + head[d] * c.page_size;
                    store_row<FORMAT, kPiece>(c, x[d], raw[d], turned, what[d] == 2, row, first, inside, l, lanes, cached && active[d] && in);
                }
            }
        }
        base += kDeep * at_once;
        if (base < end) load(base);
    }
}

using Kernel = void (*)(KvCache, RotaryRows);

// kernels: [MODE][WHOLE] of the types at hand.
int32_t launch_rows(fe2o3_ctx *ctx, cudaStream_t s, const Kernel (&kernels)[3][2], bool whole, bool interleaved, uint32_t eb, bool quantised, bool four, const KvCache &c, RotaryRows r,
                    std::atomic<int> (&per_sm)[3][2], fe2o3_geometry *geo, bool plan_only, const char *what) {
    const uint32_t piece = 16 / eb;
    // Partners lie in pieces of their own where half of the turned columns is a whole number of pieces (4 bits: of blocks, which stay with
    // neighbouring lanes).
    const int mode = interleaved ? kNeighbours : r.pairs % (four ? 16 : piece) == 0 ? kPieces : kAnywhere;
    r.groups = mode == kNeighbours ? (2 * r.pairs + piece - 1) / piece : mode == kPieces ? r.pairs / piece : 0;
    r.token_turns = mode == kNeighbours ? r.groups * (piece / 2) : (r.pairs + 1) & ~1u;
    r.lanes = r.dim / (2 * piece);   // 1 to 32; where a row's magnitudes are compared, a power of two
    if (quantised) {
        uint32_t lanes = 2;
        while (lanes < r.lanes) lanes *= 2;
        r.lanes = lanes;
    }
    int fit = per_sm[mode][whole].load(std::memory_order_relaxed);
    if (fit == 0) {
        const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kernels[mode][whole], kThreads, mode == kAnywhere ? 20480 : 4096);   // (about)
        if (e != cudaSuccess) return fe2o3_cuda_status(e, what);
        if (fit < 1) fit = 1;
        per_sm[mode][whole].store(fit, std::memory_order_relaxed);
    }
    const uint32_t at_once = kThreads / 32 * (32 / r.lanes);   // rows
    const uint32_t resident = (ctx->sm_count > 0 ? ctx->sm_count : 1) * fit;
    r.per_block = 1;
    r.parts = 1;
    if (r.tokens >= resident) {
        const uint64_t waves = (r.tokens + (uint64_t)resident * kMostTokens - 1) / ((uint64_t)resident * kMostTokens);
        r.per_block = ceil_div_u32(r.tokens, resident * waves);
    } else if (r.tokens) {
        const uint32_t rounds = ceil_div_u32(r.rows, at_once);   // of a token's rows
        r.parts = resident / r.tokens < rounds ? resident / r.tokens : rounds;
        if (r.parts == 0) r.parts = 1;
    }
    r.rows_inverse = r.rows <= 1 || (uint64_t)r.per_block * r.rows > 65536 || r.rows > 65536 ? 0 : (uint32_t)((0x100000000ull + r.rows - 1) / r.rows);
    const uint32_t in_flight = mode == kAnywhere ? at_once * 2 * r.dim * 4 : 0;   // at most 32 KiB
    const uint32_t grid = ceil_div_u32(r.tokens, r.per_block) * r.parts, shared = r.per_block * r.token_turns * (uint32_t)sizeof(float2) + in_flight;
    if (geo) *geo = fe2o3_geometry{{grid, 1, 1}, {kThreads, 1, 1}, shared, 1};
    if (plan_only || r.tokens == 0 || r.rows == 0) return FE2O3_OK;
    const cudaError_t e = fe2o3_launch_early(kernels[mode][whole], grid, kThreads, shared, s, 1, c, r);
    fe2o3_count_launch(1);
    return fe2o3_cuda_status(e, what);
}

template <typename... P>
bool on_16(uint64_t bits, P... strides) { return ((bits | ... | strides) & 15u) == 0; }

}  // namespace

#define ROTARY_MODES(FORMAT, F32)                                                                                        \
    {{rotary_kernel<FORMAT, F32, kPieces, false>, rotary_kernel<FORMAT, F32, kPieces, true>},                            \
     {rotary_kernel<FORMAT, F32, kAnywhere, false>, rotary_kernel<FORMAT, F32, kAnywhere, true>},                        \
     {rotary_kernel<FORMAT, F32, kNeighbours, false>, rotary_kernel<FORMAT, F32, kNeighbours, true>}}
#define ROTARY_FORMAT(FORMAT) {ROTARY_MODES(FORMAT, false), ROTARY_MODES(FORMAT, true)}

int32_t launch_rotary(fe2o3_ctx *ctx, cudaStream_t s, const void *args, fe2o3_geometry *geo, bool plan_only) {
    static const Kernel kernels[2][3][2] = ROTARY_FORMAT(kPlain);
    static std::atomic<int> per_sm[2][3][2];
    const fe2o3_rotary_v1_args *a = static_cast<const fe2o3_rotary_v1_args *>(args);
    const uint64_t eb = a->dtype == FE2O3_DTYPE_F32 ? 4 : 2;
    RotaryRows r{};
    r.from[0] = reinterpret_cast<const uint8_t *>(a->q.ptr);
    r.from[1] = reinterpret_cast<const uint8_t *>(a->k.ptr);
    r.to[0] = reinterpret_cast<uint8_t *>(a->q_output.ptr);
    r.to[1] = reinterpret_cast<uint8_t *>(a->k_output.ptr);
    r.token_stride[0] = a->q_token_stride, r.token_stride[1] = a->k_token_stride;
    r.head_stride[0] = a->q_head_stride, r.head_stride[1] = a->k_head_stride;
    r.to_token_stride[0] = a->q_output_token_stride, r.to_token_stride[1] = a->k_output_token_stride;
    r.to_head_stride[0] = a->q_output_head_stride, r.to_head_stride[1] = a->k_output_head_stride;
    r.positions = reinterpret_cast<const uint32_t *>(a->positions.ptr);
    r.frequencies = reinterpret_cast<const float *>(a->frequencies.ptr);
    r.tokens = a->tokens;
    r.heads = a->heads;
    r.kv_heads = a->kv_heads;
    r.rows = a->heads + a->kv_heads;
    r.dim = a->dim;
    r.pairs = a->rotary_dim / 2;
    r.scale = a->scale;
    r.sign = a->backward ? -1.f : 1.f;
    bool whole = true;
    if (a->heads) whole = on_16(a->q.ptr | a->q_output.ptr, eb * a->q_token_stride, eb * a->q_head_stride, eb * a->q_output_token_stride, eb * a->q_output_head_stride);
    if (a->kv_heads) whole = whole && on_16(a->k.ptr | a->k_output.ptr, eb * a->k_token_stride, eb * a->k_head_stride, eb * a->k_output_token_stride, eb * a->k_output_head_stride);
    return launch_rows(ctx, s, kernels[eb == 4], whole, a->layout == FE2O3_ROTARY_INTERLEAVED, (uint32_t)eb, false, false, KvCache{}, r, per_sm[eb == 4], geo, plan_only, "rotary_v1");
}

int32_t launch_kv_cache_rotary_append(fe2o3_ctx *ctx, cudaStream_t s, const void *args, fe2o3_geometry *geo, bool plan_only) {
    static const Kernel kernels[4][2][3][2] = {ROTARY_FORMAT(FE2O3_KV_BF16), ROTARY_FORMAT(FE2O3_KV_E4M3), ROTARY_FORMAT(FE2O3_KV_I8), ROTARY_FORMAT(FE2O3_KV_E2M1)};
    static std::atomic<int> per_sm[4][2][3][2];   // of each kernel, found once
    const fe2o3_kv_cache_rotary_append_v1_args *a = static_cast<const fe2o3_kv_cache_rotary_append_v1_args *>(args);
    const uint64_t eb = a->input_dtype == FE2O3_DTYPE_F32 ? 4 : 2;
    const bool four = a->format == FE2O3_KV_E2M1;
    RotaryRows r{};
    r.from[0] = reinterpret_cast<const uint8_t *>(a->q.ptr);
    r.from[1] = reinterpret_cast<const uint8_t *>(a->k.ptr);
    r.from[2] = reinterpret_cast<const uint8_t *>(a->v.ptr);
    r.to[0] = reinterpret_cast<uint8_t *>(a->q_output.ptr);
    r.token_stride[0] = a->q_token_stride, r.token_stride[1] = a->k_token_stride, r.token_stride[2] = a->v_token_stride;
    r.head_stride[0] = a->q_head_stride, r.head_stride[1] = a->k_head_stride, r.head_stride[2] = a->v_head_stride;
    r.to_token_stride[0] = a->q_output_token_stride;
    r.to_head_stride[0] = a->q_output_head_stride;
    r.positions = reinterpret_cast<const uint32_t *>(a->positions.ptr);
    r.slots = reinterpret_cast<const uint32_t *>(a->slots.ptr);
    r.frequencies = reinterpret_cast<const float *>(a->frequencies.ptr);
    r.tokens = a->tokens;
    r.heads = a->heads;
    r.kv_heads = a->kv_heads;
    r.rows = a->heads + 2 * a->kv_heads;
    r.dim = a->dim;
    r.pairs = a->rotary_dim / 2;
    r.scale = a->scale;
    r.sign = 1.f;
    bool whole = on_16(a->k.ptr | a->v.ptr, eb * a->k_token_stride, eb * a->k_head_stride, eb * a->v_token_stride, eb * a->v_head_stride);
    if (a->heads) whole = whole && on_16(a->q.ptr | a->q_output.ptr, eb * a->q_token_stride, eb * a->q_head_stride, eb * a->q_output_token_stride, eb * a->q_output_head_stride);
    const uint32_t format = four ? 3 : a->format;   // in the tables
    return launch_rows(ctx, s, kernels[format][eb == 4], whole, a->layout == FE2O3_ROTARY_INTERLEAVED, (uint32_t)eb, a->format != FE2O3_KV_BF16, four, kv_storage_of(ctx, a), r, per_sm[format][eb == 4], geo, plan_only, "kv_cache_rotary_append_v1");
}

static Fe2o3KernelRegistration reg_rotary("rotary_v1", reinterpret_cast<const void *>(rotary_kernel<kPlain, false, kPieces, true>));
static Fe2o3KernelRegistration reg_rotary_append("kv_cache_rotary_append_v1", reinterpret_cast<const void *>(rotary_kernel<FE2O3_KV_BF16, false, kPieces, true>));
