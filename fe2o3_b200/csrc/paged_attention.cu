// Attention of one new token a sequence over a paged key-value cache; the formulas stand at
// fe2o3_paged_attention_v1_args.
//
// HBM-bound: the K and V rows of a (sequence, key head) are read once, for all query heads that share them (4 * group
// flop a byte of a bf16 cache, 8 * group of an 8-bit one).
//   Work.  An item is a (sequence, key head, up to 8 * NT query heads); its keys fall into tiles of KT.  All tiles of all
//   items form one line, cut into equal shares, one a block: the lengths are known on the device only, and a launch is the
//   same whatever they are.  A block's share covers whole items and at most two pieces of items that other blocks work
//   on too.  Pieces are left in the workspace, and the block that comes last to an item (a counter) joins them in
//   their order: the same bits whoever is last.
//   Tiles.  Each warp has a ring of stages of its own, filled by 16-byte asynchronous copies row by row through the
//   page table (any page size; rows outside the sequence are filled with zeros and never read), so that nothing but
//   its own copies stops a warp between the ends of items.  The warps of a block take its tiles in turn and each keeps
//   the maximum, the sum and the output of what it has seen (one pass, f32); at an item's end they are added up in
//   pairs through shared memory, lane for lane.
//   Products.  mma.sync with the keys (and then the output's columns) as rows and the query heads as columns: of
//   the 8 columns of a tile few are wasted for small groups, and P is turned into an operand by movmatrix.  The
//   tensor unit's own sums span one tile, longer ones are f32 additions.  A bf16 cache is multiplied as it is, with the
//   probabilities as three bf16 terms that add up to the f32 value exactly (two for a bf16 output) and an f32 query as
//   three as well.  Terms are cut off, not rounded, and held above 0, so that an infinity in V stays one.  8-bit
//   codes become f16 exactly; the probabilities then carry the row's scale, against a power of two that follows the
//   largest scale seen, and are two f16 terms (22 bits); queries are brought
//   to f16's range by a power of two a row.
#include <new>

#include "kv_cache.cuh"

namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kQueryExponent = 14;   // f16 queries: the largest of a row lies in [2^14, 2^15)

struct PagedArgs {
    KvCache c;
    const void *q;
    void *o;
    float *lse;
    float4 *slots;        // two partial results a block
    uint32_t *arrived;    // pieces that have come in, by the block where the item begins; zero between launches
    uint32_t group, chunks, q_stride, q_head_stride, window, stages;
    float scale;
    bool q_f32, o_f32;
};

template <uint32_t FORMAT, int DP, int NT>
struct Shape {
    static constexpr bool kF16 = FORMAT != FE2O3_KV_BF16;
    static constexpr int kRow = DP * (kF16 ? 1 : 2);                                        // bytes of a row in a stage
    static constexpr int kKeys = kF16 ? (DP == 256 ? 16 : 32) : (DP == 64 ? 32 : 16);       // of a tile
    static constexpr int kStage = 2 * kKeys * kRow + (kF16 ? 8 * kKeys : 0);                // K, V, their scales
    static constexpr int kHeads = 8 * NT;
    static constexpr int kQueryRow = 2 * DP + 16;                                           // bytes, padded against bank conflicts
    static constexpr int kPart = (DP / 16 + 1) * NT;                                        // float4 a lane of a partial result
    static constexpr int query_bytes(int terms) { return terms * kHeads * kQueryRow; }
};

__device__ __forceinline__ void copy16(uint32_t to, const void *from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void *from, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(there ? 4u : 0u) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the youngest `behind` groups of this thread's copies have landed.
__device__ __forceinline__ void copies_wait(uint32_t behind) {
    if (behind == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (behind == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else if (behind == 3) asm volatile("cp.async.wait_group 3;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float lds_f32(uint32_t at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
// The 8x8 matrix of 16-bit values that a warp holds (row lane / 4, columns 2 (lane % 4) and the next), transposed.
__device__ __forceinline__ uint32_t turned(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <bool F16>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t f16_pair(float lo, float hi) {   // both rounded to nearest even
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 f16_values(uint32_t p) {
    float2 r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}" : "=f"(r.x), "=f"(r.y) : "r"(p));
    return r;
}
__device__ __forceinline__ float cut_bf16(float v) { return __uint_as_float(__float_as_uint(v) & 0xffff0000u); }
__device__ __forceinline__ uint32_t bf16_pair_cut(float lo, float hi) { return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632); }

// Two 8-bit codes, byte BYTE of `a` and byte BYTE + STEP of `b`, as an f16 pair: i8 exactly, e4m3 times 2^-8.
template <uint32_t FORMAT, int BYTE, int STEP>
__device__ __forceinline__ uint32_t codes_f16(uint32_t a, uint32_t b) {
    if constexpr (FORMAT == FE2O3_KV_I8) {
        // 1024 + (code + 128) has the code in its low bits: f16's step is 1 there
        const uint32_t x = __byte_perm(a, b, BYTE | (4 + BYTE + STEP) << 8);
        uint32_t r = (x & 0x00ff00ffu) ^ 0x64806480u;
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(r) : "r"(0x64806480u));
        return r;
    } else {
        // the exponent's field is one bit longer: the same bits one place lower stand for 2^(7 - 15) times the value, subnormals too
        const uint32_t x = __byte_perm(a, b, BYTE << 4 | (4 + BYTE + STEP) << 12);
        return (x & 0x80008000u) | (x >> 1 & 0x3f803f80u);
    }
}

// Where 16-byte piece c of row r lies in a stage's K or V part.  Rows that the lanes of one shared-memory access touch
// fall on different banks: 8 rows a matrix for ldmatrix; rows g, g + 1 (K) or 2t (V) for the 8-bit formats.
template <uint32_t FORMAT, int DP, bool VALUES>
__device__ __forceinline__ uint32_t piece_at(uint32_t r, uint32_t c) {
    if constexpr (FORMAT == FE2O3_KV_BF16) return r * (2 * DP) + ((c ^ (r & 7)) << 4);
    else if constexpr (DP == 64) return (r >> 1) * 128 + ((((r & 1) << 2 | c) ^ (r >> 1 & 3) << 1) << 4);
    else return r * DP + ((c ^ (VALUES ? r & 6 : (r & 1) << 2)) << 4);
}

// Column of the output that row m of tile i of the second product stands for.
template <uint32_t FORMAT, int DP>
__device__ __forceinline__ uint32_t column_of(uint32_t i, uint32_t m) {
    if constexpr (FORMAT == FE2O3_KV_BF16) return 16 * i + m;
    else return (DP == 64 ? 8 * (m & 7) : 16 * (m & 7)) + (DP == 256 ? 128 * (i >> 3) + 2 * (i & 7) : 2 * i) + (m >> 3);
}

// A sequence's keys as tiles.  One that does not fit its table is reported and has none; one tile at least, so that an
// item without keys has a block that writes its zeros.
template <int KT>
struct Span {
    uint32_t first, n, tiles;
    bool valid;
    __device__ __forceinline__ Span() {}
    __device__ __forceinline__ Span(const PagedArgs &a, uint32_t b) {
        n = a.c.lengths[b];
        valid = kv_fits(a.c, n);
        if (!valid) {
            kstatus_set(a.c.status, FE2O3_KSTATUS_LENGTH);
            n = 0;
        }
        first = a.window && n > a.window ? n - a.window : 0;
        tiles = max(1u, (n - first + KT - 1) / KT);
    }
};

// Running result of one warp over some of an item's keys: output columns (rows of tile i) by two heads a lane.
template <int MD, int NT>
struct Part {
    float m[NT][2], l[NT][2], o[MD][NT][4];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            m[t][0] = m[t][1] = -INFINITY;
            l[t][0] = l[t][1] = 0.f;
#pragma unroll
            for (int i = 0; i < MD; ++i) o[i][t][0] = o[i][t][1] = o[i][t][2] = o[i][t][3] = 0.f;
        }
    }
    // Adds another part, one float4 a lane at `at`, `at` + 32, ...
    template <typename Load>
    __device__ __forceinline__ void add(Load load) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float4 ml = load(MD * NT + t);
            const float om[2] = {ml.x, ml.y}, ol[2] = {ml.z, ml.w};
            float keep[2], take[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float top = fmaxf(m[t][e], om[e]), base = top == -INFINITY ? 0.f : top;
                keep[e] = ex2_approx(m[t][e] - base);
                take[e] = ex2_approx(om[e] - base);
                l[t][e] = l[t][e] * keep[e] + ol[e] * take[e];
                m[t][e] = top;
            }
#pragma unroll
            for (int i = 0; i < MD; ++i) {
                const float4 v = load(i * NT + t);
                o[i][t][0] = o[i][t][0] * keep[0] + v.x * take[0];
                o[i][t][1] = o[i][t][1] * keep[1] + v.y * take[1];
                o[i][t][2] = o[i][t][2] * keep[0] + v.z * take[0];
                o[i][t][3] = o[i][t][3] * keep[1] + v.w * take[1];
            }
        }
    }
    template <typename Store>
    __device__ __forceinline__ void leave(Store store) const {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            store(MD * NT + t, make_float4(m[t][0], m[t][1], l[t][0], l[t][1]));
#pragma unroll
            for (int i = 0; i < MD; ++i) store(i * NT + t, make_float4(o[i][t][0], o[i][t][1], o[i][t][2], o[i][t][3]));
        }
    }
};

template <uint32_t FORMAT, int DP, int NT>
__global__ void __launch_bounds__(kThreads) paged_attention_kernel(const PagedArgs a) {
    using S = Shape<FORMAT, DP, NT>;
    constexpr int KT = S::kKeys, MT = KT / 16, MD = DP / 16, kPieces = S::kRow / 16;
    constexpr bool F16 = S::kF16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float head_scale[S::kHeads];
    __shared__ uint32_t last_flag;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * a.stages * S::kStage;
    float4 *const parts = reinterpret_cast<float4 *>(smem + kWarps * a.stages * S::kStage);   // two of them
    uint8_t *const query = reinterpret_cast<uint8_t *>(parts + 2 * S::kPart * 32);
    const uint32_t query_s = smem_u32(query);
    const uint32_t terms = a.q_f32 ? (F16 ? 2 : 3) : 1;
    const uint32_t row_pieces = a.c.dim * (F16 ? 1 : 2) / 16;
    const uint32_t per_seq = a.c.kv_heads * a.chunks;   // items of a sequence

    begin_after_previous();

    // ---- this block's share of the line of tiles: every warp adds up the sequences' tiles for itself ----
    uint64_t total = 0;
    for (uint32_t b = lane; b < a.c.batch; b += 32) total += Span<KT>(a, b).tiles;
#pragma unroll
    for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(~0u, total, d);
    total *= per_seq;
    const uint64_t wanted = (total + 2 * kWarps - 1) / (2 * kWarps);   // a block has two tiles a warp at least
    const uint32_t blocks = wanted < gridDim.x ? (uint32_t)wanted : gridDim.x;
    if (blockIdx.x >= blocks) return;
    const uint64_t begin = total * blockIdx.x / blocks;
    const uint32_t share = (uint32_t)(total * (blockIdx.x + 1) / blocks - begin);
    Span<KT> span;
    uint32_t seq = 0, item = 0, tile = 0;
    {
        uint64_t base = 0;
        for (uint32_t b0 = 0;; b0 += 32) {
            const uint64_t mine = b0 + lane < a.c.batch ? (uint64_t)Span<KT>(a, b0 + lane).tiles * per_seq : 0;
            uint64_t upto = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint64_t v = __shfl_up_sync(~0u, upto, d);
                if (lane >= d) upto += v;
            }
            const uint32_t past = __ballot_sync(~0u, base + upto > begin);
            if (past) {
                const int at = __ffs(past) - 1;
                seq = b0 + at;
                base += __shfl_sync(~0u, upto - mine, at);
                span = Span<KT>(a, seq);
                const uint64_t in = begin - base;
                item = (uint32_t)(in / span.tiles);
                tile = (uint32_t)(in - (uint64_t)item * span.tiles);
                break;
            }
            base += __shfl_sync(~0u, upto, 31);
            if (b0 + 32 >= a.c.batch) return;   // not reached while the lengths stay as they are
        }
    }

    // ---- copies: a cursor of its own runs ahead over this warp's tiles ----
    Span<KT> lspan = span;
    uint32_t lseq = seq, litem = item, ltile = tile, lrel = 0, lslot = 0;
    auto step_copies = [&](uint32_t by) {   // moves the cursor on by `by` tiles
        lrel += by;
        ltile += by;
        while (lrel < share && ltile >= lspan.tiles) {
            ltile -= lspan.tiles;
            if (++litem == per_seq) {
                litem = 0;
                if (++lseq >= a.c.batch) {
                    lrel = share;
                    break;
                }
                lspan = Span<KT>(a, lseq);
            }
        }
    };
    auto copy_tile = [&] {
        if (lrel < share) {
            const uint32_t key = lspan.first + ltile * KT + lane, head = litem / a.chunks;
            uint64_t row = ~0ull;
            if (lane < KT && key < lspan.n) row = kv_row(a.c, lseq, head, key);
            const uint32_t to = ring + lslot * S::kStage;
            if constexpr (F16) {
                if (lane < KT) {
                    copy4(to + 2 * KT * S::kRow + 4 * lane, a.c.k_scales + (row == ~0ull ? 0 : row), row != ~0ull);
                    copy4(to + 2 * KT * S::kRow + 4 * KT + 4 * lane, a.c.v_scales + (row == ~0ull ? 0 : row), row != ~0ull);
                }
            }
            const uint32_t c = lane % kPieces;
#pragma unroll
            for (uint32_t i = 0; i < KT * kPieces / 32; ++i) {
                const uint32_t r = i * (32 / kPieces) + lane / kPieces;
                const uint64_t from = __shfl_sync(~0u, row, r);
                const bool there = from != ~0ull && c < row_pieces;
                const uint64_t at = there ? (from * row_pieces + c) * 16 : 0;
                copy16(to + piece_at<FORMAT, DP, false>(r, c), a.c.k + at, there);
                copy16(to + KT * S::kRow + piece_at<FORMAT, DP, true>(r, c), a.c.v + at, there);
            }
            lslot = lslot + 1 == a.stages ? 0 : lslot + 1;
            step_copies(kWarps);
        }
        copies_commit();
    };
    step_copies(warp);
    for (uint32_t s = 0; s < a.stages; ++s) copy_tile();

    // ---- queries of an item: a warp a row; fetched into registers, laid down as 16-bit terms ----
    constexpr int kRows = S::kHeads / kWarps, kEach = DP / 32;
    float qv[kRows][kEach];
    auto fetch_query = [&](uint32_t b, uint32_t it) {
        const uint32_t head = it / a.chunks, chunk = it % a.chunks;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const uint32_t in_group = chunk * S::kHeads + warp + kWarps * r;
            const uint64_t from = (uint64_t)b * a.q_stride + (uint64_t)(head * a.group + in_group) * a.q_head_stride;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const uint32_t d = lane + 32 * i;
                qv[r][i] = in_group >= a.group || d >= a.c.dim ? 0.f
                           : a.q_f32                           ? static_cast<const float *>(a.q)[from + d]
                                                               : bf16_bits_to_f32(static_cast<const uint16_t *>(a.q)[from + d]);
            }
        }
    };
    auto lay_query = [&] {
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const uint32_t row = warp + kWarps * r;
            float by = 1.f, back = 1.f;
            if constexpr (F16) {
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < kEach; ++i) top = fmaxf(top, isfinite(qv[r][i]) ? fabsf(qv[r][i]) : 0.f);
#pragma unroll
                for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
                const int e = min(120, max(-100, (int)(__float_as_uint(top) >> 23) - 127 - kQueryExponent));
                by = __uint_as_float((uint32_t)(127 - e) << 23);
                back = __uint_as_float((uint32_t)(127 + e) << 23) * (FORMAT == FE2O3_KV_E4M3 ? 256.f : 1.f);
            }
            if (lane == 0) head_scale[row] = a.scale * 1.4426950408889634f * back;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                uint16_t *to = reinterpret_cast<uint16_t *>(query + row * S::kQueryRow) + lane + 32 * i;
                float v = qv[r][i] * by;
                if constexpr (F16) {
                    const uint32_t hi = f16_pair(v, 0.f);
                    to[0] = (uint16_t)hi;
                    const float left = v - f16_values(hi).x;
                    if (terms > 1) to[S::kHeads * S::kQueryRow / 2] = (uint16_t)f16_pair(isfinite(v) ? left : 0.f, 0.f);
                } else {
                    to[0] = (uint16_t)(__float_as_uint(v) >> 16);   // a bf16 value as it is; an f32 one cut off
                    if (terms > 1) {
                        const float tiny = copysignf(1.1754944e-38f, v);   // of the value's sign, so that an infinity in K stays one
                        const float mid = v - cut_bf16(v), low = mid - cut_bf16(mid);
                        const bool rest = isfinite(v) && v != 0.f;
                        to[S::kHeads * S::kQueryRow / 2] = (uint16_t)(__float_as_uint(rest ? (cut_bf16(mid) == 0.f ? tiny : mid) : v) >> 16);
                        to[S::kHeads * S::kQueryRow] = (uint16_t)(__float_as_uint(rest ? (low == 0.f ? tiny : low) : v) >> 16);
                    }
                }
            }
        }
    };
    fetch_query(seq, item);
    lay_query();
    __syncthreads();

    // ---- items ----
    uint32_t rel = warp, slot = 0;
    for (uint32_t at = 0;;) {   // `at`: where in the share the item's part of it begins
        const uint32_t here = min(span.tiles - tile, share - at), end = at + here;
        Part<MD, NT> p;
        p.clear();
        float vref = 1.1754944e-38f;   // a power of two above every scale of V so far
        for (; rel < end; rel += kWarps) {
            copies_wait(a.stages - 1);
            __syncwarp();
            const uint32_t from = ring + slot * S::kStage;
            const uint32_t left = span.n - span.first - min(span.n - span.first, (tile + rel - at) * KT);   // keys from here on

            // scores: rows are keys, columns heads
            float s[MT][NT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.f;
            if constexpr (!F16) {
                float odd[MT][NT][4];   // every other step: two chains
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) odd[mt][nt][0] = odd[mt][nt][1] = odd[mt][nt][2] = odd[mt][nt][3] = 0.f;
#pragma unroll
                for (int ks = 0; ks < MD; ks += 2) {
                    uint32_t ka[MT][2][4];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            ldsm4(ka[mt][e], from + piece_at<FORMAT, DP, false>(16 * mt + (lane & 15), 2 * (ks + e) + (lane >> 4)));
                    for (uint32_t term = 0; term < terms; ++term) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            uint32_t qb[4];
                            ldsm4(qb, query_s + (term * S::kHeads + 8 * nt + (lane & 7)) * S::kQueryRow + (2 * ks + (lane >> 3)) * 16);
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) {
                                mma<false>(s[mt][nt], ka[mt][0], qb[0], qb[1]);
                                mma<false>(odd[mt][nt], ka[mt][1], qb[2], qb[3]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[mt][nt][e] += odd[mt][nt][e];
            } else {
#pragma unroll
                for (int j = 0; j < DP / 64; ++j) {   // 64 columns: the lanes of a row hold 16 each, four a step
                    uint4 ka[MT][2];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) ka[mt][e] = lds128(from + piece_at<FORMAT, DP, false>(16 * mt + 8 * e + g, 4 * j + t4));
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t kf[MT][2][4];
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const uint32_t w0 = half ? (e ? ka[mt][0].w : ka[mt][0].z) : (e ? ka[mt][0].y : ka[mt][0].x);
                                const uint32_t w1 = half ? (e ? ka[mt][1].w : ka[mt][1].z) : (e ? ka[mt][1].y : ka[mt][1].x);
                                kf[mt][e][0] = codes_f16<FORMAT, 0, 1>(w0, w0);
                                kf[mt][e][1] = codes_f16<FORMAT, 0, 1>(w1, w1);
                                kf[mt][e][2] = codes_f16<FORMAT, 2, 1>(w0, w0);
                                kf[mt][e][3] = codes_f16<FORMAT, 2, 1>(w1, w1);
                            }
                        for (uint32_t term = 0; term < terms; ++term) {
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                const uint4 qb = lds128(query_s + (term * S::kHeads + 8 * nt + g) * S::kQueryRow + 128 * j + 32 * t4 + 16 * half);
#pragma unroll
                                for (int mt = 0; mt < MT; ++mt) {
                                    mma<true>(s[mt][nt], kf[mt][0], qb.x, qb.y);
                                    mma<true>(s[mt][nt], kf[mt][1], qb.z, qb.w);
                                }
                            }
                        }
                    }
                }
            }

            // the running maximum, in units of log2; weights
            float vs[MT][2];
            float grow = 1.f;   // of the output's unit
            if constexpr (F16) {
                const uint32_t scales = from + 2 * KT * S::kRow;
                float top = 0.f;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float ks = lds_f32(scales + 4 * (16 * mt + 8 * e + g));
                        vs[mt][e] = lds_f32(scales + 4 * KT + 4 * (16 * mt + 8 * e + g));
                        top = fmaxf(top, vs[mt][e]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            s[mt][nt][2 * e] *= ks;
                            s[mt][nt][2 * e + 1] *= ks;
                        }
                    }
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
                if (top >= vref) {
                    const float next = __uint_as_float((__float_as_uint(top) & 0x7f800000u) + 0x00800000u);
                    grow = vref / next;
                    vref = next;
                }
                const float inv = 1.f / vref;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) vs[mt][0] *= inv, vs[mt][1] *= inv;
            }
            uint32_t pb[MT][NT][3][2];   // weights as the second product's operand, by terms
            float scale_o[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float c[2] = {head_scale[8 * nt + 2 * t4], head_scale[8 * nt + 2 * t4 + 1]};
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[mt][nt][e] *= c[e & 1];
                        if (left < KT && 16 * mt + 8 * (e >> 1) + g >= left) s[mt][nt][e] = -INFINITY;
                        top[e & 1] = fmaxf(top[e & 1], s[mt][nt][e]);
                    }
                float base[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(~0u, top[e], d));
                    top[e] = fmaxf(top[e], p.m[nt][e]);
                    base[e] = top[e] == -INFINITY ? 0.f : top[e];
                    const float keep = ex2_approx(p.m[nt][e] - base[e]);
                    p.m[nt][e] = top[e];
                    p.l[nt][e] *= keep;
                    scale_o[nt][e] = keep * grow;
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        w[e] = ex2_approx(s[mt][nt][e] - base[e & 1]);
                        p.l[nt][e & 1] += w[e];
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float w0 = w[2 * e], w1 = w[2 * e + 1];
                        if constexpr (F16) {
                            w0 *= vs[mt][e];
                            w1 *= vs[mt][e];
                            const uint32_t hi = f16_pair(w0, w1);
                            pb[mt][nt][0][e] = turned(hi);
                            const float2 h = f16_values(hi);
                            pb[mt][nt][1][e] = turned(f16_pair(w0 - h.x, w1 - h.y));
                        } else {
                            pb[mt][nt][0][e] = turned(bf16_pair_cut(w0, w1));
                            const float m0 = fmaxf(w0 - cut_bf16(w0), 1.1754944e-38f), m1 = fmaxf(w1 - cut_bf16(w1), 1.1754944e-38f);
                            if (a.o_f32) {
                                pb[mt][nt][1][e] = turned(bf16_pair_cut(m0, m1));
                                pb[mt][nt][2][e] = turned(bf16_pair_cut(fmaxf(m0 - cut_bf16(m0), 1.1754944e-38f), fmaxf(m1 - cut_bf16(m1), 1.1754944e-38f)));
                            } else {
                                uint32_t r;
                                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(m1), "f"(m0));
                                pb[mt][nt][1][e] = turned(r);
                            }
                        }
                    }
                }
            }

            // output: rows are its columns, columns heads; the tile's sum is the tensor unit's, the rest f32
            uint4 v4[MT][4][F16 && DP == 256 ? 2 : 1];
            if constexpr (F16) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t r = 16 * mt + 8 * (e >> 1) + 2 * t4 + (e & 1), base = from + KT * S::kRow;
                        if constexpr (DP == 64) {
                            const uint2 v = lds64(base + piece_at<FORMAT, DP, true>(r, g >> 1) + 8 * (g & 1));
                            v4[mt][e][0] = make_uint4(v.x, v.y, 0, 0);
                        } else {
#pragma unroll
                            for (int x = 0; x < DP / 128; ++x) v4[mt][e][x] = lds128(base + piece_at<FORMAT, DP, true>(r, 8 * x + g));
                        }
                    }
            }
#pragma unroll
            for (int i = 0; i < MD; ++i) {
                uint32_t va[MT][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    if constexpr (F16) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint4 v = v4[mt][e][DP == 256 ? i >> 3 : 0];
                            const int word = (DP == 256 ? i & 7 : i) >> 1;
                            w[e] = word == 0 ? v.x : word == 1 ? v.y : word == 2 ? v.z : v.w;
                        }
                        if (i & 1) {
                            va[mt][0] = codes_f16<FORMAT, 2, 0>(w[0], w[1]);
                            va[mt][1] = codes_f16<FORMAT, 3, 0>(w[0], w[1]);
                            va[mt][2] = codes_f16<FORMAT, 2, 0>(w[2], w[3]);
                            va[mt][3] = codes_f16<FORMAT, 3, 0>(w[2], w[3]);
                        } else {
                            va[mt][0] = codes_f16<FORMAT, 0, 0>(w[0], w[1]);
                            va[mt][1] = codes_f16<FORMAT, 1, 0>(w[0], w[1]);
                            va[mt][2] = codes_f16<FORMAT, 0, 0>(w[2], w[3]);
                            va[mt][3] = codes_f16<FORMAT, 1, 0>(w[2], w[3]);
                        }
                    } else {
                        ldsm4_trans(va[mt], from + KT * S::kRow + piece_at<FORMAT, DP, true>(16 * mt + (lane & 7) + (lane >> 4) * 8, 2 * i + (lane >> 3 & 1)));
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        if constexpr (F16) {
                            mma<true>(d, va[mt], pb[mt][nt][1][0], pb[mt][nt][1][1]);
                            mma<true>(d, va[mt], pb[mt][nt][0][0], pb[mt][nt][0][1]);
                        } else {
                            if (a.o_f32) mma<false>(d, va[mt], pb[mt][nt][2][0], pb[mt][nt][2][1]);
                            mma<false>(d, va[mt], pb[mt][nt][1][0], pb[mt][nt][1][1]);
                            mma<false>(d, va[mt], pb[mt][nt][0][0], pb[mt][nt][0][1]);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) p.o[i][nt][e] = p.o[i][nt][e] * scale_o[nt][e & 1] + d[e];
                }
            }
            slot = slot + 1 == a.stages ? 0 : slot + 1;
            __syncwarp();   // every lane has read the stage
            copy_tile();
        }

        // ---- the item's end: lanes of a row add up, then the warps, then the blocks ----
        {
            const float unit = F16 ? vref * (FORMAT == FE2O3_KV_E4M3 ? 256.f : 1.f) : 1.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) p.l[nt][e] += __shfl_xor_sync(~0u, p.l[nt][e], d);
                if constexpr (F16) {
#pragma unroll
                    for (int i = 0; i < MD; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) p.o[i][nt][e] *= unit;
                }
            }
        }
        uint32_t nseq = seq, nitem = item + 1;
        if (nitem == per_seq) nitem = 0, ++nseq;
        const bool more = end < share && nseq < a.c.batch;
        if (more) fetch_query(nseq, nitem);
        auto in_pairs = [&] {   // warps 2, 3 to 0, 1, then 1 to 0
            __syncthreads();    // warp 0 has read what warp 1 left last time
            if (warp >= 2) p.leave([&](int i, float4 v) { parts[(warp - 2) * S::kPart * 32 + i * 32 + lane] = v; });
            __syncthreads();
            if (warp < 2) p.add([&](int i) { return parts[warp * S::kPart * 32 + i * 32 + lane]; });
            if (warp == 1) p.leave([&](int i, float4 v) { parts[S::kPart * 32 + i * 32 + lane] = v; });
        };
        in_pairs();
        if (more) lay_query();   // nobody needs the last item's any more
        const bool whole = here == span.tiles;
        uint32_t c0 = 0, pieces = 1;
        if (!whole) {
            const uint64_t i0 = begin + at - tile;   // the item's tiles on the line, and the blocks that share them
            c0 = (uint32_t)(((i0 + 1) * blocks - 1) / total);
            pieces = (uint32_t)(((i0 + span.tiles) * blocks - 1) / total) - c0 + 1;
        }
        __syncthreads();
        if (warp == 0) {
            p.add([&](int i) { return parts[S::kPart * 32 + i * 32 + lane]; });
            if (!whole) {
                float4 *const to = a.slots + (uint64_t)(2 * blockIdx.x + (c0 == blockIdx.x)) * S::kPart * 32 + lane;
                p.leave([&](int i, float4 v) { to[i * 32] = v; });
                __threadfence();
                __syncwarp();
                if (lane == 0) {
                    const bool last = atomicAdd(&a.arrived[c0], 1u) == pieces - 1;
                    if (last) a.arrived[c0] = 0;
                    last_flag = last;
                }
            }
        }
        bool write = warp == 0 && whole;
        if (!whole) {
            __syncthreads();
            if (last_flag) {
                __threadfence();
                p.clear();
                for (uint32_t i = warp; i < pieces; i += kWarps) {
                    const float4 *const from = a.slots + (uint64_t)(2 * (c0 + i) + (i == 0)) * S::kPart * 32 + lane;
                    p.add([&](int k) { return __ldcg(from + k * 32); });
                }
                in_pairs();
                __syncthreads();
                if (warp == 0) p.add([&](int i) { return parts[S::kPart * 32 + i * 32 + lane]; });
                write = warp == 0;
            }
        }
        if (write && span.valid) {
            const uint32_t head = item / a.chunks, chunk = item % a.chunks;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t in_group = chunk * S::kHeads + 8 * nt + 2 * t4 + e;
                    if (in_group >= a.group) continue;
                    const uint64_t row = (uint64_t)seq * a.c.kv_heads * a.group + head * a.group + in_group;
                    const float l = p.l[nt][e];
#pragma unroll
                    for (int i = 0; i < MD; ++i)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const uint32_t d = column_of<FORMAT, DP>(i, g + 8 * x);
                            if (d >= a.c.dim) continue;
                            const float v = span.n ? p.o[i][nt][2 * x + e] / l : 0.f;
                            if (a.o_f32) static_cast<float *>(a.o)[row * a.c.dim + d] = v;
                            else static_cast<uint16_t *>(a.o)[row * a.c.dim + d] = f32_to_bf16_bits(v);
                        }
                    if (a.lse && g == 0) a.lse[row] = span.n ? (p.m[nt][e] + log2f(l)) * 0.6931471805599453f : -INFINITY;
                }
        }
        if (!more) break;
        at = end;
        tile = 0;
        item = nitem;
        if (nseq != seq) span = Span<KT>(a, nseq);
        seq = nseq;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

using Kernel = void (*)(PagedArgs);
struct Build {
    Kernel kernel;
    uint32_t stage, part, query;   // bytes: a stage of one warp, a partial result, one term of the queries
};
template <uint32_t FORMAT, int DP, int NT>
constexpr Build build_of() {
    using S = Shape<FORMAT, DP, NT>;
    return Build{paged_attention_kernel<FORMAT, DP, NT>, (uint32_t)S::kStage, (uint32_t)S::kPart * 512u, (uint32_t)S::query_bytes(1)};
}
template <uint32_t FORMAT>
Build build_for(uint32_t dim, uint32_t nt) {
    if (dim <= 64) return nt == 1 ? build_of<FORMAT, 64, 1>() : build_of<FORMAT, 64, 2>();
    if (dim <= 128) return nt == 1 ? build_of<FORMAT, 128, 1>() : build_of<FORMAT, 128, 2>();
    return nt == 1 ? build_of<FORMAT, 256, 1>() : build_of<FORMAT, 256, 2>();
}

}  // namespace

struct PagedPlan {
    Kernel kernel;
    PagedArgs args;
    uint32_t grid, shared;
    void *workspace;
};

void paged_attention_free(PagedPlan *p) {
    if (!p) return;
    if (p->workspace) cudaFree(p->workspace);   // (waits for launches in flight)
    delete p;
}
void paged_attention_geometry(const PagedPlan *p, fe2o3_geometry *geo) {
    *geo = fe2o3_geometry{{p->grid, 1, 1}, {kThreads, 1, 1}, p->shared, 1};
}

int32_t paged_attention_plan(fe2o3_ctx *ctx, const fe2o3_paged_attention_v1_args *a, PagedPlan **out) {
    const uint32_t group = a->heads / a->kv_heads, nt = group <= 8 ? 1 : 2;
    const Build b = a->format == FE2O3_KV_BF16 ? build_for<0>(a->dim, nt) : a->format == FE2O3_KV_E4M3 ? build_for<1>(a->dim, nt) : build_for<2>(a->dim, nt);
    const uint32_t terms = a->q_dtype == FE2O3_DTYPE_BF16 ? 1 : a->format == FE2O3_KV_BF16 ? 3 : 2;
    FE2O3_CUDA(cudaSetDevice(ctx->device));
    // three stages a warp and two blocks an SM where they fit, else what fits of it
    const uint32_t fixed = 2 * b.part + terms * b.query, half = 115712 - 512, all = 231000;
    uint32_t stages = 3;
    if (kWarps * stages * b.stage + fixed > half) {
        stages = (all - fixed) / (kWarps * b.stage);
        stages = stages > 4 ? 4 : stages;
        if (kWarps * 2 * b.stage + fixed <= half) stages = 2;
    }
    PagedPlan *p = new (std::nothrow) PagedPlan();
    if (!p) return FE2O3_ERR_SIZE_OVERFLOW;
    p->kernel = b.kernel;
    p->shared = kWarps * stages * b.stage + fixed;
    int per_sm = 0;
    cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void *>(b.kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)all);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, b.kernel, kThreads, p->shared);
    p->grid = (uint32_t)(per_sm > 0 ? per_sm : 1) * ctx->sm_count;
    const size_t slots = (size_t)2 * p->grid * b.part;
    if (e == cudaSuccess) e = cudaMalloc(&p->workspace, slots + p->grid * sizeof(uint32_t));
    if (e == cudaSuccess) e = cudaMemset(static_cast<uint8_t *>(p->workspace) + slots, 0, p->grid * sizeof(uint32_t));
    if (e == cudaSuccess) e = cudaStreamSynchronize(cudaStreamLegacy);   // no other stream is ordered behind the clear
    if (e != cudaSuccess) {
        paged_attention_free(p);
        return fe2o3_cuda_status(e, "paged_attention_v1 workspace");
    }
    p->args = PagedArgs{kv_cache_of(ctx, a), reinterpret_cast<const void *>(a->q.ptr), reinterpret_cast<void *>(a->output.ptr),
                        reinterpret_cast<float *>(a->lse.ptr), static_cast<float4 *>(p->workspace),
                        reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(p->workspace) + slots), group, (group + 8 * nt - 1) / (8 * nt),
                        a->q_stride, a->q_head_stride, a->window, stages, a->scale, a->q_dtype == FE2O3_DTYPE_F32,
                        a->output_dtype == FE2O3_DTYPE_F32};
    *out = p;
    return FE2O3_OK;
}

int32_t paged_attention_launch(const PagedPlan *p, cudaStream_t s) {
    if (p->args.c.batch == 0) return FE2O3_OK;
    const cudaError_t e = fe2o3_launch_early(p->kernel, p->grid, kThreads, p->shared, s, 1, p->args);
    fe2o3_count_launch(1);
    return fe2o3_cuda_status(e, "paged_attention_v1");
}

static Fe2o3KernelRegistration reg_paged("paged_attention_v1", reinterpret_cast<const void *>(paged_attention_kernel<0, 128, 1>));
