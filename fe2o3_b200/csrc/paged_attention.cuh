// Attention of one new token a sequence over a paged key-value cache: the kernel (paged_attention.cu plans and
// launches it, one source a format builds it); the formulas stand at fe2o3_paged_attention_v1_args.
//
// HBM-bound: the K and V rows of a (sequence, key head) are read once, for all query heads that share them (4 * group
// flop a byte of a bf16 cache, 8 * group of an 8-bit one, 14 * group of a 4-bit one).
//   Work.  An item is a (sequence, key head, up to 8 * NT query heads); its keys fall into tiles of KT.  The tiles of all
//   items form one line, an item's behind kEnd places that stand for what its end costs, and the line is cut into equal
//   shares, one a warp: the lengths are known on the device only, and a launch is the same whatever they are.  A warp
//   writes the results of items that lie in its share by itself.  Others meet twice: the warps of a block when all
//   have done their share, through shared memory, and the blocks in the workspace, where the one that comes last to an
//   item (a counter) joins the pieces.  Both go by the pieces' order: the same bits whoever is last.  A share a warp and not
//   a block: with a block at every item's end, 64 sequences of 1 to 4096 tokens took 167 us where warps took 99 (of that time).
//   Tiles.  Each warp has a ring of stages of its own, so that nothing but its own copies stops a warp, and keeps the
//   maximum, the sum and the output of what it has seen (one pass, f32).  The copy engine fetches a tile as boxes of
//   rows that lie in one page (page sizes that are multiples of 8); other page sizes go row by row in 16-byte copies (i8, 64
//   sequences of 4096: 131 us, and 173 with pages of one row; 32 of bf16 95 and 99).  Rows outside the sequence are zeros.
//   Products.  mma.sync with the keys (and then the output's columns) as rows and the query heads as columns: of
//   the 8 columns of a tile few are wasted for small groups, and P is turned into an operand by movmatrix.  (The tensor unit
//   is 20 % busy: tcgen05, whose tiles are 128 rows, would have nothing to give but its rate.)  The tensor unit's own
//   sums span one tile, longer ones are f32 additions.  A bf16 cache is multiplied as it is, with the
//   probabilities as three bf16 terms that add up to the f32 value exactly, whatever the output's type (two terms, 16 bits, take
//   64 ragged sequences from 100.7 to 99.4 us and put four bf16 outputs in a thousand on another side of their rounding), and an
//   f32 query as three as well, the lower two in a sum of their own.  Terms are cut off, not rounded, and held above 2^-40
//   of the number, so that an infinity in V stays one.  8-bit codes become f16 exactly; the probabilities then carry the row's scale and are two f16
//   terms (22 bits), in units of a power of two a head that follows the largest product of the two.  (One unit for all heads, of
//   the largest scale: e4m3 74.6 us for 74.7, 16 heads on one i8 head 53.4 for 54.2; but a large row of no weight takes the
//   others' bits, all of them from 2^40 on.)  f32 queries are two f16 terms, bf16 ones a single one, in units of a power of two
//   a row.  Error against 64 bits, f32 output: 1e-7 to 5e-7, as plain f32 arithmetic has.
//   4 bits.  Codes become f16 two at a time and are multiplied by their block's scale, 6 bits together: exact, so the rest is as for 8 bits, the
//   row's scale included.  A lane takes neighbouring columns of its keys, 16 of V (one block) and 32 of K, and the queries lie in that order.
//   What is left of a byte is two instructions an element pair, so what a tile costs beside its conversions counts for more: maxima and units are
//   compared between lanes only where one finds more than kSlack (kFull) above what is kept, copies are issued by several lanes at once, and
//   rows that may be long go by 64 keys a tile on two blocks an SM (690 instructions for 32 keys; 940 with 32 a tile, 1014 without these).
// Measured (32 query heads of 128 on 8, on 4 for e4m3): 64 ragged sequences of up to 4096 tokens 98 to 102 us, 5.3 to 5.6 TB/s; two of 131071
// 178 to 193 us, 5.6 to 6.0 TB/s by machine; 96 ragged ones of up to 6000, e4m3, 73 to 75 us, 4.2 TB/s; 16 heads of 64 on 512 tokens 9.6 us.  In
// the middle of a launch bf16 and e4m3 tiles come at 7.1 TB/s.  What is left: 4 us until the first tile is there (lengths,
// page table, rows: three trips to memory), 3 us of ends and joins, and that some SMs (40 of 148 here) end a tenth later than
// the others; a share drawn from a counter by those that are done was tried and costs more than it gives (a drawn share pays
// beginning and end again: 98 -> 105 us).  The 8-bit builds of 65 to 128 columns spill (168 registers at three blocks an SM, 178
// bytes a thread stored and 184 loaded).  16 query heads on an 8-bit head (NT 2, 54 us) are bound by latency: 255 registers leave two warps a
// scheduler, each one dependent chain of some 1150 instructions a tile of 32 keys, at a third of the issue slots; the loop no longer
// fits the first instruction cache.  Half tiles on three blocks an SM come to the same time.
// 4 bits: two sequences of 131071 (319 MB) 94 to 96 us, 3.4 TB/s, where a sum over as many bytes takes 70; 96 ragged ones of up to 6000 on 4 heads 70 us; 16 heads
// of 64 on 512 tokens 11.  Copies alone take 75 of them, products alone 73: what is left is what the two do not hide of each other with
// eight warps an SM and two tiles of 64 keys each in its ring, and about 12 us of beginning and end.  By events, which add 6: three blocks of 32
// keys 113 us where these take 102; 48 keys, or four blocks, spill (117, 129); scales by the lanes' 16-byte copies, so fewer requests to the
// copy engine, 115; pages in order the same.
#pragma once
#include "kv_cache.cuh"

constexpr int kPagedWarps = 4, kPagedThreads = 32 * kPagedWarps;

struct PagedArgs {
    KvCache c;
    const void *q;
    void *o;
    float *lse;
    float4 *slots;        // kPagedSlots partial results a block
    uint32_t *arrived;    // pieces that have come in (see the joins), three counters a block; zero between launches
    uint32_t group, chunks, q_stride, q_head_stride, window, stages;
    uint32_t q_rows;      // of the queries of a chunk in shared memory: its heads, and a row of zeros that stands for those it lacks
    uint32_t room;        // blocks that the GPU holds at once (the grid is smaller where the page table cannot fill it)
    int32_t page_shift;   // log2 of page_size, or -1
    uint32_t box;         // rows of a page that the copy engine takes at once; 1: rows go by 16-byte copies
    float scale;
    bool q_f32, o_f32, q_whole;   // q_whole: rows of the queries start on 16 bytes
};
// The partial results of a block in the workspace: the end of an item that began in an earlier block, the beginning of one that
// goes on in the next, and the ends that its warps 1 to 3 found of items that an earlier warp of the block began.
constexpr uint32_t kPagedSlots = 5, kSlotFirst = 0, kSlotLast = 1, kSlotEnds = 2;
constexpr uint32_t kPagedMaxStages = 4, kPagedMaxStages4 = 6, kPagedMeeting = 512;   // kPagedMaxStages4: of 4-bit rows, whose stages are small

using PagedKernel = void (*)(CUtensorMap, CUtensorMap, PagedArgs);
struct PagedBuild {
    PagedKernel kernel;
    uint32_t stage, part, query;   // bytes: a stage of one warp, a partial result, a row of the queries
    uint32_t scales, keys;         // bytes of a stage's scales; keys of a tile
};
PagedBuild paged_build_bf16(uint32_t dim, uint32_t nt);
PagedBuild paged_build_e4m3(uint32_t dim, uint32_t nt);
PagedBuild paged_build_i8(uint32_t dim, uint32_t nt);
PagedBuild paged_build_e2m1(uint32_t dim, uint32_t nt, bool long_rows);

namespace {

// f16 weights (probability times the row's scale): the largest of a head so far lies in [2^14, 2^15), what is rounded away is at most
// 2^-25, half of f16's smallest number: weights from 2^-17 of the largest have 22 bits, those below 2^-39 are lost.
constexpr int kWeightExponent = 15;
constexpr float kLeastWeight = 0x1p-112f, kMostWeight = 0x1.fffffep125f;   // the largest weight is held in between: powers of two and their reciprocals stay normal numbers
constexpr float kLeastTerm = 0x1p-40f;   // of a number, the least that its lower bf16 terms are: far below its last bit, and nothing where it is 0
// 4 bits: what a score may lie above the maximum kept (log2) before that moves; a probability is up to 2^8 then, and its product with the
// unit of the least weight still a number (where every row so far was zeros: 2^(8 + 103 + 15)).
constexpr float kSlack = 8.f, kLeastWeight4 = 0x1p-104f;
constexpr int kQueryExponent = 14;    // f16 queries: the largest of a row lies in [2^14, 2^15)

// LONG: tiles of 64 keys on two blocks an SM, for long rows of a 4-bit cache (see paged_attention_plan).
template <uint32_t FORMAT, int DP, int NT, bool LONG = false>
struct Shape {
    static constexpr bool kF16 = FORMAT != FE2O3_KV_BF16, kFour = FORMAT == FE2O3_KV_E2M1;
    static constexpr int kRow = kv_bytes<FORMAT>(DP);                                       // bytes of a row in a stage
    static constexpr int kKeys = LONG ? 64 : kF16 ? (DP == 256 ? 16 : 32) : (DP == 64 ? 32 : 16);       // of a tile
    static constexpr int kStage = 2 * kKeys * kRow;                                         // K, V: whole swizzle patterns
    static constexpr int kBlocks = kFour ? kKeys * DP / 16 : 0;                             // block scales of K, and of V
    static constexpr int kScales = (kF16 ? 8 * kKeys : 0) + 2 * kBlocks;                    // of the rows of K, of V; then the blocks'
    static constexpr int kPitch = kRow < 128 ? kRow : 128;                                  // a row lies in parts of at most 128 bytes
    static constexpr int kHeads = 8 * NT;
    static constexpr int kQueryRow = 2 * DP + 16;                                           // bytes, padded against bank conflicts
    static constexpr int kPart = (DP / 16 + 1) * NT;                                        // float4 a lane of a partial result
};

__device__ __forceinline__ void copy16(uint32_t to, const void *from, bool there) {   // or zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void copies_arrive(uint64_t *bar) {   // this thread's copies so far, when they have landed
    asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void *from, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(there ? 4u : 0u) : "memory");
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
// The same with nothing to add to.
template <bool F16>
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
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

__device__ __forceinline__ uint32_t bf16_max(uint32_t a, uint32_t b) {   // of a pair
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t bf16_least(uint32_t v) {   // kLeastTerm of a pair
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"((__float_as_uint(kLeastTerm) >> 16) * 0x10001u));
    return r;
}
// The next power of two above v.
__device__ __forceinline__ float above(float v) { return __uint_as_float((__float_as_uint(v) & 0x7f800000u) + 0x00800000u); }
__device__ __forceinline__ float lg2_approx(float v) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ uint16_t bf16_of(float v) {   // to nearest even
    uint16_t r;
    asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(v));
    return r;
}

// Two 8-bit codes, byte BYTE of `a` and byte BYTE + STEP of `b`, as an f16 pair (both formats exactly).  With STEP 1, a and b are one word.
template <uint32_t FORMAT, int BYTE, int STEP>
__device__ __forceinline__ uint32_t codes_f16(uint32_t a, uint32_t b) {
    if constexpr (FORMAT == FE2O3_KV_I8) {
        // 1024 + (code + 128) has the code in its low bits: f16's step is 1 there
        const uint32_t x = __byte_perm(a, b, BYTE | (4 + BYTE + STEP) << 8);
        uint32_t r = (x & 0x00ff00ffu) ^ 0x64806480u;
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(r) : "r"(0x64806480u));
        return r;
    } else {
        const uint32_t x = STEP == 1 && BYTE == 0 ? a : __byte_perm(a, b, BYTE | (4 + BYTE + STEP) << 4);
        uint32_t r;
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(x));
        return r;
    }
}

// The four codes of a word as two f16 pairs: of the first product, whose columns may come in any order that the queries share
// (lay_query).  i8 takes even and odd bytes: no permutation.
template <uint32_t FORMAT>
__device__ __forceinline__ void word_f16(uint32_t w, uint32_t &a, uint32_t &b) {
    if constexpr (FORMAT == FE2O3_KV_I8) {
        a = (w & 0x00ff00ffu) ^ 0x64806480u;
        b = (w >> 8 & 0x00ff00ffu) ^ 0x64806480u;
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(a) : "r"(0x64806480u));
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(b) : "r"(0x64806480u));
    } else {
        a = codes_f16<FORMAT, 0, 1>(w, w);
        b = codes_f16<FORMAT, 2, 1>(w, w);
    }
}

// ---- 4 bits ----
// The eight codes of a word as f16 pairs, exactly.
__device__ __forceinline__ void codes4_f16(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}" : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
__device__ __forceinline__ uint32_t code4_pair(uint32_t w, int byte) {   // the two of one byte
    uint32_t h[4];
    codes4_f16(w, h);   // (what is not asked for falls away)
    return byte == 0 ? h[0] : byte == 1 ? h[1] : byte == 2 ? h[2] : h[3];
}
__device__ __forceinline__ uint32_t scales_f16(uint32_t two) {   // of two blocks, a byte each
    uint32_t r;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(r) : "r"(two));
    return r;
}
__device__ __forceinline__ uint32_t times_f16(uint32_t a, uint32_t b) {   // (a code times its block's scale has 6 bits: exact)
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t at) {
    uint32_t v;
    asm volatile("{\n\t.reg .b16 t;\n\tld.shared.u16 t, [%1];\n\tcvt.u32.u16 %0, t;\n\t}" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t at) {
    uint32_t v;
    asm volatile("{\n\t.reg .b16 t;\n\tld.shared.u8 t, [%1];\n\tcvt.u32.u16 %0, t;\n\t}" : "=r"(v) : "r"(at) : "memory");
    return v;
}
// The key that row r of eight stands for.  With 4 bits two neighbours change places for half of the rows, so that the rows of V that the
// lanes of one access touch (2 t and its neighbour) lie on banks of their own; K's follow.
template <uint32_t FORMAT, int DP>
__device__ __forceinline__ uint32_t key_of(uint32_t r) {
    if constexpr (FORMAT != FE2O3_KV_E2M1 || DP == 256) return r;
    else return r ^ (r >> (DP == 64 ? 2 : 1) & 1);
}

// Where 16-byte piece c of row r lies in a stage's K or V part: as the copy engine's swizzle has it, rows in parts of 128 bytes.
// Of what the lanes of one access touch, nothing meets on a bank but K of the 8-bit formats, in twos.
template <uint32_t FORMAT, int DP>
__device__ __forceinline__ uint32_t piece_at(uint32_t r, uint32_t c) {
    using S = Shape<FORMAT, DP, 1>;
    if constexpr (S::kRow == 32) return r * 32 + (c << 4);
    else if constexpr (S::kRow == 64) return r * 64 + ((c ^ (r >> 1 & 3)) << 4);
    else return (c >> 3) * S::kKeys * 128 + r * 128 + (((c ^ r) & 7) << 4);
}

// Column of the output that row m of tile i of the second product stands for.
template <uint32_t FORMAT, int DP>
__device__ __forceinline__ uint32_t column_of(uint32_t i, uint32_t m) {
    if constexpr (FORMAT == FE2O3_KV_BF16) return 16 * i + m;
    else return (DP == 64 ? 8 * (m & 7) : 16 * (m & 7)) + (DP == 256 ? 128 * (i >> 3) + 2 * (i & 7) : 2 * i) + (m >> 3);
}

// places on the line in front of an item's tiles.  With 1, 2, 3: 96 ragged e4m3 sequences 80, 76, 74 us; 64 ragged ones of bf16 105,
// 100, 100; 256 of 128 tokens 41.3, 42.0, 42.5 (one box, in turn)
constexpr uint32_t kEnd = 2;
constexpr uint32_t kLeast = 1;   // places a warp has at least (10 to 2000 keys a block: 9.9 us for 16 heads of 512 keys, 11.1 with 2, the same 25.3 for 8 sequences of 2048)
constexpr uint32_t kGroup = 16;   // pieces joined by one block
constexpr uint32_t kInvalid = ~0u;
// What a warp's share ends in: whole items only; an item that begins in the share and goes on; one that goes on on both sides; no places.
enum : uint32_t { kNone, kBegun, kWithin, kEmpty };
struct Left {
    uint32_t kind, end_of_first, seq, item, n, places;   // end_of_first: an item that began before the share ended in it
    uint64_t i0;                                         // where on the line the open item begins
};
struct Job {
    uint32_t seq, item, n, pieces;   // pieces 0: none; before the count: the item's places
    uint32_t block, first, groups;   // where the item begins, and the group of pieces; groups of the item
    uint64_t i0;
};
__device__ __forceinline__ uint32_t running_sum(uint32_t v, uint32_t lane) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t u = __shfl_up_sync(~0u, v, d);
        if (lane >= d) v += u;
    }
    return v;
}
// How the line is cut: an equal share a warp.
struct Line {
    uint64_t total;          // places
    uint32_t blocks, q, r;   // at work; total / (4 blocks) and what is over
    uint32_t whole;          // items of up to so many places are not cut: they go to the warp that would have their larger half
    __device__ __forceinline__ Line(const PagedArgs &a, uint64_t total, uint32_t per_seq) : total(total) {
        // (several blocks: no warp is without a place, so that what an earlier block began is seen by warp 0)
        const uint64_t wanted = max(total / (kLeast * kPagedWarps), (uint64_t)1);
        blocks = wanted < gridDim.x ? (uint32_t)wanted : gridDim.x;
        // as many blocks an item for all, where that leaves few idle or there is little to do: items of one length then end with a block
        const uint32_t items = a.c.batch * per_seq;
        if (items <= blocks && (wanted < a.room || blocks % items * 16 <= blocks)) blocks -= blocks % items;
        const uint32_t warps = blocks * kPagedWarps;
        const uint64_t each = total >> 32 ? total / warps : (uint32_t)total / warps;
        q = (uint32_t)each;
        r = (uint32_t)(total - each * warps);
        whole = wanted < a.room ? kEnd + 1 : max(4u, q / 8);   // (SMs to spare: two tiles are sooner done by two warps)
    }
    __device__ __forceinline__ void share(uint32_t me, uint64_t &begin, uint32_t &n) const {
        const uint32_t warps = blocks * kPagedWarps, over = r * me / warps;
        begin = (uint64_t)q * me + over;
        n = q + r * (me + 1) / warps - over;
    }
    // Places of an item that a share takes which would end (or begin) behind `some` of its places: none or all where it is not cut.
    __device__ __forceinline__ uint32_t taken(uint32_t some, uint32_t places) const {
        return places > whole || some >= places ? min(some, places) : 2 * some >= places ? places : 0;
    }
    __device__ static __forceinline__ uint32_t block_of(uint64_t place, uint64_t total, uint32_t blocks) { return (uint32_t)(((place + 1) * blocks - 1) / total); }
};
// What a block has in shared memory beside rings and queries (all of it in the dynamic part, which then starts on a swizzle pattern).
template <bool FOUR>
struct Meeting {
    uint64_t arrivals[kPagedWarps][FOUR ? kPagedMaxStages4 : kPagedMaxStages];
    Left left[kPagedWarps];
    Job first;       // where warp 0 begins, should an item of an earlier block end there
    uint64_t total;  // of the line (kept here and not in registers through all tiles)
    uint32_t blocks;
    Job jobs[2];
    bool goes_on;
};
static_assert(sizeof(Meeting<false>) <= kPagedMeeting && sizeof(Meeting<true>) <= kPagedMeeting, "");
// A sequence's keys as tiles, counted from a multiple of KT.  One that does not fit its table is reported and has none.
template <int KT>
struct Span {
    uint32_t first, n, tiles;
    bool valid;
    __device__ __forceinline__ Span() : first(0), n(0), tiles(0), valid(false) {}
    __device__ __forceinline__ Span(const PagedArgs &a, uint32_t b) {
        n = a.c.lengths[b];
        valid = kv_fits(a.c, n);
        if (!valid) {
            kstatus_set(a.c.status, FE2O3_KSTATUS_LENGTH);
            n = 0;
        }
        first = a.window && n > a.window ? n - a.window : 0;
        tiles = (n + KT - 1) / KT - first / KT;
    }
    __device__ __forceinline__ uint32_t places() const { return tiles + kEnd; }
    __device__ __forceinline__ uint32_t key(uint32_t tile) const { return (first / KT + tile) * KT; }
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
    // Adds another part, float4 by float4 in leave()'s order.
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

template <uint32_t FORMAT, int DP, int NT, bool LONG = false>
__global__ void __launch_bounds__(kPagedThreads, DP == 256 || NT == 2 ? 1 : LONG ? 2 : 3)
paged_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PagedArgs a) {
    using S = Shape<FORMAT, DP, NT, LONG>;
    using P = Part<DP / 16, NT>;
    constexpr int KT = S::kKeys, MT = KT / 16, MD = DP / 16, kPieces = S::kRow / 16, kRowsAtOnce = 32 / kPieces;
    constexpr bool F16 = S::kF16, F4 = S::kFour;
    extern __shared__ __align__(1024) uint8_t smem[];   // (swizzle patterns are 1 KiB)
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
    uint8_t *const my_ring = smem + warp * a.stages * S::kStage;
    const uint32_t ring = smem_u32(my_ring);
    const uint32_t terms = a.q_f32 ? (F16 ? 2 : 3) : 1;
    uint8_t *const my_scales = smem + kPagedWarps * a.stages * S::kStage + warp * a.stages * S::kScales;
    uint8_t *const queries = smem + kPagedWarps * a.stages * (S::kStage + S::kScales);
    const uint32_t term_bytes = a.q_rows * S::kQueryRow;
    uint8_t *const query = queries + warp * terms * term_bytes;
    Meeting<F4> &meeting = *reinterpret_cast<Meeting<F4> *>(queries + kPagedWarps * terms * term_bytes);
    const uint32_t query_s = smem_u32(query);
    const uint32_t row_bytes = kv_bytes<FORMAT>(a.c.dim), row_blocks = a.c.dim / 16;   // (4 bits: block scales of a row)
    const uint32_t per_seq = a.c.kv_heads * a.chunks;   // items of a sequence

    uint64_t *const bars = meeting.arrivals[warp];
    for (uint32_t term = 0; term < terms; ++term)
        for (uint32_t i = lane; i < S::kQueryRow / 16; i += 32)
            *reinterpret_cast<uint4 *>(query + term * term_bytes + (a.q_rows - 1) * S::kQueryRow + 16 * i) = make_uint4(0, 0, 0, 0);
    if (lane < a.stages) mbar_init(&bars[lane], a.box > 1 ? 1 : 32);
    mbar_fence_init();
    if (a.box > 1) {
        if (lane == 0) {
            tma_prefetch_desc(&map_k);
            tma_prefetch_desc(&map_v);
        }
    } else if (F4) {   // (a cache without pages: nothing is ever copied)
        for (uint32_t i = lane; i < a.stages * S::kScales / 4; i += 32) reinterpret_cast<uint32_t *>(my_scales)[i] = 0;
    } else if (a.c.dim < DP) {   // the columns past the head's: zeros, which no copy goes over
        for (uint32_t i = lane; i < 2 * KT * a.stages * kPieces; i += 32) {
            const uint32_t c = i % kPieces, row = i / kPieces, r = row % KT, side = row / KT % 2, stage = row / (2 * KT);
            if (16 * c >= row_bytes) *reinterpret_cast<uint4 *>(my_ring + stage * S::kStage + side * KT * S::kRow + piece_at<FORMAT, DP>(r, c)) = make_uint4(0, 0, 0, 0);
        }
    }
    __syncwarp();
    begin_after_previous();

    // ---- the line: every warp adds up the sequences for itself, a run of them a lane ----
    const uint32_t run = (a.c.batch + 31) / 32;
    uint32_t own = 0, before;
    for (uint32_t i = 0; i < run; ++i)
        if (lane * run + i < a.c.batch) own += Span<KT>(a, lane * run + i).places();
    const uint64_t total = (uint64_t)__shfl_sync(~0u, before = running_sum(own, lane), 31) * per_seq;
    before -= own;
    const Line line(a, total, per_seq);
    if (blockIdx.x >= line.blocks) return;

    // ---- copies: the places of the share, by a cursor that runs ahead over its tiles ----
    Span<KT> lspan;
    uint32_t lseq = 0, litem = 0, lslot = 0, lrest = 0, ltile = 0, lend = 0;   // lrest: places of the share behind its present item
    auto enter = [&](uint32_t from) {   // the cursor's item, from this place on
        const uint32_t take = from ? min(lspan.places() - from, lrest) : line.taken(lrest, lspan.places());
        ltile = max(from, kEnd) - kEnd;
        lend = max(from + take, kEnd) - kEnd;
        lrest = take ? lrest - min(take, lrest) : 0;
    };
    uint32_t entry = 0, entries_from = 0, entries_of = ~0u;   // 32 entries of a sequence's table, a lane each
    const uint32_t lrow = lane / kPieces, lpiece = lane % kPieces, boxes = KT / a.box;
    // 4 bits: six copies a box, of rows, row scales and block scales.  Eight lanes take the boxes, four such sets the kinds: K's and V's row scales
    // and block scales, and two of them the rows.  (One lane after another, as with the other formats, is 120 instructions a tile more.)
    const uint32_t lbox = F4 ? lane & 7 : lane, lset = lane >> 3;
    const uint8_t *const scales_from = !F4 ? nullptr : lset == 0 ? reinterpret_cast<const uint8_t *>(a.c.k_scales) : lset == 1 ? reinterpret_cast<const uint8_t *>(a.c.v_scales)
                                                     : (lset == 2 ? a.c.k : a.c.v) + a.c.blocks;
    const uint32_t scales_row = lset < 2 ? 4 : row_blocks;   // bytes
    const uint32_t scales_to = (lset < 2 ? lset * 4 * KT : 8 * KT + (lset & 1) * S::kBlocks) + lbox * a.box * scales_row;
    const CUtensorMap *const lmap = lset & 1 ? &map_v : &map_k;
    const uint32_t scales_bytes = a.box * scales_row, rows_to = lset * (KT * S::kRow) + lbox * a.box * S::kPitch, box_bytes = a.box * (2 * S::kRow + 8 + 2 * row_blocks);
    uint32_t lhead = 0;   // of the cursor's item
    // Zeros for a row of a stage: K and V, and their scales.
    auto no_row = [&](uint32_t slot, uint32_t r, bool k_too) {
        for (uint32_t i = lane; i < 2 * kPieces; i += 32)
            if (k_too || i >= kPieces)
                *reinterpret_cast<uint4 *>(my_ring + slot * S::kStage + (i >= kPieces ? KT * S::kRow : 0) + piece_at<FORMAT, DP>(r, i % kPieces)) = make_uint4(0, 0, 0, 0);
        if (F16 && lane < 2) reinterpret_cast<float *>(my_scales + slot * S::kScales)[lane * KT + r] = 0.f;
        if constexpr (F4)
            if (lane < row_blocks) {   // (K's rows that count nothing are never added up: their scales may be what they are)
                uint8_t *const blocks = my_scales + slot * S::kScales + 8 * KT + r * row_blocks + lane;
                if (k_too) blocks[0] = 0;
                blocks[S::kBlocks] = 0;
            }
    };
    auto next_item = [&] {
        while (ltile == lend && lrest) {
            if (++litem == per_seq) {
                litem = 0;
                if (++lseq >= a.c.batch) {
                    lrest = 0;
                    break;
                }
                lspan = Span<KT>(a, lseq);
            }
            enter(0);
        }
        if constexpr (F4) lhead = litem / a.chunks;
    };
    auto copy_any = [&] {
        next_item();
        if (ltile >= lend) return;
        // a lane a box, or a row
        const uint32_t key = lspan.key(ltile) + min(lbox, boxes - 1) * a.box, head = litem / a.chunks;
        const uint32_t at = a.page_shift >= 0 ? key >> a.page_shift : key / a.c.page_size;   // in the table
        const uint32_t first_at = __shfl_sync(~0u, at, 0), last_at = __shfl_sync(~0u, at, 31);
        if (entries_of != lseq || first_at < entries_from || last_at >= entries_from + 32) {
            entries_of = lseq;
            entries_from = first_at;
            entry = ~0u;
            if (entries_from + lane < a.c.table_width) entry = a.c.page_table[(uint64_t)lseq * a.c.table_width + entries_from + lane];
        }
        const uint32_t page = __shfl_sync(~0u, entry, at - entries_from), in_page = key - at * a.c.page_size;
        const bool wanted = lbox < boxes && key < lspan.n && key + a.box > lspan.first, there = wanted && page < a.c.pages;
        if (wanted && !there) kstatus_set(a.c.status, FE2O3_KSTATUS_SLOT_RANGE);
        const uint32_t found = __ballot_sync(~0u, there) & (F4 ? 0xffu : ~0u);
        uint64_t *const bar = &bars[lslot];
        const uint32_t row = there ? (page * a.c.kv_heads + head) * a.c.page_size + in_page : ~0u;
        if (a.box > 1) {
            if (lane == 0) mbar_arrive_expect_tx(bar, __popc(found) * a.box * (2 * S::kRow + (F16 ? 8 : 0) + (F4 ? 2 * row_blocks : 0)));
            __syncwarp();
            if (F4) {
                if (there) {
                    bulk_load_1d(my_scales + lslot * S::kScales + scales_to, scales_from + (uint64_t)row * scales_row, a.box * scales_row, bar);
                    if (lset < 2)
                        tma_load_3d(my_ring + lslot * S::kStage + lset * (KT * S::kRow) + lbox * a.box * S::kPitch, lmap, bar, 0, in_page, page * a.c.kv_heads + head);
                }
            } else if (there) {
                uint8_t *const to = my_ring + lslot * S::kStage + lane * a.box * S::kPitch;
#pragma unroll
                for (int half = 0; half < S::kRow / S::kPitch; ++half) {
                    tma_load_3d(to + half * KT * 128, &map_k, bar, half * (F16 ? 128 : 64), in_page, page * a.c.kv_heads + head);
                    tma_load_3d(to + KT * S::kRow + half * KT * 128, &map_v, bar, half * (F16 ? 128 : 64), in_page, page * a.c.kv_heads + head);
                }
                if constexpr (F16) {
                    uint8_t *const scales = my_scales + lslot * S::kScales + lane * a.box * 4;
                    bulk_load_1d(scales, a.c.k_scales + row, a.box * 4, bar);
                    bulk_load_1d(scales + KT * 4, a.c.v_scales + row, a.box * 4, bar);
                }
            }
            __syncwarp();
            if (found != (boxes == 32 ? ~0u : (1u << boxes) - 1)) {   // at an end of the sequence, or reported
                for (uint32_t r = 0; r < KT; ++r)
                    if (!(found >> r / a.box & 1)) no_row(lslot, r, true);
                fence_proxy_async_smem();   // before the next box goes there
            }
        } else {
            const uint32_t to = ring + lslot * S::kStage, to_k = to + piece_at<FORMAT, DP>(lrow, lpiece), to_v = to_k + KT * S::kRow;
            if constexpr (F16) {
                if (lane < KT) {
                    const uint32_t scales = smem_u32(my_scales + lslot * S::kScales) + 4 * lane;
                    copy4(scales, a.c.k_scales + (row == ~0u ? 0 : row), row != ~0u);
                    copy4(scales + 4 * KT, a.c.v_scales + (row == ~0u ? 0 : row), row != ~0u);
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < KT / kRowsAtOnce; ++i) {
                // (the rows of one step and of another differ in bits of their own, so the swizzle falls apart)
                const uint32_t x = S::kRow == 64 ? 0 : (i * kRowsAtOnce & 7) << 4, down = i * kRowsAtOnce * S::kPitch;
                const uint32_t r = __shfl_sync(~0u, row, i * kRowsAtOnce + lrow);
                const uint64_t from = r == ~0u ? 0 : (uint64_t)r * row_bytes + 16 * lpiece;
                if (16 * lpiece < row_bytes) {
                    copy16((to_k ^ x) + down, a.c.k + from, r != ~0u);
                    copy16((to_v ^ x) + down, a.c.v + from, r != ~0u);
                }
            }
            copies_arrive(bar);
        }
        lslot = lslot + 1 == a.stages ? 0 : lslot + 1;
        ++ltile;
    };
    // Long rows of 4 bits: the same in fewer steps (two sequences of 131071 104 us, by events, where these take 100; short rows take 3 % longer so).
    auto copy_long = [&] {
        if (ltile == lend) {
            next_item();
            if (ltile >= lend) return;
        }
        const uint32_t key = (lspan.first / KT + ltile) * KT + min(lbox, boxes - 1) * a.box;
        const uint32_t at = a.page_shift >= 0 ? key >> a.page_shift : key / a.c.page_size, in_page = key - at * a.c.page_size;
        uint32_t of_entries = at - entries_from;
        if (entries_of != lseq || __any_sync(~0u, of_entries >= 32)) {
            entries_of = lseq;
            entries_from = __shfl_sync(~0u, at, 0);
            entry = ~0u;
            if (entries_from + lane < a.c.table_width) entry = a.c.page_table[(uint64_t)lseq * a.c.table_width + entries_from + lane];
            of_entries = at - entries_from;
        }
        const uint32_t page = __shfl_sync(~0u, entry, of_entries);
        const bool wanted = lbox < boxes && key < lspan.n && key + a.box > lspan.first, there = wanted && page < a.c.pages;
        const uint32_t found = __ballot_sync(~0u, there) & 0xffu, all = (1u << boxes) - 1;
        uint64_t *const bar = &bars[lslot];
        if (lane == 0) mbar_arrive_expect_tx(bar, __popc(found) * box_bytes);
        __syncwarp();
        if (there) {
            const uint32_t head_of_page = page * a.c.kv_heads + lhead, row = head_of_page * a.c.page_size + in_page;
            bulk_load_1d(my_scales + lslot * S::kScales + scales_to, scales_from + (uint64_t)row * scales_row, scales_bytes, bar);
            if (lset < 2) tma_load_3d(my_ring + lslot * S::kStage + rows_to, lmap, bar, 0, in_page, head_of_page);
        }
        if (found != all) {   // at an end of the sequence, or reported
            if (wanted && !there) kstatus_set(a.c.status, FE2O3_KSTATUS_SLOT_RANGE);
            __syncwarp();
            for (uint32_t r = 0; r < KT; ++r)
                if (!(found >> r / a.box & 1)) no_row(lslot, r, true);
            fence_proxy_async_smem();   // before the next box goes there
        }
        lslot = lslot + 1 == a.stages ? 0 : lslot + 1;
        ++ltile;
    };
    auto copy_tile = [&] {
        if (LONG && a.box > 1) copy_long();
        else copy_any();
    };
    uint32_t seq, item;   // at work
    // ---- the queries of an item, as 16-bit terms: a lane takes eight columns of a row at a time ----
    auto lay_query = [&] {
        constexpr int kLanes = DP / 8, kAtOnce = 32 / kLanes, kPasses = S::kHeads / kAtOnce;
        // where a lane's eight columns go.  4 bits: the lanes of a row of K hold 16 or 32 neighbours each (two runs of them for 256 columns), a
        // word of eight at a time, and read the queries of two words at 32 bytes from one another
        const uint32_t chunk_of_row = lane % kLanes, in_run = chunk_of_row & 15;
        const uint32_t word = DP == 64 ? chunk_of_row & 1 : (in_run & 3) + (chunk_of_row >> 4) * 4, of_lane = DP == 64 ? chunk_of_row >> 1 : in_run >> 2;
        const uint32_t place_of_chunk = F4 ? 8 * (word >> 1) + 2 * of_lane + (word & 1) : chunk_of_row;
        const uint32_t head = item / a.chunks, chunk = item % a.chunks, d = lane % kLanes * 8, r0 = lane / kLanes;
        const uint64_t base = (uint64_t)seq * a.q_stride + (uint64_t)(head * a.group) * a.q_head_stride + d;
        const uint32_t stored = min(a.group, (uint32_t)S::kHeads);
        uint4 raw[kPasses][2];
#pragma unroll
        for (int x = 0; x < kPasses; ++x) {
            raw[x][0] = raw[x][1] = make_uint4(0, 0, 0, 0);
            const uint32_t in_group = chunk * S::kHeads + x * kAtOnce + r0;
            if (in_group >= a.group || d >= a.c.dim) continue;
            const uint64_t from = base + (uint64_t)in_group * a.q_head_stride;
            const uint8_t *const at = static_cast<const uint8_t *>(a.q) + from * (a.q_f32 ? 4 : 2);
            if (a.q_whole) {   // rows start on 16 bytes
                raw[x][0] = *reinterpret_cast<const uint4 *>(at);
                if (a.q_f32) raw[x][1] = *reinterpret_cast<const uint4 *>(at + 16);
            } else if (a.q_f32) {
                const uint32_t *const v = reinterpret_cast<const uint32_t *>(at);
                raw[x][0] = make_uint4(v[0], v[1], v[2], v[3]);
                raw[x][1] = make_uint4(v[4], v[5], v[6], v[7]);
            } else {
                const uint16_t *const v = reinterpret_cast<const uint16_t *>(at);
                raw[x][0] = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
            }
        }
#pragma unroll
        for (int x = 0; x < kPasses; ++x) {
            if (x * kAtOnce >= stored) continue;
            const uint32_t row = min(x * kAtOnce + r0, a.q_rows - 1);   // (zeros again, where the rows are odd in number)
            uint8_t *const to = query + row * S::kQueryRow + 16 * place_of_chunk;
            float back = 1.f;
            if constexpr (!F16) {
                if (!a.q_f32) *reinterpret_cast<uint4 *>(to) = raw[x][0];
            }
            if (F16 || a.q_f32) {
                float v[8];
                const uint32_t w[8] = {raw[x][0].x, raw[x][0].y, raw[x][0].z, raw[x][0].w, raw[x][1].x, raw[x][1].y, raw[x][1].z, raw[x][1].w};
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(a.q_f32 ? w[i] : i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
                if constexpr (F16) {
                    float top = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]) < INFINITY ? fabsf(v[i]) : 0.f);
#pragma unroll
                    for (int i = 1; i < kLanes; i <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, i));
                    const int e = min(120, max(-100, (int)(__float_as_uint(top) >> 23) - 127 - kQueryExponent));
                    const float by = __uint_as_float((uint32_t)(127 - e) << 23);
                    back = __uint_as_float((uint32_t)(127 + e) << 23);
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        // the order of word_f16: of i8 columns 0 and 2, then 1 and 3
                        constexpr bool kEvenOdd = FORMAT == FE2O3_KV_I8;
                        const float v0 = v[kEvenOdd ? 4 * (i / 2) + i % 2 : 2 * i] * by, v1 = v[kEvenOdd ? 4 * (i / 2) + i % 2 + 2 : 2 * i + 1] * by;
                        hi[i] = f16_pair(v0, v1);
                        const float2 h = f16_values(hi[i]);
                        lo[i] = f16_pair(fabsf(v0) < INFINITY ? v0 - h.x : 0.f, fabsf(v1) < INFINITY ? v1 - h.y : 0.f);
                    }
                    *reinterpret_cast<uint4 *>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if (terms > 1) *reinterpret_cast<uint4 *>(to + term_bytes) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                } else {
                    // cut off; where nothing is left it is next to nothing with the value's sign, so that an infinity in K stays one
                    float least[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) least[i] = fabsf(v[i]) * kLeastTerm;
#pragma unroll
                    for (int term = 0; term < 3; ++term) {
                        *reinterpret_cast<uint4 *>(to + term * term_bytes) =
                            make_uint4(bf16_pair_cut(v[0], v[1]), bf16_pair_cut(v[2], v[3]), bf16_pair_cut(v[4], v[5]), bf16_pair_cut(v[6], v[7]));
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float left = v[i] - cut_bf16(v[i]);
                            if (fabsf(v[i]) < INFINITY) v[i] = fabsf(left) < least[i] ? copysignf(least[i], v[i]) : left;
                        }
                    }
                }
            }
            if (lane % kLanes == 0) *reinterpret_cast<float *>(query + row * S::kQueryRow + 2 * DP) = a.scale * 1.4426950408889634f * back;   // (in the padding)
        }
        __syncwarp();
    };

    // Writes an item's result, or the columns of it from output tile i0 on.
    auto write = [&](const auto &p, uint32_t seq, uint32_t item, uint32_t n, uint32_t i0) {
        constexpr int kTiles = sizeof(p.o) / sizeof(p.o[0]);
        const uint32_t head = item / a.chunks, chunk = item % a.chunks;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t in_group = chunk * S::kHeads + 8 * nt + 2 * t4 + e;
                if (in_group >= a.group) continue;
                const uint64_t row = (uint64_t)seq * a.c.kv_heads * a.group + head * a.group + in_group;
                const float l = p.l[nt][e], inv = n ? 1.f / l : 0.f;
                float *const o32 = static_cast<float *>(a.o) + row * a.c.dim;
                uint16_t *const o16 = static_cast<uint16_t *>(a.o) + row * a.c.dim;
#pragma unroll
                for (int i = 0; i < kTiles; ++i) {
                    const float v0 = p.o[i][nt][e] * inv, v1 = p.o[i][nt][2 + e] * inv;
                    const uint32_t d = column_of<FORMAT, DP>(i0 + i, g);   // the other row's column: 8 further, or the next
                    constexpr uint32_t kNext = F16 ? 1 : 8;
                    if (d >= a.c.dim) continue;
                    if (a.o_f32) {
                        o32[d] = v0;
                        o32[d + kNext] = v1;
                    } else {
                        o16[d] = bf16_of(v0);
                        o16[d + kNext] = bf16_of(v1);
                    }
                }
                if (a.lse && g == 0 && i0 == 0) a.lse[row] = n ? (p.m[nt][e] + log2f(l)) * 0.6931471805599453f : -INFINITY;
            }
    };
    const uint32_t gk = key_of<FORMAT, DP>(g);
    // where a lane reads K and V in a stage; a lane's offsets for further steps differ by constants
    uint32_t k_off[4], v_off[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        if constexpr (F4) {
            const uint32_t row = key_of<FORMAT, DP>(2 * t4 + (x & 1));
            k_off[x] = piece_at<FORMAT, DP>(gk, DP == 64 ? t4 >> 1 : t4 + 4 * (x & 1)) + (DP == 64 ? 8 * (t4 & 1) : 0);   // (256 columns: two pieces)
            if constexpr (DP == 64) v_off[x] = KT * S::kRow + piece_at<FORMAT, DP>(row, g >> 2) + 4 * (g & 3);
            else v_off[x] = KT * S::kRow + piece_at<FORMAT, DP>(row, (g >> 1) + (x >> 1) * 4) + 8 * (g & 1);   // (256 columns: two runs)
        } else if constexpr (!F16) {
            k_off[x] = piece_at<FORMAT, DP>(lane & 15, 2 * x + (lane >> 4));
            v_off[x] = KT * S::kRow + piece_at<FORMAT, DP>((lane & 7) + (lane >> 4) * 8, 2 * x + (lane >> 3 & 1));
        } else if constexpr (DP == 64) {
            k_off[x] = piece_at<FORMAT, DP>(g, t4);
            v_off[x] = KT * S::kRow + piece_at<FORMAT, DP>(2 * t4 + (x & 1), g >> 1) + 8 * (g & 1);
        } else {
            k_off[x] = piece_at<FORMAT, DP>(g, 4 * (x & 1) + t4);
            v_off[x] = KT * S::kRow + piece_at<FORMAT, DP>(2 * t4 + (x & 1), g);
        }
    }

    uint32_t slot = 0, phase = 0;
    bool waiting = true;
    uint64_t begin;
    uint32_t share;
    line.share(blockIdx.x * kPagedWarps + warp, begin, share);
    float4 *const slots = a.slots + (uint64_t)blockIdx.x * kPagedSlots * S::kPart * 32 + lane;
    uint32_t place = 0;   // of the item, where the share begins
    {
        const uint32_t in = __ffs(__ballot_sync(~0u, (uint64_t)(before + own) * per_seq > begin)) - 1;   // the lane whose run it is
        uint64_t base = (uint64_t)__shfl_sync(~0u, before, in) * per_seq;
        seq = min(in * run, a.c.batch - 1);
        for (uint32_t b0 = 0; run > 1 && b0 < run; b0 += 32) {
            const uint32_t b = in * run + b0 + lane, places = b0 + lane < run && b < a.c.batch ? Span<KT>(a, b).places() : 0;
            const uint32_t upto = running_sum(places, lane), past = __ballot_sync(~0u, base + (uint64_t)upto * per_seq > begin);
            if (past) {
                const int at = __ffs(past) - 1;
                seq = in * run + b0 + at;
                base += (uint64_t)__shfl_sync(~0u, upto - places, at) * per_seq;
                break;
            }
            base += (uint64_t)__shfl_sync(~0u, upto, 31) * per_seq;
        }
        lspan = Span<KT>(a, seq);
        const uint64_t into = min(begin - base, (uint64_t)lspan.places() * per_seq - 1);
        item = into >> 32 ? (uint32_t)(into / lspan.places()) : (uint32_t)into / lspan.places();
        place = (uint32_t)(into - (uint64_t)item * lspan.places());
    }
    if (place && line.taken(place, lspan.places()) != place) {   // an item that is not cut: the last warp has it, or this one
        if (line.taken(place, lspan.places())) {
            const uint32_t rest = lspan.places() - place;
            share = share > rest ? share - rest : 0;
            begin += rest;
            if (++item == per_seq && share) {
                item = 0;
                lspan = Span<KT>(a, seq = min(seq + 1, a.c.batch - 1));
            }
        } else {
            share += place;
            begin -= place;
        }
        place = 0;
    }
    Span<KT> span = lspan;
    // (4 bits: what is wanted at the end lies in shared memory until then, and the products have its registers.)
    const Span<KT> first_span = span;
    const uint32_t first_seq = seq, first_item = item, first_place = place;
    if (F4 && threadIdx.x == 0) {
        meeting.first = Job{seq, item, span.valid ? span.n : kInvalid, span.places(), 0, 0, 0, begin - place};
        meeting.total = line.total;
        meeting.blocks = line.blocks;
    }
    lseq = seq;
    litem = item;
    lrest = share;
    if constexpr (F4) lhead = litem / a.chunks;
    enter(place);
    for (uint32_t s = 0; s < a.stages; ++s) copy_tile();

    uint32_t q_off[NT], c_off[NT][2];   // and of the queries: rows, and the factors of two heads in their padding
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const uint32_t row = min(8 * nt + (F16 ? g : lane & 7), a.q_rows - 1);
        q_off[nt] = query_s + row * S::kQueryRow + (F16 ? 32 * t4 : (lane >> 3) * 16);
#pragma unroll
        for (int e = 0; e < 2; ++e) c_off[nt][e] = query_s + min(8 * nt + 2 * t4 + e, a.q_rows - 1) * S::kQueryRow + 2 * DP;
    }

    // ---- the share, item by item ----
    P p;
    uint32_t kind = share ? kNone : kEmpty;
    uint32_t end_of_first = 0;
    uint64_t i0 = 0;        // where on the line the last item begins
    if (F4 && lane == 0) meeting.left[warp].i0 = 0;
    for (uint32_t at = 0; at < share;) {
        const uint32_t here = place ? min(span.places() - place, share - at) : line.taken(share - at, span.places());
        if (here == 0) break;   // the next warp has it all
        const uint32_t last_tile = max(place + here, kEnd) - kEnd;
        p.clear();
        lay_query();
        float heaviest[NT][2];   // 8-bit caches: the largest weight of a head so far, as p.m is the largest score
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) heaviest[nt][0] = heaviest[nt][1] = F4 ? kLeastWeight4 : kLeastWeight;
        float unit4[NT][2];      // 4 bits: of the weights, and the maxima with a minus, as the last tiles left them
        uint64_t minus4[NT];
        float peak[NT][2];       // the largest score that this lane has seen: p.m may lie kSlack below it
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            peak[nt][0] = peak[nt][1] = -INFINITY;
            unit4[nt][0] = unit4[nt][1] = __uint_as_float(0x7f000000u - __float_as_uint(above(kLeastWeight4)) + (kWeightExponent << 23));
            minus4[nt] = 0;
        }
        for (uint32_t tile = max(place, kEnd) - kEnd; tile < last_tile; ++tile) {
            if (waiting && !mbar_wait_warp(&bars[slot], phase)) {   // (not seen: a copy that never lands)
                if (lane == 0) kstatus_set(a.c.status, FE2O3_KSTATUS_WAIT_EXPIRED);
                waiting = false;
            }
            const uint32_t from = ring + slot * S::kStage;
            // rows of the tile that are keys of the sequence: [ahead, left)
            const uint32_t key0 = span.key(tile), left = span.n - key0, ahead = max(span.first, key0) - key0;
            const bool edge = left < KT || ahead;
            if (edge) {   // the others count nothing: not even what an infinity times 0 would
                if (a.box > 1) {
                    for (uint32_t r = 0; r < KT; ++r)
                        if (r < ahead || r >= left) no_row(slot, r, false);
                    fence_proxy_async_smem();
                }
                __syncwarp();
            }

            // scores: rows are keys, columns heads
            float s[MT][NT][4];
            if constexpr (!F16) {
                float odd[MT][NT][4], low[MT][NT][4];   // every other step: two chains; the lower terms of f32 queries
#pragma unroll
                for (int ks = 0; ks < MD; ks += 2) {
                    uint32_t ka[MT][2][4];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) ldsm4(ka[mt][e], from + k_off[(ks + e) & 3] + (ks >> 2) * KT * 128 + mt * 16 * S::kPitch);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint32_t at_q = q_off[nt] + ks * 32;
                        uint32_t qb[4];
                        ldsm4(qb, at_q);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            if (ks == 0) {
                                mma_first<false>(s[mt][nt], ka[mt][0], qb[0], qb[1]);
                                mma_first<false>(odd[mt][nt], ka[mt][1], qb[2], qb[3]);
                            } else {
                                mma<false>(s[mt][nt], ka[mt][0], qb[0], qb[1]);
                                mma<false>(odd[mt][nt], ka[mt][1], qb[2], qb[3]);
                            }
                        }
                        if (terms > 1) {
#pragma unroll
                            for (int term = 2; term; --term) {
                                ldsm4(qb, at_q + term * term_bytes);
#pragma unroll
                                for (int mt = 0; mt < MT; ++mt) {
                                    if (ks == 0 && term == 2) mma_first<false>(low[mt][nt], ka[mt][0], qb[0], qb[1]);
                                    else mma<false>(low[mt][nt], ka[mt][0], qb[0], qb[1]);
                                    mma<false>(low[mt][nt], ka[mt][1], qb[2], qb[3]);
                                }
                            }
                        }
                    }
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[mt][nt][e] += odd[mt][nt][e];
                            if (terms > 1) s[mt][nt][e] += low[mt][nt][e];
                        }
            } else if constexpr (F4) {
                float low[MT][NT][4];
                constexpr int kAtOnce = MT < 2 ? MT : 2, kRuns = DP == 256 ? 2 : 1, kWords = DP == 64 ? 2 : 4;   // runs of a lane's columns, words of eight in one
                const uint32_t blocks = smem_u32(my_scales) + slot * S::kScales + 8 * KT;
#pragma unroll
                for (int m0 = 0; m0 < MT; m0 += kAtOnce)   // (more rows at once cost registers)
#pragma unroll
                for (int run = 0; run < kRuns; ++run) {
                    uint4 ka[kAtOnce][2];
                    uint32_t ks[kAtOnce][2];   // scales of the run's blocks (of 64 columns one)
#pragma unroll
                    for (int mt = 0; mt < kAtOnce; ++mt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t row = 16 * (m0 + mt) + 8 * e, at = from + k_off[run] + row * S::kPitch, scale = blocks + (row + gk) * row_blocks;
                            if constexpr (DP == 64) {
                                const uint2 v = lds64(at);
                                ka[mt][e] = make_uint4(v.x, v.y, 0, 0);
                                ks[mt][e] = scales_f16(t4 < row_blocks ? lds8(scale + t4) * 0x101u : 0u);
                            } else {
                                ka[mt][e] = lds128(at);
                                ks[mt][e] = scales_f16(2 * t4 + 8 * run < row_blocks ? lds16(scale + 2 * t4 + 8 * run) : 0u);
                            }
                        }
#pragma unroll
                    for (int word = 0; word < kWords; ++word) {
                        uint32_t kf[kAtOnce][2][4];
#pragma unroll
                        for (int mt = 0; mt < kAtOnce; ++mt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const uint4 &v = ka[mt][e];
                                uint32_t h[4];
                                codes4_f16(word == 0 ? v.x : word == 1 ? v.y : word == 2 ? v.z : v.w, h);
                                const uint32_t by = DP == 64 ? ks[mt][e] : __byte_perm(ks[mt][e], 0, word < 2 ? 0x1010 : 0x3232);
                                kf[mt][0][e] = times_f16(h[0], by);
                                kf[mt][0][e + 2] = times_f16(h[1], by);
                                kf[mt][1][e] = times_f16(h[2], by);
                                kf[mt][1][e + 2] = times_f16(h[3], by);
                            }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const int all = 4 * run + word;
                            const bool first = all == 0;
                            const uint32_t at_q = q_off[nt] + 128 * (all >> 1) + 16 * (all & 1);
                            const uint4 qb = lds128(at_q);
#pragma unroll
                            for (int mt = 0; mt < kAtOnce; ++mt) {
                                if (first) mma_first<true>(s[m0 + mt][nt], kf[mt][0], qb.x, qb.y);
                                else mma<true>(s[m0 + mt][nt], kf[mt][0], qb.x, qb.y);
                                mma<true>(s[m0 + mt][nt], kf[mt][1], qb.z, qb.w);
                            }
                            if (terms > 1) {
                                const uint4 ql = lds128(at_q + term_bytes);
#pragma unroll
                                for (int mt = 0; mt < kAtOnce; ++mt) {
                                    if (first) mma_first<true>(low[m0 + mt][nt], kf[mt][0], ql.x, ql.y);
                                    else mma<true>(low[m0 + mt][nt], kf[mt][0], ql.x, ql.y);
                                    mma<true>(low[m0 + mt][nt], kf[mt][1], ql.z, ql.w);
                                }
                            }
                        }
                    }
                }
                if (terms > 1) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[mt][nt][e] += low[mt][nt][e];
                }
            } else {
                float low[MT][NT][4];
#pragma unroll
                for (int j = 0; j < DP / 64; ++j) {   // 64 columns: the lanes of a row hold 16 each, four a step
                    uint4 ka[MT][2];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) ka[mt][e] = lds128(from + k_off[j & 1] + (j >> 1) * KT * 128 + (16 * mt + 8 * e) * S::kPitch);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t kf[MT][2][4];
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const uint32_t w0 = half ? (e ? ka[mt][0].w : ka[mt][0].z) : (e ? ka[mt][0].y : ka[mt][0].x);
                                const uint32_t w1 = half ? (e ? ka[mt][1].w : ka[mt][1].z) : (e ? ka[mt][1].y : ka[mt][1].x);
                                word_f16<FORMAT>(w0, kf[mt][e][0], kf[mt][e][2]);
                                word_f16<FORMAT>(w1, kf[mt][e][1], kf[mt][e][3]);
                            }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const uint32_t at_q = q_off[nt] + 128 * j + 16 * half;
                            const uint4 qb = lds128(at_q);
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) {
                                if (j == 0 && half == 0) mma_first<true>(s[mt][nt], kf[mt][0], qb.x, qb.y);
                                else mma<true>(s[mt][nt], kf[mt][0], qb.x, qb.y);
                                mma<true>(s[mt][nt], kf[mt][1], qb.z, qb.w);
                            }
                            if (terms > 1) {
                                const uint4 ql = lds128(at_q + term_bytes);
#pragma unroll
                                for (int mt = 0; mt < MT; ++mt) {
                                    if (j == 0 && half == 0) mma_first<true>(low[mt][nt], kf[mt][0], ql.x, ql.y);
                                    else mma<true>(low[mt][nt], kf[mt][0], ql.x, ql.y);
                                    mma<true>(low[mt][nt], kf[mt][1], ql.z, ql.w);
                                }
                            }
                        }
                    }
                }
                if (terms > 1) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[mt][nt][e] += low[mt][nt][e];
                }
            }

            // the running maximum, in units of log2; weights
            float vs[MT][2], vs_log[MT][2];   // (4 bits: no logarithms)
            if constexpr (F16) {
                const uint32_t scales = smem_u32(my_scales) + slot * S::kScales + 4 * gk;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float ks = lds_f32(scales + 4 * (16 * mt + 8 * e));
                        vs[mt][e] = lds_f32(scales + 4 * KT + 4 * (16 * mt + 8 * e));
                        if constexpr (!F4) vs_log[mt][e] = lg2_approx(vs[mt][e]);   // (of 0 the lowest there is: such a row weighs nothing)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            float (&x)[4] = s[mt][nt];
                            unpack_f32x2(mul_f32x2(pack_f32x2(x[2 * e], x[2 * e + 1]), pack_f32x2(ks, ks)), x[2 * e], x[2 * e + 1]);
                        }
                    }
            }
            uint32_t pb[MT][NT][3][2];   // weights as the second product's operand, by terms
            uint64_t scale_o[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float c[2] = {lds_f32(c_off[nt][0]), lds_f32(c_off[nt][1])};
                float top[2] = {p.m[nt][0], p.m[nt][1]};
                const uint64_t c2 = pack_f32x2(c[0], c[1]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float (&x)[4] = s[mt][nt];
                    unpack_f32x2(mul_f32x2(pack_f32x2(x[0], x[1]), c2), x[0], x[1]);
                    unpack_f32x2(mul_f32x2(pack_f32x2(x[2], x[3]), c2), x[2], x[3]);
                }
                if (edge) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (16 * mt + 8 * (e >> 1) + gk - ahead >= left - ahead) s[mt][nt][e] = -INFINITY;
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) top[e] = max3(top[e], s[mt][nt][e], s[mt][nt][e + 2]);
                if constexpr (F4) {
                    // Once some tiles are done, a tile seldom moves a maximum or a unit: the lanes look at what they have themselves, and only where
                    // one of them finds more do they compare notes.  (The 8-bit order, both trees at every tile: see below.)
                    float keep[2] = {1.f, 1.f};
                    peak[nt][0] = fmaxf(peak[nt][0], top[0]);
                    peak[nt][1] = fmaxf(peak[nt][1], top[1]);
                    const bool higher = __any_sync(~0u, top[0] > p.m[nt][0] + kSlack || top[1] > p.m[nt][1] + kSlack);
                    if (higher) {
                        float base[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(~0u, top[e], d));
                            base[e] = top[e] == -INFINITY ? 0.f : top[e];
                            keep[e] = ex2_approx(p.m[nt][e] - base[e]);
                            p.m[nt][e] = top[e];
                            p.l[nt][e] *= keep[e];
                        }
                        minus4[nt] = pack_f32x2(-base[0], -base[1]);
                    }
                    float w[MT][4], z[MT][4], largest[2] = {0.f, 0.f};
                    auto weigh = [&] {   // (in this order: a scale of no weight may be beyond f32 in these units)
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                            for (int e = 0; e < 4; e += 2)
                                unpack_f32x2(mul_f32x2(mul_f32x2(pack_f32x2(w[mt][e], w[mt][e + 1]), pack_f32x2(unit4[nt][0], unit4[nt][1])), pack_f32x2(vs[mt][e / 2], vs[mt][e / 2])),
                                             z[mt][e], z[mt][e + 1]);
                    };
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            float x0, x1;
                            unpack_f32x2(add_f32x2(pack_f32x2(s[mt][nt][e], s[mt][nt][e + 1]), minus4[nt]), x0, x1);
                            w[mt][e] = ex2_approx(x0);
                            w[mt][e + 1] = ex2_approx(x1);
                            unpack_f32x2(add_f32x2(pack_f32x2(p.l[nt][0], p.l[nt][1]), pack_f32x2(w[mt][e], w[mt][e + 1])), p.l[nt][0], p.l[nt][1]);
                        }
                    weigh();
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) largest[e] = max3(largest[e], z[mt][e], z[mt][e + 2]);
                    constexpr float kFull = 65504.f;   // f16's largest number: an octave above where the largest weight is put
                    scale_o[nt] = pack_f32x2(1.f, 1.f);
                    if (higher || __any_sync(~0u, largest[0] >= kFull || largest[1] >= kFull)) {
                        float by[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float most = 0.f;
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) most = max3(most, w[mt][e] * vs[mt][0], w[mt][e + 2] * vs[mt][1]);
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
                            const float before = keep[e] * above(heaviest[nt][e]);
                            heaviest[nt][e] = fminf(fmaxf(fmaxf(heaviest[nt][e] * keep[e], most), kLeastWeight4), kMostWeight);
                            const uint32_t inverse = 0x7f000000u - __float_as_uint(above(heaviest[nt][e]));
                            by[e] = before * __uint_as_float(inverse);
                            unit4[nt][e] = __uint_as_float(inverse + (kWeightExponent << 23));
                        }
                        scale_o[nt] = pack_f32x2(by[0], by[1]);
                        weigh();
                    }
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float w0 = z[mt][2 * e], w1 = z[mt][2 * e + 1];
                            const uint32_t hi = f16_pair(w0, w1);
                            pb[mt][nt][0][e] = turned(hi);
                            const float2 h = f16_values(hi);
                            pb[mt][nt][1][e] = turned(f16_pair(w0 - h.x, w1 - h.y));
                        }
                    continue;
                }
                float base[2], keep[2], unit[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(~0u, top[e], d));
                    base[e] = top[e] == -INFINITY ? 0.f : top[e];
                    keep[e] = ex2_approx(p.m[nt][e] - base[e]);
                    p.m[nt][e] = top[e];
                    p.l[nt][e] *= keep[e];
                }
                scale_o[nt] = pack_f32x2(keep[0], keep[1]);
                const uint64_t minus = pack_f32x2(-base[0], -base[1]);
                if constexpr (F16) {   // the output counts in units of a power of two just above the largest weight
                    float weight[2] = {-INFINITY, -INFINITY}, by[2];   // weight: the tile's largest, as a logarithm
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        float (&x)[4] = s[mt][nt];
                        float y[4];
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            const uint64_t score = add_f32x2(pack_f32x2(x[e], x[e + 1]), minus);
                            unpack_f32x2(score, x[e], x[e + 1]);
                            unpack_f32x2(add_f32x2(score, pack_f32x2(vs_log[mt][e / 2], vs_log[mt][e / 2])), y[e], y[e + 1]);
                        }
#pragma unroll
                        for (int e = 0; e < 2; ++e) weight[e] = max3(weight[e], y[e], y[e + 2]);
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) weight[e] = fmaxf(weight[e], __shfl_xor_sync(~0u, weight[e], d));
                        const float before = keep[e] * above(heaviest[nt][e]);
                        heaviest[nt][e] = fminf(fmaxf(fmaxf(heaviest[nt][e] * keep[e], ex2_approx(weight[e])), kLeastWeight), kMostWeight);
                        const uint32_t inverse = 0x7f000000u - __float_as_uint(above(heaviest[nt][e]));
                        by[e] = before * __uint_as_float(inverse);
                        unit[e] = __uint_as_float(inverse + (kWeightExponent << 23));
                    }
                    scale_o[nt] = pack_f32x2(by[0], by[1]);
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        float x0 = s[mt][nt][e], x1 = s[mt][nt][e + 1];
                        if constexpr (!F16) unpack_f32x2(add_f32x2(pack_f32x2(x0, x1), minus), x0, x1);
                        w[e] = ex2_approx(x0);
                        w[e + 1] = ex2_approx(x1);
                        unpack_f32x2(add_f32x2(pack_f32x2(p.l[nt][0], p.l[nt][1]), pack_f32x2(w[e], w[e + 1])), p.l[nt][0], p.l[nt][1]);
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float w0 = w[2 * e], w1 = w[2 * e + 1];
                        if constexpr (F16) {
                            // (in this order: a scale of no weight may be beyond f32 in these units)
                            unpack_f32x2(mul_f32x2(mul_f32x2(pack_f32x2(w0, w1), pack_f32x2(unit[0], unit[1])), pack_f32x2(vs[mt][e], vs[mt][e])), w0, w1);
                            const uint32_t hi = f16_pair(w0, w1);
                            pb[mt][nt][0][e] = turned(hi);
                            const float2 h = f16_values(hi);
                            pb[mt][nt][1][e] = turned(f16_pair(w0 - h.x, w1 - h.y));
                        } else {
                            const uint32_t hi = bf16_pair_cut(w0, w1), least = bf16_least(hi);
                            const float m0 = w0 - cut_bf16(w0), m1 = w1 - cut_bf16(w1);
                            pb[mt][nt][0][e] = turned(hi);
                            pb[mt][nt][1][e] = turned(bf16_max(bf16_pair_cut(m0, m1), least));
                            pb[mt][nt][2][e] = turned(bf16_max(bf16_pair_cut(m0 - cut_bf16(m0), m1 - cut_bf16(m1)), least));
                        }
                    }
                }
            }

            // output: rows are its columns, columns heads; the tile's sum is the tensor unit's, the rest f32
            uint4 v4[F4 ? 1 : MT][4][F16 && DP == 256 ? 2 : 1];
            if constexpr (F4) {
                constexpr int kAtOnce = MT < 2 ? MT : 2, kRuns = DP == 256 ? 2 : 1, kTiles = MD / kRuns;   // kTiles: of a run of the lane's columns
                const uint32_t blocks = smem_u32(my_scales) + slot * S::kScales + 8 * KT + S::kBlocks, k0 = key_of<FORMAT, DP>(2 * t4);
#pragma unroll
                for (int m0 = 0; m0 < MT; m0 += kAtOnce)
#pragma unroll
                    for (int run = 0; run < kRuns; ++run) {
                        const uint32_t block = (DP == 64 ? g >> 1 : g) + 8 * run;
                        uint2 w4[kAtOnce][4];       // the lane's columns of four keys
                        uint32_t vs4[kAtOnce][2];   // and the scales of two keys' blocks
#pragma unroll
                        for (int mt = 0; mt < kAtOnce; ++mt) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t at = from + v_off[(e & 1) + 2 * run] + (16 * (m0 + mt) + 8 * (e >> 1)) * S::kPitch;
                                if constexpr (DP == 64) w4[mt][e] = make_uint2(lds32(at), 0);
                                else w4[mt][e] = lds64(at);
                            }
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const uint32_t at = blocks + (16 * (m0 + mt) + 8 * e) * row_blocks + block;
                                vs4[mt][e] = scales_f16(block < row_blocks ? lds8(at + k0 * row_blocks) | lds8(at + (k0 ^ 1) * row_blocks) << 8 : 0u);
                            }
                        }
                        uint32_t lo4[kAtOnce][2], hi4[kAtOnce][2];   // codes of two keys side by side: even columns, odd ones
#pragma unroll
                        for (int i = 0; i < kTiles; ++i) {
                            uint32_t va[kAtOnce][4];
#pragma unroll
                            for (int mt = 0; mt < kAtOnce; ++mt)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    if (i % 4 == 0) {
                                        const uint32_t w0 = i / 4 ? w4[mt][2 * e].y : w4[mt][2 * e].x, w1 = i / 4 ? w4[mt][2 * e + 1].y : w4[mt][2 * e + 1].x;
                                        lo4[mt][e] = (w0 & 0x0f0f0f0fu) | (w1 << 4 & 0xf0f0f0f0u);
                                        hi4[mt][e] = (w0 >> 4 & 0x0f0f0f0fu) | (w1 & 0xf0f0f0f0u);
                                    }
                                    va[mt][2 * e] = times_f16(code4_pair(lo4[mt][e], i % 4), vs4[mt][e]);
                                    va[mt][2 * e + 1] = times_f16(code4_pair(hi4[mt][e], i % 4), vs4[mt][e]);
                                }
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                float d[4];
#pragma unroll
                                for (int mt = 0; mt < kAtOnce; ++mt) {
                                    if (mt == 0) mma_first<true>(d, va[mt], pb[m0 + mt][nt][1][0], pb[m0 + mt][nt][1][1]);
                                    else mma<true>(d, va[mt], pb[m0 + mt][nt][1][0], pb[m0 + mt][nt][1][1]);
                                    mma<true>(d, va[mt], pb[m0 + mt][nt][0][0], pb[m0 + mt][nt][0][1]);
                                }
                                float (&o)[4] = p.o[run * kTiles + i][nt];
                                const uint64_t d01 = pack_f32x2(d[0], d[1]), d23 = pack_f32x2(d[2], d[3]), o01 = pack_f32x2(o[0], o[1]), o23 = pack_f32x2(o[2], o[3]);
                                unpack_f32x2(m0 ? add_f32x2(o01, d01) : fma_f32x2(o01, scale_o[nt], d01), o[0], o[1]);
                                unpack_f32x2(m0 ? add_f32x2(o23, d23) : fma_f32x2(o23, scale_o[nt], d23), o[2], o[3]);
                            }
                        }
                    }
            } else if constexpr (F16) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (DP == 64) {
                            const uint2 v = lds64(from + v_off[e & 1] + (16 * mt + 8 * (e >> 1)) * S::kPitch);
                            v4[mt][e][0] = make_uint4(v.x, v.y, 0, 0);
                        } else {
#pragma unroll
                            for (int x = 0; x < DP / 128; ++x) v4[mt][e][x] = lds128(from + v_off[e & 1] + x * KT * 128 + (16 * mt + 8 * (e >> 1)) * S::kPitch);
                        }
                    }
            }
#pragma unroll
            for (int i = 0; i < (F4 ? 0 : MD); ++i) {
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
                        ldsm4_trans(va[mt], from + v_off[i & 3] + (i >> 2) * KT * 128 + mt * 16 * S::kPitch);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float d[4];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        if (mt == 0) mma_first<F16>(d, va[mt], pb[mt][nt][1][0], pb[mt][nt][1][1]);
                        else mma<F16>(d, va[mt], pb[mt][nt][1][0], pb[mt][nt][1][1]);
                        if constexpr (!F16) mma<false>(d, va[mt], pb[mt][nt][2][0], pb[mt][nt][2][1]);
                        mma<F16>(d, va[mt], pb[mt][nt][0][0], pb[mt][nt][0][1]);
                    }
                    float (&o)[4] = p.o[i][nt];
                    unpack_f32x2(fma_f32x2(pack_f32x2(o[0], o[1]), scale_o[nt], pack_f32x2(d[0], d[1])), o[0], o[1]);
                    unpack_f32x2(fma_f32x2(pack_f32x2(o[2], o[3]), scale_o[nt], pack_f32x2(d[2], d[3])), o[2], o[3]);
                }
            }
            __syncwarp();   // every lane has read the stage
            if (waiting) {
                if (++slot == a.stages) slot = 0, phase ^= 1;
                copy_tile();
            }
        }

        // the lanes of a row add up
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) p.l[nt][e] += __shfl_xor_sync(~0u, p.l[nt][e], d);
            float back[2] = {1.f, 1.f};
            if constexpr (F4) {   // from here on probabilities are at most 1 again: sums of the largest values stay in range
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) peak[nt][e] = fmaxf(peak[nt][e], __shfl_xor_sync(~0u, peak[nt][e], d));
                    if (peak[nt][e] > p.m[nt][e]) {
                        back[e] = ex2_approx(p.m[nt][e] - peak[nt][e]);
                        p.l[nt][e] *= back[e];
                        p.m[nt][e] = peak[nt][e];
                    }
                }
            }
            if constexpr (F16) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float unit = __uint_as_float(__float_as_uint(above(heaviest[nt][e & 1])) - (kWeightExponent << 23));
                    if constexpr (F4) unit *= back[e & 1];
#pragma unroll
                    for (int i = 0; i < MD; ++i) p.o[i][nt][e] *= unit;
                }
            }
        }
        const bool begins = place == 0, ended = place + here == span.places();
        if constexpr (!F4) i0 = begin + at - place;
        else if (lane == 0) meeting.left[warp].i0 = begin + at - place;
        if (ended) {
            if (!begins) {
                float4 *const to = slots + (warp ? kSlotEnds + warp - 1 : kSlotFirst) * S::kPart * 32;
                p.leave([&](int i, float4 v) { to[i * 32] = v; });
                end_of_first = 1;
            } else if (span.valid) {
                write(p, seq, item, span.n, 0);
            }
        } else {
            kind = begins ? kBegun : kWithin;
        }
        at += here;
        if (at < share) {
            place = 0;
            if (++item == per_seq) {
                item = 0;
                if (++seq >= a.c.batch) break;   // not reached while the lengths stay as they are
                span = Span<KT>(a, seq);
            }
        }
    }
    if (!waiting) {   // what was under way when a wait ran out gets its time; nothing was asked for since
        while ((slot + 1 == a.stages ? 0 : slot + 1) != lslot) {
            if (++slot == a.stages) slot = 0, phase ^= 1;
            mbar_wait_warp(&bars[slot], phase);
        }
    }

    // ---- the block: what its warps left open, each of them a quarter of the columns ----
    float4 *const my_part = reinterpret_cast<float4 *>(my_ring) + lane;   // the ring is free now
    if (kind == kBegun || kind == kWithin) {
        __syncwarp();
        p.leave([&](int i, float4 v) { my_part[i * 32] = v; });
    }
    if (lane == 0) meeting.left[warp] = Left{kind, end_of_first, seq, item, span.valid ? span.n : kInvalid, span.places(), F4 ? meeting.left[warp].i0 : i0};
    if (threadIdx.x < 2) meeting.jobs[threadIdx.x].pieces = 0;
    __threadfence_block();
    __syncthreads();
    constexpr int kQuarter = MD / kPagedWarps;
    Part<kQuarter, NT> part;
    auto add = [&](const float4 *from) {   // a whole part lies there
        part.add([&](int i) { return from[(i < kQuarter * NT ? warp * kQuarter * NT + i : MD * NT + (i - kQuarter * NT)) * 32]; });
    };
    auto leave_quarter = [&](const auto &part, float4 *to) {
        part.leave([&](int i, float4 v) {
            if (i < kQuarter * NT) to[(warp * kQuarter * NT + i) * 32] = v;
            else if (warp == 0) to[(MD * NT + (i - kQuarter * NT)) * 32] = v;
        });
    };
#pragma unroll 1
    for (uint32_t w = 0; w < kPagedWarps; ++w) {   // an item that warp w was the first of the block to leave open
        const Left left = meeting.left[w];
        if (left.kind != kBegun && (left.kind != kWithin || w)) continue;
        part.clear();
        add(reinterpret_cast<const float4 *>(smem + w * a.stages * S::kStage) + lane);
        bool open = true;
#pragma unroll 1
        for (uint32_t v = w + 1; v < kPagedWarps && open; ++v) {
            const Left &other = meeting.left[v];
            if (other.kind != kWithin && !other.end_of_first) continue;   // (no places)
            open = other.kind == kWithin;
            add(open ? reinterpret_cast<const float4 *>(smem + v * a.stages * S::kStage) + lane : slots + (kSlotEnds + v - 1) * S::kPart * 32);
        }
        if (left.kind == kBegun && !open) {
            if (left.n != kInvalid) write(part, left.seq, left.item, left.n, warp * kQuarter);
        } else {
            leave_quarter(part, slots + (left.kind == kBegun ? kSlotLast : kSlotFirst) * S::kPart * 32);
            if (threadIdx.x == 0) meeting.jobs[left.kind == kBegun] = Job{left.seq, left.item, left.n, left.places, 0, 0, 0, left.i0};
        }
    }
    if (threadIdx.x == 0 && end_of_first)   // an item of an earlier block that ended in warp 0: it lies in its slot
        meeting.jobs[0] = F4 ? meeting.first : Job{first_seq, first_item, first_span.valid ? first_span.n : kInvalid, first_span.places(), 0, 0, 0, begin - first_place};

    // ---- the blocks: the last one to come joins the pieces, of many pieces in two steps: 16 neighbours, then those ----
    __threadfence();
    __syncthreads();
    if (threadIdx.x < 2) {
        Job &job = meeting.jobs[threadIdx.x];
        if (job.pieces) {
            const uint64_t total = F4 ? meeting.total : line.total;
            const uint32_t blocks = F4 ? meeting.blocks : line.blocks;
            const uint32_t b0 = Line::block_of(job.i0, total, blocks), pieces = Line::block_of(job.i0 + job.pieces - 1, total, blocks) - b0 + 1;
            const uint32_t group = (blockIdx.x - b0) / kGroup, groups = (pieces + kGroup - 1) / kGroup;
            job.block = b0;
            job.first = b0 + group * kGroup;
            job.groups = groups;
            job.pieces = min(kGroup, pieces - group * kGroup);
            // (a block may be in the first group of one item and begin the second, or a later, of another)
            uint32_t *const count = a.arrived + (group ? gridDim.x : 0) + job.first;
            if (atomicAdd(count, 1u) == job.pieces - 1) *count = 0;
            else job.pieces = 0;
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int role = 0; role < 2; ++role) {
        const Job job = meeting.jobs[role];
        if (!job.pieces) continue;
        uint32_t from = job.first, step = 1, n = job.pieces;
        auto slot_of = [&](uint32_t block) { return a.slots + ((uint64_t)block * kPagedSlots + (block == job.block ? kSlotLast : kSlotFirst)) * S::kPart * 32 + lane; };
        for (bool whole = job.groups == 1;; whole = true) {
            __threadfence();
            part.clear();
            constexpr int kAtOnce = kQuarter * NT <= 2 ? 8 : kQuarter * NT <= 4 ? 4 : 2, kLoads = (kQuarter + 1) * NT;
#pragma unroll 1
            for (uint32_t i = 0; i < n; i += kAtOnce) {
                float4 v[kAtOnce][kLoads];
#pragma unroll
                for (int x = 0; x < kAtOnce; ++x) {   // (beyond the last one: that again, which is not added)
                    const float4 *const at = slot_of(from + min(i + x, n - 1) * step);
#pragma unroll
                    for (int k = 0; k < kLoads; ++k) v[x][k] = __ldcg(at + (k < kQuarter * NT ? warp * kQuarter * NT + k : MD * NT + (k - kQuarter * NT)) * 32);
                }
#pragma unroll
                for (int x = 0; x < kAtOnce; ++x)
                    if (i + x < n) part.add([&](int k) { return v[x][k]; });
            }
            if (whole) {
                if (job.n != kInvalid) write(part, job.seq, job.item, job.n, warp * kQuarter);
                break;
            }
            __syncthreads();   // (all warps have read the first piece's maxima)
            leave_quarter(part, slot_of(from));
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                uint32_t *const count = a.arrived + 2 * gridDim.x + job.block;
                meeting.goes_on = atomicAdd(count, 1u) == job.groups - 1;
                if (meeting.goes_on) *count = 0;
            }
            __syncthreads();
            if (!meeting.goes_on) break;
            from = job.block;
            step = kGroup;
            n = job.groups;
        }
    }
}

template <uint32_t FORMAT, int DP, int NT, bool LONG = false>
PagedBuild paged_build() {
    using S = Shape<FORMAT, DP, NT, LONG>;
    return PagedBuild{paged_attention_kernel<FORMAT, DP, NT, LONG>, (uint32_t)S::kStage, (uint32_t)S::kPart * 512u, (uint32_t)S::kQueryRow,
                      (uint32_t)S::kScales, (uint32_t)S::kKeys};
}
template <uint32_t FORMAT>
PagedBuild paged_build_for(uint32_t dim, uint32_t nt) {
    if (dim <= 64) return nt == 1 ? paged_build<FORMAT, 64, 1>() : paged_build<FORMAT, 64, 2>();
    if (dim <= 128) return nt == 1 ? paged_build<FORMAT, 128, 1>() : paged_build<FORMAT, 128, 2>();
    return nt == 1 ? paged_build<FORMAT, 256, 1>() : paged_build<FORMAT, 256, 2>();
}

}  // namespace
