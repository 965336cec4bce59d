// Page tables and slot maps of a step, planned on the device; the rules stand at fe2o3_kv_pages_v1_args.
//
// Latency-bound: a step of some hundred sequences moves a few KB, prompts of 131072 tokens 1 MB of slots and positions.  One launch: a
// block with a token a thread, or a cluster of kBlocks blocks.  Every block adds up all sequences for itself (pages that come back, new
// pages, new tokens), so that each knows whether the step fits before anything is written; blocks meet once, when all have read what is
// replaced in place and the released pages lie on the stack.  Then pages and tokens are dealt out evenly, whatever sequence
// they are of: a thread finds the sequence of its first token by bisection in shared memory and goes on from there.  The page
// of a position comes from the table's row or straight from the stack, so tables and slots are written at the same time.
// A step of 48 sequences 3.3 us, where an empty launch takes 3; 131072 tokens of 512 sequences, 61 of which leave their pages, 10.7 us
// (eight blocks, four tokens a thread and a warp to every released sequence: 37; eight tokens a thread 19; sixteen blocks 10.7).  What is left is a chain of trips
// to memory, lengths, table, stack, and 1100 instructions a warp on sixteen SMs.  More blocks in one launch would need a meeting in memory
// that stays between launches, which two captured graphs would share; positions and slots could be a second launch's, over all SMs, from what the first has
// written.
#include "common.cuh"

namespace {

constexpr uint32_t kMostSequences = 8192, kMaxThreads = 1024, kBlocks = 16;

struct PagesArgs {
    const uint32_t *counts, *release, *lengths, *free_count;
    uint32_t *table, *free_pages, *next_lengths, *next_free_count, *offsets, *positions, *slots, *attended, *status;
    uint32_t batch, width, page_size, tokens, pages;
    int32_t shift;   // log2 of page_size, or negative
};

// A sequence as it comes in: pages it gives back, its length after that, its new tokens, its pages then and in the end.
struct Sequence {
    uint32_t back, length, count, held, need;
    bool fits;
};

__device__ __forceinline__ uint32_t page_of(const PagesArgs &a, uint32_t position) { return a.shift >= 0 ? position >> a.shift : position / a.page_size; }
__device__ __forceinline__ uint32_t pages_for(const PagesArgs &a, uint32_t length) { return length ? page_of(a, length - 1) + 1 : 0; }

__device__ __forceinline__ Sequence sequence_of(const PagesArgs &a, uint32_t b) {
    Sequence s{0, a.lengths[b], 0, 0, 0, true};
    uint32_t pages = pages_for(a, s.length);
    s.fits = s.length <= 0x7fffffffu && pages <= a.width;
    if (a.release && a.release[b]) {
        s.back = pages;
        s.length = pages = 0;
    }
    s.held = pages;
    s.count = a.counts ? a.counts[b] : s.length ? 1 : 0;
    const uint64_t after = (uint64_t)s.length + s.count;
    s.fits = s.fits && after <= 0x7fffffffu;
    s.need = s.fits ? pages_for(a, (uint32_t)after) : 0;
    s.fits = s.fits && s.need <= a.width;
    return s;
}

struct Sums {   // (pages of sequences that fit are fewer than the table's entries, which 32 bits count)
    uint32_t back, fresh;
    uint64_t tokens;
    __device__ __forceinline__ Sums operator+(const Sums &o) const { return {back + o.back, fresh + o.fresh, tokens + o.tokens}; }
};

// What a sequence's pages and tokens are found by, in shared memory.
struct Place {
    uint32_t length, first_page, first_token, first_back;
};

template <uint32_t kAtOnce>   // tokens that a thread writes at once
__global__ void __launch_bounds__(kMaxThreads) kv_pages_kernel(PagesArgs a) {
    extern __shared__ Place places[];   // [batch]
    __shared__ Sums warps[32];
    __shared__ Sums carry;
    __shared__ uint32_t bad;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t thread = blockIdx.x * blockDim.x + threadIdx.x, threads = gridDim.x * blockDim.x;
    if (threadIdx.x == 0) {
        carry = Sums{0, 0, 0};
        bad = 0;
    }
    begin_after_previous();
    __syncthreads();
    const uint32_t count = *a.free_count;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += blockDim.x) {
        const uint32_t b = b0 + threadIdx.x;
        Sequence s{0, 0, 0, 0, 0, true};
        if (b < a.batch) s = sequence_of(a, b);
        if (!s.fits) bad = 1;
        const Sums own{s.fits ? s.back : 0, s.fits ? s.need - s.held : 0, s.count};
        Sums sum = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const Sums up{__shfl_up_sync(~0u, sum.back, d), __shfl_up_sync(~0u, sum.fresh, d), __shfl_up_sync(~0u, sum.tokens, d)};
            if (lane >= d) sum = sum + up;
        }
        if (lane == 31) warps[warp] = sum;
        __syncthreads();
        Sums before = carry;
        for (uint32_t w = 0; w < warp; ++w) before = before + warps[w];
        sum = before + sum;
        if (b < a.batch) places[b] = Place{s.length, sum.fresh - own.fresh, (uint32_t)(sum.tokens - own.tokens), sum.back - own.back};
        __syncthreads();
        if (threadIdx.x == blockDim.x - 1) carry = sum;
    }
    __syncthreads();
    const Sums total = carry;
    const bool too_long = bad || total.tokens > 0xffffffffull || (a.counts && (a.positions || a.slots) && total.tokens > a.tokens);
    const uint64_t top = (uint64_t)count + total.back;
    const bool fits = !too_long && top <= a.pages && total.fresh <= top;
    if (!fits && thread == 0) kstatus_set(a.status, too_long ? FE2O3_KSTATUS_LENGTH : FE2O3_KSTATUS_PAGES);

    // the last sequence that begins at or before x
    auto find = [&](uint32_t x, uint32_t Place::*first) {
        uint32_t low = 0, high = a.batch;
        while (high - low > 1) {
            const uint32_t mid = (low + high) / 2;
            if (places[mid].*first <= x) low = mid;
            else high = mid;
        }
        return low;
    };
    if (fits)   // the released pages: place i on the stack, of a row of n entries, is its entry n - 1 - i
        for (uint32_t i = thread; i < total.back; i += threads) {
            const uint32_t b = find(i, &Place::first_back), end = b + 1 < a.batch ? places[b + 1].first_back : total.back;
            a.free_pages[count + i] = a.table[(uint64_t)b * a.width + (end - 1 - i)];
        }
    if (gridDim.x > 1) {
        __threadfence();
        cluster_sync();
    } else {
        __syncthreads();
    }

    // what the sequences become
    if (a.offsets && thread == 0) a.offsets[a.batch] = fits ? (uint32_t)total.tokens : 0;
    if (thread == 0) *a.next_free_count = fits ? (uint32_t)(top - total.fresh) : count;
    for (uint32_t b = thread; b < a.batch; b += threads) {
        const uint32_t end = b + 1 < a.batch ? places[b + 1].first_token : (uint32_t)total.tokens;
        const uint32_t length = places[b].length + (end - places[b].first_token);
        if (fits) a.next_lengths[b] = length;
        else if (a.next_lengths != a.lengths) a.next_lengths[b] = a.lengths[b];
        if (a.attended) a.attended[b] = fits ? length : 0;
        if (a.offsets) a.offsets[b] = fits ? places[b].first_token : 0;
    }
    if (fits)
        for (uint32_t i = thread; i < total.fresh; i += threads) {
            const uint32_t b = find(i, &Place::first_page);
            a.table[(uint64_t)b * a.width + pages_for(a, places[b].length) + (i - places[b].first_page)] = a.free_pages[top - 1 - i];
        }
    if (!a.positions && !a.slots) return;
    const uint32_t tokens = !fits ? 0 : a.counts ? (uint32_t)total.tokens : a.batch;   // (without counts row b is sequence b's)
    const bool whole = ((reinterpret_cast<uint64_t>(a.positions) | reinterpret_cast<uint64_t>(a.slots)) & 15) == 0;
    for (uint64_t t0 = (uint64_t)thread * kAtOnce; t0 < a.tokens; t0 += (uint64_t)threads * kAtOnce) {
        uint32_t position[kAtOnce], slot[kAtOnce];
        const uint32_t *from[kAtOnce];   // the number of the position's page
        uint32_t b = t0 >= tokens ? 0 : a.counts ? find((uint32_t)t0, &Place::first_token) : (uint32_t)t0;
        Place p{0, 0, 0, 0};
        uint32_t end = 0, held = 0;
        if (t0 < tokens) {
            p = places[b];
            end = !a.counts ? b + 1 : b + 1 < a.batch ? places[b + 1].first_token : tokens;
            held = pages_for(a, p.length);
        }
#pragma unroll
        for (uint32_t i = 0; i < kAtOnce; ++i) {
            const uint32_t t = (uint32_t)t0 + i;
            position[i] = 0;
            slot[i] = FE2O3_SLOT_NONE;
            from[i] = nullptr;
            if (t0 + i >= tokens) continue;
            while (t >= end) {
                p = places[++b];
                end = !a.counts ? b + 1 : b + 1 < a.batch ? places[b + 1].first_token : tokens;
                held = pages_for(a, p.length);
            }
            if (!a.counts && !p.length) continue;
            position[i] = p.length + (a.counts ? t - p.first_token : 0);
            const uint32_t page = page_of(a, position[i]);
            from[i] = page < held ? a.table + (uint64_t)b * a.width + page : a.free_pages + (top - 1 - p.first_page - (page - held));
            slot[i] = position[i] - page * a.page_size;
        }
#pragma unroll
        for (uint32_t i = 0; i < kAtOnce; ++i) {
            if (!from[i]) continue;
            const uint32_t number = *from[i];
            if (number < a.pages) {
                slot[i] += number * a.page_size;
            } else {
                slot[i] = FE2O3_SLOT_NONE;
                kstatus_set(a.status, FE2O3_KSTATUS_SLOT_RANGE);
            }
        }
        auto put = [&](uint32_t *to, const uint32_t (&v)[kAtOnce]) {
            if (!to) return;
            if (kAtOnce % 4 == 0 && whole && t0 + kAtOnce <= a.tokens) {
#pragma unroll
                for (uint32_t i = 0; i + 3 < kAtOnce; i += 4) *reinterpret_cast<uint4 *>(to + t0 + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            } else {
#pragma unroll
                for (uint32_t i = 0; i < kAtOnce; ++i)
                    if (t0 + i < a.tokens) to[t0 + i] = v[i];
            }
        };
        put(a.positions, position);
        put(a.slots, slot);
    }
}

}  // namespace

int32_t launch_kv_pages(fe2o3_ctx *ctx, cudaStream_t s, const void *args, fe2o3_geometry *geo, bool plan_only) {
    const fe2o3_kv_pages_v1_args *a = static_cast<const fe2o3_kv_pages_v1_args *>(args);
    // one block for as many tokens and sequences as it has threads, a thread each; else a cluster, eight tokens a thread
    const uint32_t work = a->batch > a->tokens ? a->batch : a->tokens, threads = work <= 256 ? 256 : work <= 512 ? 512 : kMaxThreads;
    const bool one = work <= kMaxThreads;
    const uint32_t grid = one ? 1 : kBlocks, shared = a->batch * (uint32_t)sizeof(Place);
    const auto kernel = one ? kv_pages_kernel<1> : kv_pages_kernel<8>;
    if (geo) *geo = fe2o3_geometry{{grid, 1, 1}, {threads, 1, 1}, shared, 1};
    if (plan_only) {
        FE2O3_CUDA(cudaSetDevice(ctx->device));
        for (const auto each : {kv_pages_kernel<1>, kv_pages_kernel<8>}) {   // (both: a patched batch or number of tokens may take the other)
            FE2O3_CUDA(cudaFuncSetAttribute(reinterpret_cast<const void *>(each), cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSequences * sizeof(Place)));
            FE2O3_CUDA(cudaFuncSetAttribute(reinterpret_cast<const void *>(each), cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        }
        return FE2O3_OK;
    }
    int32_t shift = -1;
    if ((a->page_size & (a->page_size - 1)) == 0) shift = __builtin_ctz(a->page_size);
    auto at = [](const fe2o3_slice &x) { return reinterpret_cast<uint32_t *>(x.ptr); };
    const PagesArgs p{at(a->counts), at(a->release), at(a->lengths), at(a->free_count), at(a->page_table), at(a->free_pages), at(a->next_lengths),
                      at(a->next_free_count), at(a->token_offsets), at(a->positions), at(a->slots), at(a->attended), ctx->status_word, a->batch, a->table_width,
                      a->page_size, a->tokens, (uint32_t)a->free_pages.len, shift};
    const cudaError_t e = fe2o3_launch_early(kernel, grid, threads, shared, s, grid, p);
    fe2o3_count_launch(1);
    return fe2o3_cuda_status(e, "kv_pages_v1");
}

static Fe2o3KernelRegistration reg_pages("kv_pages_v1", reinterpret_cast<const void *>(kv_pages_kernel<1>));
