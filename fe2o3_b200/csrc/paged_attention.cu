// Plans and launches of attention over a paged key-value cache (the kernel: paged_attention.cuh).
#include <mutex>
#include <new>

#include "gemm_tc.h"
#include "paged_attention.cuh"

// Workspaces of one device: pieces of slabs that stay until the process ends, so that preparing a launch seldom waits for
// the allocator (half a millisecond to tens of them).  Pieces are powers of two from 64 KiB on, and what is given back goes to the next
// plan of the same power: a program that prepares for many geometries, a few at a time, keeps a few pieces of each.
namespace {

struct Workspaces {
    struct Piece {
        void *at;
        size_t bytes;
        Piece *next;
    };
    std::mutex lock;
    Piece *returned = nullptr;
    uint8_t *slab = nullptr;
    size_t left = 0;

    static size_t size_of(size_t bytes) {
        size_t size = 65536;
        while (size < bytes) size *= 2;
        return size;
    }
    cudaError_t take(size_t bytes, void **out) {   // (bytes as size_of gives them)
        std::lock_guard<std::mutex> held(lock);
        for (Piece **p = &returned; *p; p = &(*p)->next) {
            if ((*p)->bytes != bytes) continue;
            Piece *const found = *p;
            *out = found->at;
            *p = found->next;
            delete found;
            return cudaSuccess;
        }
        if (bytes > left) {
            const size_t size = bytes > (64u << 20) ? bytes : 64u << 20;
            void *fresh = nullptr;
            const cudaError_t e = cudaMalloc(&fresh, size);
            if (e != cudaSuccess) return e;
            for (size_t part = 64u << 20; part >= 65536; part /= 2)   // what is left of the last one, as pieces
                while (left >= part) {
                    put(slab, part);
                    slab += part;
                    left -= part;
                }
            slab = static_cast<uint8_t *>(fresh);
            left = size;
        }
        *out = slab;
        slab += bytes;
        left -= bytes;
        return cudaSuccess;
    }
    void give(void *at, size_t bytes) {   // no launch uses it any more
        std::lock_guard<std::mutex> held(lock);
        put(at, bytes);
    }

private:
    void put(void *at, size_t bytes) {
        Piece *const p = new (std::nothrow) Piece{at, bytes, returned};
        if (p) returned = p;
    }
};
Workspaces *workspaces_of(int device) {
    static Workspaces all[64];
    return device >= 0 && device < 64 ? &all[device] : nullptr;
}

}  // namespace

struct PagedPlan {
    CUtensorMap map_k, map_v;
    int device;
    size_t bytes;
    PagedKernel kernel;
    PagedArgs args;
    uint32_t grid, shared;
    void *workspace;
};

void paged_attention_free(PagedPlan *p) {
    if (!p) return;
    if (p->workspace) {
        // a launch in flight may still use it; when the device cannot say, the workspace is not used again
        int current = -1;
        cudaGetDevice(&current);
        if (current != p->device) cudaSetDevice(p->device);
        if (cudaDeviceSynchronize() == cudaSuccess) workspaces_of(p->device)->give(p->workspace, p->bytes);
        if (current >= 0 && current != p->device) cudaSetDevice(current);
    }
    delete p;
}
void paged_attention_geometry(const PagedPlan *p, fe2o3_geometry *geo) {
    *geo = fe2o3_geometry{{p->grid, 1, 1}, {kPagedThreads, 1, 1}, p->shared, 1};
}

int32_t paged_attention_plan(fe2o3_ctx *ctx, const fe2o3_paged_attention_v1_args *a, PagedPlan **out) {
    const uint32_t group = a->heads / a->kv_heads;
    // 16 query heads at once for a group of more than 8 (three terms of f32 queries of such long rows would not fit a block)
    const uint32_t nt = group <= 8 || (a->dim > 128 && a->format == FE2O3_KV_BF16 && a->q_dtype == FE2O3_DTYPE_F32) ? 1 : 2;
    const PagedBuild b = a->format == FE2O3_KV_BF16 ? paged_build_bf16(a->dim, nt) : a->format == FE2O3_KV_E4M3 ? paged_build_e4m3(a->dim, nt) : paged_build_i8(a->dim, nt);
    const uint32_t terms = a->q_dtype == FE2O3_DTYPE_BF16 ? 1 : a->format == FE2O3_KV_BF16 ? 3 : 2;
    FE2O3_CUDA(cudaSetDevice(ctx->device));
    cudaFuncAttributes attr;
    FE2O3_CUDA(cudaFuncGetAttributes(&attr, reinterpret_cast<const void *>(b.kernel)));
    // as many blocks an SM as registers and two stages a warp allow, then as many stages as fit; a partial result has to fit a
    // warp's ring.  Full stages of bf16 rows: two blocks of three stages (32 sequences of 4096, 32 heads of 128 on 8: 95 us, three
    // blocks of two 101; 64 ragged ones 100 and 105; two of 131071 178 and 181).  Rows of 112 columns take 94 us so and 92 with three
    // blocks, of 96 columns 94 and 77, pages that take several boxes a tile 101 and 99, e4m3 135 and 113, i8 147 and 131.
    const uint32_t q_rows = group < 8 * nt ? group + 1 : 8 * nt;
    const uint32_t fixed = kPagedWarps * terms * q_rows * b.query + kPagedMeeting, least = b.part > 2 * b.stage ? (b.part + b.stage - 1) / b.stage : 2;
    auto stages_of = [&](uint32_t blocks) -> uint32_t {   // 0: not so many blocks
        const uint32_t room = 233472 / blocks - 1024;   // an SM's, less what the system keeps of each block's
        if (blocks > 1 && (uint32_t)attr.numRegs * kPagedThreads * blocks > 65536) return 0;
        const uint32_t fit = room < fixed ? 0 : (room - fixed) / (kPagedWarps * (b.stage + b.scales));
        return fit < least ? 0 : fit;
    };
    uint32_t stages = a->format == FE2O3_KV_BF16 && a->dim == 128 && a->page_size % b.keys == 0 && stages_of(2) >= 3 ? stages_of(2) : 0;
    for (uint32_t blocks = 3; blocks && !stages; --blocks) stages = stages_of(blocks);
    if (!stages) return FE2O3_ERR_UNSUPPORTED_SHAPE;   // (not reached: one block fits for every build)
    if (stages > kPagedMaxStages) stages = kPagedMaxStages;
    PagedPlan *p = new (std::nothrow) PagedPlan();
    if (!p) return FE2O3_ERR_SIZE_OVERFLOW;
    p->kernel = b.kernel;
    p->shared = kPagedWarps * stages * (b.stage + b.scales) + fixed;
    int per_sm = 0;
    cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void *>(b.kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);   // (all: plans of one kernel differ)
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, b.kernel, kPagedThreads, p->shared);
    const uint32_t at_once = (uint32_t)(per_sm > 0 ? per_sm : 1) * ctx->sm_count;
    p->grid = at_once;
    // no more blocks than sequences that fill their rows of the table give work to (kEnd and a tile begun come on top)
    const double tiles = (double)a->table_width * a->page_size / b.keys + 4;
    const double most = tiles * a->batch * a->kv_heads * ((group + 8 * nt - 1) / (8 * nt)) / kPagedWarps;
    if (most < p->grid) p->grid = most < 1 ? 1 : (uint32_t)most;
    const size_t slots = (size_t)kPagedSlots * p->grid * b.part;   // behind them: counters
    p->device = ctx->device;
    p->bytes = Workspaces::size_of(slots + 3 * p->grid * sizeof(uint32_t));
    Workspaces *const workspaces = workspaces_of(ctx->device);
    if (e == cudaSuccess) e = workspaces ? workspaces->take(p->bytes, &p->workspace) : cudaErrorInvalidDevice;
    if (e == cudaSuccess) e = cudaMemset(static_cast<uint8_t *>(p->workspace) + slots, 0, 3 * p->grid * sizeof(uint32_t));
    if (e == cudaSuccess) e = cudaStreamSynchronize(cudaStreamLegacy);   // no other stream is ordered behind the clear
    if (e != cudaSuccess) {
        paged_attention_free(p);
        return fe2o3_cuda_status(e, "paged_attention_v1 workspace");
    }
    p->args.c = kv_cache_of(ctx, a);
    const uint32_t qb = a->q_dtype == FE2O3_DTYPE_F32 ? 4 : 2;
    const bool whole = a->q.ptr % 16 == 0 && (uint64_t)a->q_stride * qb % 16 == 0 && (uint64_t)a->q_head_stride * qb % 16 == 0;
    // boxes of the copy engine: rows that no page's end cuts, of whole swizzle patterns
    uint32_t box = b.keys;
    while (a->page_size % box) box /= 2;
    if (box < 8 || p->args.c.pages == 0 || (a->format != FE2O3_KV_BF16 && ((a->k_scales.ptr | a->v_scales.ptr) & 15u))) box = 1;
    if (box > 1) {
        const uint32_t eb = a->format == FE2O3_KV_BF16 ? 2 : 1, columns = eb == 2 ? 64 : a->dim <= 64 ? 64 : 128;
        const uint64_t dims[3] = {a->dim, a->page_size, (uint64_t)p->args.c.pages * a->kv_heads};
        const uint64_t strides[2] = {(uint64_t)a->dim * eb, (uint64_t)a->dim * eb * a->page_size};
        const uint32_t shape[3] = {columns, box, 1};
        const auto make = eb == 2 ? fe2o3_make_tmap_bf16 : fe2o3_make_tmap_u8;
        if (make(&p->map_k, a->k_cache.ptr, 3, dims, strides, shape) != FE2O3_OK || make(&p->map_v, a->v_cache.ptr, 3, dims, strides, shape) != FE2O3_OK) box = 1;
    }
    uint32_t *const counters = reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(p->workspace) + slots);
    int32_t shift = -1;
    if ((a->page_size & (a->page_size - 1)) == 0) shift = __builtin_ctz(a->page_size);
    p->args = PagedArgs{kv_cache_of(ctx, a), reinterpret_cast<const void *>(a->q.ptr), reinterpret_cast<void *>(a->output.ptr),
                        reinterpret_cast<float *>(a->lse.ptr), static_cast<float4 *>(p->workspace),
                        counters, group, (group + 8 * nt - 1) / (8 * nt),
                        a->q_stride, a->q_head_stride, a->window, stages, q_rows, at_once, shift, box, a->scale, a->q_dtype == FE2O3_DTYPE_F32,
                        a->output_dtype == FE2O3_DTYPE_F32, whole};
    *out = p;
    return FE2O3_OK;
}

int32_t paged_attention_launch(const PagedPlan *p, cudaStream_t s) {
    if (p->args.c.batch == 0) return FE2O3_OK;
    const cudaError_t e = fe2o3_launch_early(p->kernel, p->grid, kPagedThreads, p->shared, s, 1, p->map_k, p->map_v, p->args);
    fe2o3_count_launch(1);
    return fe2o3_cuda_status(e, "paged_attention_v1");
}
