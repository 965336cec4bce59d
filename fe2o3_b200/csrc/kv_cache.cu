// Paged key-value cache: new rows written (rounded or quantised) and rows read back.  The formulas stand at
// fe2o3_kv_cache_append_v1_args and fe2o3_kv_cache_read_v1_args.
#include "kv_cache.cuh"

namespace {

constexpr int kThreads = 256;

struct KvRows {
    void *p[2];   // k, v: sources of an append, destinations of a read
    uint32_t token_stride[2], head_stride[2];
    const uint32_t *offsets;
    uint32_t tokens;
    bool f32;
};

// Sequence and position of a token's row; false (reported) where the sequence's length does not allow it.
__device__ __forceinline__ bool place_of(const KvCache &c, const KvRows &r, uint32_t t, uint32_t &b, uint32_t &position) {
    uint32_t before = 1, own = 1;   // new tokens of the sequence: from this one on, and all
    b = t;
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
    position = length - before;
    return true;
}

// One block a token, a warp for each head's row of K and of V.
template <uint32_t FORMAT>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(KvCache c, KvRows r) {
    begin_after_previous();
    const uint32_t t = blockIdx.x, lane = threadIdx.x & 31;
    uint32_t b, position;
    if (!place_of(c, r, t, b, position)) return;
    for (uint32_t w = threadIdx.x >> 5; w < 2 * c.kv_heads; w += kThreads / 32) {
        const uint32_t side = w & 1, h = w >> 1;
        const uint32_t row = kv_row(c, b, h, position);
        if (row == ~0u) continue;
        const uint64_t from = (uint64_t)t * r.token_stride[side] + (uint64_t)h * r.head_stride[side];
        float x[8], top = 0.f;
        bool finite = true;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            const uint32_t at = lane + 32 * i;
            x[i] = at >= c.dim ? 0.f : r.f32 ? static_cast<const float *>(r.p[side])[from + at]
                                            : bf16_bits_to_f32(static_cast<const uint16_t *>(r.p[side])[from + at]);
            finite = finite && isfinite(x[i]);
            top = fmaxf(top, fabsf(x[i]));
        }
        uint8_t *to = (side ? c.v : c.k) + (uint64_t)row * c.dim * kKvBytes<FORMAT>;
        if constexpr (FORMAT == FE2O3_KV_BF16) {
            for (uint32_t i = 0; i < 8; ++i)
                if (lane + 32 * i < c.dim) reinterpret_cast<uint16_t *>(to)[lane + 32 * i] = f32_to_bf16_bits(x[i]);
        } else {
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
            finite = __all_sync(~0u, finite);
            const float scale = finite ? __fdiv_rn(top, kKvTop<FORMAT>) : __int_as_float(0x7fc00000);
            for (uint32_t i = 0; i < 8; ++i) {
                if (lane + 32 * i >= c.dim) continue;
                const float y = scale > 0.f ? __fdiv_rn(x[i], scale) : 0.f;
                to[lane + 32 * i] = FORMAT == FE2O3_KV_E4M3 ? f32_to_e4m3(y) : (uint8_t)(int8_t)fminf(fmaxf(rintf(y), -127.f), 127.f);
            }
            if (lane == 0) (side ? c.v_scales : c.k_scales)[row] = scale;
        }
    }
}

template <uint32_t FORMAT>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(KvCache c, KvRows r) {
    begin_after_previous();
    const uint32_t t = blockIdx.x, lane = threadIdx.x & 31;
    uint32_t b, position;
    if (!place_of(c, r, t, b, position)) return;
    for (uint32_t w = threadIdx.x >> 5; w < 2 * c.kv_heads; w += kThreads / 32) {
        const uint32_t side = w & 1, h = w >> 1;
        const uint32_t row = kv_row(c, b, h, position);
        const uint64_t to = (uint64_t)t * r.token_stride[side] + (uint64_t)h * r.head_stride[side];
        const uint8_t *from = (side ? c.v : c.k) + (uint64_t)(row == ~0u ? 0 : row) * c.dim * kKvBytes<FORMAT>;
        const float scale = FORMAT == FE2O3_KV_BF16 ? 1.f : row == ~0u ? 0.f : (side ? c.v_scales : c.k_scales)[row];
        for (uint32_t i = lane; i < c.dim; i += 32) {
            const float v = row == ~0u ? 0.f : __fmul_rn(kv_element<FORMAT>(from, i), scale);
            if (r.f32) static_cast<float *>(r.p[side])[to + i] = v;
            else static_cast<uint16_t *>(r.p[side])[to + i] = f32_to_bf16_bits(v);
        }
    }
}

template <typename Args>
KvRows rows_of(const Args *a, uint32_t dtype) {
    return KvRows{{reinterpret_cast<void *>(a->k.ptr), reinterpret_cast<void *>(a->v.ptr)},
                  {a->k_token_stride, a->v_token_stride},
                  {a->k_head_stride, a->v_head_stride},
                  reinterpret_cast<const uint32_t *>(a->token_offsets.ptr),
                  a->tokens,
                  dtype == FE2O3_DTYPE_F32};
}

template <typename Args>
int32_t launch_rows(fe2o3_ctx *ctx, cudaStream_t s, const Args *a, uint32_t dtype, fe2o3_geometry *geo, bool plan_only,
                    void (*const kernels[3])(KvCache, KvRows), const char *what) {
    if (geo) *geo = fe2o3_geometry{{a->tokens, 1, 1}, {kThreads, 1, 1}, 0, 1};
    if (plan_only || a->tokens == 0) return FE2O3_OK;
    const cudaError_t e = fe2o3_launch_early(kernels[a->format], a->tokens, kThreads, 0, s, 1, kv_cache_of(ctx, a), rows_of(a, dtype));
    fe2o3_count_launch(1);
    return fe2o3_cuda_status(e, what);
}

}  // namespace

int32_t launch_kv_cache_append(fe2o3_ctx *ctx, cudaStream_t s, const void *args, fe2o3_geometry *geo, bool plan_only) {
    static void (*const kernels[3])(KvCache, KvRows) = {kv_append_kernel<0>, kv_append_kernel<1>, kv_append_kernel<2>};
    const fe2o3_kv_cache_append_v1_args *a = static_cast<const fe2o3_kv_cache_append_v1_args *>(args);
    return launch_rows(ctx, s, a, a->input_dtype, geo, plan_only, kernels, "kv_cache_append_v1");
}
int32_t launch_kv_cache_read(fe2o3_ctx *ctx, cudaStream_t s, const void *args, fe2o3_geometry *geo, bool plan_only) {
    static void (*const kernels[3])(KvCache, KvRows) = {kv_read_kernel<0>, kv_read_kernel<1>, kv_read_kernel<2>};
    const fe2o3_kv_cache_read_v1_args *a = static_cast<const fe2o3_kv_cache_read_v1_args *>(args);
    return launch_rows(ctx, s, a, a->output_dtype, geo, plan_only, kernels, "kv_cache_read_v1");
}

static Fe2o3KernelRegistration reg_append("kv_cache_append_v1", reinterpret_cast<const void *>(kv_append_kernel<0>));
static Fe2o3KernelRegistration reg_read("kv_cache_read_v1", reinterpret_cast<const void *>(kv_read_kernel<0>));
