// Attention of one new token a sequence over a paged key-value cache; the formulas stand at
// fe2o3_paged_attention_v1_args.
#include "kv_cache.cuh"

namespace {

struct PagedArgs {
    KvCache c;
    const void *q;
    void *o;
    float *lse;
    uint32_t heads, q_stride, q_head_stride, window;
    float scale;
    bool q_f32, o_f32;
};

// One warp a query head: the running maximum and sum of its row, one key at a time.
template <uint32_t FORMAT>
__global__ void __launch_bounds__(32) paged_attention_row_kernel(PagedArgs a) {
    begin_after_previous();
    const KvCache &c = a.c;
    const uint32_t b = blockIdx.x / a.heads, hq = blockIdx.x % a.heads, h = hq / (a.heads / c.kv_heads), lane = threadIdx.x;
    const uint32_t n = c.lengths[b];
    if (!kv_fits(c, n)) {
        kstatus_set(c.status, FE2O3_KSTATUS_LENGTH);
        return;
    }
    float q[8], o[8] = {}, m = -INFINITY, l = 0.f;
    const uint64_t from = (uint64_t)b * a.q_stride + (uint64_t)hq * a.q_head_stride;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t at = lane + 32 * i;
        q[i] = at >= c.dim ? 0.f : a.q_f32 ? static_cast<const float *>(a.q)[from + at] : bf16_bits_to_f32(static_cast<const uint16_t *>(a.q)[from + at]);
    }
    for (uint32_t j = a.window && n > a.window ? n - a.window : 0; j < n; ++j) {
        const uint64_t row = kv_row(c, b, h, j);
        const uint64_t at = (row == ~0ull ? 0 : row) * c.dim * kKvBytes<FORMAT>;
        const float ks = FORMAT == FE2O3_KV_BF16 ? 1.f : row == ~0ull ? 0.f : c.k_scales[row];
        const float vs = FORMAT == FE2O3_KV_BF16 ? 1.f : row == ~0ull ? 0.f : c.v_scales[row];
        float s = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            if (lane + 32 * i < c.dim && row != ~0ull) s += q[i] * kv_element<FORMAT>(c.k + at, lane + 32 * i);
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
        s *= ks * a.scale;
        const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;   // (fmaxf takes the number beside a NaN: p is NaN then)
        const float p = expf(s - base), keep = expf(m - base);
        l = l * keep + p;
        m = top;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            if (lane + 32 * i < c.dim) o[i] = o[i] * keep + (row == ~0ull ? 0.f : p * (kv_element<FORMAT>(c.v + at, lane + 32 * i) * vs));
    }
    const uint64_t to = (uint64_t)blockIdx.x * c.dim;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        if (lane + 32 * i >= c.dim) continue;
        const float v = n ? o[i] / l : 0.f;
        if (a.o_f32) static_cast<float *>(a.o)[to + lane + 32 * i] = v;
        else static_cast<uint16_t *>(a.o)[to + lane + 32 * i] = f32_to_bf16_bits(v);
    }
    if (a.lse && lane == 0) a.lse[blockIdx.x] = n ? m + logf(l) : -INFINITY;
}

}  // namespace

int32_t launch_paged_attention(fe2o3_ctx *ctx, cudaStream_t s, const void *args, fe2o3_geometry *geo, bool plan_only) {
    static void (*const kernels[3])(PagedArgs) = {paged_attention_row_kernel<0>, paged_attention_row_kernel<1>, paged_attention_row_kernel<2>};
    const fe2o3_paged_attention_v1_args *a = static_cast<const fe2o3_paged_attention_v1_args *>(args);
    const uint32_t grid = a->batch * a->heads;
    if (geo) *geo = fe2o3_geometry{{grid, 1, 1}, {32, 1, 1}, 0, 1};
    if (plan_only || grid == 0) return FE2O3_OK;
    const PagedArgs p{kv_cache_of(ctx, a), reinterpret_cast<const void *>(a->q.ptr), reinterpret_cast<void *>(a->output.ptr),
                      reinterpret_cast<float *>(a->lse.ptr), a->heads, a->q_stride, a->q_head_stride, a->window, a->scale,
                      a->q_dtype == FE2O3_DTYPE_F32, a->output_dtype == FE2O3_DTYPE_F32};
    const cudaError_t e = fe2o3_launch_early(kernels[a->format], grid, 32, 0, s, 1, p);
    fe2o3_count_launch(1);
    return fe2o3_cuda_status(e, "paged_attention_v1");
}

static Fe2o3KernelRegistration reg_paged("paged_attention_v1", reinterpret_cast<const void *>(paged_attention_row_kernel<0>));
