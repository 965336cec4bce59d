// The paged attention kernels over a cache of this format.
#include "paged_attention.cuh"

PagedBuild paged_build_e2m1(uint32_t dim, uint32_t nt, bool long_rows) {
    if (long_rows) return dim <= 64 ? paged_build<FE2O3_KV_E2M1, 64, 1, true>() : paged_build<FE2O3_KV_E2M1, 128, 1, true>();
    return paged_build_for<FE2O3_KV_E2M1>(dim, nt);
}
