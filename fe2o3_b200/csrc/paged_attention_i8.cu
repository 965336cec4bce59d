// The paged attention kernels over a cache of this format.
#include "paged_attention.cuh"

PagedBuild paged_build_i8(uint32_t dim, uint32_t nt) { return paged_build_for<FE2O3_KV_I8>(dim, nt); }
