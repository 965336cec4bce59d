// The paged attention kernels over a cache of this format.
#include "paged_attention.cuh"

PagedBuild paged_build_bf16(uint32_t dim, uint32_t nt) { return paged_build_for<FE2O3_KV_BF16>(dim, nt); }

static Fe2o3KernelRegistration reg_paged("paged_attention_v1", reinterpret_cast<const void *>(paged_attention_kernel<FE2O3_KV_BF16, 128, 1>));
