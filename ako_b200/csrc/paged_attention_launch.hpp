// Host side of the attention kernels: which one a call runs, and its launch.
#pragma once

#include <atomic>

#include "paged_attention.cuh"

namespace ako_b200 {

struct AttnPlan {
    int dtype;
    bool quant, wide;  // e4m3 cache; head_dim above 64
    int kernel, tile_rows, ctas;
    int64_t workspace;  // bytes: an int4 per CTA, then two partial blocks per CTA
};

constexpr int kMostDevices = 64;  // that launches remember something of
using PerDevice = std::atomic<bool>[kMostDevices];

// Raises a kernel's limit of dynamic shared memory once per device. Any number of threads may call
// it at once: the limit is then raised more than once, to the same value.
template <typename K>
int allow_smem(K kernel, int bytes, PerDevice& done, const char* name) {
    int dev = -1;
    const bool known = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < kMostDevices;
    if (known && done[dev].load(std::memory_order_relaxed)) return AKO_B200_OK;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_error(AKO_B200_ERR_CUDA, "%s: %d bytes of shared memory: %s", name, bytes, cudaGetErrorString(e));
    }
    if (known) done[dev].store(true, std::memory_order_relaxed);
    return AKO_B200_OK;
}

// Bytes of workspace for `ctas` CTAs that keep blocks of `rows` rows.
inline int64_t attention_workspace(int ctas, int rows, bool wide) {
    return static_cast<int64_t>(ctas) * (sizeof(int4) + 2 * sizeof(float) * rows * (2 + (wide ? 128 : 64)));
}

// Kernel 0, for few rows: tile_rows is 8, 16 or 32.
void plan_rows(AttnPlan& p);
int launch_rows(const AttnArgs& a, const AttnPlan& p, cudaStream_t st);

// Kernel 1, on the tensor cores.
void plan_tiles(AttnPlan& p);
int launch_tiles(const AttnArgs& a, const AttnPlan& p, cudaStream_t st);

}  // namespace ako_b200
