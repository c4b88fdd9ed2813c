// Host side of the attention kernels: which one a call runs, and its launch.
#pragma once

#include "paged_attention.cuh"

namespace ako_b200 {

struct AttnPlan {
    int dtype;
    bool quant, wide;  // e4m3 cache; head_dim above 64
    int kernel, tile_rows, ctas;
    int64_t workspace;  // bytes: an int4 per CTA, then two partial blocks per CTA
};

// Fills kernel, tile_rows, ctas and workspace for calls whose longest
// sequence has `rows` rows (new tokens times q heads) per kv head.
void make_plan(int64_t rows, AttnPlan& p);

int launch_attention(const AttnArgs& a, const AttnPlan& p, cudaStream_t st);

}  // namespace ako_b200
