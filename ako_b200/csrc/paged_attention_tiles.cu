// Instantiations and launches of the kernel on the tensor cores.
#include <cmath>

#include "paged_attention_launch.hpp"
#include "paged_attention_tiles.cuh"

namespace ako_b200 {
namespace {

template <typename T, bool QUANT, int DPAD>
int launch(const TilesArgs& t, const AttnPlan& p, cudaStream_t st) {
    using Shape = TilesShape<DPAD>;
    const char* name = "paged_attention";
    auto kernel = attn_tiles_kernel<T, QUANT, DPAD>;
    static bool done[64] = {};
    static int regs = 0;
    if (regs == 0) {
        // The warps' registers are shares of what the block is launched with.
        cudaFuncAttributes f{};
        const cudaError_t e = cudaFuncGetAttributes(&f, kernel);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return set_error(AKO_B200_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
        }
        regs = f.numRegs;
    }
    if (regs * kTilesThreads < 128 * (2 * kSoftmaxRegs + kLoadRegs + kIssueRegs))
        return set_error(AKO_B200_ERR_CUDA, "%s: built with %d registers a thread, too few to share out", name, regs);
    int rc = allow_smem(kernel, Shape::kSmem, done, name);
    if (rc) return rc;
    rc = launch_ex(kernel, dim3(p.ctas), dim3(kTilesThreads), Shape::kSmem, 1, st, t, name);
    if (rc) return rc;
    constexpr int STEP = 128 / (DPAD / 4);
    return launch_ex(attn_join_kernel<T, kTilesRows, DPAD>, dim3(p.ctas, kTilesRows / STEP), dim3(128), 0, 1, st, t.a,
                     name);
}

template <typename T>
int with_type(const TilesArgs& t, const AttnPlan& p, cudaStream_t st) {
    if (p.quant) return p.wide ? launch<T, true, 128>(t, p, st) : launch<T, true, 64>(t, p, st);
    return p.wide ? launch<T, false, 128>(t, p, st) : launch<T, false, 64>(t, p, st);
}

}  // namespace

void plan_tiles(AttnPlan& p) {
    p.kernel = 1;
    p.tile_rows = kTilesRows;
    p.ctas = sm_count();
    p.workspace = attention_workspace(p.ctas, kTilesRows, p.wide);
}

int launch_tiles(const AttnArgs& a, const AttnPlan& p, double scale, cudaStream_t st) {
    TilesArgs t{a, device_status_word(), wait_polls(), scale < 0 ? -1.0f : scale == 0 ? 0.0f : 1.0f};
    if (t.status == nullptr) return AKO_B200_ERR_CUDA;
    // The softmax follows the largest score, so the scale's sign goes into q;
    // a scale of zero is a q of zero.
    t.a.scale = scale == 0 ? 1.0f : std::fabs(a.scale);
    return p.dtype == AKO_B200_F16 ? with_type<__half>(t, p, st) : with_type<__nv_bfloat16>(t, p, st);
}

}  // namespace ako_b200
