// Instantiations and launches of the kernel on the tensor cores.
#include <cmath>

#include "paged_attention_launch.hpp"
#include "paged_attention_tiles.cuh"

namespace ako_b200 {
namespace {

using EncodeTiled = decltype(&cuTensorMapEncodeTiled);

// The driver's encoder, or null.
EncodeTiled encoder() {
    static const EncodeTiled f = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found);
        if (e != cudaSuccess) cudaGetLastError();
        return e == cudaSuccess && found == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiled>(p) : nullptr;
    }();
    return f;
}

// Keys or values as a 4-D tensor in boxes of `box` slots and 64 columns; columns past head_dim read as zeros.
bool make_map(const PagedTensor& t, const PagedCache& c, bool half, int box, CUtensorMap& map) {
    const EncodeTiled encode = encoder();
    if (encode == nullptr) return false;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c.head_dim), static_cast<cuuint64_t>(c.page_size),
                                static_cast<cuuint64_t>(c.kv_heads), static_cast<cuuint64_t>(c.num_pages)};
    // the stride of an axis of one element plays no part, but has to be a valid one
    auto bytes = [&](uint32_t stride, int n) { return n > 1 ? static_cast<cuuint64_t>(stride) * 16 : 256; };
    const cuuint64_t strides[3] = {bytes(t.slot, c.page_size), bytes(t.head, c.kv_heads), bytes(t.page, c.num_pages)};
    const cuuint32_t boxes[4] = {64, static_cast<cuuint32_t>(box), 1, 1}, steps[4] = {1, 1, 1, 1};
    return encode(&map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, t.p, dims, strides,
                  boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, bool QUANT, int DPAD>
int launch(const TilesArgs& t, const AttnPlan& p, cudaStream_t st) {
    using Shape = TilesShape<DPAD>;
    const char* name = "paged_attention";
    auto kernel = attn_tiles_kernel<T, QUANT, DPAD>;
    static PerDevice done{};
    static std::atomic<int> launch_regs{0};
    int regs = launch_regs.load(std::memory_order_relaxed);
    if (regs == 0) {
        // The warps' registers are shares of what the block is launched with.
        cudaFuncAttributes f{};
        const cudaError_t e = cudaFuncGetAttributes(&f, kernel);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return set_error(AKO_B200_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
        }
        regs = f.numRegs;
        launch_regs.store(regs, std::memory_order_relaxed);
    }
    if (regs * kTilesThreads < 128 * (2 * kSoftmaxRegs + kLoadRegs + kIssueRegs))
        return set_error(AKO_B200_ERR_CUDA, "%s: built with %d registers a thread, too few to share out", name, regs);
    int rc = allow_smem(kernel, Shape::kSmem, done, name);
    if (rc) return rc;
    rc = launch_ex(kernel, dim3(p.ctas), dim3(kTilesThreads), Shape::kSmem, 1, st, t, name);
    if (rc) return rc;
    constexpr int EACH = 32;  // rows of a CTA that joins
    return launch_ex(attn_join_kernel<T, kTilesRows, DPAD, EACH>, dim3(p.ctas, kTilesRows / EACH), dim3(128), 0, 1, st,
                     t.a, name);
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

int launch_tiles(const AttnArgs& a, const AttnPlan& p, cudaStream_t st) {
    TilesArgs t{};
    t.a = a;
    t.status = device_status_word();
    t.wait_polls = wait_polls();
    t.q_factor = a.scale < 0 ? -1.0f : a.scale == 0 ? 0.0f : 1.0f;
    if (t.status == nullptr) return AKO_B200_ERR_CUDA;
    // The softmax follows the largest score, so the scale's sign goes into q;
    // a scale of zero is a q of zero.
    t.a.scale = a.scale == 0 ? 1.0f : std::fabs(a.scale);
    // Boxes start on multiples of eight rows, the swizzle's period, and 64 rows are made of whole ones.
    const int page = a.cache.page_size;
    if (!p.quant && page % 8 == 0 && (page % 64 == 0 || 64 % page == 0)) {
        t.box = page < 64 ? page : 64;
        const bool half = p.dtype == AKO_B200_F16;
        if (!make_map(a.cache.k, a.cache, half, t.box, t.k_map) || !make_map(a.cache.v, a.cache, half, t.box, t.v_map))
            t.box = 0;
    }
    return p.dtype == AKO_B200_F16 ? with_type<__half>(t, p, st) : with_type<__nv_bfloat16>(t, p, st);
}

}  // namespace ako_b200
