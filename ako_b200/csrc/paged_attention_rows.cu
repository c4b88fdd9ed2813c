// Instantiations and launches of the kernel for few rows.
#include "paged_attention_launch.hpp"
#include "paged_attention_rows.cuh"

namespace ako_b200 {
namespace {

template <typename T, bool QUANT, int DPAD, int NT>
int launch(const AttnArgs& a, const AttnPlan& p, cudaStream_t st) {
    using Shape = RowsShape<T, QUANT, DPAD, NT>;
    static PerDevice done{};
    const char* name = "paged_attention";
    int rc = allow_smem(attn_rows_kernel<T, QUANT, DPAD, NT>, Shape::kSmem, done, name);
    if (rc) return rc;
    rc = launch_ex(attn_rows_kernel<T, QUANT, DPAD, NT>, dim3(p.ctas), dim3(kRowsThreads), Shape::kSmem, 1, st, a, name);
    if (rc) return rc;
    constexpr int EACH = 8;  // rows of a CTA that joins
    return launch_ex(attn_join_kernel<T, Shape::kRows, DPAD, EACH>, dim3(p.ctas, Shape::kRows / EACH), dim3(128), 0, 1, st,
                     a, name);
}

template <typename T, bool QUANT, int DPAD, int NT>
void plan(AttnPlan& p) {
    using Shape = RowsShape<T, QUANT, DPAD, NT>;
    p.kernel = 0;
    p.ctas = sm_count() * Shape::kCtas;
    p.workspace = attention_workspace(p.ctas, Shape::kRows, DPAD == 128);
    static_assert(sizeof(PartialBlock<Shape::kRows, DPAD>) == sizeof(float) * Shape::kRows * (2 + DPAD), "block size");
}

// f.run<T, QUANT, DPAD, NT>() for the instantiation of `p`.
template <typename T, bool QUANT, int DPAD, typename F>
int with_rows(const AttnPlan& p, F f) {
    switch (p.tile_rows) {
        case 8: return f.template run<T, QUANT, DPAD, 1>();
        case 16: return f.template run<T, QUANT, DPAD, 2>();
        default: return f.template run<T, QUANT, DPAD, 4>();
    }
}

template <typename T, typename F>
int with_type(const AttnPlan& p, F f) {
    if (p.quant) return p.wide ? with_rows<T, true, 128>(p, f) : with_rows<T, true, 64>(p, f);
    return p.wide ? with_rows<T, false, 128>(p, f) : with_rows<T, false, 64>(p, f);
}

template <typename F>
int with_plan(const AttnPlan& p, F f) {
    return p.dtype == AKO_B200_F16 ? with_type<__half>(p, f) : with_type<__nv_bfloat16>(p, f);
}

struct Plan {
    AttnPlan& p;
    template <typename T, bool QUANT, int DPAD, int NT>
    int run() const {
        plan<T, QUANT, DPAD, NT>(p);
        return AKO_B200_OK;
    }
};

struct Launch {
    const AttnArgs& a;
    const AttnPlan& p;
    cudaStream_t st;
    template <typename T, bool QUANT, int DPAD, int NT>
    int run() const {
        return launch<T, QUANT, DPAD, NT>(a, p, st);
    }
};

}  // namespace

void plan_rows(AttnPlan& p) { with_plan(p, Plan{p}); }

int launch_rows(const AttnArgs& a, const AttnPlan& p, cudaStream_t st) { return with_plan(p, Launch{a, p, st}); }

}  // namespace ako_b200
