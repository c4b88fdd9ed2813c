// Entry points of attention over a paged cache: argument checks, the choice
// of a kernel and its launch.
#include <climits>
#include <cmath>

#include "paged_attention.cuh"
#include "paged_attention_launch.hpp"

namespace ako_b200 {
namespace {

// Rows per sequence and kv head up to which the kernel for few rows runs. At
// 32 rows (16 contexts of 2048 tokens) it takes 48 us in bf16, as the other
// does with up to 128 rows, and 46 us in e4m3 where the other takes 80; at 34
// it would need a tile more.
constexpr int kFewRows = 32;

// Checks that need no pointer of the call; fills the sizes of `a`.
int check_sizes(const char* op, const ako_b200_paged_kv* cache, const ako_b200_paged_batch* batch, int64_t tokens,
                int64_t q_len, int64_t q_heads, int dtype, AttnArgs& a, AttnPlan& p) {
    if (dtype == AKO_B200_F32)
        return set_error(AKO_B200_ERR_UNSUPPORTED_DTYPE, "%s: q must be fp16 or bf16", op);
    int es = 0;
    int rc = make_cache(op, cache, dtype, a.cache, es);
    if (rc) return rc;
    if ((rc = make_seqs(op, batch, a.cache, tokens, q_len, a.seqs))) return rc;
    if (q_heads < 1 || q_heads > INT_MAX || q_heads % a.cache.kv_heads != 0)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: q_heads must be a multiple of kv_heads (%d), got %lld", op,
                         a.cache.kv_heads, static_cast<long long>(q_heads));
    if (tokens > 0 && q_heads > (INT_MAX - 4096) / tokens)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: tokens * q_heads must be < 2^31 - 4096", op);
    a.group = static_cast<int>(q_heads / a.cache.kv_heads);
    a.by_group = FastDiv::make(static_cast<uint32_t>(a.group));
    int64_t most = a.seqs.cu == nullptr ? q_len : batch->max_q_len;
    if (most < 1) most = 1;
    if (most > tokens) most = tokens;
    p.dtype = dtype;
    p.quant = cache->dtype == AKO_B200_E4M3;
    p.wide = a.cache.head_dim > 64;
    const int64_t rows = most * a.group;
    if (rows <= kFewRows) {
        p.tile_rows = rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
        plan_rows(p);
    } else {
        plan_tiles(p);
    }
    return AKO_B200_OK;
}

bool rows16(const void* p, int64_t s0, int64_t n0, int64_t s1, int64_t n1, int64_t s2, int64_t n2) {
    auto ok = [](int64_t s, int64_t n) { return n <= 1 || (s & 7) == 0; };
    return aligned16(p) && ok(s0, n0) && ok(s1, n1) && ok(s2, n2);
}

}  // namespace
}  // namespace ako_b200

using namespace ako_b200;

extern "C" int ako_b200_paged_attention(const void* q, int64_t q_stride_b, int64_t q_stride_s, int64_t q_stride_h,
                                        const ako_b200_paged_kv* cache, const ako_b200_paged_batch* batch,
                                        int64_t tokens, int64_t q_len, int64_t q_heads, double scale, int64_t window,
                                        int64_t sinks, void* out, int64_t out_stride_b, int64_t out_stride_s,
                                        int64_t out_stride_h, void* workspace, int64_t workspace_bytes, int dtype,
                                        void* stream) {
    clear_error();
    const char* op = "ako_b200_paged_attention";
    AttnArgs a{};
    AttnPlan p{};
    int rc = check_sizes(op, cache, batch, tokens, q_len, q_heads, dtype, a, p);
    if (rc) return rc;
    if (window < 0 || sinks < 0)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: window and sinks must be >= 0", op);
    a.scale = static_cast<float>(scale * 1.4426950408889634);
    if (!std::isfinite(a.scale))
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: scale must be finite, in fp32 too", op);
    if ((rc = refuse_if_wait_expired(op))) return rc;
    if (tokens == 0 || a.seqs.batch == 0) return AKO_B200_OK;
    if (q == nullptr || out == nullptr)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: q or out is a null pointer", op);
    const bool uniform = a.seqs.cu == nullptr;
    const int64_t nb = uniform ? a.seqs.batch : 1, ns = uniform ? q_len : tokens;
    if (!rows16(q, q_stride_b, nb, q_stride_s, ns, q_stride_h, q_heads) ||
        !rows16(out, out_stride_b, nb, out_stride_s, ns, out_stride_h, q_heads))
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: q, out and their strides must be multiples of 16 bytes",
                         op);
    if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < p.workspace)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: workspace must be 16-byte aligned and hold %lld bytes", op,
                         static_cast<long long>(p.workspace));
    a.q = q;
    a.out = out;
    a.qb = q_stride_b;
    a.qs = q_stride_s;
    a.qh = q_stride_h;
    a.ob = out_stride_b;
    a.os = out_stride_s;
    a.oh = out_stride_h;
    // A window that reaches behind every position is none.
    a.window = static_cast<int>(window >= a.seqs.max_kv ? 0 : window);
    a.sinks = static_cast<int>(a.window == 0 ? 0 : sinks < a.seqs.max_kv ? sinks : a.seqs.max_kv);
    a.joins = static_cast<int4*>(workspace);
    a.partial = reinterpret_cast<float*>(a.joins + p.ctas);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return p.kernel == 0 ? launch_rows(a, p, st) : launch_tiles(a, p, st);
}

extern "C" int ako_b200_paged_attention_plan(const ako_b200_paged_kv* cache, const ako_b200_paged_batch* batch,
                                             int64_t tokens, int64_t q_len, int64_t q_heads, int dtype, int* kernel,
                                             int* tile_rows, int* ctas, int64_t* workspace_bytes) {
    clear_error();
    const char* op = "ako_b200_paged_attention_plan";
    if (kernel == nullptr || tile_rows == nullptr || ctas == nullptr || workspace_bytes == nullptr)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: null output pointer", op);
    AttnArgs a{};
    AttnPlan p{};
    const int rc = check_sizes(op, cache, batch, tokens, q_len, q_heads, dtype, a, p);
    if (rc) return rc;
    *kernel = p.kernel;
    *tile_rows = p.tile_rows;
    *ctas = p.ctas;
    *workspace_bytes = p.workspace;
    return AKO_B200_OK;
}
