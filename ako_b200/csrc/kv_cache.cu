// Writing new tokens into a paged key/value cache and reading sequences back.
//
// Both move each value once and compute next to nothing, so both are bound by
// memory: by HBM where there are megabytes to move, by the chain
// lengths -> page number -> access where there are few.
#include <climits>

#include <cuda_fp8.h>

#include "paged.cuh"

namespace ako_b200 {

// ------------------------------------------------------------ argument checks
namespace {

bool multiple16(int64_t stride, int64_t extent, int es) { return extent <= 1 || ((stride * es) & 15) == 0; }

// A stride of `stride` elements in units of `unit` bytes; false if it is none that fits.
bool stride_units(int64_t stride, int es, int unit, uint32_t& out) {
    if (stride < 0 || stride > INT64_MAX / 16 || stride * es % unit != 0 || stride * es / unit > UINT32_MAX) return false;
    out = static_cast<uint32_t>(stride * es / unit);
    return true;
}

// A cache tensor's view; strides of axes of one element play no part.
bool make_tensor(void* p, const int64_t (&strides)[3], const ako_b200_paged_kv& c, int es, int unit, PagedTensor& out) {
    out.p = p;
    return stride_units(c.num_pages > 1 ? strides[0] : 0, es, unit, out.page) &&
           stride_units(c.kv_heads > 1 ? strides[1] : 0, es, unit, out.head) &&
           stride_units(c.page_size > 1 ? strides[2] : 0, es, unit, out.slot);
}

}  // namespace

int make_cache(const char* op, const ako_b200_paged_kv* c, int dtype, PagedCache& out, int& cache_es) {
    if (c == nullptr) return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: cache is a null pointer", op);
    if (dtype_size(dtype) == 0)
        return set_error(AKO_B200_ERR_UNSUPPORTED_DTYPE, "%s: unsupported dtype code %d", op, dtype);
    const bool e4m3 = c->dtype == AKO_B200_E4M3;
    if (!e4m3 && (c->dtype < 0 || c->dtype > AKO_B200_BF16))
        return set_error(AKO_B200_ERR_UNSUPPORTED_DTYPE, "%s: unsupported cache dtype code %lld", op,
                         static_cast<long long>(c->dtype));
    if (!e4m3 && c->dtype != dtype)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: dtype %d differs from the cache's %lld", op, dtype,
                         static_cast<long long>(c->dtype));
    cache_es = e4m3 ? 1 : dtype_size(dtype);
    if (c->num_pages < 1 || c->num_pages > INT_MAX || c->kv_heads < 1 || c->kv_heads > 65535 || c->page_size < 1 ||
        c->page_size > INT_MAX)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: num_pages, kv_heads and page_size must be >= 1 (and "
                                                        "kv_heads <= 65535)", op);
    const int step = e4m3 ? 16 : 8;
    if (c->head_dim < step || c->head_dim > 128 || c->head_dim % step != 0)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: head_dim must be a multiple of %d up to 128, got %lld", op,
                         step, static_cast<long long>(c->head_dim));
    if (c->k == nullptr || c->v == nullptr)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: k or v of the cache is a null pointer", op);
    if (e4m3 && (c->k_scale == nullptr || c->v_scale == nullptr))
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: an e4m3 cache needs k_scale and v_scale", op);
    const int64_t k[3] = {c->k_stride_page, c->k_stride_head, c->k_stride_slot};
    const int64_t v[3] = {c->v_stride_page, c->v_stride_head, c->v_stride_slot};
    if (!aligned16(c->k) || !aligned16(c->v) || !make_tensor(c->k, k, *c, cache_es, 16, out.k) ||
        !make_tensor(c->v, v, *c, cache_es, 16, out.v))
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: k and v of the cache and their strides must be multiples "
                                                        "of 16 bytes, and strides within 0 .. 64 GB", op);
    const int64_t ks[3] = {c->ks_stride_page, c->ks_stride_head, c->ks_stride_slot};
    const int64_t vs[3] = {c->vs_stride_page, c->vs_stride_head, c->vs_stride_slot};
    if (e4m3 && (!make_tensor(c->k_scale, ks, *c, 4, 4, out.ks) || !make_tensor(c->v_scale, vs, *c, 4, 4, out.vs)))
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: strides of the scales must be within 0 .. 16 GB", op);
    out.num_pages = static_cast<int>(c->num_pages);
    out.kv_heads = static_cast<int>(c->kv_heads);
    out.head_dim = static_cast<int>(c->head_dim);
    out.page_size = static_cast<int>(c->page_size);
    out.by_page = FastDiv::make(static_cast<uint32_t>(c->page_size));
    return AKO_B200_OK;
}

int make_seqs(const char* op, const ako_b200_paged_batch* b, const PagedCache& c, int64_t tokens, int64_t q_len,
              PagedSeqs& out) {
    if (b == nullptr) return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: batch is a null pointer", op);
    if (b->batch < 0 || b->batch > 65535 || b->max_pages < 0)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: batch must be within 0 .. 65535 and max_pages >= 0", op);
    if (b->max_pages > 0 && b->max_pages > (INT_MAX - 4096) / c.page_size)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: max_pages * page_size must be < 2^31 - 4096", op);
    if (tokens < 0 || q_len < 0 || tokens > INT_MAX)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: tokens and q_len must be within 0 .. 2^31 - 1", op);
    if (b->cu_seqlens == nullptr && (q_len > INT_MAX || b->batch * q_len != tokens))
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: without cu_seqlens tokens must be batch * q_len", op);
    if (b->batch > 0 && (b->kv_lens == nullptr || (b->max_pages > 0 && b->page_table == nullptr)))
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: page_table or kv_lens is a null pointer", op);
    if (b->batch > 1 && b->page_table_stride < b->max_pages)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: page_table_stride %lld is smaller than max_pages", op,
                         static_cast<long long>(b->page_table_stride));
    out.table = b->page_table;
    out.table_stride = b->page_table_stride;
    out.kv_lens = b->kv_lens;
    out.cu = b->cu_seqlens;
    out.batch = static_cast<int>(b->batch);
    out.q_len = static_cast<int>(q_len);
    out.tokens = static_cast<int>(tokens);
    out.max_kv = static_cast<int>(b->max_pages * c.page_size);
    return AKO_B200_OK;
}

namespace {

// ------------------------------------------------------------------ e4m3
__device__ __forceinline__ float2 from_e4m3(uint32_t pair) {
    return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(pair), __NV_E4M3)));
}

// Exponent of the least power of two s with top / s <= 448 = 1.75 * 2^8, at
// least -126 (so that s and 1 / s are normal); top is finite and positive.
__device__ __forceinline__ int scale_exponent(float top) {
    const uint32_t u = __float_as_uint(top);
    const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(e, -126);
}

__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// ------------------------------------------------------------ row accesses
// Eight elements of T (one 16-byte access for 16-bit types, two for fp32).
template <typename T>
struct Row8 {
    static constexpr int N = 8 * sizeof(T) / 16;
    uint4 w[N];

    __device__ __forceinline__ void load(const void* base, int64_t at) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const T*>(base) + at);
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = p[i];
    }
    __device__ __forceinline__ void store(void* base, int64_t at) const {
        uint4* p = reinterpret_cast<uint4*>(static_cast<T*>(base) + at);
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = w[i];
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const T* v = reinterpret_cast<const T*>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(v[i]);
    }
    __device__ __forceinline__ void put(const float (&x)[8]) {
        auto& v = *reinterpret_cast<Packed<T, 8>*>(w);
#pragma unroll
        for (int i = 0; i < 8; i += 2) put2(v, i, x[i], x[i + 1]);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = make_uint4(0, 0, 0, 0);
    }
    // Times 2^e, as e4m3: to nearest even, saturating. The product is exact, or
    // below 2^-14 and so rounds to zero either way.
    __device__ __forceinline__ uint2 scaled_e4m3(int e) const {
        uint32_t y[4];
        if (std::is_same_v<T, __half> && e >= -14 && e <= 15) {
            const uint32_t u[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
            const __half2 f = __half2half2(__float2half_rn(exp2_int(e)));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __half2 p = __hmul2(*reinterpret_cast<const __half2*>(&u[i]), f);
                y[i] = __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(p), __NV_SATFINITE, __NV_E4M3);
            }
        } else {
            const float f = exp2_int(e);
            float x[8];
            get(x);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                y[i] = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(x[2 * i], f), __fmul_rn(x[2 * i + 1], f)),
                                                __NV_SATFINITE, __NV_E4M3);
        }
        return make_uint2(y[0] | (y[1] << 16), y[2] | (y[3] << 16));
    }
    // The largest finite magnitude, or 0. Magnitudes of 16-bit types compare as
    // integers, two at a time; infinities and NaN, which are the largest of
    // them, are looked for only where there are any.
    __device__ __forceinline__ float largest() const {
        if constexpr (sizeof(T) == 2) {
            constexpr uint32_t INF = std::is_same_v<T, __half> ? 0x7c00 : 0x7f80;
            const uint32_t m = 0x7fff7fffu;
            uint32_t t = __vmaxu2(__vmaxu2(w[0].x & m, w[0].y & m), __vmaxu2(w[0].z & m, w[0].w & m));
            t = max(t >> 16, t & 0xffffu);
            if (t < INF) {
                const uint16_t bits = static_cast<uint16_t>(t);
                return to_f32(*reinterpret_cast<const T*>(&bits));
            }
        }
        float x[8], top = 0.0f;
        get(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = fabsf(x[i]);
            if (a < INFINITY) top = fmaxf(top, a);  // false for NaN too
        }
        return top;
    }
};

constexpr int kThreads = 256;

// Lanes that share a row of head_dim elements, `each` to a lane: a power of
// two, as its logarithm.
int lanes_log2(int head_dim, int each) {
    int l = 0;
    while ((each << l) < head_dim) ++l;
    return l;
}

// ------------------------------------------------------------------- write
// Rows of new tokens: strides over sequences, tokens and heads, in 16 bytes.
struct NewRows {
    const void* p;
    uint32_t b, s, h;

    __device__ __forceinline__ const uint8_t* row(uint32_t bi, uint32_t si, uint32_t hi) const {
        return static_cast<const uint8_t*>(p) +
               (static_cast<uint64_t>(b) * bi + static_cast<uint64_t>(s) * si + static_cast<uint64_t>(h) * hi) * 16;
    }
};

struct WriteArgs {
    NewRows k, v;
    PagedCache cache;
    PagedSeqs seqs;
    FastDiv heads, q_len;
    uint32_t rows;  // tokens * kv_heads
    int lanes_log2;
};

// Sequence of token `t` under cu_seqlens: the last b with cu[b] <= t, or 0.
// All lanes of a warp call it: they search together for their least token,
// 32 entries at a time, then each walks on to its own.
__device__ __forceinline__ int find_sequence(const int* cu, int batch, int t) {
    const int least = __reduce_min_sync(0xffffffffu, t);
    const int lane = static_cast<int>(threadIdx.x & 31);
    int lo = 0, hi = batch;  // the answer for `least` lies in [lo, hi)
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) >> 5;
        const int at = lo + step * (lane + 1);
        // cu is not decreasing, so these are the first lanes
        const int n = __popc(__ballot_sync(0xffffffffu, at < hi && cu[at] <= least));
        lo += n * step;
        hi = min(hi, lo + step);
    }
    while (lo + 1 < batch && cu[lo + 1] <= t) ++lo;
    return lo;
}

// Quantises the row that 2^lanes_log2 lanes hold sixteen values each of, and stores it.
template <typename T>
__device__ __forceinline__ void store_quantised(const Row8<T> (&x)[2], const PagedTensor& to, const PagedTensor& scale,
                                                bool store, int page, int h, int slot, int lane_of_row, int lanes_log2,
                                                bool active) {
    float top = fmaxf(x[0].largest(), x[1].largest());  // idle lanes hold zeros
    for (int off = 1 << lanes_log2 >> 1; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    const int e = top > 0.0f ? scale_exponent(top) : 0;
    if (!store) return;
    if (active) {
        const uint2 lo = x[0].scaled_e4m3(-e), hi = x[1].scaled_e4m3(-e);
        *reinterpret_cast<uint4*>(to.row(page, h, slot) + lane_of_row * 16) = make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
    if (lane_of_row == 0) *scale.scale(page, h, slot) = exp2_int(e);
}

// A lane moves eight values, sixteen where they are quantised, of a token's
// keys and of its values in one head; 2^lanes_log2 lanes share such a row
// (those behind head_dim idle). The loads are under way while the thread finds
// the row's page.
// Bound: HBM for prompts as they are (82.6 MB in 15.3 us, 5.4 TB/s); for
// quantised ones the issue of instructions, of which sixteen values to a lane
// take fewer than eight (216 MB of fp16: 38 us against 54); the chain
// cu_seqlens -> length -> page for a step.
template <typename T, bool QUANT>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const WriteArgs a) {
    pdl_enter();
    constexpr int PARTS = QUANT ? 2 : 1;
    const int c = static_cast<int>(threadIdx.x) & ((1 << a.lanes_log2) - 1);
    const uint32_t at_row = blockIdx.x * (kThreads >> a.lanes_log2) + (threadIdx.x >> a.lanes_log2);
    const bool active = c * PARTS * 8 < a.cache.head_dim;
    // rows behind the last repeat it and are not stored
    const uint32_t row = min(at_row, a.rows - 1);
    const uint32_t t = a.heads.div(row);
    const int h = static_cast<int>(row - t * a.heads.d);
    uint32_t b = 0, s = t;
    if (a.seqs.cu == nullptr) {
        b = a.q_len.div(t);
        s -= b * a.q_len.d;
    }
    Row8<T> k[PARTS], v[PARTS];
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        k[i].zero();
        v[i].zero();
        if (active) {
            k[i].load(a.k.row(b, s, h), (c * PARTS + i) * 8);
            v[i].load(a.v.row(b, s, h), (c * PARTS + i) * 8);
        }
    }
    if (a.seqs.cu != nullptr) b = find_sequence(a.seqs.cu, a.seqs.batch, static_cast<int>(t));
    int first, n;
    new_tokens(a.seqs, static_cast<int>(b), first, n);
    const int at = static_cast<int>(t) - first;
    int slot = 0, page = -1;
    if (at_row < a.rows && at >= 0 && at < n) {
        const int pos = new_position(a.seqs.kv_lens[b], n, at, a.seqs.max_kv);
        if (pos >= 0) page = page_of(a.seqs, a.cache, static_cast<int>(b), pos, slot);
    }
    if constexpr (QUANT) {
        store_quantised(k, a.cache.k, a.cache.ks, page >= 0, page, h, slot, c, a.lanes_log2, active);
        store_quantised(v, a.cache.v, a.cache.vs, page >= 0, page, h, slot, c, a.lanes_log2, active);
    } else if (page >= 0 && active) {
        k[0].store(a.cache.k.row(page, h, slot), c * 8);
        v[0].store(a.cache.v.row(page, h, slot), c * 8);
    }
}

template <typename T>
int launch_write(WriteArgs& a, bool quant, cudaStream_t st) {
    a.lanes_log2 = lanes_log2(a.cache.head_dim, quant ? 16 : 8);
    const int64_t pass = kThreads >> a.lanes_log2;
    const char* name = "kv_cache_write";
    const dim3 grid(static_cast<unsigned>((a.rows + pass - 1) / pass));
    return quant ? launch_ex(kv_write_kernel<T, true>, grid, dim3(kThreads), 0, 1, st, a, name)
                 : launch_ex(kv_write_kernel<T, false>, grid, dim3(kThreads), 0, 1, st, a, name);
}

// -------------------------------------------------------------------- read
struct ReadArgs {
    void *k, *v;
    int64_t kb, kh, ks, vb, vh, vs;
    PagedCache cache;
    PagedSeqs seqs;
    FastDiv length, heads;
    int64_t start;
    uint32_t rows;  // batch * kv_heads * length
    int lanes_log2;
};

// 16 e4m3 values (one 16-byte access).
struct Row16Q {
    uint4 w;

    __device__ __forceinline__ void load(const void* base, int64_t at) {
        w = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + at);
    }
    __device__ __forceinline__ void zero() { w = make_uint4(0, 0, 0, 0); }
    template <typename T>
    __device__ __forceinline__ void store(void* base, int64_t at, float scale) const {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = from_e4m3((u[half * 2 + i / 2] >> (16 * (i & 1))) & 0xffffu);
                x[2 * i] = __fmul_rn(f.x, scale);
                x[2 * i + 1] = __fmul_rn(f.y, scale);
            }
            Row8<T> r;
            r.put(x);
            r.store(base, at + half * 8);
        }
    }
};

// A lane moves 16 bytes of a row of the cache (a position's keys in one head)
// and the same of its values. Rows run over positions first, along a page and
// along the output. One row to a thread: with two the same bytes are under way
// in half the CTAs, which measured 144 us against 131 for 744 MB (e4m3 to bf16).
template <typename T, bool QUANT>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const ReadArgs a) {
    pdl_enter();
    using Held = std::conditional_t<QUANT, Row16Q, Row8<T>>;
    constexpr int EACH = QUANT ? 16 : 8;
    const int c = static_cast<int>(threadIdx.x) & ((1 << a.lanes_log2) - 1);
    const uint32_t row = blockIdx.x * (kThreads >> a.lanes_log2) + (threadIdx.x >> a.lanes_log2);
    if (c * EACH >= a.cache.head_dim || row >= a.rows) return;
    const uint32_t bh = a.length.div(row);
    const uint32_t j = row - bh * a.length.d;
    const int b = static_cast<int>(a.heads.div(bh));
    const int h = static_cast<int>(bh - b * a.heads.d);
    const int64_t pos = a.start + j;
    int page = -1, slot = 0;
    if (pos < cached_tokens(a.seqs, b)) page = page_of(a.seqs, a.cache, b, static_cast<int>(pos), slot);
    Held k, v;
    [[maybe_unused]] float ks = 0.0f, vs = 0.0f;
    k.zero();
    v.zero();
    if (page >= 0) {
        k.load(a.cache.k.row(page, h, slot), c * EACH);
        v.load(a.cache.v.row(page, h, slot), c * EACH);
        if constexpr (QUANT) {
            ks = *a.cache.ks.scale(page, h, slot);
            vs = *a.cache.vs.scale(page, h, slot);
        }
    }
    const int64_t ko = b * a.kb + h * a.kh + j * a.ks + c * EACH;
    const int64_t vo = b * a.vb + h * a.vh + j * a.vs + c * EACH;
    if constexpr (QUANT) {
        k.template store<T>(a.k, ko, ks);
        v.template store<T>(a.v, vo, vs);
    } else {
        k.store(a.k, ko);
        v.store(a.v, vo);
    }
}

template <typename T>
int launch_read(ReadArgs& a, bool quant, cudaStream_t st) {
    a.lanes_log2 = lanes_log2(a.cache.head_dim, quant ? 16 : 8);
    const int64_t pass = kThreads >> a.lanes_log2;
    const dim3 grid(static_cast<unsigned>((int64_t{a.rows} + pass - 1) / pass));
    const char* name = "kv_cache_read";
    return quant ? launch_ex(kv_read_kernel<T, true>, grid, dim3(kThreads), 0, 1, st, a, name)
                 : launch_ex(kv_read_kernel<T, false>, grid, dim3(kThreads), 0, 1, st, a, name);
}

bool make_rows(const void* p, int64_t sb, int64_t nb, int64_t ss, int64_t ns, int64_t sh, int64_t nh, int es,
               NewRows& out) {
    const int64_t strides[3] = {nb > 1 ? sb : 0, ns > 1 ? ss : 0, nh > 1 ? sh : 0};
    uint32_t units[3];
    for (int i = 0; i < 3; ++i)
        if (!stride_units(strides[i], es, 16, units[i])) return false;
    out = NewRows{p, units[0], units[1], units[2]};
    return aligned16(p);
}

// Whether places of a cache's tensor are one place: which write is left there would be chance.
bool repeats(const PagedTensor& t, const PagedCache& c) {
    return (c.num_pages > 1 && t.page == 0) || (c.kv_heads > 1 && t.head == 0) || (c.page_size > 1 && t.slot == 0);
}

// Pointer and the strides of axes longer than one are multiples of 16 bytes.
bool rows16(const void* p, int64_t s0, int64_t n0, int64_t s1, int64_t n1, int64_t s2, int64_t n2, int es) {
    return aligned16(p) && multiple16(s0, n0, es) && multiple16(s1, n1, es) && multiple16(s2, n2, es);
}

}  // namespace
}  // namespace ako_b200

using namespace ako_b200;

extern "C" int ako_b200_kv_cache_write(const void* k, int64_t k_stride_b, int64_t k_stride_s, int64_t k_stride_h,
                                       const void* v, int64_t v_stride_b, int64_t v_stride_s, int64_t v_stride_h,
                                       const ako_b200_paged_kv* cache, const ako_b200_paged_batch* batch,
                                       int64_t tokens, int64_t q_len, int dtype, void* stream) {
    clear_error();
    const char* op = "ako_b200_kv_cache_write";
    WriteArgs a{};
    int es = 0;
    int rc = make_cache(op, cache, dtype, a.cache, es);
    if (rc) return rc;
    if ((rc = make_seqs(op, batch, a.cache, tokens, q_len, a.seqs))) return rc;
    if ((rc = refuse_if_wait_expired(op))) return rc;
    if (tokens == 0 || a.seqs.batch == 0 || a.seqs.max_kv == 0) return AKO_B200_OK;
    if (tokens * a.cache.kv_heads > INT_MAX)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: tokens * kv_heads must be < 2^31", op);
    if (k == nullptr || v == nullptr)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: k or v is a null pointer", op);
    const bool quant = cache->dtype == AKO_B200_E4M3;
    if (repeats(a.cache.k, a.cache) || repeats(a.cache.v, a.cache) ||
        (quant && (repeats(a.cache.ks, a.cache) || repeats(a.cache.vs, a.cache))))
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: a cache that repeats its elements along an axis (a stride "
                                                        "of 0) cannot be written", op);
    const bool uniform = a.seqs.cu == nullptr;
    const int64_t nb = uniform ? a.seqs.batch : 1, ns = uniform ? q_len : tokens;
    const int in = dtype_size(dtype);
    const bool fit = make_rows(k, k_stride_b, nb, k_stride_s, ns, k_stride_h, a.cache.kv_heads, in, a.k) &&
                     make_rows(v, v_stride_b, nb, v_stride_s, ns, v_stride_h, a.cache.kv_heads, in, a.v);
    if (!fit)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT,
                         "%s: k, v and their strides must be multiples of 16 bytes, and strides within 0 .. 64 GB", op);
    a.heads = FastDiv::make(static_cast<uint32_t>(a.cache.kv_heads));
    a.rows = static_cast<uint32_t>(tokens * a.cache.kv_heads);
    a.q_len = FastDiv::make(static_cast<uint32_t>(uniform ? q_len : 1));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case AKO_B200_F32: return launch_write<float>(a, quant, st);
        case AKO_B200_F16: return launch_write<__half>(a, quant, st);
        default: return launch_write<__nv_bfloat16>(a, quant, st);
    }
}

extern "C" int ako_b200_kv_cache_read(const ako_b200_paged_kv* cache, const ako_b200_paged_batch* batch,
                                      int64_t start, int64_t length, void* k_out, int64_t k_stride_b,
                                      int64_t k_stride_h, int64_t k_stride_s, void* v_out, int64_t v_stride_b,
                                      int64_t v_stride_h, int64_t v_stride_s, int dtype, void* stream) {
    clear_error();
    const char* op = "ako_b200_kv_cache_read";
    ReadArgs a{};
    int es = 0;
    int rc = make_cache(op, cache, dtype, a.cache, es);
    if (rc) return rc;
    // the new tokens' rows play no part in a read
    if ((rc = make_seqs(op, batch, a.cache, 0, 0, a.seqs))) return rc;
    if ((rc = refuse_if_wait_expired(op))) return rc;
    if (start < 0 || length < 0 || start > INT_MAX || length > INT_MAX)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: start and length must be within 0 .. 2^31 - 1", op);
    if (length == 0 || a.seqs.batch == 0) return AKO_B200_OK;
    if (int64_t{a.seqs.batch} * a.cache.kv_heads > INT_MAX / length)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: batch * kv_heads * length must be < 2^31", op);
    if (k_out == nullptr || v_out == nullptr)
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT, "%s: k_out or v_out is a null pointer", op);
    const int out = dtype_size(dtype);
    if (!rows16(k_out, k_stride_b, a.seqs.batch, k_stride_h, a.cache.kv_heads, k_stride_s, length, out) ||
        !rows16(v_out, v_stride_b, a.seqs.batch, v_stride_h, a.cache.kv_heads, v_stride_s, length, out))
        return set_error(AKO_B200_ERR_INVALID_ARGUMENT,
                         "%s: k_out, v_out and their strides must be multiples of 16 bytes", op);
    a.k = k_out;
    a.v = v_out;
    a.kb = k_stride_b;
    a.kh = k_stride_h;
    a.ks = k_stride_s;
    a.vb = v_stride_b;
    a.vh = v_stride_h;
    a.vs = v_stride_s;
    a.length = FastDiv::make(static_cast<uint32_t>(length));
    a.heads = FastDiv::make(static_cast<uint32_t>(a.cache.kv_heads));
    a.start = start;
    a.rows = static_cast<uint32_t>(int64_t{a.seqs.batch} * a.cache.kv_heads * length);
    const bool quant = cache->dtype == AKO_B200_E4M3;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case AKO_B200_F32: return launch_read<float>(a, quant, st);
        case AKO_B200_F16: return launch_read<__half>(a, quant, st);
        default: return launch_read<__nv_bfloat16>(a, quant, st);
    }
}
