// Attention of few rows per sequence and kv head over a paged cache: the
// decoding step, and the general form of the operator.
//
// Each warp takes 16 keys at a time through its own ring of asynchronous
// copies and keeps a running maximum, sum and weighted sum of values; a CTA's
// four warps take neighbouring 16 keys of each 64-key tile and join their
// sums once per item, so nothing in the loop waits for another warp.
//
// The products are taken transposed, keys along M: S^T = K Q^T and
// O^T = V^T P^T with m16n8k16, so that the rows, of which there are few, fill
// an N of 8 and not an M of 16. S^T's accumulators become P^T's operand by one
// 8x8 transpose in registers (movmatrix).
//
// Bound: HBM, by the keys and values read once. 32 contexts of 2048 tokens (32
// heads of 128, 8 kv heads, bf16, 252 MB): 48 us, 5.2 TB/s with the launch's
// begin and end; 16 e4m3 contexts of 2000 to 65536 tokens (849 MB): 149 to 159
// us by the card, 5.7 to 5.3 TB/s. Instructions count for almost as much:
// addresses made of constants took those two from 51 and 157 us (the latter, at
// the clock of a long run, from 169).
#pragma once

#include <utility>

#include <cuda_fp8.h>

#include "paged_attention.cuh"

namespace ako_b200 {

constexpr int kRowsWarps = 4;
constexpr int kRowsThreads = kRowsWarps * 32;
constexpr int kWarpKeys = 16;
constexpr int kRowsKeys = kRowsWarps * kWarpKeys;  // keys of a tile
// Tiles that an item's begin and end take as long as. 64 sequences under a window of 1024: 15.4 us
// with 2 or 3, 17.1 with 1, 19.7 with 0.
constexpr int kRowsCost = 2;

// 16-byte asynchronous copy; zeros instead when `real` is false.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t smem, const void* gmem, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(real ? 16 : 0)
                 : "memory");
}

// The same without the choice, at constant offsets.
template <int TO, int FROM>
__device__ __forceinline__ void cp_async16_at(uint32_t smem, const void* gmem) {
    asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(smem), "l"(gmem), "n"(TO), "n"(FROM)
                 : "memory");
}

__device__ __forceinline__ void cp_async4_or_zero(uint32_t smem, const void* gmem, bool real) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem), "l"(gmem), "r"(real ? 4 : 0) : "memory");
}

template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// d += a b, m16n8k16, fp32 sums.
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<T, __half>) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    Packed<T, 2> p;
    put2(p, 0, lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
}

// Four e4m3 values as two pairs of fp16 (exact).
__device__ __forceinline__ uint2 e4m3x4_to_half2x2(uint32_t four) {
    uint2 r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(r.x), "=r"(r.y)
        : "r"(four));
    return r;
}

template <typename T>
struct Half16;  // bit patterns of a 16-bit type
template <>
struct Half16<__half> {
    static constexpr uint32_t inf = 0x7c00, one = 0x3c00;
};
template <>
struct Half16<__nv_bfloat16> {
    static constexpr uint32_t inf = 0x7f80, one = 0x3f80;
};

// Shape of an instantiation: T the activations' type, QUANT an e4m3 cache,
// DPAD the head's width rounded up, NT tiles of 8 rows.
template <typename T, bool QUANT, int DPAD, int NT>
struct RowsShape {
    // An e4m3 cache is multiplied in fp16, which holds its values exactly; q
    // is scaled by a power of two per row to fit.
    using M = std::conditional_t<QUANT, __half, T>;
    static constexpr int kRows = NT * 8;
    static constexpr int kRowBytes = DPAD * (QUANT ? 1 : 2);
    static constexpr int kChunks = kRowBytes / 16;
    // keys, values, scales, and which keys are there; a multiple of 128, so that swizzles are exclusive ors
    static constexpr int kStageBytes = 2 * kWarpKeys * kRowBytes + 2 * kWarpKeys * 4 + 128;
    // Warps on an SM count for more than stages: a warp's 16 keys are a chain of reads, products and
    // exponentials. Head 128, before the copies of dense pages were shortened: with 16 bits two CTAs of
    // 3 stages took 51 us for 32 contexts of 2048 tokens, three of 2 stages 54, one of 4 stages 64; in
    // e4m3 four CTAs of 3 stages 172 us where three of 4 took 179, two of 6 216.
    static constexpr int kStages = 3;
    static constexpr int kRing = kRowsWarps * kStages * kStageBytes;
    static constexpr int kJoinStride = DPAD + 4;  // floats; keeps the four column groups on different banks
    static constexpr int kJoin = kRowsWarps * kRows * (kJoinStride + 2) * 4;
    static constexpr int kQStride = DPAD + 8;
    static constexpr int kSmem = (kRing > kJoin ? kRing : kJoin) + kRows * (kQStride * 2 + 8);
    static constexpr int kFit = 227 * 1024 / (kSmem + 2048);
    static constexpr int kMost = NT >= 4 ? 2 : NT == 2 ? 3 : 4;
    static constexpr int kCtas = kFit < kMost ? kFit : kMost;  // per SM
};

// Chunk c of a key's row in shared memory, so that eight rows' chunks that are
// read together lie in different banks. K of a quantised cache is read as two
// rows of four chunks at a time, everything else as eight rows of one.
template <bool QUANT, int DPAD, bool KEYS>
__device__ __forceinline__ int swizzled(int row, int c) {
    if constexpr (!QUANT) return c ^ (row & 7);
    if constexpr (KEYS) return DPAD == 128 ? c ^ ((row & 1) << 2) : c;
    return DPAD == 128 ? c ^ (row & 7) : c ^ ((row >> 1) & 3);
}

// Copies 16 rows that lie one behind the other, in the cache as in the stage:
// every address is a lane's own and a constant. Row r of chunk c goes to chunk
// swizzled(r, c), which differs from that of the lane's first row by an
// exclusive or that the row's distance alone gives.
template <bool QUANT, int DPAD, bool KEYS, int... I>
__device__ __forceinline__ void copy_dense(uint32_t to, const uint8_t* from, int lane, std::integer_sequence<int, I...>) {
    constexpr int ROWB = DPAD * (QUANT ? 1 : 2), CHUNKS = ROWB / 16, TAKEN = 32 / CHUNKS;
    const int row = lane / CHUNKS, c = lane % CHUNKS;
    const uint32_t first = to + row * ROWB + swizzled<QUANT, DPAD, KEYS>(row, c) * 16;
    (cp_async16_at<I * TAKEN * ROWB, I * TAKEN * ROWB>(
         first ^ (swizzled<QUANT, DPAD, KEYS>(I * TAKEN, 0) * 16), from),
     ...);
}

// An e4m3 cache's rows that are all zero (of either sign): bit r for row r of the 32 / CHUNKS * N rows
// whose 16-byte chunks a warp holds, lane L chunk L % CHUNKS of the rows L / CHUNKS + i * 32 / CHUNKS.
template <int CHUNKS, int N>
__device__ __forceinline__ uint32_t empty_rows(const uint4 (&v)[N]) {
    constexpr int TAKEN = 32 / CHUNKS;
    const int lane = static_cast<int>(threadIdx.x & 31);
    uint32_t held = 1;  // of the lane's row, a chunk with something in it; lanes past the rows count as held
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t any = __ballot_sync(0xffffffffu, ((v[i].x | v[i].y | v[i].z | v[i].w) & 0x7f7f7f7fu) != 0);
        if (lane / TAKEN == i) held = any >> (lane % TAKEN * CHUNKS) & ((1u << CHUNKS) - 1u);
    }
    return __ballot_sync(0xffffffffu, held == 0);
}

template <typename T, bool QUANT, int DPAD, int NT>
__global__ void __launch_bounds__(kRowsThreads, (RowsShape<T, QUANT, DPAD, NT>::kCtas))
    attn_rows_kernel(const AttnArgs a) {
    pdl_enter();
    using Shape = RowsShape<T, QUANT, DPAD, NT>;
    using M = typename Shape::M;
    using Block = PartialBlock<Shape::kRows, DPAD>;
    constexpr int ROWS = Shape::kRows, KS = DPAD / 16, STAGES = Shape::kStages, CHUNKS = Shape::kChunks;
    constexpr int ROWB = Shape::kRowBytes;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ ShareScratch scratch;
    M* const sq = reinterpret_cast<M*>(smem + Shape::kSmem - ROWS * (Shape::kQStride * 2 + 8));
    float* const row_factor = reinterpret_cast<float*>(sq + ROWS * Shape::kQStride);
    int* const row_pos = reinterpret_cast<int*>(row_factor + ROWS);

    const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t4 = lane & 3;  // row and column pair of a fragment
    const int dim = a.cache.head_dim;

    if (tid == 0) a.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
    Share<kRowsCost> share;
    if (!find_share<ROWS, kRowsKeys, kRowsCost, kRowsThreads>(a, kRowsCost + 1, scratch, share)) return;
    Item& it = share.it;

    uint8_t* const ring = smem + warp * (STAGES * Shape::kStageBytes);
    const uint32_t ring_addr = smem_addr(ring);

    while (true) {
        const int t0 = share.first(), t_end = share.last();

        // ------------------------------------------------ keys under way
        // Lanes 0-15 look after the 16 keys' rows of K, lanes 16-31 of V.
        const PagedTensor& mine = lane < 16 ? a.cache.k : a.cache.v;
        const bool one_page = a.cache.page_size % kWarpKeys == 0;
        const bool dense = one_page && dim == DPAD && a.cache.k.slot * 16 == ROWB && a.cache.v.slot * 16 == ROWB;
        int next_page = -1, next_slot = 0;
        auto look_up = [&](int t) {
            const int key = key_tile(it, t) * kRowsKeys + warp * kWarpKeys + (lane & 15);
            next_page = -1;
            if (t < t_end && key <= it.p_hi && (key >= it.win_lo || key < a.sinks))
                next_page = page_of(a.seqs, a.cache, it.b, key, next_slot);
        };
        auto issue = [&](int t, int stage) {
            if (t < t_end) {
                const int page = next_page, slot = next_slot;
                look_up(t + 1);
                const uint32_t to = ring_addr + stage * Shape::kStageBytes;
                const unsigned there = __ballot_sync(0xffffffffu, page >= 0) & 0xffffu;
                constexpr int BYTES = QUANT ? 1 : 2, TAKEN = 32 / CHUNKS;  // rows that the warp takes at once
                if (dense && there == 0xffffu) {
                    using Times = std::make_integer_sequence<int, kWarpKeys / TAKEN>;
                    const int first = slot - (lane & 15);  // the first key's slot
                    copy_dense<QUANT, DPAD, true>(to, a.cache.k.row(page, it.h, first) + lane * 16, lane, Times{});
                    copy_dense<QUANT, DPAD, false>(to + kWarpKeys * ROWB, a.cache.v.row(page, it.h, first) + lane * 16, lane,
                                                   Times{});
                } else if (one_page && there == 0xffffu) {
                    // 16 rows of one page, a slot apart: no lane needs another's place.
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        const PagedTensor& t = kv == 0 ? a.cache.k : a.cache.v;
                        const int c = lane % CHUNKS, row = lane / CHUNKS;
                        const int first = slot - (lane & 15);  // the first key's slot
                        const uint8_t* from = t.row(page, it.h, first + row) + c * 16;
                        const uint64_t step = static_cast<uint64_t>(t.slot) * (TAKEN * 16);
                        const bool real = c * 16 < dim * BYTES;
#pragma unroll
                        for (int i = 0; i < kWarpKeys / TAKEN; ++i) {
                            const int r = row + i * TAKEN;
                            const int sc = kv == 0 ? swizzled<QUANT, DPAD, true>(r, c) : swizzled<QUANT, DPAD, false>(r, c);
                            cp_async16_or_zero(to + (kv * kWarpKeys + r) * ROWB + sc * 16, real ? from : t.p, real);
                            from += step;
                        }
                    }
                } else {
                    const int64_t off = page >= 0 ? static_cast<int64_t>(mine.offset(page, it.h, slot)) : -1;
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        const uint8_t* base = static_cast<const uint8_t*>(kv == 0 ? a.cache.k.p : a.cache.v.p);
#pragma unroll
                        for (int i = 0; i < kWarpKeys / TAKEN; ++i) {
                            const int row = i * TAKEN + lane / CHUNKS, c = lane % CHUNKS;
                            const int64_t o = __shfl_sync(0xffffffffu, off, kv * 16 + row);
                            const bool real = o >= 0 && c * 16 < dim * BYTES;
                            const int sc =
                                kv == 0 ? swizzled<QUANT, DPAD, true>(row, c) : swizzled<QUANT, DPAD, false>(row, c);
                            cp_async16_or_zero(to + (kv * kWarpKeys + row) * ROWB + sc * 16,
                                               real ? base + o * 16 + c * 16 : base, real);
                        }
                    }
                }
                if constexpr (QUANT) {
                    const PagedTensor& st = lane < 16 ? a.cache.ks : a.cache.vs;
                    cp_async4_or_zero(to + 2 * kWarpKeys * ROWB + lane * 4,
                                      page >= 0 ? st.scale(page, it.h, slot) : static_cast<float*>(st.p), page >= 0);
                }
                if (lane == 0)
                    *reinterpret_cast<volatile uint32_t*>(ring + (stage + 1) * Shape::kStageBytes - 16) = there;
            }
            cp_async_commit();
        };
        look_up(t0);
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) issue(t0 + i, i);

        // ------------------------------------------------------------ rows
        for (int r = warp; r < ROWS; r += kRowsWarps) {
            constexpr int EACH = DPAD / 32;  // 4 or 2 elements per lane
            float x[EACH] = {};
            if (r < it.rows && lane * EACH < dim) {
                const T* p = static_cast<const T*>(a.q) + row_offset(a, it, it.row0 + r, a.qb, a.qs, a.qh) + lane * EACH;
                const Packed<T, EACH> v = *reinterpret_cast<const Packed<T, EACH>*>(p);
#pragma unroll
                for (int i = 0; i < EACH; ++i) x[i] = to_f32(v.v[i]);
            }
            float factor = 1.0f;
            if constexpr (QUANT && !std::is_same_v<T, __half>) {
                // power of two that takes the row's largest value into [2^8, 2^9): what fp16 then
                // flushes is 2^-33 of it
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < EACH; ++i) top = fmaxf(top, fabsf(x[i]));
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                if (top > 0.0f && top < INFINITY) {
                    const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127 - 8, -126), 118);
                    const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
                    for (int i = 0; i < EACH; ++i) x[i] = __fmul_rn(x[i], inv);
                    factor = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
                }
            }
            Packed<M, EACH> w;
#pragma unroll
            for (int i = 0; i < EACH; i += 2) put2(w, i, x[i], x[i + 1]);
            *reinterpret_cast<Packed<M, EACH>*>(sq + r * Shape::kQStride + lane * EACH) = w;
            if (lane == 0) {
                row_factor[r] = factor;
                row_pos[r] = r < it.rows ? it.kv - it.n + static_cast<int>(a.by_group.div(it.row0 + r)) : it.p_hi;
            }
        }
        __syncthreads();

        // B operand of S^T: q's rows along N. With an e4m3 cache a k-step
        // takes its head columns in the order that K's 16-byte reads give.
        auto q_fragment = [&](int ks, int nt, uint32_t& b0, uint32_t& b1) {
            const M* p = sq + (nt * 8 + g) * Shape::kQStride;
            if constexpr (QUANT) {
                p += (ks >> 2) * 64 + t4 * 16 + (ks & 3) * 4;
                b0 = *reinterpret_cast<const uint32_t*>(p);
                b1 = *reinterpret_cast<const uint32_t*>(p + 2);
            } else {
                p += ks * 16 + t4 * 2;
                b0 = *reinterpret_cast<const uint32_t*>(p);
                b1 = *reinterpret_cast<const uint32_t*>(p + 8);
            }
        };
        constexpr bool HOLD = NT <= 2;  // q's fragments stay in registers
        uint32_t qf[HOLD ? KS : 1][HOLD ? NT : 1][2];
        if constexpr (HOLD) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) q_fragment(ks, nt, qf[ks][nt][0], qf[ks][nt][1]);
        }
        // m: what weights are relative to; limit: scores above it move m (m plus a factor of 2^8,
        // which the 16-bit types have room for)
        float m[NT][2], limit[NT][2], l[NT][2], factor[NT][2];
        int pos[NT][2];
        float o[KS][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m[nt][e] = 0.0f;
                limit[nt][e] = -INFINITY;
                l[nt][e] = 0.0f;
                factor[nt][e] = QUANT ? row_factor[nt * 8 + t4 * 2 + e] : 1.0f;
                pos[nt][e] = row_pos[nt * 8 + t4 * 2 + e];
            }
#pragma unroll
            for (int mt = 0; mt < KS; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[mt][nt][e] = 0.0f;
        }

        // ------------------------------------------------------------ keys
        int stage = 0;
        for (int t = t0; t < t_end; ++t) {
            const int to = stage == 0 ? STAGES - 1 : stage - 1;
            issue(t + STAGES - 1, to);
            cp_async_wait<STAGES - 1>();
            __syncwarp();
            const uint8_t* const st = ring + stage * Shape::kStageBytes;
            const uint32_t k_addr = ring_addr + stage * Shape::kStageBytes, v_addr = k_addr + kWarpKeys * ROWB;
            const uint32_t there = *reinterpret_cast<const volatile uint32_t*>(st + Shape::kStageBytes - 16);
            const int key0 = key_tile(it, t) * kRowsKeys + warp * kWarpKeys;

            // A product waits for the one before it on the same sum, and a warp has little else to do
            // meanwhile: few rows take their scores as two sums, and fragments are read ahead.
            constexpr int SUMS = NT == 1 ? 2 : 1;
            float xs[SUMS][NT][4];
#pragma unroll
            for (int c = 0; c < SUMS; ++c)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) xs[c][nt][e] = 0.0f;
            auto scores = [&](int ks, const uint32_t(&kf)[4]) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if constexpr (HOLD) {
                        mma16816<M>(xs[ks % SUMS][nt], kf, qf[ks][nt][0], qf[ks][nt][1]);
                    } else {
                        uint32_t b0, b1;
                        q_fragment(ks, nt, b0, b1);
                        mma16816<M>(xs[0][nt], kf, b0, b1);
                    }
                }
            };
            if constexpr (QUANT) {
#pragma unroll
                for (int j = 0; j < DPAD / 64; ++j) {
                    const uint4 lo = *reinterpret_cast<const uint4*>(
                        st + g * ROWB + swizzled<QUANT, DPAD, true>(g, j * 4 + t4) * 16);
                    const uint4 hi = *reinterpret_cast<const uint4*>(
                        st + (g + 8) * ROWB + swizzled<QUANT, DPAD, true>(g + 8, j * 4 + t4) * 16);
                    const uint32_t u[4] = {lo.x, lo.y, lo.z, lo.w}, w[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint2 f = e4m3x4_to_half2x2(u[i]), f8 = e4m3x4_to_half2x2(w[i]);
                        const uint32_t kf[4] = {f.x, f8.x, f.y, f8.y};
                        scores(j * 4 + i, kf);
                    }
                }
            } else {
                constexpr int AHEAD = NT <= 2 ? KS : 2;
                const int row = lane & 15;
#pragma unroll
                for (int k0 = 0; k0 < KS; k0 += AHEAD) {
                    uint32_t kf[AHEAD][4];
#pragma unroll
                    for (int i = 0; i < AHEAD; ++i)
                        ldmatrix4(kf[i],
                                  k_addr + row * ROWB + swizzled<QUANT, DPAD, true>(row, 2 * (k0 + i) + (lane >> 4)) * 16);
#pragma unroll
                    for (int i = 0; i < AHEAD; ++i) scores(k0 + i, kf[i]);
                }
            }
            float x[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[nt][e] = SUMS == 2 ? xs[0][nt][e] + xs[SUMS - 1][nt][e] : xs[0][nt][e];
            // The values of few rows are asked for before the softmax.
            constexpr int MATRICES = QUANT ? KS / 2 : KS;  // of 16 keys and 16 or 32 columns
            constexpr int VAHEAD = NT == 1 ? MATRICES : 2;
            uint32_t vr[VAHEAD][4];
            auto read_values = [&](int first) {
#pragma unroll
                for (int i = 0; i < VAHEAD; ++i) {
                    if constexpr (QUANT) {
                        const int r = (lane & 7) + 8 * ((lane >> 3) & 1), c = 2 * (first + i) + (lane >> 4);
                        ldmatrix4_trans(vr[i], v_addr + r * ROWB + swizzled<QUANT, DPAD, false>(r, c) * 16);
                    } else {
                        const int r = (lane & 7) + 8 * (lane >> 4), c = 2 * (first + i) + ((lane >> 3) & 1);
                        ldmatrix4_trans(vr[i], v_addr + r * ROWB + swizzled<QUANT, DPAD, false>(r, c) * 16);
                    }
                }
            };
            if constexpr (NT == 1) read_values(0);

            // Scores in units of log2(e). A quantised value's scale joins its key's
            // score as a logarithm: the weights of the second product, exp2(x - max) of
            // the joint score, are relative to what contributes most, and the sum of
            // weights takes the scale out again. That holds where an element of the row
            // comes near 448, as kv_cache_write's do; rows of zeros, which contribute
            // nothing, count with kEmptyLog below where it would matter. A scale of
            // zero counts as 2^-100.
            float kc[2] = {a.scale, a.scale}, lv[2] = {0.0f, 0.0f}, unscale[2] = {1.0f, 1.0f};
            if constexpr (QUANT) {
                const float* sc = reinterpret_cast<const float*>(st + 2 * kWarpKeys * ROWB);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    kc[e] = a.scale * sc[g + 8 * e];
                    const float v = fmaxf(sc[16 + g + 8 * e], 0x1p-100f);
                    lv[e] = __log2f(v);
                    unscale[e] = __fdividef(1.0f, v);
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // the powers of two of q's row and of the key first: one may be as large as the other is small
                    if constexpr (QUANT) x[nt][e] = fmaf(x[nt][e], factor[nt][e & 1] * kc[e >> 1], lv[e >> 1]);
                    else x[nt][e] *= a.scale;
                }
            const bool whole = there == 0xffffu && key0 + kWarpKeys - 1 <= it.p_lo &&
                               (a.window == 0 || key0 > it.p_hi - a.window || key0 + kWarpKeys <= a.sinks);
            unsigned seen = 0xffffffffu;
            if (!whole) {
                seen = 0;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = g + 8 * (e >> 1), key = key0 + i, p = pos[nt][e & 1];
                        const bool sees = (there >> i & 1) != 0 && key <= p &&
                                          (a.window == 0 || key > p - a.window || key < a.sinks);
                        if (sees) seen |= 1u << (nt * 4 + e);
                        else x[nt][e] = -INFINITY;
                    }
            }
            bool grew = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) grew |= x[nt][e] > limit[nt][e & 1];
            if (__any_sync(0xffffffffu, grew)) {
                // Values that are all zero matter only here, where a maximum is about to move.
                if constexpr (QUANT) {
                    constexpr int TIMES = kWarpKeys * CHUNKS / 32;
                    uint4 w[TIMES];
#pragma unroll
                    for (int i = 0; i < TIMES; ++i)
                        w[i] = *reinterpret_cast<const uint4*>(st + kWarpKeys * ROWB + i * 512 + lane * 16);
                    const uint32_t empty = empty_rows<CHUNKS>(w) >> g;  // bits 0 and 8: of the lane's keys
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if ((empty >> 8 * i & 1) != 0 && lv[i] > kEmptyLog) {
                            const float by = kEmptyLog - lv[i];
                            unscale[i] = 0x1p64f;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                x[nt][2 * i] += by;
                                x[nt][2 * i + 1] += by;
                            }
                        }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = fmaxf(x[nt][e], x[nt][e + 2]);
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        if (top > limit[nt][e]) {
                            // nothing has been summed yet where there was no limit
                            const float to = top - kLift<M>;
                            const float alpha = limit[nt][e] == -INFINITY ? 0.0f : ex2(m[nt][e] - to);
                            m[nt][e] = to;
                            limit[nt][e] = top + kGrowth;
                            l[nt][e] *= alpha;
#pragma unroll
                            for (int mt = 0; mt < KS; ++mt) {
                                o[mt][nt][e] *= alpha;
                                o[mt][nt][e + 2] *= alpha;
                            }
                        }
                    }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    x[nt][e] = ex2(x[nt][e] - m[nt][e]);
                    x[nt][e + 2] = ex2(x[nt][e + 2] - m[nt][e]);
                    l[nt][e] += QUANT ? fmaf(x[nt][e], unscale[0], x[nt][e + 2] * unscale[1]) : x[nt][e] + x[nt][e + 2];
                }
            // The weights go to the 16-bit operand type, as the values are; the sum above took them in fp32.
            uint32_t pf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                pf[nt][0] = transpose8x8(pack2<M>(x[nt][0], x[nt][1]));
                pf[nt][1] = transpose8x8(pack2<M>(x[nt][2], x[nt][3]));
            }
            auto values = [&](auto check, int mt, uint32_t(&vf)[4]) {
                if constexpr (check.value) {
                    // A weight of zero does not keep an infinity or NaN out of a product, so a
                    // value that is not finite is taken out of the operand and, for the rows that
                    // see it, counted by a product of its own.
                    using B = Half16<M>;
                    uint32_t bad[4], any = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        bad[i] = __vcmpgeu2(vf[i] & 0x7fff7fffu, B::inf | B::inf << 16);
                        any |= bad[i];
                    }
                    if (__any_sync(0xffffffffu, any != 0)) {
                        constexpr uint32_t ONE = B::one | B::one << 16;
                        uint32_t kind[3][4];  // +inf, -inf, NaN as ones
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            kind[0][i] = __vcmpeq2(vf[i], B::inf | B::inf << 16) & ONE;
                            kind[1][i] = __vcmpeq2(vf[i], (B::inf | B::inf << 16) | 0x80008000u) & ONE;
                            kind[2][i] = __vcmpgtu2(vf[i] & 0x7fff7fffu, B::inf | B::inf << 16) & ONE;
                            vf[i] &= ~bad[i];
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            auto one = [&](int e) { return seen >> (nt * 4 + e) & 1 ? 1.0f : 0.0f; };
                            const uint32_t b0 = transpose8x8(pack2<M>(one(0), one(1)));
                            const uint32_t b1 = transpose8x8(pack2<M>(one(2), one(3)));
#pragma unroll
                            for (int k = 0; k < 3; ++k) {
                                float n[4] = {};
                                mma16816<M>(n, kind[k], b0, b1);
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (n[e] > 0.0f) o[mt][nt][e] += k == 0 ? INFINITY : k == 1 ? -INFINITY : NAN;
                            }
                        }
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816<M>(o[mt][nt], vf, pf[nt][0], pf[nt][1]);
            };
            auto weigh = [&](auto check) {
#pragma unroll
                for (int first = 0; first < MATRICES; first += VAHEAD) {
                    if constexpr (NT != 1) read_values(first);
#pragma unroll
                    for (int i = 0; i < VAHEAD; ++i) {
                        if constexpr (QUANT) {
                            // A 16-bit element of V is the pair (2u, 2u + 1) of a tile's 16 head columns:
                            // its transposed matrices give rows 2u and 2u + 1, which are taken as rows
                            // u and u + 8 of the operand.
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                uint32_t vf[4];
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const uint2 f = e4m3x4_to_half2x2(__byte_perm(vr[i][2 * k + e], 0, 0x3120));
                                    vf[2 * e] = f.x;
                                    vf[2 * e + 1] = f.y;
                                }
                                values(check, 2 * (first + i) + k, vf);
                            }
                        } else {
                            values(check, first + i, vr[i]);
                        }
                    }
                }
            };
            if (whole) weigh(std::false_type{});
            else weigh(std::true_type{});
            stage = stage == STAGES - 1 ? 0 : stage + 1;
            __syncwarp();  // the stage is read before the next copies into it
        }

        // ------------------------------------------------------------ join
        __syncthreads();  // the rings become the warps' results
        float* const join_o = reinterpret_cast<float*>(smem);
        float* const join_m = join_o + kRowsWarps * ROWS * Shape::kJoinStride;
        float* const join_l = join_m + kRowsWarps * ROWS;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float s = l[nt][e];
                s += __shfl_xor_sync(0xffffffffu, s, 4);
                s += __shfl_xor_sync(0xffffffffu, s, 8);
                s += __shfl_xor_sync(0xffffffffu, s, 16);
                const int r = nt * 8 + t4 * 2 + e;
                if (g == 0) {
                    join_m[warp * ROWS + r] = limit[nt][e] == -INFINITY ? -INFINITY : m[nt][e];
                    join_l[warp * ROWS + r] = s;
                }
                float* const to = join_o + (warp * ROWS + r) * Shape::kJoinStride;
#pragma unroll
                for (int mt = 0; mt < KS; ++mt) {
                    to[mt * 16 + (QUANT ? 2 * g : g)] = o[mt][nt][e];
                    to[mt * 16 + (QUANT ? 2 * g + 1 : g + 8)] = o[mt][nt][e + 2];
                }
            }
        __syncthreads();
        const bool begins = t0 == 0, ends = t_end == it.tiles;
        Block* const block = reinterpret_cast<Block*>(a.partial) + 2 * blockIdx.x + (begins ? 1 : 0);
        constexpr int LANES = DPAD / 4;  // of a row
        for (int r = tid / LANES; r < it.rows; r += kRowsThreads / LANES) {
            const int c = (tid % LANES) * 4;
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) top = fmaxf(top, join_m[w * ROWS + r]);
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) {
                const float f = ex2(join_m[w * ROWS + r] - ref);
                const float4 v = *reinterpret_cast<const float4*>(join_o + (w * ROWS + r) * Shape::kJoinStride + c);
                sum = fmaf(f, join_l[w * ROWS + r], sum);
                acc.x = fmaf(f, v.x, acc.x);
                acc.y = fmaf(f, v.y, acc.y);
                acc.z = fmaf(f, v.z, acc.z);
                acc.w = fmaf(f, v.w, acc.w);
            }
            if (begins && ends) {
                write_row<T>(a, it, r, c, acc, sum);
            } else {
                *reinterpret_cast<float4*>(&block->o[r][c]) = acc;
                if (c == 0) {
                    block->m[r] = top;
                    block->l[r] = sum;
                }
            }
        }
        if (begins && !ends && tid == 0) a.joins[blockIdx.x] = make_int4(it.b, it.rt, it.h, share.last_cta());
        if (!next_item<ROWS, kRowsKeys>(a, share)) return;
        __syncthreads();  // before the rings and the rows are filled again
    }
}

}  // namespace ako_b200
