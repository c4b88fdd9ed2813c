// Attention of many rows per sequence and kv head over a paged cache: chunks
// of prompts, on the tensor cores.
//
// A CTA holds 256 rows of one sequence and kv head (new tokens times the q
// heads that share it) as two halves of 128 and goes over the keys in tiles of
// 128, one CTA per SM. The scores S = Q K^T of a half go to tensor memory; its
// four warps, a row to a thread, take them from there, write the weights P
// over them in 16 bits, and O += P V reads P from tensor memory. While one
// half's warps work on their softmax the tensor cores work for the other:
//
//   tensor cores  | O_a += P_a V, S_a | O_b += P_b V, S_b | O_a += ...
//   half a's warps|                   | softmax of S_a    |
//   half b's warps| softmax of S_b    |                   | softmax of S_b
//
// Four more warps bring keys and values into shared memory (rows anywhere in
// the cache, swizzled for the products), and one thread issues the products.
// O stays in tensor memory. A row's maximum is followed only when it grows by
// more than a factor of 2^8: weights relative to an older maximum are the same
// numbers after the division by their sum, and fit the 16-bit types; O is then
// rescaled rarely.
//
// Bound: per tile and half, two products of 128 x 128 x head_dim take 8 *
// head_dim cycles and the 16384 exponentials 1024 cycles of the SM's 16 a
// cycle; for a head of 128 the two are equal.
//
// Every wait is bounded. If one runs out, all roles stop waiting, the rows not
// yet written become NaN, and the status word is set.
#pragma once

#include "paged_attention_rows.cuh"
#include "tcgen05.cuh"

namespace ako_b200 {

constexpr int kTilesThreads = 512;
constexpr int kTilesRows = 256;
constexpr int kTilesKeys = 128;
// Tiles whose key data are kept: the loading warps find a tile's keys one tile
// before they bring them, at most STAGES + 2 tiles ahead of the softmax.
constexpr int kMetaStages = 8;
constexpr int kOffsetStages = 4;
constexpr uint32_t kDrainLimit = 1u << 24;
// Registers per thread of the softmax, loading and issuing warps. The block is
// launched with 128 a thread, and 2 * 184 + 96 + 48 = 4 * 128.
constexpr int kSoftmaxRegs = 184, kLoadRegs = 96, kIssueRegs = 48;
constexpr float kGrowth = 8.0f;  // log2 of the factor by which a maximum may lag

struct TilesArgs {
    AttnArgs a;
    int* status;
    uint32_t wait_polls;
    float q_factor;  // -1, 0 or 1: the sign of the scale, taken into q
};

template <int DPAD>
struct TilesShape {
    static constexpr int kOperand = 128 * DPAD * 2;  // a tile of 128 rows
    static constexpr int kStages = DPAD == 128 ? 2 : 3;
    static constexpr int kSmem = 1024 + (2 + 2 * kStages) * kOperand;
};

// Data of a tile's keys that the softmax needs.
struct TileMeta {
    float kc[kTilesKeys], lv[kTilesKeys], unscale[kTilesKeys];  // of an e4m3 cache, as in the kernel for few rows
    uint32_t there[4];  // keys whose page exists and which some row may see
};

template <int STAGES>
struct TilesShared {
    TileMeta meta[kMetaStages];
    int64_t offset[kOffsetStages][2][kTilesKeys];  // of the keys' rows in k and v, or -1
    uint64_t k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES];
    uint64_t q_full[2], s_full[2], p_full[2], o_full[2], drained;
    uint32_t tmem;
    volatile int stop;     // a wait ran out
    volatile int odd;      // a value that is not finite was taken out of a tile that not every row sees
    ShareScratch scratch;
};

// Waits for a phase of `bar`; false when the limit ran out, here or in another role.
template <typename S>
__device__ __forceinline__ bool tile_wait(S& sm, uint64_t* bar, uint32_t phase, uint32_t polls) {
    for (uint32_t i = 0; i < polls; ++i) {
        if (mbar_try_wait(bar, phase)) return true;
        if (sm.stop) return false;
    }
    sm.stop = 1;
    return false;
}

// Whether every row of the item sees every key of a tile, as far as positions go.
__device__ __forceinline__ bool whole_tile(const AttnArgs& a, const Item& it, int key0) {
    return key0 + kTilesKeys - 1 <= it.p_lo &&
           (a.window == 0 || key0 > it.p_hi - a.window || key0 + kTilesKeys <= a.sinks);
}

__device__ __forceinline__ bool sees_key(const AttnArgs& a, int pos, int key) {
    return key <= pos && (a.window == 0 || key > pos - a.window || key < a.sinks);
}

// Adds to row r's result, at `out`, the values that are not finite of the keys
// that it sees in the part [t0, t1) of the item's tiles and that were taken
// out of their tiles: those that not every row sees.
template <typename T, bool QUANT, typename O>
__device__ __forceinline__ void add_odd_values(const AttnArgs& a, const Item& it, int t0, int t1, int r, O* out) {
    const int pos = it.kv - it.n + static_cast<int>(a.by_group.div(it.row0 + r));
    for (int t = t0; t < t1; ++t) {
        const int key0 = key_tile(it, t) * kTilesKeys;
        if (whole_tile(a, it, key0)) continue;
        for (int key = key0; key < key0 + kTilesKeys; ++key) {
            int slot;
            if (!sees_key(a, pos, key)) continue;
            const int page = page_of(a.seqs, a.cache, it.b, key, slot);
            if (page < 0) continue;
            const int64_t at = a.cache.v.offset(page, it.h, slot);
            for (int d = 0; d < a.cache.head_dim; ++d) {
                float x;
                if constexpr (QUANT) {
                    const uint8_t e = static_cast<const uint8_t*>(a.cache.v.p)[at + d];
                    x = (e & 0x7f) == 0x7f ? NAN : 0.0f;
                } else {
                    x = to_f32(static_cast<const T*>(a.cache.v.p)[at + d]);
                }
                if (!isfinite(x)) out[d] = from_f32<O>(to_f32(out[d]) + x);
            }
        }
    }
}

// ------------------------------------------------------------------ loading
// Eight 16-bit patterns: those that are not finite become 0; true if any was.
template <typename M>
__device__ __forceinline__ bool scrub(uint4& v) {
    constexpr uint32_t INF = Half16<M>::inf | Half16<M>::inf << 16;
    uint32_t* const w = reinterpret_cast<uint32_t*>(&v);
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t bad = __vcmpgeu2(w[i] & 0x7fff7fffu, INF);
        w[i] &= ~bad;
        any |= bad;
    }
    return any != 0;
}

template <typename T, bool QUANT, int DPAD>
struct TileLoader {
    using Shape = TilesShape<DPAD>;
    using Shared = TilesShared<Shape::kStages>;
    static constexpr int ES = QUANT ? 1 : 2;
    static constexpr int CHUNKS = DPAD * ES / 16;      // 16-byte chunks of a cached row
    static constexpr int ROWS = 128 / CHUNKS;          // rows that the 128 threads take at once
    static constexpr int EACH = kTilesKeys / ROWS;     // chunks of a thread
    const AttnArgs& a;
    Shared& sm;
    int tid, chunk, row0;
    bool real;  // the chunk lies within head_dim

    __device__ TileLoader(const AttnArgs& args, Shared& shared, int t)
        : a(args), sm(shared), tid(t), chunk(t % CHUNKS), row0(t / CHUNKS), real(chunk * 16 < args.cache.head_dim * ES) {}

    // Where the 16-bit chunk c of a row goes in a tile.
    static __device__ __forceinline__ uint32_t place(int row, int c) {
        return static_cast<uint32_t>((c >> 3) * (kTilesKeys * 128) + row * 128 + ((c & 7) ^ (row & 7)) * 16);
    }

    // Finds the rows of a tile's keys and fills its meta data; every thread looks after one key.
    __device__ __forceinline__ void find(const Item& it, int key0, int64_t (&offset)[2][kTilesKeys], TileMeta& meta) {
        const int key = key0 + tid;
        int page = -1, slot = 0;
        if (key <= it.p_hi && (key >= it.win_lo || key < a.sinks)) page = page_of(a.seqs, a.cache, it.b, key, slot);
        offset[0][tid] = page >= 0 ? a.cache.k.offset(page, it.h, slot) : -1;
        offset[1][tid] = page >= 0 ? a.cache.v.offset(page, it.h, slot) : -1;
        const unsigned there = __ballot_sync(0xffffffffu, page >= 0);
        if ((tid & 31) == 0) meta.there[tid >> 5] = there;
        if constexpr (QUANT) {
            float ks = 0.0f, vs = 1.0f;
            if (page >= 0) {
                ks = static_cast<const float*>(a.cache.ks.p)[a.cache.ks.offset(page, it.h, slot)];
                vs = fmaxf(static_cast<const float*>(a.cache.vs.p)[a.cache.vs.offset(page, it.h, slot)], 0x1p-100f);
            }
            meta.kc[tid] = ks * a.scale;
            meta.lv[tid] = __log2f(vs);
            meta.unscale[tid] = __fdividef(1.0f, vs);
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
    }

    // 16-bit caches: copies straight into the tile.
    __device__ __forceinline__ void copy(const void* base, const int64_t* offset, uint32_t tile) const {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int row = row0 + i * ROWS;
            const int64_t o = offset[row];
            const bool there = o >= 0 && real;
            cp_async16_or_zero(tile + place(row, chunk),
                               there ? static_cast<const uint8_t*>(base) + (o + chunk * 8) * 2 : base, there);
        }
    }

    // Takes what is not finite out of this thread's chunks of a tile of values.
    __device__ __forceinline__ void scrub_copied(uint8_t* tile) {
        bool any = false;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            uint4* const p = reinterpret_cast<uint4*>(tile + place(row0 + i * ROWS, chunk));
            uint4 v = *p;
            if (scrub<T>(v)) {
                *p = v;
                any = true;
            }
        }
        if (any) sm.odd = 1;
    }

    // e4m3 caches: into registers, and from there as fp16.
    __device__ __forceinline__ void fetch(const void* base, const int64_t* offset, uint4 (&v)[EACH]) const {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int64_t o = offset[row0 + i * ROWS];
            v[i] = make_uint4(0, 0, 0, 0);
            if (o >= 0 && real) v[i] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + o + chunk * 16);
        }
    }

    __device__ __forceinline__ void convert(const uint4 (&v)[EACH], uint8_t* tile, bool clean) {
        bool any = false;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint4 w = make_uint4(e4m3x2_to_half2(u[2 * half]), e4m3x2_to_half2(u[2 * half] >> 16),
                                     e4m3x2_to_half2(u[2 * half + 1]), e4m3x2_to_half2(u[2 * half + 1] >> 16));
                if (clean && scrub<__half>(w)) any = true;
                *reinterpret_cast<uint4*>(tile + place(row0 + i * ROWS, chunk * 2 + half)) = w;
            }
        }
        if (any) sm.odd = 1;
    }
};

template <typename T, bool QUANT, int DPAD>
__global__ void __launch_bounds__(kTilesThreads, 1) attn_tiles_kernel(const TilesArgs args) {
    pdl_enter();
    using Shape = TilesShape<DPAD>;
    using M = std::conditional_t<QUANT, __half, T>;
    using Block = PartialBlock<kTilesRows, DPAD>;
    constexpr int STAGES = Shape::kStages;
    constexpr int TYPE = std::is_same_v<M, __half> ? 0 : 1;
    constexpr uint32_t O_COL = 256;
    const AttnArgs& a = args.a;
    extern __shared__ __align__(1024) uint8_t raw[];
    __shared__ TilesShared<STAGES> sm;
    uint8_t* const tiles = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
    uint8_t* const q_tile = tiles;                        // two halves
    uint8_t* const k_tile = tiles + 2 * Shape::kOperand;  // STAGES of keys, then of values
    uint8_t* const v_tile = k_tile + STAGES * Shape::kOperand;
    const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31, wg = tid >> 7;
    const uint32_t polls = args.wait_polls;

    if (tid == 0) a.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
    Share share;
    if (!find_share<kTilesRows, kTilesKeys, kTilesThreads>(a, 1, sm.scratch, share)) return;
    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&sm.k_full[i], 128);
            mbar_init(&sm.v_full[i], 128);
            mbar_init(&sm.k_empty[i], 1);
            mbar_init(&sm.v_empty[i], 1);
        }
        for (int h = 0; h < 2; ++h) {
            mbar_init(&sm.q_full[h], 128);
            mbar_init(&sm.s_full[h], 1);
            mbar_init(&sm.p_full[h], 128);
            mbar_init(&sm.o_full[h], 1);
        }
        mbar_init(&sm.drained, 1);
        fence_mbar_init();
        sm.stop = 0;
        sm.odd = 0;
    }
    if (warp == 12) tmem_alloc<512>(&sm.tmem);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = sm.tmem;
    Item& it = share.it;
    int64_t at = share.begin;
    auto part_end = [&] { return static_cast<int>(min(static_cast<int64_t>(it.tiles), share.t + (share.end - at))); };
    // moves on to the next item; false when the share is done
    auto advance = [&](int t_end) {
        at += t_end - share.t;
        share.t = 0;
        return at < share.end && next_item<kTilesRows, kTilesKeys>(a, it);
    };

    if (wg == 3) {
        // ---------------------------------------------------------- products
        give_registers<kIssueRegs>();
        if (warp == 12 && lane == 0) {
            const int steps = (a.cache.head_dim + 15) / 16;
            const uint32_t s_shape = mma_shape(128, kTilesKeys, TYPE, false);
            const uint32_t o_shape = mma_shape(128, steps * 16, TYPE, true);
            constexpr uint32_t BLOCK = kTilesKeys * 128;  // bytes of 64 columns of a tile
            const uint32_t q_addr = smem_addr(q_tile), k_addr = smem_addr(k_tile), v_addr = smem_addr(v_tile);
            uint32_t n = 0;            // tiles so far
            uint32_t ns[2] = {0, 0};   // of a half
            uint32_t nq[2] = {0, 0};   // items of a half
            bool ok = true;
            auto weigh = [&](int h, uint32_t tile, bool add) {  // O_h (+)= P_h V
                ok = ok && tile_wait(sm, &sm.p_full[h], (ns[h] - 1) & 1, polls);
                ok = ok && tile_wait(sm, &sm.v_full[tile % STAGES], (tile / STAGES) & 1, polls);
                if (!ok) return;
                tmem_fence_after();
                const uint32_t v = v_addr + (tile % STAGES) * Shape::kOperand;
#pragma unroll
                for (int k = 0; k < kTilesKeys / 16; ++k)
                    mma_ts(tmem + O_COL + h * 128, tmem + h * 128 + k * 8, smem_operand(v + k * 16 * 128, BLOCK), o_shape,
                           add || k > 0);
            };
            do {
                const int t_end = part_end();
                const int halves = it.rows > 128 ? 2 : 1;
                for (int t = share.t; t < t_end && ok; ++t, ++n) {
                    ok = ok && tile_wait(sm, &sm.k_full[n % STAGES], (n / STAGES) & 1, polls);
                    for (int h = 0; h < halves && ok; ++h) {
                        if (t == share.t) {
                            ok = tile_wait(sm, &sm.q_full[h], nq[h] & 1, polls);
                            ++nq[h];
                        } else {
                            weigh(h, n - 1, t - 1 > share.t);
                            if (h == halves - 1) mma_commit(&sm.v_empty[(n - 1) % STAGES]);
                        }
                        if (!ok) break;
                        tmem_fence_after();
                        const uint32_t q = q_addr + h * Shape::kOperand, k = k_addr + (n % STAGES) * Shape::kOperand;
                        for (int s = 0; s < steps; ++s) {
                            const uint32_t to = (s >> 2) * BLOCK + (s & 3) * 32;
                            mma_ss(tmem + h * 128, smem_operand(q + to, 16), smem_operand(k + to, 16), s_shape, s > 0);
                        }
                        ++ns[h];
                        mma_commit(&sm.s_full[h]);
                    }
                    mma_commit(&sm.k_empty[n % STAGES]);
                }
                for (int h = 0; h < halves && ok; ++h) {
                    weigh(h, n - 1, t_end - 1 > share.t);
                    mma_commit(&sm.o_full[h]);
                }
                mma_commit(&sm.v_empty[(n - 1) % STAGES]);
                if (!advance(t_end)) break;
            } while (ok);
            // nothing of this CTA's is under way when it gives its tensor memory back
            mma_commit(&sm.drained);
            mbar_wait_bounded(&sm.drained, 0, kDrainLimit);
        }
        __syncwarp();
    } else if (wg == 2) {
        // ----------------------------------------------------------- loading
        give_registers<kLoadRegs>();
        TileLoader<T, QUANT, DPAD> load(a, sm, tid - 256);
        const uint32_t k_addr = smem_addr(k_tile), v_addr = smem_addr(v_tile);
        uint32_t n = 0;
        bool ok = true;
        uint64_t* pending = nullptr;  // full barrier of the copies under way before the last
        uint8_t* dirty = nullptr;     // their tile, if its values are to be cleaned
        auto landed = [&] {
            if (dirty != nullptr) load.scrub_copied(dirty);
            fence_proxy_async_smem();
            mbar_arrive(pending);
            pending = nullptr;
        };
        // Waits until a stage is free, handing on first what has been copied.
        auto acquire = [&](uint64_t* empty, uint32_t use) {
            const uint32_t phase = ((use / STAGES) & 1) ^ 1;
            if (mbar_try_wait(empty, phase)) return;
            if (pending != nullptr) {
                cp_async_wait<0>();
                landed();
            }
            ok = ok && tile_wait(sm, empty, phase, polls);
        };
        auto issued = [&](uint64_t* full, uint8_t* clean) {
            cp_async_commit();
            if (pending != nullptr) {
                cp_async_wait<1>();
                landed();
            }
            pending = full;
            dirty = clean;
        };
        // A tile's keys are found while the tile before is on its way.
        int t_end = part_end();
        int t = share.t;
        bool whole;
        auto find = [&] {
            const int key0 = key_tile(it, t) * kTilesKeys;
            whole = whole_tile(a, it, key0);
            load.find(it, key0, sm.offset[n % kOffsetStages], sm.meta[n % kMetaStages]);
        };
        auto next = [&] {
            ++n;
            if (++t == t_end) {
                if (!advance(t_end)) return false;
                t = 0;
                t_end = part_end();
            }
            find();
            return true;
        };
        find();
        bool more = true;
        [[maybe_unused]] uint4 kv[TileLoader<T, QUANT, DPAD>::EACH], vv[TileLoader<T, QUANT, DPAD>::EACH];
        if constexpr (QUANT) {
            load.fetch(a.cache.k.p, sm.offset[0][0], kv);
            load.fetch(a.cache.v.p, sm.offset[0][1], vv);
        }
        while (more) {
            const int st = n % STAGES;
            const uint32_t use = n;
            const bool clean = !whole;
            uint8_t* const vt = v_tile + st * Shape::kOperand;
            acquire(&sm.k_empty[st], use);
            if (!ok) break;
            if constexpr (!QUANT) {
                load.copy(a.cache.k.p, sm.offset[use % kOffsetStages][0], k_addr + st * Shape::kOperand);
                issued(&sm.k_full[st], nullptr);
                more = next();
                acquire(&sm.v_empty[st], use);
                if (!ok) break;
                load.copy(a.cache.v.p, sm.offset[use % kOffsetStages][1], v_addr + st * Shape::kOperand);
                issued(&sm.v_full[st], clean ? vt : nullptr);
            } else {
                load.convert(kv, k_tile + st * Shape::kOperand, false);
                fence_proxy_async_smem();
                mbar_arrive(&sm.k_full[st]);
                more = next();
                if (more) load.fetch(a.cache.k.p, sm.offset[n % kOffsetStages][0], kv);
                acquire(&sm.v_empty[st], use);
                if (!ok) break;
                load.convert(vv, vt, clean);
                fence_proxy_async_smem();
                mbar_arrive(&sm.v_full[st]);
                if (more) load.fetch(a.cache.v.p, sm.offset[n % kOffsetStages][1], vv);
            }
        }
        cp_async_wait<0>();
        if (pending != nullptr) landed();
    } else {
        // ----------------------------------------------------------- softmax
        take_registers<kSoftmaxRegs>();
        const int h = wg, row = tid & 127;
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // first lane of the warp, in bits 16 up
        const uint32_t s_at = tmem + lanes + h * 128, o_at = tmem + lanes + O_COL + h * 128;
        uint8_t* const my_q = q_tile + h * Shape::kOperand;
        uint32_t n = 0, ns = 0, no = 0;
        bool ok = true;
        int pos = 0;
        float factor = 1.0f;
        // Brings this thread's row of q into the half's tile; `factor` takes out what it was scaled by.
        auto load_q = [&] {
            const int r = h * 128 + row;
            const bool real = r < it.rows;
            pos = real ? it.kv - it.n + static_cast<int>(a.by_group.div(it.row0 + r)) : it.p_hi;
            const T* const p = static_cast<const T*>(a.q) + (real ? row_offset(a, it, it.row0 + r, a.qb, a.qs, a.qh) : 0);
            float top = 0.0f;
            factor = 1.0f;
            float inv = args.q_factor;
            if constexpr (QUANT && !std::is_same_v<T, __half>) {
                if (real) {
                    for (int c = 0; c < a.cache.head_dim; c += 8) {
                        const Packed<T, 8> x = ld_cached<T, 8>(p + c);
#pragma unroll
                        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(to_f32(x.v[i])));
                    }
                }
                if (top > 0.0f && top < INFINITY) {  // as in the kernel for few rows
                    const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127 - 8, -126), 118);
                    inv *= __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                    factor = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
                }
            }
#pragma unroll 4
            for (int c = 0; c < DPAD / 8; ++c) {
                Packed<M, 8> y;
                Packed<T, 8> x;
                *reinterpret_cast<uint4*>(&x) = make_uint4(0, 0, 0, 0);
                if (real && c * 8 < a.cache.head_dim) x = ld_cached<T, 8>(p + c * 8);
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float2 f = get2(x, i);
                    put2(y, i, f.x * inv, f.y * inv);
                }
                *reinterpret_cast<uint4*>(my_q + TileLoader<T, QUANT, DPAD>::place(row, c)) = *reinterpret_cast<uint4*>(&y);
            }
            fence_proxy_async_smem();
            mbar_arrive(&sm.q_full[h]);
        };
        bool loaded = false;
        while (true) {
            const int t0 = share.t, t_end = part_end();
            const bool mine = it.rows > h * 128;
            if (!mine) {  // the other half's rows are all there are
                n += t_end - t0;
                loaded = false;
                if (!advance(t_end)) break;
                continue;
            }
            if (!loaded) load_q();
            // Warps without a row take part in the barriers alone.
            const bool rows = h * 128 + (warp & 3) * 32 < it.rows;
            float ref = -INFINITY, sum = 0.0f;
            for (int t = t0; t < t_end && ok; ++t, ++n, ++ns) {
                const int key0 = key_tile(it, t) * kTilesKeys;
                const TileMeta& meta = sm.meta[n % kMetaStages];
                ok = tile_wait(sm, &sm.s_full[h], ns & 1, polls);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tmem_fence_after();
                if (rows) {
                    float x[kTilesKeys];
#pragma unroll
                    for (int c = 0; c < kTilesKeys; c += 32) tmem_load32(s_at + c, reinterpret_cast<uint32_t*>(x + c));
                    tmem_wait_load();
                    if constexpr (QUANT) {
#pragma unroll
                        for (int c = 0; c < kTilesKeys; c += 4) {
                            const float4 kc = *reinterpret_cast<const float4*>(meta.kc + c);
                            const float4 lv = *reinterpret_cast<const float4*>(meta.lv + c);
                            x[c] = fmaf(x[c], kc.x * factor, lv.x);
                            x[c + 1] = fmaf(x[c + 1], kc.y * factor, lv.y);
                            x[c + 2] = fmaf(x[c + 2], kc.z * factor, lv.z);
                            x[c + 3] = fmaf(x[c + 3], kc.w * factor, lv.w);
                        }
                    }
                    const uint32_t there[4] = {meta.there[0], meta.there[1], meta.there[2], meta.there[3]};
                    const bool full = (there[0] & there[1] & there[2] & there[3]) == 0xffffffffu;
                    if (!full || !whole_tile(a, it, key0)) {
#pragma unroll
                        for (int c = 0; c < kTilesKeys; ++c)
                            if ((there[c / 32] >> (c % 32) & 1) == 0 || !sees_key(a, pos, key0 + c)) x[c] = -INFINITY;
                    }
                    float top = x[0];
#pragma unroll
                    for (int c = 1; c < kTilesKeys; ++c) top = fmaxf(top, x[c]);
                    const float scale = QUANT ? 1.0f : a.scale;
                    top *= scale;
                    const bool grew = top > ref + (ref == -INFINITY ? 0.0f : kGrowth);
                    if (__any_sync(0xffffffffu, grew)) {
                        const float to = grew ? top : ref;
                        const float alpha = grew ? ex2(ref - to) : 1.0f;
                        ref = to;
                        sum *= alpha;
                        if (t > t0) {
#pragma unroll
                            for (int c = 0; c < DPAD; c += 32) {
                                uint32_t o[32];
                                tmem_load32(o_at + c, o);
                                tmem_wait_load();
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                                tmem_store32(o_at + c, o);
                            }
                        }
                    }
                    const float base = ref == -INFINITY ? 0.0f : ref;
                    float part[4] = {};
#pragma unroll
                    for (int c = 0; c < kTilesKeys; c += 32) {
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float p0 = ex2(fmaf(x[c + i], scale, -base)), p1 = ex2(fmaf(x[c + i + 1], scale, -base));
                            if constexpr (QUANT) {
                                const float2 un = *reinterpret_cast<const float2*>(meta.unscale + c + i);
                                part[i & 2] = fmaf(p0, un.x, part[i & 2]);
                                part[(i & 2) + 1] = fmaf(p1, un.y, part[(i & 2) + 1]);
                            } else {
                                part[i & 2] += p0;
                                part[(i & 2) + 1] += p1;
                            }
                            // the weights in the values' 16 bits; their sum above in fp32
                            w[i / 2] = pack2<M>(p0, p1);
                        }
                        tmem_store16(s_at + c / 2, w);
                    }
                    sum += (part[0] + part[1]) + (part[2] + part[3]);
                    tmem_wait_store();
                }
                tmem_fence_before();
                mbar_arrive(&sm.p_full[h]);
            }
            // The next item's rows while this one's last product runs.
            const Item done = it;
            const int64_t after = at + (t_end - t0);
            const bool more = advance(t_end);
            loaded = false;
            if (more && it.rows > h * 128 && ok) {
                load_q();
                loaded = true;
            }
            ok = ok && tile_wait(sm, &sm.o_full[h], no & 1, polls);
            ok = __all_sync(0xffffffffu, ok);
            ++no;
            tmem_fence_after();
            const bool begins = t0 == 0, ends = t_end == done.tiles;
            const int r = h * 128 + row;
            if (rows) {
                Block* const block = reinterpret_cast<Block*>(a.partial) + 2 * blockIdx.x + (begins ? 1 : 0);
                const float nan = __int_as_float(0x7fffffff);
                const float inv = !ok ? nan : sum == 0.0f ? 0.0f : __fdividef(1.0f, sum);
                T* const to = static_cast<T*>(a.out) +
                              (r < done.rows ? row_offset(a, done, done.row0 + r, a.ob, a.os, a.oh) : 0);
#pragma unroll
                for (int c = 0; c < DPAD; c += 32) {
                    uint32_t o[32];
                    __syncwarp();
                    tmem_load32(o_at + c, o);
                    tmem_wait_load();
                    if (r >= done.rows) {
                        // a row of the tile that the item does not have
                    } else if (begins && ends) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            if (c + i >= a.cache.head_dim) break;
                            Packed<T, 8> y;
#pragma unroll
                            for (int e = 0; e < 8; e += 2)
                                put2(y, e, __uint_as_float(o[i + e]) * inv, __uint_as_float(o[i + e + 1]) * inv);
                            *reinterpret_cast<uint4*>(to + c + i) = *reinterpret_cast<uint4*>(&y);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<uint4*>(&block->o[r][c + i]) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                }
                if (r < done.rows) {
                    if (!(begins && ends)) {
                        block->m[r] = ref;
                        block->l[r] = ok ? sum : nan;
                    }
                    if (sm.odd) {
                        if (begins && ends) add_odd_values<T, QUANT, T>(a, done, t0, t_end, r, to);
                        else add_odd_values<T, QUANT, float>(a, done, t0, t_end, r, block->o[r]);
                    }
                }
            }
            tmem_fence_before();
            if (begins && !ends && row == 0 && h == 0)
                a.joins[blockIdx.x] = make_int4(done.b, done.rt, done.h, owner(share, after + (done.tiles - t_end) - 1));
            if (!more) break;
        }
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (tid == 0 && sm.stop) *reinterpret_cast<volatile int*>(args.status) = kStatusWaitTimeout;
    if (warp == 12) tmem_free<512>(tmem);
}

}  // namespace ako_b200
