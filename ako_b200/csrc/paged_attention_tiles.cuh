// Attention of many rows per sequence and kv head over a paged cache: chunks
// of prompts, on the tensor cores.
//
// A CTA holds 256 rows of one sequence and kv head (new tokens times the q
// heads that share it) as two halves of 128 and goes over the keys in tiles of
// 128, one CTA per SM. The scores S = Q K^T of a half go to tensor memory; its
// four warps, a row to a thread, take them from there, write the weights P over
// them in 16 bits, and O += P V reads P from tensor memory, the first 96 keys'
// (PV) as soon as they are there and the last 32 keys' (pv) with the next S.
// While one half's warps work on their softmax the tensor cores work for the
// other's:
//
//   tensor cores  | PV_a | pv_a, S_a | PV_b | pv_b, S_b | PV_a | pv_a, S_a | ...
//   half a's warps| soft-|           | softmax of S_a          |
//   half b's warps| softmax              |              | softmax of S_b ...
//
// S is taken 128 keys at a time because a product of 128 x 64 reads shared
// memory for its first operand at more than the tensor cores' own rate (391
// cycles measured against 260, and 520 for 128 x 128).
//
// Four more warps bring keys and values into shared memory (rows anywhere in
// the cache, swizzled for the products), and one thread issues the products.
// O stays in tensor memory. A row's maximum is followed only when it grows by
// more than a factor of 2^8: weights relative to an older maximum are the same
// numbers after the division by their sum, and fit the 16-bit types; O is then
// rescaled rarely.
//
// Where items change, what the next one needs is found while the last products
// run, and that code is kept short: it took 8 prompts of 2048 tokens from 382 to
// 347 us on one card. Over the cards and clocks met they take 345 to 397 us.
//
// Bound: per tile and half, two products of 128 x 128 x head_dim take 8 *
// head_dim cycles and the 16384 exponentials 1024 cycles of the SM's 16 a
// cycle; for a head of 128 the two are equal, 2080 cycles a tile for both
// halves. Measured, a tile takes about 3500: a half's softmax (2000 from the
// scores' arrival to the last weights) and its products do not overlap, and
// the halves' products wait for one another. 2048 new tokens on 16384 cached
// ones, 32 heads of 128 and 8 kv heads: 498 to 585 us in bf16 by the card and its
// clock, 1.17 to 1.00 PFLOP/s; 826 to 841 us in e4m3 (786 to 796 with fp16
// queries), where the softmax reads three more numbers for each key from shared
// memory and four warps convert every tile through registers.
//
// A key of an e4m3 cache whose values are all zero must not set a row's maximum
// (kEmptyLog). The loading warps note such keys with the values, and the softmax
// waits for that where a maximum is about to move, once or a few times an item:
// 83 to 87 us for 12 mixed sequences, 650 to 670 for e4m3 prompts of 8 x 2048.
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
// Tiles that an item's begin and end take as long as: 9,000 cycles for its
// queries, first scores, last products and output, several times what their
// instructions would take; likely they have left the instruction cache by the
// time they run again, since making the code shorter helped. Counting it
// when the work is shared out took prompts of 8 x 2048 from 549 to 424 us; 2, 3
// and 4 are within 1% of one another.
constexpr int kTilesCost = 4;
constexpr int kEarly = 96;  // keys whose weights are handed on before the tile's others
// Tiles whose key data are kept: the loading warps find a tile's keys one tile
// before they bring them, at most STAGES + 2 tiles ahead of the softmax.
constexpr int kMetaStages = 8;
constexpr uint32_t kWaitCycles = 1u << 31;  // of a wait, about a second
constexpr uint32_t kDrainPolls = 1u << 24;
// Registers per thread of the softmax, loading and issuing warps. The block is
// launched with 128 a thread, and 2 * 192 + 88 + 40 = 4 * 128. An e4m3 cache's
// loading warps hold a tile's keys or values in them: with 80 and 48, 2048 tokens
// on 16384 took 863 us where these took 784.
constexpr int kSoftmaxRegs = 192, kLoadRegs = 88, kIssueRegs = 40;

struct TilesArgs {
    // The cache's keys and values as (page, head, slot, column) in boxes of `box` slots and 64
    // columns, swizzled as the tiles are; box is 0 where pages do not divide into such boxes.
    CUtensorMap k_map, v_map;
    int box;
    AttnArgs a;
    int* status;
    uint32_t wait_polls;
    float q_factor;  // -1, 0 or 1: the sign of the scale, taken into q
};

template <int DPAD>
struct TilesShape {
    static constexpr int kOperand = 128 * DPAD * 2;  // a tile of 128 rows
    static constexpr int kStages = DPAD == 128 ? 2 : 3;  // what shared memory holds next to q
    static constexpr int kSmem = 1024 + (2 + 2 * kStages) * kOperand;
};

// Data of a tile's keys that the softmax needs.
struct TileMeta {
    float kc[kTilesKeys], lv[kTilesKeys], unscale[kTilesKeys];  // of an e4m3 cache, as in the kernel for few rows
    uint32_t there[4];  // keys whose page exists and which some row may see
    uint32_t empty[4];  // of an e4m3 cache, keys whose values are all zero; known when the values are there
};

template <int STAGES>
struct TilesShared {
    TileMeta meta[kMetaStages];
    uint64_t k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES];
    uint64_t q_full[2], s_full[2], p_full[2][2], o_full[2], drained;
    uint4 staging[8][128];  // of a softmax warp: 32 rows of 64 bytes on their way out
    uint32_t tmem;
    volatile int stop;     // a wait ran out
    volatile int odd;      // a value that is not finite was taken out of a tile that not every row sees
    ShareScratch scratch;
};

// Waits for a phase of `bar`, at most `polls` polls and a second or so (a poll
// may sleep).
__device__ __forceinline__ bool wait_bounded(uint64_t* bar, uint32_t phase, uint32_t polls, const volatile int* stop) {
    const uint32_t begin = static_cast<uint32_t>(clock());
    for (uint32_t i = 0; i < polls; ++i) {
        if (mbar_try_wait(bar, phase)) return true;
        if (*stop || static_cast<uint32_t>(clock()) - begin > kWaitCycles) break;
    }
    return false;
}

// The same for a role: when its limit runs out, all roles stop.
template <typename S>
__device__ __forceinline__ bool tile_wait(S& sm, uint64_t* bar, uint32_t phase, uint32_t polls) {
    if (wait_bounded(bar, phase, polls, &sm.stop)) return true;
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
            const uint8_t* const row = a.cache.v.row(page, it.h, slot);
            for (int d = 0; d < a.cache.head_dim; ++d) {
                float x;
                if constexpr (QUANT) {
                    const uint8_t e = row[d];
                    x = (e & 0x7f) == 0x7f ? NAN : 0.0f;
                } else {
                    x = to_f32(reinterpret_cast<const T*>(row)[d]);
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

// One of the four loading warps. In an e4m3 cache each brings 32 keys of every
// tile and their values; in a 16-bit cache, whose copies need no registers,
// two warps bring 64 keys each and two 64 values each, so that neither waits
// for the other's stage. A lane looks after one place in the cache (or two)
// and copies chunks of several rows; 64 rows of which every row of q sees every
// key come as boxes of a tensor map instead, where the pages allow it.
template <typename T, bool QUANT, int DPAD>
struct TileLoader {
    static constexpr int ES = QUANT ? 1 : 2;
    static constexpr int CHUNKS = DPAD * ES / 16;  // 16-byte chunks of a cached row
    static constexpr int ROWS = 32 / CHUNKS;       // rows that the warp takes at once
    static constexpr int EACH = 32 / ROWS;         // chunks of a lane
    const AttnArgs& a;
    int rows0, lane, chunk, row0;  // the warp's first row of a tile; the lane's among those taken at once
    bool real;  // the chunk lies within head_dim

    // A key's place, as far as it is known: its table entry is on the way.
    struct Place {
        int page, slot, h;
        bool whole;  // of the tile
    };
    // Where its row is.
    struct Rows {
        int64_t k, v;  // offsets in 16 bytes, or -1
        float ks, vs;
        bool whole;
    };

    __device__ TileLoader(const AttnArgs& args, int first, int l)
        : a(args), rows0(first), lane(l), chunk(l % CHUNKS), row0(l / CHUNKS), real(chunk * 16 < args.cache.head_dim * ES) {}

    // Where the 16-bit chunk c of a row goes in a tile.
    static __device__ __forceinline__ uint32_t place(int row, int c) {
        return static_cast<uint32_t>((c >> 3) * (kTilesKeys * 128) + row * 128 + ((c & 7) ^ (row & 7)) * 16);
    }

    // Of the lane's key, `more` rows behind its first.
    __device__ __forceinline__ Place look_up(const Item& it, int key0, int more = 0) const {
        Place p{-1, 0, it.h, whole_tile(a, it, key0)};
        const int key = key0 + rows0 + more + lane;
        if (key <= it.p_hi && (key >= it.win_lo || key < a.sinks)) {
            const int i = static_cast<int>(a.cache.by_page.div(static_cast<uint32_t>(key)));
            p.slot = key - i * a.cache.page_size;
            p.page = a.seqs.table[it.b * a.seqs.table_stride + i];
        }
        return p;
    }

    __device__ __forceinline__ bool there(const Place& p) const { return p.page >= 0 && p.page < a.cache.num_pages; }

    // Notes which of 32 keys, `more` rows behind the warp's first, are there.
    __device__ __forceinline__ void put_there(const Place& p, TileMeta& meta, int more = 0) const {
        const unsigned bits = __ballot_sync(0xffffffffu, there(p));
        if (lane == 0) meta.there[(rows0 + more) / 32] = bits;
    }

    __device__ __forceinline__ Rows find(const Place& p) const {
        Rows r{-1, -1, 0.0f, 1.0f, p.whole};
        if (there(p)) {
            r.k = static_cast<int64_t>(a.cache.k.offset(p.page, p.h, p.slot));
            r.v = static_cast<int64_t>(a.cache.v.offset(p.page, p.h, p.slot));
            if constexpr (QUANT) {
                r.ks = *a.cache.ks.scale(p.page, p.h, p.slot);
                r.vs = *a.cache.vs.scale(p.page, p.h, p.slot);
            }
        }
        return r;
    }

    // An e4m3 cache's scales, as the kernel for few rows has them.
    __device__ __forceinline__ void put_scales(const Rows& r, TileMeta& meta) const {
        const float vs = fmaxf(r.vs, 0x1p-100f);
        meta.kc[rows0 + lane] = r.ks * a.scale;
        meta.lv[rows0 + lane] = __log2f(vs);
        meta.unscale[rows0 + lane] = __fdividef(1.0f, vs);
    }

    // 16-bit caches: copies straight into the tile.
    __device__ __forceinline__ void copy(const PagedTensor& from, const Place& p, uint32_t tile, int more) const {
        const int64_t offset = there(p) ? static_cast<int64_t>(from.offset(p.page, p.h, p.slot)) : -1;
        // The places first: the copies' order is fixed, and each would wait for its own.
        int64_t o[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) o[i] = __shfl_sync(0xffffffffu, offset, row0 + i * ROWS);
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const bool there = o[i] >= 0 && real;
            cp_async16_or_zero(tile + place(rows0 + more + row0 + i * ROWS, chunk),
                               static_cast<const uint8_t*>(from.p) + (there ? (o[i] + chunk) * 16 : 0), there);
        }
    }

    // Takes what is not finite out of this lane's chunks of a tile of values.
    __device__ __forceinline__ bool scrub_copied(uint8_t* tile) const {
        bool any = false;
#pragma unroll
        for (int i = 0; i < 2 * EACH; ++i) {
            uint4* const p = reinterpret_cast<uint4*>(tile + place(rows0 + row0 + i * ROWS, chunk));
            uint4 v = *p;
            if (scrub<T>(v)) {
                *p = v;
                any = true;
            }
        }
        return any;
    }

    // e4m3 caches: into registers, and from there as fp16.
    __device__ __forceinline__ void fetch(const void* base, int64_t offset, uint4 (&v)[EACH]) const {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int64_t o = __shfl_sync(0xffffffffu, offset, row0 + i * ROWS);
            v[i] = make_uint4(0, 0, 0, 0);
            if (o >= 0 && real) v[i] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + (o + chunk) * 16);
        }
    }

    // True if `clean` took anything out.
    __device__ __forceinline__ bool convert(const uint4 (&v)[EACH], uint8_t* tile, bool clean) const {
        bool any = false;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint2 lo = e4m3x4_to_half2x2(u[2 * half]), hi = e4m3x4_to_half2x2(u[2 * half + 1]);
                uint4 w = make_uint4(lo.x, lo.y, hi.x, hi.y);
                if (clean && scrub<__half>(w)) any = true;
                *reinterpret_cast<uint4*>(tile + place(rows0 + row0 + i * ROWS, chunk * 2 + half)) = w;
            }
        }
        return any;
    }
};

// Bits 32 w .. 32 w + 31 of the mask whose first `n` bits (none if negative) are set.
__device__ __forceinline__ uint32_t first_bits(int n, int w) {
    const int k = min(max(n - 32 * w, 0), 32);
    return k == 32 ? 0xffffffffu : (1u << k) - 1u;
}

template <typename T, bool QUANT, int DPAD>
__global__ void __launch_bounds__(kTilesThreads, 1) attn_tiles_kernel(const __grid_constant__ TilesArgs args) {
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
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0), wg = warp >> 2;
    const uint32_t polls = args.wait_polls;

    if (tid == 0) a.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
    Share<kTilesCost> share;
    if (!find_share<kTilesRows, kTilesKeys, kTilesCost, kTilesThreads>(a, kTilesCost + 1, sm.scratch, share)) return;
    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&sm.k_full[i], QUANT ? 128 : 64 + 2);  // 16 bits: two warps' copies, and the masks they note
            mbar_init(&sm.v_full[i], QUANT ? 128 : 64);
            mbar_init(&sm.k_empty[i], 1);
            mbar_init(&sm.v_empty[i], 1);
        }
        for (int h = 0; h < 2; ++h) {
            mbar_init(&sm.q_full[h], 128);
            mbar_init(&sm.s_full[h], 1);
            mbar_init(&sm.p_full[h][0], 128);
            mbar_init(&sm.p_full[h][1], 128);
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
    // moves on to the next item; false when the share is done
    auto advance = [&] { return next_item<kTilesRows, kTilesKeys>(a, share); };

    if (wg == 3) {
        // ---------------------------------------------------------- products
        give_registers<kIssueRegs>();
        if (warp != 12) return;
        // The whole warp follows the loop, so that addresses and descriptors are uniform; one
        // elected lane issues the products and commits them.
        const int steps = (a.cache.head_dim + 15) / 16;
        const uint32_t s_shape = mma_shape(128, kTilesKeys, TYPE, false);
        const uint32_t o_shape = mma_shape(128, steps * 16, TYPE, true);
        constexpr uint32_t BLOCK = kTilesKeys * 128;  // bytes of 64 columns of a tile
        // a descriptor's address counts 16 bytes
        const uint64_t q_desc = smem_operand(smem_addr(q_tile), 16), k_desc = smem_operand(smem_addr(k_tile), 16);
        const uint64_t v_desc = smem_operand(smem_addr(v_tile), BLOCK);
        uint32_t n = 0;           // tiles so far
        uint32_t ns[2] = {0, 0};  // of a half
        uint32_t nq[2] = {0, 0};  // items of a half
        bool ok = true;
        auto await = [&](uint64_t* bar, uint32_t phase) {
            ok = ok && tile_wait(sm, bar, phase & 1, polls);
            ok = __all_sync(0xffffffffu, ok);
            return ok;
        };
        // cp.async is not the products' proxy; tensor-map copies are.
        auto order_copies = [&](bool whole) {
            if (!QUANT && !(whole && args.box != 0)) fence_proxy_async_smem();
        };
        bool before = false;  // whether every row sees every key of the tile before
        // O_h (+)= P_h V over the half's last tile of scores, the CTA's tile `tile`
        auto weigh = [&](int h, uint32_t tile, bool add) {
            const uint64_t v = v_desc + (tile % STAGES) * Shape::kOperand / 16;
            const uint32_t o = tmem + O_COL + h * 128, p = tmem + h * 128;
            if (h == 0) {
                if (!await(&sm.v_full[tile % STAGES], tile / STAGES)) return;
                order_copies(before);
            }
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                if (!await(&sm.p_full[h][part], ns[h] - 1)) return;
                tmem_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < kTilesKeys / 16; ++k)
                        if ((k < kEarly / 16) == (part == 0))
                            mma_ts(o, p + k * 8, v + k * (16 * 128 / 16), o_shape, add || k > 0);
                }
            }
        };
        do {
            const int t0 = share.first(), t_end = share.last();
            const int halves = it.rows > 128 ? 2 : 1;
            for (int t = t0; t < t_end && ok; ++t, ++n) {
                if (t == t0) {
                    await(&sm.q_full[0], nq[0]++);
                    if (halves == 2) await(&sm.q_full[1], nq[1]++);
                }
                await(&sm.k_full[n % STAGES], n / STAGES);
                const bool whole = whole_tile(a, it, key_tile(it, t) * kTilesKeys);
                order_copies(whole && t > t0);  // q is copied too
                const uint64_t k = k_desc + (n % STAGES) * Shape::kOperand / 16;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h >= halves || !ok) break;
                    if (t > t0) weigh(h, n - 1, t - 1 > t0);
                    if (!ok) break;
                    if (elect_one()) {
                        const uint64_t q = q_desc + h * Shape::kOperand / 16;
#pragma unroll
                        for (int s = 0; s < DPAD / 16; ++s) {
                            const uint32_t to = ((s >> 2) * BLOCK + (s & 3) * 32) / 16;
                            if (s < steps) mma_ss(tmem + h * 128, q + to, k + to, s_shape, s > 0);
                        }
                        mma_commit(&sm.s_full[h]);
                    }
                    ++ns[h];
                }
                if (elect_one()) {
                    if (t > t0) mma_commit(&sm.v_empty[(n - 1) % STAGES]);
                    mma_commit(&sm.k_empty[n % STAGES]);
                }
                before = whole;
            }
            const bool more = advance();  // while the softmax is at the last tile
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h >= halves || !ok) break;
                weigh(h, n - 1, t_end - 1 > t0);
                if (!ok) break;  // the last product was not issued, so these rows are not to be had
                if (elect_one()) mma_commit(&sm.o_full[h]);
            }
            if (elect_one()) mma_commit(&sm.v_empty[(n - 1) % STAGES]);
            if (!more) break;
        } while (ok);
        // nothing of this CTA's is under way when it gives its tensor memory back
        if (elect_one()) mma_commit(&sm.drained);
        const volatile int never = 0;
        wait_bounded(&sm.drained, 0, kDrainPolls, &never);
        __syncwarp();
        // the other roles are done with tensor memory
        asm volatile("bar.sync 2, 416;" ::: "memory");
        tmem_fence_after();
        if (lane == 0 && sm.stop) *reinterpret_cast<volatile int*>(args.status) = kStatusWaitTimeout;
        tmem_free<512>(tmem);
    } else if (wg == 2) {
        // ----------------------------------------------------------- loading
        give_registers<kLoadRegs>();
        using Loader = TileLoader<T, QUANT, DPAD>;
        const Loader load(a, QUANT ? (warp & 3) * 32 : (warp & 1) * 64, lane);
        bool ok = true;
        auto acquire = [&](uint64_t* empty, uint32_t use) {
            ok = ok && tile_wait(sm, empty, ((use / STAGES) & 1) ^ 1, polls);
            ok = __all_sync(0xffffffffu, ok);
        };
        // The table entries of a tile's keys are asked for ahead of the tile (by two tiles in an
        // e4m3 cache, whose scales are asked for by one), so that it does not wait for them.
        int t = share.first(), t_end = share.last();
        // moves on to the next tile; false behind the last
        auto step = [&] {
            if (++t < t_end) return true;
            if (!advance()) return false;
            t = share.first();
            t_end = share.last();
            return true;
        };
        auto key0 = [&] { return key_tile(it, t) * kTilesKeys; };
        if constexpr (!QUANT) {
            using Place = typename Loader::Place;
            const bool values = (warp & 2) != 0;
            const PagedTensor& from = values ? a.cache.v : a.cache.k;
            uint8_t* const tile = values ? v_tile : k_tile;
            const uint32_t tile_addr = smem_addr(tile);
            uint64_t* const full = values ? sm.v_full : sm.k_full;
            uint64_t* const empty = values ? sm.v_empty : sm.k_empty;
            Place p0 = load.look_up(it, key0()), p1 = load.look_up(it, key0(), 32);
            bool more = true;
            uint32_t n = 0;
            for (; more; ++n) {
                const int st = n % STAGES;
                const Place now0 = p0, now1 = p1;
                more = step();
                if (more) {
                    p0 = load.look_up(it, key0());
                    p1 = load.look_up(it, key0(), 32);
                }
                acquire(&empty[st], n);
                if (!ok) break;
                if (!values) {
                    load.put_there(now0, sm.meta[n % kMetaStages]);
                    load.put_there(now1, sm.meta[n % kMetaStages], 32);
                    // an arrival by cp.async hands on its copies, not what was stored before it
                    if (lane == 0) mbar_arrive(&full[st]);
                }
                if (args.box != 0 && now0.whole && __all_sync(0xffffffffu, load.there(now0) && load.there(now1))) {
                    // Boxes of whole pages, or of 64 rows of one, a lane to each.
                    constexpr int BLOCKS = DPAD / 64;
                    const int r = lane / BLOCKS * args.box, block = lane % BLOCKS;
                    const int page0 = __shfl_sync(0xffffffffu, now0.page, r & 31), page1 = __shfl_sync(0xffffffffu, now1.page, r & 31);
                    const int slot0 = __shfl_sync(0xffffffffu, now0.slot, r & 31), slot1 = __shfl_sync(0xffffffffu, now1.slot, r & 31);
                    if (lane == 0) mbar_expect_tx(&full[st], 64 * DPAD * 2);
                    else mbar_arrive(&full[st]);
                    __syncwarp();
                    if (r < 64)
                        tensor_load(tile_addr + st * Shape::kOperand + block * (kTilesKeys * 128) + ((warp & 1) * 64 + r) * 128,
                                    values ? &args.v_map : &args.k_map, block * 64, r < 32 ? slot0 : slot1, now0.h,
                                    r < 32 ? page0 : page1, &full[st]);
                    continue;
                }
                load.copy(from, now0, tile_addr + st * Shape::kOperand, 0);
                load.copy(from, now1, tile_addr + st * Shape::kOperand, 32);
                if (now0.whole ? args.box == 0 : !values) {
                    mbar_arrive_copied(&full[st]);
                } else {
                    cp_async_wait_everything();
                    if (!now0.whole && load.scrub_copied(tile + st * Shape::kOperand)) sm.odd = 1;
                    fence_proxy_async_smem();
                    mbar_arrive(&full[st]);
                }
            }
            // The last stages' copies by tensor map land before the CTA ends, even where whoever was to use
            // them has given up; cp.async's own wait below does not cover them.
            const volatile int never = 0;
            for (uint32_t u = n > STAGES ? n - STAGES : 0; u < n; ++u)
                wait_bounded(&full[u % STAGES], (u / STAGES) & 1, kDrainPolls, &never);
        } else {
            typename Loader::Place place = load.look_up(it, key0());
            load.put_there(place, sm.meta[0]);
            typename Loader::Rows rows = load.find(place);
            bool more = step();
            if (more) place = load.look_up(it, key0());
            for (uint32_t n = 0;; ++n) {
                const int st = n % STAGES;
                const typename Loader::Rows now = rows;
                const bool next = more;
                uint4 v[Loader::EACH];  // of keys, then of values: both at once do not fit the registers
                load.fetch(a.cache.k.p, now.k, v);
                if (next) {
                    rows = load.find(place);
                    load.put_there(place, sm.meta[(n + 1) % kMetaStages]);
                    more = step();
                    if (more) place = load.look_up(it, key0());
                }
                acquire(&sm.k_empty[st], n);
                if (!ok) break;
                load.put_scales(now, sm.meta[n % kMetaStages]);
                load.convert(v, k_tile + st * Shape::kOperand, false);
                load.fetch(a.cache.v.p, now.v, v);
                fence_proxy_async_smem();
                mbar_arrive(&sm.k_full[st]);
                acquire(&sm.v_empty[st], n);
                if (!ok) break;
                const uint32_t empties = empty_rows<Loader::CHUNKS>(v);
                if (lane == 0) sm.meta[n % kMetaStages].empty[warp & 3] = empties;
                if (load.convert(v, v_tile + st * Shape::kOperand, !now.whole)) sm.odd = 1;
                fence_proxy_async_smem();
                mbar_arrive(&sm.v_full[st]);
                if (!next) break;
            }
        }
        cp_async_wait_everything();
        asm volatile("bar.arrive 2, 416;" ::: "memory");
    } else {
        // ----------------------------------------------------------- softmax
        take_registers<kSoftmaxRegs>();
        const int h = wg, row = tid & 127, row0 = h * 128 + (warp & 3) * 32;
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // first lane of the warp, in bits 16 up
        const uint32_t s_at = tmem + lanes + h * 128, o_at = tmem + lanes + O_COL + h * 128;
        uint8_t* const my_q = q_tile + h * Shape::kOperand;
        uint4* const staging = sm.staging[warp];
        uint32_t n = 0, ns = 0, no = 0;  // tiles of the CTA and of this half, and the half's items
        bool ok = true;
        int pos = 0;
        float factor = 1.0f;
        // Brings the warp's rows of q into the half's tile, a row by DPAD / 8 lanes; `factor` takes
        // out what this thread's row was scaled by.
        auto load_q = [&](const Item& it) {
            constexpr int LANES = DPAD / 8, TAKEN = 32 / LANES, TIMES = 32 / TAKEN;
            const int r = row0 + lane, c = lane % LANES;
            const bool real = r < it.rows;
            pos = real ? it.kv - it.n + static_cast<int>(a.by_group.div(it.row0 + r)) : it.p_hi;
            const int64_t mine = real ? row_offset(a, it, it.row0 + r, a.qb, a.qs, a.qh) : -1;
            if (!QUANT && args.q_factor == 1.0f) {  // as it is
#pragma unroll 4
                for (int i = 0; i < TIMES; ++i) {
                    const int64_t o = __shfl_sync(0xffffffffu, mine, i * TAKEN + lane / LANES);
                    const bool there = o >= 0 && c * 8 < a.cache.head_dim;
                    cp_async16_or_zero(smem_addr(my_q) + TileLoader<T, QUANT, DPAD>::place(
                                                             (warp & 3) * 32 + i * TAKEN + lane / LANES, c),
                                       static_cast<const T*>(a.q) + (there ? o + c * 8 : 0), there);
                }
                mbar_arrive_copied(&sm.q_full[h]);
                return;
            }
            factor = 1.0f;
            Packed<T, 8> x[TIMES];
#pragma unroll
            for (int i = 0; i < TIMES; ++i) {
                const int64_t o = __shfl_sync(0xffffffffu, mine, i * TAKEN + lane / LANES);
                *reinterpret_cast<uint4*>(&x[i]) = make_uint4(0, 0, 0, 0);
                if (o >= 0 && c * 8 < a.cache.head_dim) x[i] = ld_cached<T, 8>(static_cast<const T*>(a.q) + o + c * 8);
            }
#pragma unroll
            for (int i = 0; i < TIMES; ++i) {
                const int to = i * TAKEN + lane / LANES;
                float inv = args.q_factor;
                if constexpr (QUANT && !std::is_same_v<T, __half>) {
                    float top = 0.0f, f = 1.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(to_f32(x[i].v[e])));
#pragma unroll
                    for (int off = LANES / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                    if (top > 0.0f && top < INFINITY) {  // as in the kernel for few rows
                        const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127 - 8, -126), 118);
                        inv *= __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                        f = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
                    }
                    const float g = __shfl_sync(0xffffffffu, f, (lane % TAKEN) * LANES);
                    if (lane / TAKEN == i) factor = g;
                }
                Packed<M, 8> y;
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float2 f = get2(x[i], e);
                    put2(y, e, f.x * inv, f.y * inv);
                }
                *reinterpret_cast<uint4*>(my_q + TileLoader<T, QUANT, DPAD>::place((warp & 3) * 32 + to, c)) =
                    *reinterpret_cast<uint4*>(&y);
            }
            fence_proxy_async_smem();
            mbar_arrive(&sm.q_full[h]);
        };
        bool loaded = false;
        while (true) {
            const int t0 = share.first(), t_end = share.last();
            if (it.rows <= h * 128) {  // the other half's rows are all there are
                n += t_end - t0;
                loaded = false;
                if (!advance()) break;
                continue;
            }
            if (!loaded) load_q(it);
            // Warps without a row take part in the barriers alone.
            const bool rows = row0 < it.rows;
            const int my_pos = pos;
            const float my_factor = factor;
            // The next item and its rows of q, which take the place of this one's once the last scores
            // are there.
            Share<kTilesCost> following = share;
            bool more = false;
            loaded = false;
            auto prepare_next = [&] {
                more = next_item<kTilesRows, kTilesKeys>(a, following);
                if (more && following.it.rows > h * 128) {
                    load_q(following.it);
                    loaded = true;
                }
            };
            const float scale = QUANT ? 1.0f : a.scale;
            float ref = -INFINITY, sum = 0.0f;
            for (int t = t0; t < t_end && ok; ++t, ++n, ++ns) {
                const TileMeta& meta = sm.meta[n % kMetaStages];
                const int key0 = key_tile(it, t) * kTilesKeys;
                ok = tile_wait(sm, &sm.s_full[h], ns & 1, polls);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tmem_fence_after();
                if (rows) {
                    float x[kTilesKeys];
#pragma unroll
                    for (int c = 0; c < kTilesKeys; c += 32) tmem_load32(s_at + c, reinterpret_cast<uint32_t*>(x + c));
                    const uint4 there = *reinterpret_cast<const uint4*>(meta.there);
                    const bool whole = (there.x & there.y & there.z & there.w) == 0xffffffffu && whole_tile(a, it, key0);
                    tmem_wait_load();
                    if constexpr (QUANT) {
#pragma unroll
                        for (int c = 0; c < kTilesKeys; c += 4) {
                            const float4 kc = *reinterpret_cast<const float4*>(meta.kc + c);
                            const float4 lv = *reinterpret_cast<const float4*>(meta.lv + c);
                            float2 k0 = make_float2(kc.x, kc.y), k1 = make_float2(kc.z, kc.w);
                            if constexpr (!std::is_same_v<T, __half>) {
                                k0 = mul2(k0, make_float2(my_factor, my_factor));
                                k1 = mul2(k1, make_float2(my_factor, my_factor));
                            }
                            const float2 x0 = fma2(make_float2(x[c], x[c + 1]), k0, make_float2(lv.x, lv.y));
                            const float2 x1 = fma2(make_float2(x[c + 2], x[c + 3]), k1, make_float2(lv.z, lv.w));
                            x[c] = x0.x;
                            x[c + 1] = x0.y;
                            x[c + 2] = x1.x;
                            x[c + 3] = x1.y;
                        }
                    }
                    if (!whole) {
                        const uint32_t seen[4] = {there.x, there.y, there.z, there.w};
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            uint32_t bits = first_bits(my_pos - key0 + 1, w);
                            if (a.window > 0)
                                bits &= ~first_bits(my_pos - a.window - key0 + 1, w) | first_bits(a.sinks - key0, w);
                            bits &= seen[w];
                            if (__all_sync(0xffffffffu, bits == 0xffffffffu)) continue;
#pragma unroll
                            for (int c = 0; c < 32; ++c)
                                x[w * 32 + c] = (bits & (1u << c)) != 0 ? x[w * 32 + c] : -INFINITY;
                        }
                    }
                    auto largest = [&] {
                        float tops[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                        for (int c = 4; c < kTilesKeys - 4; c += 8) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) tops[i] = max3(tops[i], x[c + i], x[c + 4 + i]);
                        }
                        return max3(max3(tops[0], x[124], x[125]), max3(tops[1], x[126], x[127]), fmaxf(tops[2], tops[3]));
                    };
                    float top = largest() * scale;
                    auto grows = [&] { return top > ref + (ref == -INFINITY ? 0.0f : kGrowth); };
                    bool grew = grows();
                    // Weights of keys whose values are all zero, relative to the largest of them: as in the
                    // kernel for few rows.
                    float empty_top = -INFINITY, empty_sum = 0.0f;
                    if (__any_sync(0xffffffffu, grew)) {
                        if constexpr (QUANT) {
                            ok = tile_wait(sm, &sm.v_full[n % STAGES], n / STAGES & 1, polls);
                            ok = __all_sync(0xffffffffu, ok);
                            const uint4 e4 = *reinterpret_cast<const uint4*>(meta.empty);
                            if ((e4.x | e4.y | e4.z | e4.w) != 0) {
                                // Few keys: read again from tensor memory one by one. Code for any of the 128
                                // registers would take more of them from every tile (fp16 queries, 2048 tokens on
                                // 16384: 805 us, and 788 so).
#pragma unroll 1
                                for (int w = 0; w < 4; ++w) {
#pragma unroll 1
                                    for (uint32_t bits = meta.empty[w] & meta.there[w]; bits != 0; bits &= bits - 1) {
                                        const int c = w * 32 + __ffs(bits) - 1;
                                        __syncwarp();
                                        const float s = __uint_as_float(tmem_load1(s_at + c)) * (my_factor * meta.kc[c]);
                                        if (sees_key(a, my_pos, key0 + c) && s != -INFINITY) {
                                            const float most = fmaxf(empty_top, s);
                                            empty_sum = empty_sum * ex2(empty_top - most) + ex2(s - most);
                                            empty_top = most;
                                        }
                                    }
                                }
                                const uint32_t empty[4] = {e4.x, e4.y, e4.z, e4.w};
#pragma unroll
                                for (int c = 0; c < kTilesKeys; ++c)
                                    if (empty[c / 32] >> (c % 32) & 1) x[c] = -INFINITY;
                                top = fmaxf(largest(), empty_top + kEmptyLog);
                                grew = grows();
                            }
                        }
                        const float to = grew ? top : ref;
                        const float alpha = grew ? ex2(ref - to) : 1.0f;
                        ref = to;
                        sum *= alpha;
                        if (t > t0) {  // the products of the tile before are done: this tile's scores came after them
#pragma unroll 1
                            for (int c = 0; c < DPAD; c += 16) {
                                uint32_t o[16];
                                tmem_load16(o_at + c, o);
                                tmem_wait_load();
#pragma unroll
                                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                                tmem_store16(o_at + c, o);
                            }
                        }
                    }
                    const float base = ref == -INFINITY ? 0.0f : ref - kLift<M>;
                    if (QUANT && empty_sum != 0.0f) sum += empty_sum * ex2(empty_top - base);
                    const float2 scale2 = make_float2(scale, scale), base2 = make_float2(-base, -base);
                    float2 part[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                    for (int c = 0; c < kTilesKeys; c += 32) {
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            float2 p = fma2(make_float2(x[c + i], x[c + i + 1]), scale2, base2);
                            p = make_float2(ex2(p.x), ex2(p.y));
                            if constexpr (QUANT)
                                part[i / 2 & 1] = fma2(p, *reinterpret_cast<const float2*>(meta.unscale + c + i), part[i / 2 & 1]);
                            else
                                part[i / 2 & 1] = add2(part[i / 2 & 1], p);
                            // the weights in the values' 16 bits; their sum above in fp32
                            w[i / 2] = pack2<M>(p.x, p.y);
                        }
                        tmem_store16(s_at + c / 2, w);
                        if (c + 32 == kEarly) {
                            tmem_wait_store();
                            tmem_fence_before();
                            mbar_arrive(&sm.p_full[h][0]);
                        }
                    }
                    part[0] = add2(part[0], part[1]);
                    sum += part[0].x + part[0].y;
                    tmem_wait_store();
                } else {
                    mbar_arrive(&sm.p_full[h][0]);
                }
                tmem_fence_before();
                mbar_arrive(&sm.p_full[h][1]);
                if (t == t_end - 1) prepare_next();  // while the last products run
            }
            if (!ok) {
                following = share;
                more = next_item<kTilesRows, kTilesKeys>(a, following);
                loaded = false;
            }
            const int r = row0 + lane;
            const bool real = r < it.rows, begins = t0 == 0, ends = t_end == it.tiles;
            const int64_t mine = real ? row_offset(a, it, it.row0 + r, a.ob, a.os, a.oh) : -1;
            int64_t to[4];  // rows that the lane writes eight columns of
#pragma unroll
            for (int k = 0; k < 4; ++k) to[k] = __shfl_sync(0xffffffffu, mine, k * 8 + lane / 4);
            ok = ok && tile_wait(sm, &sm.o_full[h], no++ & 1, polls);
            ok = __all_sync(0xffffffffu, ok);
            tmem_fence_after();
            if (rows) {
                // 64 bytes of a row at a time go through shared memory, so that four lanes write them.
                Block* const block = reinterpret_cast<Block*>(a.partial) + 2 * blockIdx.x + (begins ? 1 : 0);
                const float nan = __int_as_float(0x7fffffff);
                const float inv = !ok ? nan : sum == 0.0f ? 0.0f : __fdividef(1.0f, sum);
                auto put = [&](int i, const uint4& v) { staging[lane * 4 + (i ^ (lane >> 1 & 3))] = v; };
                auto get = [&](int k) {
                    const int to = k * 8 + lane / 4;
                    return staging[to * 4 + (lane % 4 ^ (to >> 1 & 3))];
                };
#pragma unroll 1
                for (int c0 = 0; c0 < DPAD; c0 += 32) {
                    uint32_t o[32];
                    tmem_load32(o_at + c0, o);
                    tmem_wait_load();
                    if (begins && ends) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            Packed<T, 8> y;
#pragma unroll
                            for (int e = 0; e < 8; e += 2)
                                put2(y, e, __uint_as_float(o[i * 8 + e]) * inv, __uint_as_float(o[i * 8 + e + 1]) * inv);
                            put(i, *reinterpret_cast<uint4*>(&y));
                        }
                        __syncwarp();
                        const int col = c0 + lane % 4 * 8;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (to[k] >= 0 && col < a.cache.head_dim)
                                *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + to[k] + col) = get(k);
                        __syncwarp();
                    } else {
#pragma unroll
                        for (int c = 0; c < 32; c += 16) {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                put(i, make_uint4(o[c + i * 4], o[c + i * 4 + 1], o[c + i * 4 + 2], o[c + i * 4 + 3]));
                            __syncwarp();
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const int r2 = row0 + k * 8 + lane / 4;
                                if (r2 < it.rows) *reinterpret_cast<uint4*>(&block->o[r2][c0 + c + lane % 4 * 4]) = get(k);
                            }
                            __syncwarp();
                        }
                    }
                }
                if (real && !(begins && ends)) {
                    block->m[r] = ref;
                    block->l[r] = ok ? sum : nan;
                }
                if (sm.odd) {
                    __syncwarp();  // orders the row's stores by other lanes before this one's
                    if (real && begins && ends) add_odd_values<T, QUANT, T>(a, it, t0, t_end, r, static_cast<T*>(a.out) + mine);
                    else if (real) add_odd_values<T, QUANT, float>(a, it, t0, t_end, r, block->o[r]);
                }
            }
            tmem_fence_before();
            if (begins && !ends && row == 0 && h == 0)
                a.joins[blockIdx.x] = make_int4(it.b, it.rt, it.h, share.last_cta());
            if (!more) break;
            share = following;
        }
        cp_async_wait_everything();  // rows of q that no product waited for
        asm volatile("bar.arrive 2, 416;" ::: "memory");
    }
}

}  // namespace ako_b200
