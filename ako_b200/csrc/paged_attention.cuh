// Attention over a paged cache: its arguments, the division of the work, and
// what its kernels share.
#pragma once

#include "paged.cuh"

namespace ako_b200 {

struct AttnArgs {
    const void* q;
    void* out;
    int64_t qb, qs, qh, ob, os, oh;
    PagedCache cache;
    PagedSeqs seqs;
    int group;       // q heads that share a kv head
    int window;      // 0: none
    int sinks;
    float scale;     // scale * log2(e)
    FastDiv by_group;
    float* partial;  // (2 * ctas) blocks of PartialBlock
    int4* joins;     // per CTA: the item that it begins and others end
};

// ------------------------------------------------------------------- work
// The rows that one kv head of one sequence answers are its new tokens times
// the q heads that share it, token by token: row r is token r / group, head
// r % group of the group. A tile of TILE rows against one kv head is an item;
// its keys come in tiles of BN. All items' key tiles, in the order (sequence,
// row tile, kv head, key tile), form one list, in which COST places that stand
// for what an item costs by itself precede its tiles. CTA c of N takes the
// part from c * total / N up to (c + 1) * total / N of it. So every CTA gets
// the same work whatever the sequences' lengths are, and a CTA shares at most
// two items with others, the one at its part's begin and the one at its end.
struct Item {
    int b, rt, h;           // sequence, row tile, kv head
    int first, n, kv;       // the sequence's first new token, new and cached tokens
    int row0, rows;         // rows of this item: row0 .. row0 + rows - 1
    int p_lo, p_hi;         // positions of its first and last row
    int win_lo;             // no row sees a key below it that is not a sink
    int sink_tiles, tile_lo, tiles;  // key tiles: [0, sink_tiles) and then from tile_lo on
};

template <int TILE, int BN>
__device__ __forceinline__ void item_geometry(const AttnArgs& a, Item& it) {
    it.row0 = it.rt * TILE;
    it.rows = min(TILE, it.n * a.group - it.row0);
    const int before = it.kv - it.n;
    it.p_lo = before + static_cast<int>(a.by_group.div(it.row0));
    it.p_hi = before + static_cast<int>(a.by_group.div(it.row0 + it.rows - 1));
    const int end = max(it.p_hi + 1, 0);
    it.win_lo = a.window > 0 ? max(max(it.p_lo, 0) - a.window + 1, 0) : 0;
    it.tile_lo = it.win_lo / BN;
    it.sink_tiles = min((min(a.sinks, end) + BN - 1) / BN, it.tile_lo);
    // an item without a key still has its rows to write: one tile, all masked
    it.tiles = max(it.sink_tiles + (end + BN - 1) / BN - it.tile_lo, 1);
}

__device__ __forceinline__ int key_tile(const Item& it, int t) {
    return t < it.sink_tiles ? t : it.tile_lo + (t - it.sink_tiles);
}

template <int TILE>
__device__ __forceinline__ int row_tiles(const AttnArgs& a, int n) { return (n * a.group + TILE - 1) / TILE; }

// Places of sequence `b` over its row tiles and heads. All lanes of a warp
// call it, with b = -1 for none: sequences with many row tiles are summed by
// the whole warp.
template <int TILE, int BN, int COST>
__device__ __forceinline__ int64_t sequence_tiles(const AttnArgs& a, int b) {
    Item it;
    it.n = 0;
    it.kv = 0;
    if (b >= 0) {
        new_tokens(a.seqs, b, it.first, it.n);
        it.kv = cached_tokens(a.seqs, b);
    }
    const int nrt = row_tiles<TILE>(a, it.n);
    int64_t sum = 0;
    if (nrt <= 4) {
        for (it.rt = 0; it.rt < nrt; ++it.rt) {
            item_geometry<TILE, BN>(a, it);
            sum += it.tiles + COST;
        }
    }
    const int lane = static_cast<int>(threadIdx.x & 31);
    for (unsigned many = __ballot_sync(0xffffffffu, nrt > 4); many != 0; many &= many - 1) {
        const int src = __ffs(many) - 1;
        Item o;
        o.n = __shfl_sync(0xffffffffu, it.n, src);
        o.kv = __shfl_sync(0xffffffffu, it.kv, src);
        const int tiles = __shfl_sync(0xffffffffu, nrt, src);
        int64_t s = 0;
        for (o.rt = lane; o.rt < tiles; o.rt += 32) {
            item_geometry<TILE, BN>(a, o);
            s += o.tiles + COST;
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        if (lane == src) sum = s;
    }
    return sum * a.cache.kv_heads;
}

// This CTA's part of the list, and the item that it is at.
template <int COST>
struct Share {
    int64_t begin, end, total;
    int ctas;  // CTAs that take part
    Item it;
    int64_t item_at;  // where the item begins in the list

    // The part's tiles of the item: first() .. last() - 1.
    __device__ __forceinline__ int first() const {
        const int64_t t = begin - item_at - COST;
        return t > 0 ? static_cast<int>(t) : 0;
    }
    __device__ __forceinline__ int last() const {
        const int64_t t = end - item_at - COST;
        return t < it.tiles ? static_cast<int>(t) : it.tiles;
    }
    // The last CTA that has a tile of the item.
    __device__ __forceinline__ int last_cta() const {
        return static_cast<int>(((item_at + COST + it.tiles) * ctas - 1) / total);
    }
};

struct ShareScratch {
    int64_t warp_sum[32];
    int64_t at;  // begin, counted from the sequence's first tile
    int b;
};

// All threads of the CTA call it (THREADS a multiple of 32). False when this
// CTA has nothing to do. No CTA takes less than `per_cta` places if it can help it.
template <int TILE, int BN, int COST, int THREADS>
__device__ bool find_share(const AttnArgs& a, int per_cta, ShareScratch& sm, Share<COST>& out) {
    constexpr int WARPS = THREADS / 32;
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
    const int chunks = (a.seqs.batch + THREADS - 1) / THREADS;
    int64_t mine = 0, total = 0;
    for (int i = 0; i < chunks; ++i) {
        const int b = i * THREADS + tid;
        mine = sequence_tiles<TILE, BN, COST>(a, b < a.seqs.batch ? b : -1);
        total += mine;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
    if (lane == 0) sm.warp_sum[warp] = total;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) total += sm.warp_sum[i];
    __syncthreads();
    const int64_t most = (total + per_cta - 1) / per_cta;
    out.ctas = static_cast<int>(most < gridDim.x ? most : gridDim.x);
    if (static_cast<int>(blockIdx.x) >= out.ctas) return false;
    out.total = total;
    out.begin = blockIdx.x * total / out.ctas;
    out.end = (blockIdx.x + 1) * total / out.ctas;
    int64_t before = 0;
    for (int i = 0; i < chunks; ++i) {
        const int b = i * THREADS + tid;
        if (chunks > 1) mine = sequence_tiles<TILE, BN, COST>(a, b < a.seqs.batch ? b : -1);
        int64_t incl = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int64_t o = __shfl_up_sync(0xffffffffu, incl, off);
            if (lane >= off) incl += o;
        }
        if (lane == 31) sm.warp_sum[warp] = incl;
        __syncthreads();
        int64_t base = before;
        for (int w = 0; w < WARPS; ++w) {
            if (w == warp) incl += base;
            base += sm.warp_sum[w];
        }
        before = base;
        if (out.begin >= incl - mine && out.begin < incl) {
            sm.b = b;
            sm.at = out.begin - (incl - mine);
        }
        __syncthreads();
        if (before > out.begin) break;
    }
    Item& it = out.it;
    it.b = sm.b;
    int64_t at = sm.at;
    new_tokens(a.seqs, it.b, it.first, it.n);
    it.kv = cached_tokens(a.seqs, it.b);
    const int last = row_tiles<TILE>(a, it.n) - 1;
    for (it.rt = 0;; ++it.rt) {
        item_geometry<TILE, BN>(a, it);
        const int64_t all = static_cast<int64_t>(it.tiles + COST) * a.cache.kv_heads;
        if (at < all || it.rt >= last) break;
        at -= all;
    }
    it.h = static_cast<int>(at / (it.tiles + COST));
    out.item_at = out.begin - (at - static_cast<int64_t>(it.h) * (it.tiles + COST));
    return out.last() > out.first();
}

// Moves on to the next item; false when the part has none of its tiles.
template <int TILE, int BN, int COST>
__device__ __forceinline__ bool next_item(const AttnArgs& a, Share<COST>& s) {
    Item& it = s.it;
    s.item_at += it.tiles + COST;
    if (s.item_at + COST >= s.end) return false;
    if (++it.h < a.cache.kv_heads) return true;
    it.h = 0;
    if (++it.rt < row_tiles<TILE>(a, it.n)) {
        item_geometry<TILE, BN>(a, it);
        return true;
    }
    it.rt = 0;
    while (++it.b < a.seqs.batch) {
        new_tokens(a.seqs, it.b, it.first, it.n);
        if (it.n > 0) {
            it.kv = cached_tokens(a.seqs, it.b);
            item_geometry<TILE, BN>(a, it);
            return true;
        }
    }
    return false;
}

// ---------------------------------------------------------------- partials
// A CTA writes at most two partial results: block 2c, of an item that an
// earlier CTA begins, and block 2c + 1, of an item that it begins and a later
// one ends. Each holds the rows' maxima (log2 domain), sums, and sums of
// weighted values. CTA c's entry of `joins` says who else has parts of the
// second: {b, rt, h, last CTA}, or {-1, ...}.
template <int ROWS, int DPAD>
struct PartialBlock {
    float m[ROWS], l[ROWS];
    float o[ROWS][DPAD];
};

// How far (as a power of two) a row's weights may exceed those that they are
// relative to before that is moved: 16-bit weights keep their precision, and
// sums are rescaled rarely.
constexpr float kGrowth = 8.0f;

// Where the weights' 16-bit type is fp16, which has few exponents, they are taken 2^7 higher: up to
// 2^15 with kGrowth, of the type's 2^16, so that a weight keeps all its bits down to 2^-21 of the
// largest, and some down to 2^-31. The sums take the factor along, and their quotient drops it.
template <typename M>
constexpr float kLift = std::is_same_v<M, __half> ? 7.0f : 0.0f;

// What a key of an e4m3 cache whose values are all zero counts with, at most, as the logarithm of its scale, which
// may be any number (kv_cache_write's is 1). Maxima are those of score + log2(scale), and weights relative to them,
// so a large scale would take bits from the weights of the keys that do have values. The key's own weight counts in
// the sum alone: relative to a maximum that follows it 2^64 below, it stays finite there, and is not lost unless it
// is 2^62 times smaller than that of a key whose scale is 1.
constexpr float kEmptyLog = -64.0f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Element offset of row r of an item in q (or out) with strides b, s, h.
__device__ __forceinline__ int64_t row_offset(const AttnArgs& a, const Item& it, int r, int64_t sb, int64_t ss,
                                              int64_t sh) {
    const int i = static_cast<int>(a.by_group.div(r));
    const int64_t head = static_cast<int64_t>(it.h) * a.group + (r - i * a.group);
    if (a.seqs.cu == nullptr) return it.b * sb + i * ss + head * sh;
    return static_cast<int64_t>(it.first + i) * ss + head * sh;
}

// Four columns of an item's row: weighted sum over sum of weights, rounded
// once; zero where no key was seen.
template <typename T>
__device__ __forceinline__ void write_row(const AttnArgs& a, const Item& it, int r, int c, const float4& acc, float sum) {
    if (c >= a.cache.head_dim) return;
    const float inv = sum == 0.0f ? 0.0f : __fdividef(1.0f, sum);
    Packed<T, 4> y;
    put2(y, 0, acc.x * inv, acc.y * inv);
    put2(y, 2, acc.z * inv, acc.w * inv);
    *reinterpret_cast<Packed<T, 4>*>(static_cast<T*>(a.out) + row_offset(a, it, it.row0 + r, a.ob, a.os, a.oh) + c) = y;
}

// Joins the parts of the items that several CTAs took: CTA (c, y) the rows
// [y * EACH, (y + 1) * EACH) of the item that CTA c of the grid before it began.
// Bound by the parts' bytes, so a thread asks for its rows of a part at once.
template <typename T, int ROWS, int DPAD, int EACH>
__global__ void __launch_bounds__(128) attn_join_kernel(const AttnArgs a) {
    pdl_enter();
    const int4 j = a.joins[blockIdx.x];
    if (j.x < 0) return;
    using Block = PartialBlock<ROWS, DPAD>;
    constexpr int LANES = DPAD / 4, STEP = 128 / LANES, TIMES = EACH / STEP;
    Item it;
    it.b = j.x;
    it.rt = j.y;
    it.h = j.z;
    new_tokens(a.seqs, it.b, it.first, it.n);
    it.row0 = it.rt * ROWS;
    it.rows = min(ROWS, it.n * a.group - it.row0);
    const int r0 = static_cast<int>(blockIdx.y) * EACH + static_cast<int>(threadIdx.x) / LANES;
    const int c = static_cast<int>(threadIdx.x) % LANES * 4;
    if (r0 >= it.rows) return;
    // block 2c + 1 of the first CTA, blocks 2i of those behind it
    const Block* const own = reinterpret_cast<const Block*>(a.partial) + 2 * blockIdx.x + 1;
    const int n = j.w - static_cast<int>(blockIdx.x);
    float top[TIMES], sum[TIMES];
    float4 acc[TIMES];
#pragma unroll
    for (int i = 0; i < TIMES; ++i) {
        const int r = min(r0 + i * STEP, it.rows - 1);
        top[i] = own->m[r];
        sum[i] = own->l[r];
        acc[i] = *reinterpret_cast<const float4*>(&own->o[r][c]);
    }
    for (int k = 0; k < n; ++k) {
        const Block& b = own[2 * k + 1];
        float m[TIMES], l[TIMES];
        float4 v[TIMES];
#pragma unroll
        for (int i = 0; i < TIMES; ++i) {
            const int r = min(r0 + i * STEP, it.rows - 1);
            m[i] = b.m[r];
            l[i] = b.l[r];
            v[i] = *reinterpret_cast<const float4*>(&b.o[r][c]);
        }
#pragma unroll
        for (int i = 0; i < TIMES; ++i) {
            const float mn = fmaxf(top[i], m[i]), ref = mn == -INFINITY ? 0.0f : mn;
            const float f = ex2(top[i] - ref), g = ex2(m[i] - ref);
            top[i] = mn;
            sum[i] = fmaf(g, l[i], f * sum[i]);
            acc[i].x = fmaf(g, v[i].x, f * acc[i].x);
            acc[i].y = fmaf(g, v[i].y, f * acc[i].y);
            acc[i].z = fmaf(g, v[i].z, f * acc[i].z);
            acc[i].w = fmaf(g, v[i].w, f * acc[i].w);
        }
    }
#pragma unroll
    for (int i = 0; i < TIMES; ++i)
        if (r0 + i * STEP < it.rows) write_row<T>(a, it, r0 + i * STEP, c, acc[i], sum[i]);
}

}  // namespace ako_b200
