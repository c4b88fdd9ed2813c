// Paged key/value caches: the views that the kernels take, position and page
// arithmetic, and the division of attention work over a grid.
//
// A cache is (num_pages, kv_heads, page_size, head_dim) with free strides for
// the first three axes. Position p of sequence b lies in page
// table[b, p / page_size], at offset p % page_size. The lengths, offsets and
// page numbers are device data that the host has not seen, so every kernel
// clamps the lengths to the table's extent and the tokens given, and treats a
// page number outside the cache as a page that is not there.
#pragma once

#include "common.cuh"
#include "host.hpp"
#include "lengths.hpp"

namespace ako_b200 {

// One of a cache's tensors, with strides over pages, heads and slots in units
// of 16 bytes (keys and values) or of a float (scales). 32-bit strides make an
// offset three multiply-adds; they reach 64 GB.
struct PagedTensor {
    void* p;
    uint32_t page, head, slot;

    __device__ __forceinline__ uint64_t offset(int pg, int h, int s) const {
        return static_cast<uint64_t>(page) * static_cast<uint32_t>(pg) +
               static_cast<uint64_t>(head) * static_cast<uint32_t>(h) +
               static_cast<uint64_t>(slot) * static_cast<uint32_t>(s);
    }
    // Of a row of keys or values.
    __device__ __forceinline__ uint8_t* row(int pg, int h, int s) const {
        return static_cast<uint8_t*>(p) + offset(pg, h, s) * 16;
    }
    __device__ __forceinline__ float* scale(int pg, int h, int s) const { return static_cast<float*>(p) + offset(pg, h, s); }
};

struct PagedCache {
    PagedTensor k, v, ks, vs;  // ks, vs: fp32 scales, null unless the cache is quantised
    int num_pages, kv_heads, head_dim, page_size;
    FastDiv by_page;
};

struct PagedSeqs {
    const int* table;
    int64_t table_stride;
    const int* kv_lens;
    const int* cu;  // null: every sequence has q_len new tokens
    int batch, q_len, tokens, max_kv;
};

// New tokens of sequence `b`: the first one's index among the call's tokens,
// and how many.
__device__ __forceinline__ void new_tokens(const PagedSeqs& s, int b, int& first, int& n) {
    if (s.cu == nullptr) {
        first = b * s.q_len;
        n = s.q_len;
    } else {
        const RowRange r = row_range(s.cu[b], s.cu[b + 1], s.tokens);
        first = r.first;
        n = r.n;
    }
}

__device__ __forceinline__ int cached_tokens(const PagedSeqs& s, int b) { return clamp_to(s.kv_lens[b], s.max_kv); }

// Page number of position p (0 <= p < max_kv) of sequence b, or -1 if the
// table's entry lies outside the cache.
__device__ __forceinline__ int page_of(const PagedSeqs& s, const PagedCache& c, int b, int p, int& slot) {
    const int i = static_cast<int>(c.by_page.div(static_cast<uint32_t>(p)));
    slot = p - i * c.page_size;
    const int page = s.table[b * s.table_stride + i];
    return page >= 0 && page < c.num_pages ? page : -1;
}

// Fill the kernels' views from the C structs, checking them; `cache_es` is
// set to the bytes of a cached element. Status as in ako_b200_status.
int make_cache(const char* op, const ako_b200_paged_kv* c, int dtype, PagedCache& out, int& cache_es);
int make_seqs(const char* op, const ako_b200_paged_batch* b, const PagedCache& c, int64_t tokens, int64_t q_len,
              PagedSeqs& out);

}  // namespace ako_b200
