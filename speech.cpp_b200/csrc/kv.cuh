// kv.cuh — the paged key/value cache as the kernels see it (b200_kv_cache, include/b200.h).
#pragma once

#include "internal.h"

namespace b200 {

// Row (page, head, slot) of an array lies at ((page * n_kv_head + head) * page_size + slot) * row elements.
struct KvView {
    const uint8_t * k;   // F16 or int8 [n_pages][n_kv_head][page_size][head_dim]
    const uint8_t * v;
    const __half * kd;   // Q8_0 scales [n_pages][n_kv_head][page_size][head_dim / 32]
    const __half * vd;
    int n_kv_head, head_dim, page_size, n_pages;
    const int32_t * table;  // [n_seq][max_pages]
    const int32_t * lens;   // [n_seq]
    int64_t max_pages;
    unsigned * err;
};

// The length of sequence s; one outside [0, max_pages * page_size] counts as 0 (and is reported by the thread whose `tell`
// is set).
__device__ __forceinline__ int64_t kv_len(const KvView & c, int64_t s, bool tell) {
    const int64_t len = c.lens[s];
    if (len >= 0 && len <= c.max_pages * c.page_size) return len;
    if (tell) atomicOr(c.err, B200_DEVERR_PAGE);
    return 0;
}

// Page number i of sequence s, or -1 (reported) when the table holds one outside the cache.
__device__ __forceinline__ int kv_page(const KvView & c, int64_t s, int64_t i, bool tell) {
    const int p = c.table[s * c.max_pages + i];
    if ((unsigned) p < (unsigned) c.n_pages) return p;
    if (tell) atomicOr(c.err, B200_DEVERR_PAGE);
    return -1;
}

// Checks what the paged calls have in common; fills the view. what: the call's name for the error text.
b200_status kv_checked_view(b200_context * ctx, const char * what, const b200_kv_cache * cache, const int32_t * table, int64_t max_pages,
                            const int32_t * lens, int64_t n_seq, int64_t n_tok, KvView * out);
b200_status kv_fail(b200_context * ctx, b200_status s, const char * what, const char * why);
b200_status kv_cuda(b200_context * ctx, cudaError_t e, const char * what);

}  // namespace b200
