// What the operators on a paged key/value cache share: the checked description of a cache and a ragged batch as the
// kernels take it, and the device helpers that find a token's sequence and a row's page. Lengths, offsets and page
// numbers live on the device (a replayed graph sees new ones), so the kernels check them: a value that is out of range is
// replaced before it forms an address, and recorded in the device error flag.
#pragma once

#include "tma.cuh"

namespace voxcuda {

constexpr unsigned int kDevErrRange = VOX_CUDA_DEVERR_RANGE;

struct PagedArgs {
    void *k, *v;
    const int32_t *table, *kv_len, *q_start;  // q_start NULL: q_per tokens a sequence
    int64_t table_stride;
    int64_t page_stride, row_stride, head_stride;  // elements
    int32_t page_shift, page_mask, pages;
    int32_t seqs, cap;                             // cap: rows that a sequence's table can hold
    int32_t tokens, q_per;
    int32_t heads, kv_heads, group;                // group: query heads a key/value head
    FastDiv qdiv;                                  // division by q_per
};

// Fills the shared part of the arguments after checking them. VOX_CUDA_OK or an error status.
int paged_args(const vox_cuda_kv_cache *c, const vox_cuda_kv_batch *b, int64_t heads, const char *name, PagedArgs &a);

__device__ __forceinline__ void range_error() { atomicOr(&g_device_error, kDevErrRange); }

// First token and number of new tokens of sequence b, held inside [0, tokens].
__device__ __forceinline__ void seq_tokens(const PagedArgs &a, int b, int &t0, int &n) {
    if (a.q_start == nullptr) {
        t0 = b * a.q_per;
        n = a.q_per;
        return;
    }
    const int s0 = __ldg(a.q_start + b), s1 = __ldg(a.q_start + b + 1);
    t0 = min(max(s0, 0), a.tokens);
    n = min(max(s1, t0), a.tokens) - t0;
    if (t0 != s0 || t0 + n != s1) range_error();
}
// Rows of sequence b in the cache, held inside what its page table can name.
__device__ __forceinline__ int seq_rows(const PagedArgs &a, int b) {
    const int n = __ldg(a.kv_len + b);
    const int m = min(max(n, 0), a.cap);
    if (m != n) range_error();
    return m;
}
// A page number taken from a table, held inside the cache.
__device__ __forceinline__ int page_checked(const PagedArgs &a, int p) {
    if (uint32_t(p) < uint32_t(a.pages)) return p;
    range_error();
    return 0;
}

}  // namespace voxcuda
