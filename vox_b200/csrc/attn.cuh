// Internal interface of the paged attention kernels: their arguments, the split of a call into jobs, and the launchers.
//
// One call is a list of jobs (rows x keys of one key/value head): the rows are query heads of tokens that share that head,
// the keys a range of one sequence's cache or of the shared prefix. A range that one block takes alone is normalised and
// stored at once; a range cut into splits leaves for each row and split the running maximum and sum of its softmax (f32)
// and the unnormalised output (f32) in the workspace, and attn_merge joins the splits of a row in ascending order:
//   M = max_s m_s,  out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s
// (all exponents base 2: the scores are scaled by scale * log2 e before the softmax).
#pragma once

#include <cuda.h>

#include "paged.cuh"

namespace voxcuda {

struct AttnArgs {
    PagedArgs p;
    const void *q;
    void *out;
    int64_t q_stride, out_stride;  // elements
    const int32_t *prefix_pages;
    int32_t prefix_len, window;    // window 0: none
    float scale_log2;              // scale * log2 e
    FastDiv gdiv;                  // division by p.group
    // the own keys of a sequence: split s takes keys [s * chunk, (s + 1) * chunk), chunk at least own_chunk
    int32_t own_splits, own_chunk, own_tiles;  // tiles: blocks over the rows of a sequence
    // the prefix: likewise, over the rows of all tokens
    int32_t pre_splits, pre_chunk, pre_tiles;
    FastDiv kvdiv, otdiv, osdiv, ptdiv, srdiv; // divisions by kv_heads, seqs * own_splits, own_splits, pre_tiles, stream_rows
    int32_t pre_blocks, splits;                // blocks of the prefix (they come first); slots of a row in the workspace
    int32_t partial;                           // results go to the workspace (a row's parts meet in a later launch)
    // the tensor-core kernel: rows a block; whether its blocks have one row tile, two of them an SM; whether the own keys
    // follow the prefix in one walk (then pre_splits is 0). own_tiles counts the row tiles of all sequences there.
    int32_t tc_rows, tc_half, concat;
    // there the scale is positive (row maxima are taken before it): a negative one flips q's signs, zero clears q
    float tc_scale;
    uint32_t q_and, q_xor;
    // few query rows (attn_rows.cuh): blocks a cluster and how many of them take the prefix; or log2 of the keys a tile of
    // the list, rows that the joining launch looks at, rows and number of the parts, and the parts themselves
    int32_t cluster, cluster_pre, stream_shift, stream_rows, stream_rb, stream_blocks;
    float *stream_o;
    float2 *stream_ml;
    CUtensorMap mk, mv;  // the cache's tensors, boxes of 16 rows of one page (attn_mma.cu)
    int2 *stream_desc;  // [seqs][kv_heads]: first and last block of a sequence's tiles
    float *part_o;                             // [tokens * heads][splits][hd]
    float2 *part_ml;                           // [tokens * heads][splits]: (maximum, sum)
};

// Which frame of attn_rows.cuh takes a part of a call.
enum RowsFrame { kFrameGrid = 0, kFrameCluster = 1, kFrameStream = 2 };

// A block's job (rows x keys).
struct AttnJob {
    int tok0, rows;        // first token; rows = tokens of the job * group
    int kvh;
    int split;             // slot of the partial results
    int base;              // causal: row of token i sees keys < base + i + 1 (own keys); prefix: every key
    bool causal;
    int k0, k1;            // keys of the split
    const int32_t *pages;  // page numbers of the keys
    int tile, tiles;       // row tiles: tile, tile + tiles, ...
};

__device__ __forceinline__ AttnJob attn_job(const AttnArgs &a, uint32_t blk) {
    AttnJob j;
    uint32_t x = blk;
    if (blk < uint32_t(a.pre_blocks)) {
        const uint32_t y = a.kvdiv.div(x);
        j.kvh = int(x - y * uint32_t(a.p.kv_heads));
        j.split = int(a.ptdiv.div(y));
        j.tile = int(y - uint32_t(j.split) * uint32_t(a.pre_tiles));
        j.tiles = a.pre_tiles;
        j.tok0 = 0, j.rows = a.p.tokens * a.p.group;
        j.base = 0, j.causal = false;
        j.pages = a.prefix_pages;
        j.k0 = min(j.split * a.pre_chunk, a.prefix_len);
        j.k1 = j.split + 1 == a.pre_splits ? a.prefix_len : min(j.k0 + a.pre_chunk, a.prefix_len);
        return j;
    }
    // row tiles in descending order over all sequences: the last rows, which see most keys, first
    x -= uint32_t(a.pre_blocks);
    const uint32_t y = a.kvdiv.div(x);
    j.kvh = int(x - y * uint32_t(a.p.kv_heads));
    const uint32_t t = a.otdiv.div(y), z = y - t * a.otdiv.d;
    j.tile = a.own_tiles - 1 - int(t);
    j.tiles = a.own_tiles;
    const uint32_t b = a.osdiv.div(z);
    const int s = int(z - b * uint32_t(a.own_splits));
    j.split = a.pre_splits + s;
    int n;
    seq_tokens(a.p, int(b), j.tok0, n);
    const int kv = seq_rows(a.p, int(b));
    j.rows = n * a.p.group;
    j.base = kv - n, j.causal = true;
    j.pages = a.p.table + int64_t(b) * a.p.table_stride;
    // a sequence longer than the host's bound gets longer splits, whole tiles of 128 keys
    const int chunk = max(a.own_chunk, ((kv + a.own_splits - 1) / a.own_splits + 127) & ~127);
    j.k0 = int(min(int64_t(s) * chunk, int64_t(kv)));
    j.k1 = int(min(int64_t(j.k0) + chunk, int64_t(kv)));
    return j;
}


// Few rows on a bf16 cache (attn_mma.cu): rows_blk 8, or 16 (bf16 activations); units: blocks, or clusters.
int attn_mma_launch(AttnArgs &a, int head_dim, int rows_blk, int dtype, int frame, int64_t units, cudaStream_t st, const char *name);
int attn_mma_resident(int head_dim, int rows_blk, int dtype);  // blocks of the stream frame on the device at once
// Many rows at f32 accuracy (attn_f32.cu): 64 rows a block, jobs of attn_job().
constexpr int kF32Rows = 64;
int attn_f32_launch(const AttnArgs &a, int head_dim, int dtype, int cache_dtype, int64_t blocks, cudaStream_t st, const char *name);
// Map of one of the cache's tensors: [pages][page rows][kv heads][hd], box 64 elements of one head x box_rows rows of one
// page, 128-byte swizzle (attn_tc.cu).
int attn_cache_map(const vox_cuda_kv_cache &c, const void *base, int box_rows, CUtensorMap &m, const char *name);
// Tiled tensor copy of such a map's box; x times the element size is a multiple of 128 bytes at every call site.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_addr(bar))
                 : "memory");
}
// Bounded wait of a converged warp, as mbar_wait_warp, in little code whose first 256 polls touch neither the timer nor
// memory: the waits of the attention kernels are short as a rule, and a poll that comes late delays all that follows it.
__device__ __forceinline__ bool wait_soon(uint64_t *bar, uint32_t parity) {
    uint64_t t0 = 0;
#pragma unroll 1
    for (uint32_t i = 1;; ++i) {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
        if ((i & 255u) == 0) {
            const uint64_t now = globaltimer_ns();
            if (t0 == 0) t0 = now;
            if (__any_sync(0xffffffffu, now - t0 > kWaitLimitNs)) break;
        }
    }
    if ((threadIdx.x & 31) == 0) atomicOr(&g_device_error, kDevErrTimeout);
    return false;
}
// The tensor-core path (attn_tc.cu).
int attn_tc_launch(const AttnArgs &a, const vox_cuda_kv_cache &c, int64_t blocks, cudaStream_t st, const char *name);

}  // namespace voxcuda
