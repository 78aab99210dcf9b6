// The frame around the kernels of few query rows (attn.cu on f32 caches, attn_mma.cu on bf16 caches): which rows and keys a
// block takes, and where its result goes. A core computes softmax statistics and unnormalised output of up to RB rows over
// a range of keys, one part a warp, into shared memory:
//   struct Core { static constexpr int HD, RB, kMinBlocks; using Q = ...;
//                 static void run(const AttnArgs &, const RowsJob &, float (*acc)[RB][HD], float2 (*ml)[RB]); };
// Three frames use it:
//   attn_grid_kernel     one block a job of attn_job() (many row tiles, or a prefix); splits meet in attn_merge_kernel.
//   attn_cluster_kernel  one cluster of blocks a sequence and key/value head: the blocks share its keys evenly and join
//                        their parts through distributed shared memory, so a small call is one launch without scratch.
//   attn_stream_kernel   every resident block takes an equal run of key tiles out of the list of all sequences' tiles
//                        (sequence, then key/value head, then tile), whatever their lengths: the lengths are on the device,
//                        so the host cannot balance them. A block that covers a sequence's keys whole stores its rows;
//                        the others leave at most two parts a block (the end of one sequence, the start of another), which
//                        attn_stream_merge_kernel joins in ascending order of keys.
#pragma once

#include "attn.cuh"
#include "sfu.cuh"

namespace voxcuda {

constexpr int kRowsThreads = 128;
constexpr int kRowsWarps = kRowsThreads / 32;

struct RowsJob {
    int tok0, rows, row0;  // tokens of the job start at tok0; the rows row0 .. row0 + RB - 1 of `rows`
    int kvh, base;         // causal: token i sees keys < base + i + 1
    bool causal;
    int k0, k1;            // keys (rows of the cache behind `pages`)
    const int32_t *pages;
};

__device__ __forceinline__ void store4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void store4(__nv_bfloat16 *p, float4 v) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}

// A running join of parts (reference m, sum l, unnormalised output o of four elements) in the order they are added.
struct Join {
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    __device__ __forceinline__ void add(float pm, float pl, float4 po) {
        if (pm == -INFINITY) {  // a part that saw no key; NaN statistics must not be lost
            l += pl;
            return;
        }
        const float mx = fmaxf(m, pm), wa = ex2_approx(m - mx), wb = ex2_approx(pm - mx);  // m = -inf: wa = 0
        m = mx;
        l = l * wa + pl * wb;
        o.x = o.x * wa + po.x * wb, o.y = o.y * wa + po.y * wb, o.z = o.z * wa + po.z * wb, o.w = o.w * wa + po.w * wb;
    }
    __device__ __forceinline__ float4 out() const {  // a row that sees no key gives zeros
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        return make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    }
};

// The warps' parts of row r, elements d .. d + 3, joined in warp order.
template <int RB, int HD>
__device__ __forceinline__ Join join_warps(const float (*acc)[RB][HD], const float2 (*ml)[RB], int r, int d) {
    Join t;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) t.add(ml[w][r].x, ml[w][r].y, *reinterpret_cast<const float4 *>(&acc[w][r][d]));
    return t;
}
// Token and query head of row r of a job.
__device__ __forceinline__ void row_of(const AttnArgs &a, int tok0, int kvh, int r, int &tok, int &h) {
    const int i = int(a.gdiv.div(uint32_t(r)));
    tok = tok0 + i;
    h = kvh * a.p.group + r - i * a.p.group;
}
// The parts that an earlier launch left for the row's shared prefix, joined in ascending order of keys.
template <int HD>
__device__ __forceinline__ void add_prefix(const AttnArgs &a, Join &t, int tok, int h, int d) {
    const int64_t slot = (int64_t(tok) * a.p.heads + h) * a.splits;
    for (int s = 0; s < a.pre_splits; s += 4) {  // four parts' loads in flight
        float2 ml[4];
        float4 o[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (s + u < a.pre_splits) {
                ml[u] = __ldcg(a.part_ml + slot + s + u);
                o[u] = __ldcg(reinterpret_cast<const float4 *>(a.part_o + (slot + s + u) * HD + d));
            }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (s + u < a.pre_splits) t.add(ml[u].x, ml[u].y, o[u]);
    }
}

// ------------------------------------------------------------------ one block a job

template <class Core>
__global__ void __launch_bounds__(kRowsThreads, Core::kMinBlocks) attn_grid_kernel(const AttnArgs a) {
    constexpr int HD = Core::HD, RB = Core::RB;
    __shared__ float s_acc[kRowsWarps][RB][HD];
    __shared__ float2 s_ml[kRowsWarps][RB];
    pdl_enter();
    const AttnJob j = attn_job(a, blockIdx.x);
    for (int row0 = j.tile * RB; row0 < j.rows; row0 += j.tiles * RB) {
        Core::run(a, RowsJob{j.tok0, j.rows, row0, j.kvh, j.base, j.causal, j.k0, j.k1, j.pages}, s_acc, s_ml);
        __syncthreads();
        for (int x = threadIdx.x; x < RB * (HD / 4); x += kRowsThreads) {
            const int r = x / (HD / 4), d = (x % (HD / 4)) * 4;
            if (row0 + r >= j.rows) break;
            const Join t = join_warps<RB, HD>(s_acc, s_ml, r, d);
            int tok, h;
            row_of(a, j.tok0, j.kvh, row0 + r, tok, h);
            if (a.splits == 1) {
                store4(static_cast<typename Core::Q *>(a.out) + int64_t(tok) * a.out_stride + int64_t(h) * HD + d, t.out());
            } else {
                const int64_t slot = (int64_t(tok) * a.p.heads + h) * a.splits + j.split;
                store4(a.part_o + slot * HD + d, t.o);
                if (d == 0) a.part_ml[slot] = make_float2(t.m, t.l);
            }
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ one cluster a sequence and key/value head

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, uint32_t rank) {  // the same shared address in block `rank`
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// Grid: clusters of a.cluster blocks; cluster c takes key/value head c % kv_heads of sequence c / kv_heads.
template <class Core>
__global__ void __launch_bounds__(kRowsThreads, Core::kMinBlocks) attn_cluster_kernel(const AttnArgs a) {
    constexpr int HD = Core::HD, RB = Core::RB;
    __shared__ float s_acc[kRowsWarps][RB][HD];
    __shared__ float2 s_ml[kRowsWarps][RB];
    pdl_enter();
    const uint32_t rank = cluster_rank(), c = blockIdx.x / uint32_t(a.cluster);
    const uint32_t b = a.kvdiv.div(c);
    const int kvh = int(c - b * uint32_t(a.p.kv_heads));
    int tok0, n;
    seq_tokens(a.p, int(b), tok0, n);
    const int kv = seq_rows(a.p, int(b)), rows = n * a.p.group;
    int lo = 0;
    if (a.window > 0) lo = max(kv - n + 1 - a.window, 0) & ~15;
    const int per = ((kv - lo + a.cluster - 1) / a.cluster + 15) & ~15;
    const int k0 = min(lo + int(rank) * per, kv), k1 = min(k0 + per, kv);
    const int32_t *pages = a.p.table + int64_t(b) * a.p.table_stride;
    for (int row0 = 0; row0 < rows; row0 += RB) {  // the same rows in every block of the cluster
        Core::run(a, RowsJob{tok0, rows, row0, kvh, kv - n, true, k0, k1, pages}, s_acc, s_ml);
        __syncthreads();
        Join mine[(RB * (HD / 4) + kRowsThreads - 1) / kRowsThreads];
#pragma unroll
        for (int y = 0; y < (RB * (HD / 4) + kRowsThreads - 1) / kRowsThreads; ++y) {
            const int x = threadIdx.x + y * kRowsThreads;
            if (x < RB * (HD / 4)) mine[y] = join_warps<RB, HD>(s_acc, s_ml, x / (HD / 4), (x % (HD / 4)) * 4);
        }
        __syncthreads();
#pragma unroll
        for (int y = 0; y < (RB * (HD / 4) + kRowsThreads - 1) / kRowsThreads; ++y) {
            const int x = threadIdx.x + y * kRowsThreads, r = x / (HD / 4), d = (x % (HD / 4)) * 4;
            if (x < RB * (HD / 4)) {
                store4(&s_acc[0][r][d], mine[y].o);
                if (d == 0) s_ml[0][r] = make_float2(mine[y].m, mine[y].l);
            }
        }
        cluster_sync();
        // block `rank` joins every cluster-th quad of the rows, blocks in ascending order of keys
        const int live = min(rows - row0, RB) * (HD / 4);
        for (int x = int(rank) * kRowsThreads + threadIdx.x; x < live; x += a.cluster * kRowsThreads) {
            const int r = x / (HD / 4), d = (x % (HD / 4)) * 4;
            Join t;
            int tok, h;
            row_of(a, tok0, kvh, row0 + r, tok, h);
            add_prefix<HD>(a, t, tok, h, d);
            const uint32_t pa = smem_addr(&s_acc[0][r][d]), pm = smem_addr(&s_ml[0][r]);
            for (int s = 0; s < a.cluster; ++s) {
                const float2 ml = ld_cluster2(cluster_addr(pm, uint32_t(s)));
                t.add(ml.x, ml.y, ld_cluster4(cluster_addr(pa, uint32_t(s))));
            }
            store4(static_cast<typename Core::Q *>(a.out) + int64_t(tok) * a.out_stride + int64_t(h) * HD + d, t.out());
        }
        cluster_sync();  // the others have read this block's part
    }
}

// ------------------------------------------------------------------ equal runs of all sequences' key tiles

// Key tiles of sequence b (for one key/value head) and its first key: none for a sequence without new tokens.
__device__ __forceinline__ int stream_tiles(const AttnArgs &a, int b, int &tok0, int &n, int &kv, int &lo) {
    seq_tokens(a.p, b, tok0, n);
    kv = seq_rows(a.p, b);
    lo = a.window > 0 ? max(kv - n + 1 - a.window, 0) & ~15 : 0;
    return n > 0 ? (kv - lo + a.stream_keys - 1) / a.stream_keys : 0;
}
// Block-wide: the number of all tiles of one key/value head, and the sequence whose tiles hold tile `at / kv_heads`-wise
// position `at` of the list (every sequence's tiles times kv_heads), with the list position of its first tile.
struct StreamAt {
    int64_t total;
    int seq;
    int64_t start;
};
__device__ __forceinline__ int64_t stream_total(const AttnArgs &a, int64_t (&part)[kRowsThreads], int64_t &before, int &b0, int &b1) {
    const int per = (a.p.seqs + kRowsThreads - 1) / kRowsThreads;
    b0 = min(int(threadIdx.x) * per, a.p.seqs), b1 = min(b0 + per, a.p.seqs);
    int64_t sum = 0;
    for (int b = b0; b < b1; ++b) {
        int t, n, kv, lo;
        sum += stream_tiles(a, b, t, n, kv, lo);
    }
    sum *= a.p.kv_heads;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) part[warp] = inc;
    __syncthreads();
    int64_t total = 0;
    before = inc - sum;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) {
        if (w < warp) before += part[w];
        total += part[w];
    }
    return total;
}

template <class Core>
__global__ void __launch_bounds__(kRowsThreads, Core::kMinBlocks) attn_stream_kernel(const AttnArgs a) {
    constexpr int HD = Core::HD, RB = Core::RB;
    __shared__ float s_acc[kRowsWarps][RB][HD];
    __shared__ float2 s_ml[kRowsWarps][RB];
    __shared__ int64_t s_part[kRowsThreads], s_start;
    __shared__ int s_seq;
    pdl_enter();
    const int64_t c = blockIdx.x;
    int64_t u, u1, start;
    int b;
    {
        int64_t before;
        int b0, b1;
        const int64_t total = stream_total(a, s_part, before, b0, b1);
        const int64_t blocks = min(int64_t(gridDim.x), total);  // no block without a tile between two that share a sequence
        if (c >= blocks) return;
        u = total * c / blocks, u1 = total * (c + 1) / blocks;
        for (int x = b0; x < b1; ++x) {  // the thread whose sequences hold tile u
            int t, n, kv, lo;
            const int64_t w = int64_t(stream_tiles(a, x, t, n, kv, lo)) * a.p.kv_heads;
            if (u >= before && u < before + w) s_seq = x, s_start = before;
            before += w;
        }
        __syncthreads();
        b = s_seq, start = s_start;
    }
    int tok0, n, kv, lo, extra = 0;
    int tiles = stream_tiles(a, b, tok0, n, kv, lo);
    while (u < u1) {
        while (u >= start + int64_t(tiles) * a.p.kv_heads) {
            start += int64_t(tiles) * a.p.kv_heads;
            tiles = stream_tiles(a, ++b, tok0, n, kv, lo);
        }
        const int kvh = int((u - start) / tiles);
        const int64_t s0 = start + int64_t(kvh) * tiles;  // the list positions of this sequence and head: s0 .. s0 + tiles
        const int64_t e = min(s0 + tiles, u1);
        const bool head = u == s0, whole = head && e == s0 + tiles;
        const int rows = n * a.p.group;
        // rows past RB (a sequence with more new tokens than the host's bound): the block of the first tile takes them over
        // all keys
        const int row0 = extra * RB;
        const int k0 = extra ? lo : min(lo + int(u - s0) * a.stream_keys, kv), k1 = extra ? kv : min(lo + int(e - s0) * a.stream_keys, kv);
        Core::run(a, RowsJob{tok0, rows, row0, kvh, kv - n, true, k0, k1, a.p.table + int64_t(b) * a.p.table_stride}, s_acc, s_ml);
        __syncthreads();
        for (int x = threadIdx.x; x < RB * (HD / 4); x += kRowsThreads) {
            const int r = x / (HD / 4), d = (x % (HD / 4)) * 4;
            if (row0 + r >= rows) break;
            Join t = join_warps<RB, HD>(s_acc, s_ml, r, d);
            int tok, h;
            row_of(a, tok0, kvh, row0 + r, tok, h);
            if (whole || extra) {
                if (a.pre_splits > 0) {
                    Join p;
                    add_prefix<HD>(a, p, tok, h, d);
                    p.add(t.m, t.l, t.o);
                    t = p;
                }
                store4(static_cast<typename Core::Q *>(a.out) + int64_t(tok) * a.out_stride + int64_t(h) * HD + d, t.out());
            } else {
                const int64_t slot = (2 * c + (head ? 1 : 0)) * RB + r;
                store4(a.stream_o + slot * HD + d, t.o);
                if (d == 0) a.stream_ml[slot] = make_float2(t.m, t.l);
            }
        }
        __syncthreads();
        if (head && (extra + 1) * RB < rows) {
            ++extra;
        } else {
            extra = 0;
            u = e;
        }
    }
}

// One block a sequence and query-head row: joins the parts of the blocks that share its keys; rows that one block took
// whole are stored already. Grid: (rows of a sequence up to RB) * kv_heads * seqs.
template <typename QT, int HD>
__global__ void __launch_bounds__(kRowsThreads) attn_stream_merge_kernel(const AttnArgs a) {
    __shared__ int64_t s_part[kRowsThreads], s_total, s_before;
    __shared__ float s_o[kRowsWarps][HD];
    __shared__ float2 s_ml[kRowsWarps];
    pdl_enter();
    const int r = int(blockIdx.x % uint32_t(a.stream_rows));
    const uint32_t y = blockIdx.x / uint32_t(a.stream_rows), b = a.kvdiv.div(y);
    const int kvh = int(y - b * uint32_t(a.p.kv_heads));
    {
        int64_t before;
        int b0, b1;
        const int64_t total = stream_total(a, s_part, before, b0, b1);
        for (int x = b0; x < b1; ++x) {
            int t, n, kv, lo;
            const int64_t w = int64_t(stream_tiles(a, x, t, n, kv, lo)) * a.p.kv_heads;
            if (x == int(b)) s_before = before, s_total = total;
            before += w;
        }
        __syncthreads();
    }
    int tok0, n, kv, lo;
    const int tiles = stream_tiles(a, int(b), tok0, n, kv, lo);
    const int rows = n * a.p.group;
    if (r >= rows) return;
    const int64_t total = s_total, blocks = min(int64_t(a.stream_blocks), total);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int tok, h;
    int64_t c0 = 0, c1 = -1;
    if (tiles > 0) {
        // block of tile u: the c with total c / blocks <= u < total (c + 1) / blocks (rounded down)
        const int64_t s0 = s_before + int64_t(kvh) * tiles, s1 = s0 + tiles - 1;
        auto block_of = [&](int64_t u) { return ((u + 1) * blocks - 1) / total; };
        c0 = block_of(s0), c1 = block_of(s1);
        if (c0 == c1) return;  // stored by its block
    } else {
        for (int rr = r + a.stream_rows; rr < rows; rr += a.stream_rows) {  // rows past the bound of a sequence without keys
            row_of(a, tok0, kvh, rr, tok, h);
            for (int d = threadIdx.x * 4; d < HD; d += kRowsThreads * 4) {
                Join t;
                add_prefix<HD>(a, t, tok, h, d);
                store4(static_cast<QT *>(a.out) + int64_t(tok) * a.out_stride + int64_t(h) * HD + d, t.out());
            }
        }
    }
    // warp w joins a contiguous quarter of the parts, lane: elements E lane .. of the row
    constexpr int E = HD / 32;
    const int64_t cnt = c1 - c0 + 1, per = (cnt + kRowsWarps - 1) / kRowsWarps;
    float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    auto add = [&](float pm, float pl, const float *po) {
        if (pm == -INFINITY) {
            l += pl;
            return;
        }
        const float mx = fmaxf(m, pm), wa = ex2_approx(m - mx), wb = ex2_approx(pm - mx);
        m = mx;
        l = l * wa + pl * wb;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * wa + po[e] * wb;
    };
    for (int64_t c = c0 + warp * per; c < min(c0 + (warp + 1) * per, c1 + 1); ++c) {
        const int64_t slot = (2 * c + (c == c0 ? 1 : 0)) * a.stream_rb + r;
        const float2 ml = __ldcg(a.stream_ml + slot);
        float po[E];
#pragma unroll
        for (int e = 0; e < E; ++e) po[e] = __ldcg(a.stream_o + slot * HD + lane * E + e);
        add(ml.x, ml.y, po);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
    if (lane == 0) s_ml[warp] = make_float2(m, l);
    __syncthreads();
    row_of(a, tok0, kvh, r, tok, h);
    for (int d = threadIdx.x * 4; d < HD; d += kRowsThreads * 4) {
        Join t;
        add_prefix<HD>(a, t, tok, h, d);
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) t.add(s_ml[w].x, s_ml[w].y, *reinterpret_cast<const float4 *>(&s_o[w][d]));
        store4(static_cast<QT *>(a.out) + int64_t(tok) * a.out_stride + int64_t(h) * HD + d, t.out());
    }
}

// ------------------------------------------------------------------ launches

// Launches the frame that the shape asks for (attn.cu): blocks of the grid or stream kernel, or clusters.
template <class Core>
int launch_rows(AttnArgs &a, int frame, int64_t units, cudaStream_t st, const char *name) {
    if (frame == kFrameCluster) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(unsigned(units * a.cluster));
        cfg.blockDim = kRowsThreads;
        cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = unsigned(a.cluster), attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = pdl_enabled() ? 2 : 1;
        cudaLaunchKernelEx(&cfg, attn_cluster_kernel<Core>, a);
    } else if (frame == kFrameStream) {
        launch_k(attn_stream_kernel<Core>, dim3(unsigned(units)), kRowsThreads, 0, st, a);
        launch_k(attn_stream_merge_kernel<typename Core::Q, Core::HD>, dim3(unsigned(a.stream_rows * a.p.kv_heads * a.p.seqs)), kRowsThreads, 0, st,
                 a);
    } else {
        launch_k(attn_grid_kernel<Core>, dim3(unsigned(units)), kRowsThreads, 0, st, a);
    }
    return check_launch(name);
}

}  // namespace voxcuda
