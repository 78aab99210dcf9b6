// The frame around the kernels of few query rows (attn.cu on f32 caches, attn_mma.cu on bf16 caches): which rows and keys a
// block takes, and where its result goes. A core computes softmax statistics and unnormalised output of up to RB rows over
// a range of keys, one part a warp, into shared memory:
//   struct Core { static constexpr int HD, RB, kMinBlocks, kStreamBlocks (blocks an SM, of the stream frame); static constexpr size_t kSmem (dynamic shared memory); using Q = ...;
//                 struct State (of a thread, through all its jobs); static void init(State &); static (*acc(State &))[RB][HD];
//                 static void run(const AttnArgs &, const RowsJob &, float (*acc)[RB][HD], float2 (*ml)[RB], State &, F between); };
// (between() is called by every thread while the first copies of the job are on their way.)
// Three frames use it:
//   attn_grid_kernel     one block a job of attn_job() (many row tiles, or a prefix); splits meet in attn_merge_kernel.
//   attn_cluster_kernel  one cluster of blocks a sequence and key/value head: the blocks share its keys evenly and join
//                        their parts through distributed shared memory, so a small call is one launch without scratch.
//   attn_stream_kernel   every resident block takes an equal run of key tiles out of the list of all sequences' tiles
//                        (sequence, then key/value head, then tile), whatever their lengths: the lengths are on the device,
//                        so the host cannot balance them. A block that covers a sequence's keys whole stores its rows;
//                        the others leave at most two parts a block (the end of one sequence, the start of another), which
//                        attn_stream_merge_kernel joins in ascending order of keys. The joining launch costs
//                        some 5 us, most of it its start and the parts' way through L2; attn.cu has when it pays.
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
__global__ void __launch_bounds__(kRowsThreads, Core::kMinBlocks) attn_grid_kernel(const __grid_constant__ AttnArgs a) {
    constexpr int HD = Core::HD, RB = Core::RB;
    __shared__ float2 s_ml[kRowsWarps][RB];
    pdl_enter();
    typename Core::State core;
    Core::init(core);
    float(*s_acc)[RB][HD] = Core::acc(core);
    const AttnJob j = attn_job(a, blockIdx.x);
    for (int row0 = j.tile * RB; row0 < j.rows; row0 += j.tiles * RB) {
        Core::run(a, RowsJob{j.tok0, j.rows, row0, j.kvh, j.base, j.causal, j.k0, j.k1, j.pages}, s_acc, s_ml, core, [] {});
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

// Grid: clusters of a.cluster blocks; cluster c takes key/value head c % kv_heads of sequence c / kv_heads. The first
// a.cluster_pre blocks of each take the shared prefix, where a call is so small that its launches cost more than reading the
// prefix again for every sequence.
template <class Core>
__global__ void __launch_bounds__(kRowsThreads, Core::kMinBlocks) attn_cluster_kernel(const __grid_constant__ AttnArgs a) {
    constexpr int HD = Core::HD, RB = Core::RB;
    __shared__ float2 s_ml[kRowsWarps][RB];
    pdl_enter();
    typename Core::State core;
    Core::init(core);
    float(*s_acc)[RB][HD] = Core::acc(core);
    const uint32_t rank = cluster_rank(), c = blockIdx.x / uint32_t(a.cluster);
    const uint32_t b = a.kvdiv.div(c);
    const int kvh = int(c - b * uint32_t(a.p.kv_heads));
    int tok0, n;
    seq_tokens(a.p, int(b), tok0, n);
    const int kv = seq_rows(a.p, int(b)), rows = n * a.p.group;
    const bool pre = int(rank) < a.cluster_pre;
    const int keys = pre ? a.prefix_len : kv, blocks = pre ? a.cluster_pre : a.cluster - a.cluster_pre;
    int lo = 0;
    if (a.window > 0) lo = max(kv - n + 1 - a.window, 0) & ~15;  // there is no prefix then
    const int per = ((keys - lo + blocks - 1) / blocks + 15) & ~15;
    const int k0 = min(lo + (pre ? int(rank) : int(rank) - a.cluster_pre) * per, keys), k1 = min(k0 + per, keys);
    const int32_t *pages = pre ? a.prefix_pages : a.p.table + int64_t(b) * a.p.table_stride;
    for (int row0 = 0; row0 < rows; row0 += RB) {  // the same rows in every block of the cluster
        Core::run(a, RowsJob{tok0, rows, row0, kvh, kv - n, !pre, k0, k1, pages}, s_acc, s_ml, core, [] {});
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

// Key tiles of sequence b (for one key/value head) and its first key: none for a sequence without new tokens. The list's
// positions fit 31 bits (attn.cu).
__device__ __forceinline__ int stream_tiles(const AttnArgs &a, int b, int &tok0, int &n, int &kv, int &lo) {
    seq_tokens(a.p, b, tok0, n);
    kv = seq_rows(a.p, b);
    lo = a.window > 0 ? max(kv - n + 1 - a.window, 0) & ~15 : 0;
    return n > 0 ? (kv - lo + (1 << a.stream_shift) - 1) >> a.stream_shift : 0;
}
// The list cut into `blocks` runs of `per` tiles, the first `rem` of them one longer.
struct StreamCut {
    int blocks, per, rem;
    __device__ __forceinline__ StreamCut(int total, int grid) {
        blocks = max(min(total, grid), 1);  // no block without a tile between two that share a sequence
        per = total / blocks;
        rem = total - per * blocks;
    }
    __device__ __forceinline__ int start(int c) const { return c * per + min(c, rem); }
    __device__ __forceinline__ int block_of(int u) const {
        const int x = rem * (per + 1);
        return u < x ? u / (per + 1) : rem + (u - x) / per;
    }
};

// Where a block stands in the list, and its next job; in shared memory: the registers belong to the core.
struct StreamState {
    int u, u1, start;  // next tile, end of the block's run, first tile of sequence b
    int b, extra, tiles;
    int part[2];       // of the workspace; -1: the rows are stored
    RowsJob job[2];    // tok0 < 0: no more
};

// Writes the block's next job into slot `s` (one thread).
template <int RB>
__device__ __forceinline__ void stream_next(const AttnArgs &a, StreamState &st, const StreamCut &cut, int s) {
    const int u = st.u;
    if (u >= st.u1) {
        st.job[s].tok0 = -1;
        return;
    }
    int b = st.b, start = st.start, tok0, n, kv, lo;
    const int extra = st.extra;
    int tiles = stream_tiles(a, b, tok0, n, kv, lo);
    while (u >= start + tiles * a.p.kv_heads) {
        start += tiles * a.p.kv_heads;
        tiles = stream_tiles(a, ++b, tok0, n, kv, lo);
    }
    const int kvh = (u - start) / tiles;
    const int s0 = start + kvh * tiles;  // the list positions of this sequence and head: s0 .. s0 + tiles
    const int e = min(s0 + tiles, st.u1);
    const bool head = u == s0, whole = head && e == s0 + tiles;
    const int rows = n * a.p.group;
    // rows past RB (a sequence with more new tokens than the host's bound): the block of the first tile takes them over all
    // keys
    st.job[s] = RowsJob{tok0, rows, extra * RB, kvh, kv - n, true, extra ? lo : min(lo + ((u - s0) << a.stream_shift), kv),
                        extra ? kv : min(lo + ((e - s0) << a.stream_shift), kv), a.p.table + int64_t(b) * a.p.table_stride};
    st.part[s] = (whole && a.pre_splits == 0) || extra ? -1 : whole ? 2 * a.stream_blocks + b * a.p.kv_heads + kvh : 2 * int(blockIdx.x) + (head ? 1 : 0);
    if (head) a.stream_desc[int64_t(b) * a.p.kv_heads + kvh] = make_int2(int(blockIdx.x), whole ? int(blockIdx.x) : cut.block_of(s0 + tiles - 1));
    const bool more = head && (extra + 1) * RB < rows;
    st.extra = more ? extra + 1 : 0;
    st.u = more ? u : e;
    st.start = start, st.b = b;
}

template <class Core>
__global__ void __launch_bounds__(kRowsThreads, Core::kStreamBlocks) attn_stream_kernel(const __grid_constant__ AttnArgs a) {
    constexpr int HD = Core::HD, RB = Core::RB;
    __shared__ float2 s_ml[kRowsWarps][RB];
    __shared__ int s_part[kRowsWarps];
    __shared__ StreamState st;
    pdl_enter();
    typename Core::State core;
    Core::init(core);
    float(*s_acc)[RB][HD] = Core::acc(core);
    int total;
    {   // all tiles, and the sequence that holds the block's first: every thread sums a run of sequences, then a prefix sum
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const int per = (a.p.seqs + kRowsThreads - 1) / kRowsThreads;
        const int b0 = min(int(threadIdx.x) * per, a.p.seqs), b1 = min(b0 + per, a.p.seqs);
        int t, n, kv, lo, sum = 0;
        for (int x = b0; x < b1; ++x) sum += stream_tiles(a, x, t, n, kv, lo);
        sum *= a.p.kv_heads;
        int inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) s_part[warp] = inc;
        __syncthreads();
        int before = inc - sum;
        total = 0;
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) {
            if (w < warp) before += s_part[w];
            total += s_part[w];
        }
        const StreamCut cut(total, int(gridDim.x));
        if (total == 0 || int(blockIdx.x) >= cut.blocks) return;
        const int u = cut.start(int(blockIdx.x));
        if (u >= before && u < before + sum) {  // this thread's sequences hold it
            st.u = u, st.u1 = cut.start(int(blockIdx.x) + 1), st.extra = 0, st.b = b0, st.start = before;
            stream_next<RB>(a, st, cut, 0);
        }
    }
    for (int s = 0;; s ^= 1) {
        __syncthreads();
        if (st.job[s].tok0 < 0) return;
        Core::run(a, st.job[s], s_acc, s_ml, core, [&] {
            if (threadIdx.x == 0) stream_next<RB>(a, st, StreamCut(total, int(gridDim.x)), s ^ 1);
        });
        __syncthreads();
        const RowsJob j = st.job[s];
        const int64_t part = st.part[s];
        for (int x = threadIdx.x; x < RB * (HD / 4); x += kRowsThreads) {
            const int r = x / (HD / 4), d = (x % (HD / 4)) * 4;
            if (j.row0 + r >= j.rows) break;
            Join t = join_warps<RB, HD>(s_acc, s_ml, r, d);
            if (part >= 0) {
                store4(a.stream_o + (part * RB + r) * HD + d, t.o);
                if (d == 0) a.stream_ml[part * RB + r] = make_float2(t.m, t.l);
                continue;
            }
            int tok, h;
            row_of(a, j.tok0, j.kvh, j.row0 + r, tok, h);
            if (a.pre_splits > 0) {
                Join p;
                add_prefix<HD>(a, p, tok, h, d);
                p.add(t.m, t.l, t.o);
                t = p;
            }
            store4(static_cast<typename Core::Q *>(a.out) + int64_t(tok) * a.out_stride + int64_t(h) * HD + d, t.out());
        }
    }
}

// Joins, for each sequence and query-head row, the parts of the shared prefix and of the blocks that share the sequence's
// keys; rows that one block took whole are stored already (without a prefix). WPR warps a row (one where there are rows
// enough for the device, four where there are few): warp w of them takes parts w, w + WPR, .., lane: elements E lane .. of
// the row. Rows: (rows of a sequence up to RB) * kv_heads * seqs.
template <typename QT, int HD, int WPR>
__global__ void __launch_bounds__(kRowsThreads) attn_stream_merge_kernel(const __grid_constant__ AttnArgs a) {
    constexpr int E = HD / 32, RPB = kRowsWarps / WPR;
    __shared__ __align__(16) float s_o[kRowsWarps][HD];
    __shared__ float2 s_ml[kRowsWarps];
    pdl_enter();
    const int warp = (threadIdx.x >> 5) % WPR, lane = threadIdx.x & 31;
    const uint32_t id = blockIdx.x * RPB + (threadIdx.x >> 5) / WPR;
    const uint32_t y = a.srdiv.div(id), b = a.kvdiv.div(y);
    const int r = int(id - y * uint32_t(a.stream_rows)), kvh = int(y - b * uint32_t(a.p.kv_heads));
    if (int(b) >= a.p.seqs) return;  // the whole row's warps (WPR 4: the whole block)
    const int2 desc = __ldcg(a.stream_desc + y);
    int tok0, n, kv, lo;
    const int tiles = stream_tiles(a, int(b), tok0, n, kv, lo);
    const int rows = n * a.p.group;
    if (r >= rows) return;
    int own = 0, c0 = 0;
    if (tiles > 0) {
        c0 = desc.x, own = desc.y - desc.x + 1;
        if (own == 1 && a.pre_splits == 0) return;
    }
    // a sequence without keys: this launch alone stores its rows, those past the host's bound too
    for (int row = r; row < (tiles > 0 ? r + 1 : rows); row += a.stream_rows) {
        int tok, h;
        row_of(a, tok0, kvh, row, tok, h);
        const int64_t pre = (int64_t(tok) * a.p.heads + h) * a.splits;
        const int parts = a.pre_splits + own, mine = (parts - warp + WPR - 1) / WPR;
        // part p: a slot of the prefix, or the c0-th, .. block's part of the own keys (kept as a whole where there is one)
        auto slot = [&](int p, const float2 *&ml, const float *&o) {
            if (p < a.pre_splits) {
                ml = a.part_ml + pre + p, o = a.part_o + (pre + p) * HD;
                return;
            }
            const int c = c0 + p - a.pre_splits;
            const int64_t part = own == 1 ? 2 * int64_t(a.stream_blocks) + y : 2 * int64_t(c) + (c == c0 ? 1 : 0);
            ml = a.stream_ml + part * a.stream_rb + r, o = a.stream_o + (part * a.stream_rb + r) * HD;
        };
        float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0.f;
        for (int base = 0; base < mine; base += 32) {
            const int cnt = min(mine - base, 32);
            const float2 *ml;
            const float *po;
            slot(warp + (base + min(lane, cnt - 1)) * WPR, ml, po);
            const float2 v = lane < cnt ? __ldcg(ml) : make_float2(-INFINITY, 0.f);
            constexpr int U = 8;  // parts in flight; the first of them beside the statistics
            float x[U][E];
            auto fetch = [&](int k) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float *src = reinterpret_cast<const float *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(po), min(k + u, cnt - 1))) + lane * E;
                    if (k + u >= cnt) continue;
                    if constexpr (E == 4) {
                        const float4 f = __ldcg(reinterpret_cast<const float4 *>(src));
                        x[u][0] = f.x, x[u][1] = f.y, x[u][2] = f.z, x[u][3] = f.w;
                    } else {
                        const float2 f = __ldcg(reinterpret_cast<const float2 *>(src));
                        x[u][0] = f.x, x[u][1] = f.y;
                    }
                }
            };
            fetch(0);
            const float mx = fmaxf(m, warp_max(v.x)), ms = mx == -INFINITY ? 0.f : mx;
            const float alpha = ex2_approx(m - ms), w = ex2_approx(v.x - ms);
            m = mx;
            l = l * alpha + warp_sum(v.x == -INFINITY ? v.y : v.y * w);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] *= alpha;
            for (int k = 0; k < cnt; k += U) {
                if (k > 0) fetch(k);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float wu = __shfl_sync(0xffffffffu, w, min(k + u, 31));
                    if (k + u < cnt)
#pragma unroll
                        for (int e = 0; e < E; ++e) o[e] = fmaf(x[u][e], wu, o[e]);
                }
            }
        }
        QT *dst = static_cast<QT *>(a.out) + int64_t(tok) * a.out_stride + int64_t(h) * HD;
        if constexpr (WPR == 1) {
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            if constexpr (E == 4)
                store4(dst + lane * E, make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv));
            else if constexpr (sizeof(QT) == 4)
                *reinterpret_cast<float2 *>(dst + lane * E) = make_float2(o[0] * inv, o[1] * inv);
            else
                *reinterpret_cast<uint32_t *>(dst + lane * E) = pack_bf16(o[0] * inv, o[1] * inv);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
            if (lane == 0) s_ml[warp] = make_float2(m, l);
            __syncthreads();
            for (int d = threadIdx.x * 4; d < HD; d += kRowsThreads * 4) {
                Join t;
#pragma unroll
                for (int w = 0; w < kRowsWarps; ++w) t.add(s_ml[w].x, s_ml[w].y, *reinterpret_cast<const float4 *>(&s_o[w][d]));
                store4(dst + d, t.out());
            }
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------------ launches

// Allows a kernel its dynamic shared memory, once a device.
template <class Core>
bool rows_allow(const void *kern, uint64_t &done) {
    if (Core::kSmem <= 48 * 1024) return true;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    const uint64_t bit = uint64_t(1) << (dev & 63);
    if (__atomic_load_n(&done, __ATOMIC_RELAXED) & bit) return true;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Core::kSmem)) != cudaSuccess) return false;
    __atomic_fetch_or(&done, bit, __ATOMIC_RELAXED);
    return true;
}
template <class Core>
bool rows_ready(int frame) {
    static uint64_t done[3] = {};
    return frame == kFrameCluster  ? rows_allow<Core>((const void *)attn_cluster_kernel<Core>, done[frame])
           : frame == kFrameStream ? rows_allow<Core>((const void *)attn_stream_kernel<Core>, done[frame])
                                   : rows_allow<Core>((const void *)attn_grid_kernel<Core>, done[frame]);
}
// Blocks of the stream frame on the device at once.
template <class Core>
int rows_resident() {
    if (!rows_ready<Core>(kFrameStream)) {
        cudaGetLastError();  // without a device (a size query): what the launch will find
        return sm_count();
    }
    return resident_blocks((const void *)attn_stream_kernel<Core>, kRowsThreads, Core::kSmem);
}

// Launches the frame that the shape asks for (attn.cu): blocks of the grid or stream kernel, or clusters.
template <class Core>
int launch_rows(AttnArgs &a, int frame, int64_t units, cudaStream_t st, const char *name) {
    if (!rows_ready<Core>(frame)) return check_launch(name);
    if (frame == kFrameCluster) {
        cudaLaunchConfig_t cfg = {};
        cfg.dynamicSmemBytes = Core::kSmem;
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
        launch_k(attn_stream_kernel<Core>, dim3(unsigned(units)), kRowsThreads, Core::kSmem, st, a);
        const int64_t rows = int64_t(a.stream_rows) * a.p.kv_heads * a.p.seqs;
        if (rows >= int64_t(sm_count()) * 4)
            launch_k(attn_stream_merge_kernel<typename Core::Q, Core::HD, 1>, dim3(unsigned((rows + kRowsWarps - 1) / kRowsWarps)), kRowsThreads, 0, st, a);
        else
            launch_k(attn_stream_merge_kernel<typename Core::Q, Core::HD, 4>, dim3(unsigned(rows)), kRowsThreads, 0, st, a);
    } else {
        launch_k(attn_grid_kernel<Core>, dim3(unsigned(units)), kRowsThreads, Core::kSmem, st, a);
    }
    return check_launch(name);
}

}  // namespace voxcuda
