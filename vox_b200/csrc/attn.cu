// Attention over a paged key/value cache: vox_cuda_attn_paged and vox_cuda_attn_prefix, their split of the work, the
// CUDA-core kernel (f32 caches) and the join of split rows.
#include <algorithm>
#include <cmath>

#include "attn_rows.cuh"

namespace voxcuda {
namespace {

__device__ __forceinline__ float load_f(const float *p) { return *p; }
__device__ __forceinline__ float load_f(const __nv_bfloat16 *p) { return __bfloat162float(*p); }

// Sums c values over 2 o lanes, each lane left with c / (2 o) whole sums (at least one): at every exchange a lane gives half of its
// values away and adds what it gets to the other half, the upper for the upper lane.
template <int O, int CNT, int N>
__device__ __forceinline__ void halve(float (&s)[N], int lane) {
    if constexpr (O > 0) {
        constexpr int H = CNT > 1 ? CNT / 2 : 1;
        if constexpr (CNT > 1) {
            const bool up = lane & O;
#pragma unroll
            for (int i = 0; i < H; ++i) {
                const float give = up ? s[i] : s[i + H], keep = up ? s[i + H] : s[i];
                s[i] = keep + __shfl_xor_sync(0xffffffffu, give, O);
            }
        } else {
            s[0] += __shfl_xor_sync(0xffffffffu, s[0], O);
        }
        halve<O / 2, H>(s, lane);
    }
}

// softmax(scale q k^T) v on the CUDA cores for an f32 cache, f32 throughout: R rows (query heads that share a key/value
// head, of one or more tokens) against a range of keys. Lane layout: a key's row of HD elements takes LPK lanes of 16
// bytes, so a warp load brings KPW keys (one a group of LPK lanes); a step takes U of them. The U R dot products of a step are
// summed over the group by halving: a lane gives half of its values away at each exchange and adds what it gets to the
// other half, so it ends with the whole sum of one (row, key) pair (or C of them, or D lanes with the same one), takes its
// 2^x alone, keeps the sum of its weights, and hands the weights to the group through shared memory. That is about one
// exchange a score. (A butterfly for each, every lane taking every 2^x: 201 us against 139 at 32 sequences of 2000-4000 keys
// and 4 rows, 369 against 227 at 8.) The rows' references are the warp's and move only when a score exceeds one by 8 (base 2):
// the common step has one vote. Every warp takes each kRowsWarps-th run of KPI keys; from four rows on, the next step's K is
// loaded while this one's weights and products are worked on (without it 169 us for 139, 297 for 225).
// At that size, 8 heads of 128: 1 row 135 us (5.9 TB/s), 2 rows 126 (6.3), 4 rows 139, 8 rows 186 (4.3, bound by the exchanges and
// additions). One token over 650 keys takes 8.4 us in a graph: latency (its 5 MB would need 0.8).
template <typename QT, int HD_, int R>
struct VecCore {
    using Q = QT;
    // of 8 rows, three blocks an SM spill 150 bytes and still pay in long runs (192 us against 225 at the size above, 14 heads on
    // 2 of 64 55 against 63), but not in small calls (26 against 24 at 8 sequences of 1000 keys). Four blocks an SM of 2 and 4 rows
    // spill too: 28-80 bytes in the stream frame, and 36-72 in the cluster frame, which never has as many on an SM and would not
    // need the bound (what that costs there is not measured).
    static constexpr int HD = HD_, RB = R, kMinBlocks = R <= 4 ? 4 : 2, kStreamBlocks = R <= 4 ? 4 : 3;
    static constexpr size_t kSmem = 0;
    struct State {};
    static __device__ __forceinline__ void init(State &) {}
    static __device__ __forceinline__ float (*acc(State &))[RB][HD] {
        __shared__ float s_acc[kRowsWarps][RB][HD];
        return s_acc;
    }

    template <typename F>
    static __device__ __forceinline__ void run(const AttnArgs &a, const RowsJob &j, float (*s_acc)[RB][HD], float2 (*s_ml)[RB], State &, F between) {
        between();
        constexpr int V = 4;                        // elements a lane holds of a key
        constexpr int LPK = HD / V, KPW = 32 / LPK; // lanes a key, keys a warp load
        constexpr int U = R <= 2 ? 8 : 4;           // loads of K (and of V) in flight
        constexpr int KPI = KPW * U;                // keys a step; divides or is a multiple of 16
        constexpr int N = U * R, C = N >= LPK ? N / LPK : 1, D = N >= LPK ? 1 : LPK / N;
        constexpr int kRowLanes = LPK / R;          // of a group
        constexpr bool kAhead = R >= 4;
        __shared__ __align__(16) float s_p[kRowsWarps][2][KPW][N + 4];
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, grp = lane / LPK, li = lane % LPK, e0 = li * V, row0 = j.row0;
        const int mine = li * C / D, row = mine / U, u0 = mine % U;  // this lane's scores: row `row`, keys u0 .. u0 + C - 1 of the group
        const float *K = static_cast<const float *>(a.p.k) + int64_t(j.kvh) * a.p.head_stride + e0;
        const float *Vp = static_cast<const float *>(a.p.v) + int64_t(j.kvh) * a.p.head_stride + e0;
        float2 q[R][V / 2], acc[R][V / 2];
        int kmin = j.k1, kend = j.k0, hi = 0, lo = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int rr = min(row0 + r, j.rows - 1);
            const int i = int(a.gdiv.div(uint32_t(rr))), h = j.kvh * a.p.group + rr - i * a.p.group;
            const QT *src = static_cast<const QT *>(a.q) + int64_t(j.tok0 + i) * a.q_stride + int64_t(h) * HD + e0;
#pragma unroll
            for (int e = 0; e < V / 2; ++e) {
                q[r][e] = make_float2(load_f(src + 2 * e) * a.scale_log2, load_f(src + 2 * e + 1) * a.scale_log2);
                acc[r][e] = make_float2(0.f, 0.f);
            }
            const int h1 = j.causal ? min(j.base + i + 1, j.k1) : j.k1;
            const int l0 = a.window > 0 && j.causal ? max(j.base + i + 1 - a.window, j.k0) : j.k0;
            kmin = min(kmin, l0), kend = max(kend, h1);
            if (r == row) hi = h1, lo = l0;
        }
        float m = -INFINITY, l = 0.f;  // the row's reference; this lane's weights
        uint4 kr[U], vr[U];
        int64_t off[U];
        auto load_k = [&](int base) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int key = base + u * KPW + grp;
                kr[u] = make_uint4(0, 0, 0, 0), off[u] = -1;  // rows outside the range are never read: zero weight times zero
                if (key >= kmin && key < kend) {
                    const int page = page_checked(a.p, __ldg(j.pages + (key >> a.p.page_shift)));
                    off[u] = int64_t(page) * a.p.page_stride + int64_t(key & a.p.page_mask) * a.p.row_stride;
                    kr[u] = ld_stream(K + off[u]);
                }
            }
        };
        int base = (kmin & ~15) + warp * KPI, buf = 0;
        if (kAhead && base < kend) load_k(base);
        for (; base < kend; base += kRowsWarps * KPI, buf ^= 1) {
            if (!kAhead) load_k(base);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                vr[u] = make_uint4(0, 0, 0, 0);
                if (off[u] >= 0) vr[u] = ld_stream(Vp + off[u]);
            }
            float s[N];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float2 kf[V / 2];
                unpack2<VOX_CUDA_F32>(kr[u], kf);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    float2 d = mul2(q[r][0], kf[0]);
#pragma unroll
                    for (int e = 1; e < V / 2; ++e) d = fma2(q[r][e], kf[e], d);
                    s[r * U + u] = d.x + d.y;
                }
            }
            if (kAhead && base + kRowsWarps * KPI < kend) load_k(base + kRowsWarps * KPI);
            halve<LPK / 2, N>(s, lane);
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const int key = base + (u0 + i) * KPW + grp;
                if (key < lo || key >= hi) s[i] = -INFINITY;
                top = fmaxf(top, s[i]);
            }
            if (__any_sync(0xffffffffu, top > m + 8.f)) {
#pragma unroll
                for (int o = 1; o < kRowLanes; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
                for (int o = LPK; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                top = fmaxf(top, m);
                const float alpha = ex2_approx(m - (top == -INFINITY ? 0.f : top));  // nothing seen before: 0
                m = top;
                l *= alpha;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float w = __shfl_sync(0xffffffffu, alpha, r * kRowLanes);
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) acc[r][e] = mul2(acc[r][e], bc2(w));
                }
            }
            const float ref = m == -INFINITY ? 0.f : m;  // nothing seen yet: the weights are 2^-inf = 0
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const float p = ex2_approx(s[i] - ref);
                l += p;
                if (D == 1 || li % D == 0) s_p[warp][buf][grp][mine + i] = p;
            }
            __syncwarp();  // the other buffer's readers are past the last one
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int u = 0; u < U; u += 4) {
                    const float4 p = *reinterpret_cast<const float4 *>(&s_p[warp][buf][grp][r * U + u]);
                    const float w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        float2 vf[V / 2];
                        unpack2<VOX_CUDA_F32>(vr[u + k], vf);
#pragma unroll
                        for (int e = 0; e < V / 2; ++e) acc[r][e] = fma2(vf[e], bc2(w[k]), acc[r][e]);
                    }
                }
        }
        if (D > 1 && li % D != 0) l = 0.f;  // counted by the lane's twin
#pragma unroll
        for (int o = 1; o < kRowLanes; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
        for (int o = LPK; o < 32; o <<= 1) {
            l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    acc[r][e].x += __shfl_xor_sync(0xffffffffu, acc[r][e].x, o);
                    acc[r][e].y += __shfl_xor_sync(0xffffffffu, acc[r][e].y, o);
                }
        }
        if (grp == 0) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < V / 2; ++e) *reinterpret_cast<float2 *>(&s_acc[warp][r][e0 + 2 * e]) = acc[r][e];
            if (li % kRowLanes == 0) s_ml[warp][row] = make_float2(m, l);
        }
    }
};

template <typename QT, typename F>
int with_vec(int head_dim, int rows_blk, F f) {
    if (head_dim == 64)
        return rows_blk == 1 ? f(VecCore<QT, 64, 1>()) : rows_blk == 2 ? f(VecCore<QT, 64, 2>()) : rows_blk == 4 ? f(VecCore<QT, 64, 4>()) : f(VecCore<QT, 64, 8>());
    return rows_blk == 1 ? f(VecCore<QT, 128, 1>()) : rows_blk == 2 ? f(VecCore<QT, 128, 2>()) : rows_blk == 4 ? f(VecCore<QT, 128, 4>()) : f(VecCore<QT, 128, 8>());
}
template <typename F>
int with_vec(int dtype, int head_dim, int rows_blk, F f) {
    return dtype == VOX_CUDA_F32 ? with_vec<float>(head_dim, rows_blk, f) : with_vec<__nv_bfloat16>(head_dim, rows_blk, f);
}

// Joins the splits of each row: one warp a row, lanes over the splits for the weights, then over the head's elements.
template <typename QT, int HD>
__global__ void __launch_bounds__(128) attn_merge_kernel(const AttnArgs a) {
    constexpr int E = HD / 32;
    pdl_enter();
    const int lane = threadIdx.x & 31;
    const int64_t rows = int64_t(a.p.tokens) * a.p.heads;
    for (int64_t row = (int64_t(blockIdx.x) * 128 + threadIdx.x) >> 5; row < rows; row += int64_t(gridDim.x) * 4) {
        const float2 *ml = a.part_ml + row * a.splits;
        const float *po = a.part_o + row * a.splits * HD + lane * E;
        float mx = -INFINITY;
        for (int s = lane; s < a.splits; s += 32) mx = fmaxf(mx, __ldcg(&ml[s]).x);
        mx = warp_max(mx);
        const float ms = mx == -INFINITY ? 0.f : mx;
        float o[E], lt = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0.f;
        for (int s = 0; s < a.splits; ++s) {
            const float2 t = __ldcg(&ml[s]);
            const float w = ex2_approx(t.x - ms);
            lt = fmaf(t.y, w, lt);
            if (t.x == -INFINITY) continue;  // a split without a visible key
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf(__ldcg(po + int64_t(s) * HD + e), w, o[e]);
        }
        const float inv = lt == 0.f ? 0.f : 1.0f / lt;
        const int64_t tok = row / a.p.heads, h = row - tok * a.p.heads;
        QT *dst = static_cast<QT *>(a.out) + tok * a.out_stride + h * HD + lane * E;
        if constexpr (E == 4)
            store4(dst, make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv));
        else if constexpr (sizeof(QT) == 4)
            *reinterpret_cast<float2 *>(dst) = make_float2(o[0] * inv, o[1] * inv);
        else
            *reinterpret_cast<uint32_t *>(dst) = pack_bf16(o[0] * inv, o[1] * inv);
    }
}

int ceil_div(int64_t x, int64_t y) { return int((x + y - 1) / y); }

// How a call is cut: which kernels take its parts, rows a block, row tiles, key splits.
struct AttnShape {
    bool own_tc, pre_tc, concat, mma;  // mma: what the tensor-core kernel does not take goes to attn_mma.cu, else to the CUDA cores
    bool wide, pre_wide;               // or, many rows at f32 accuracy, to attn_f32.cu (the prefix alone, in a launch of its own)
    int frame;                         // of the own keys, where the tensor-core kernel does not take them
    int rows_blk, tc_rows;
    bool tc_half;                      // blocks of one row tile of the tensor-core kernel
    int own_tiles, own_splits, own_chunk;
    int pre_tiles, pre_splits, pre_chunk;
    int cluster, cluster_pre, stream_shift, stream_rows;
    int64_t own_units, pre_blocks;     // blocks, or clusters
    int slots;                         // of a row in the workspace
};

// Keys cut into at most `want` splits of whole 128-key tiles.
void cut_keys(int64_t keys, int64_t want, int &splits, int &chunk) {
    const int64_t tiles = keys > 0 ? (keys + 127) / 128 : 1;
    int64_t n = want < 1 ? 1 : want > tiles ? tiles : want;
    const int64_t per = (tiles + n - 1) / n;
    splits = int((tiles + per - 1) / per);
    chunk = int(per * 128);
}

//
// Times beside a rule: of a 16-head call on 8 key/value heads of 128, in a graph, by the rule and by the other side.
AttnShape attn_shape(const PagedArgs &p, int head_dim, int dtype, bool bf16_cache, int64_t max_q, int64_t max_kv, int64_t prefix_len) {
    AttnShape s = {};
    const int64_t rows = max_q * p.group, all = int64_t(p.tokens) * p.group, sms = sm_count(), base = int64_t(p.seqs) * p.kv_heads;
    const bool f32 = dtype == VOX_CUDA_F32, tc_types = !f32 && bf16_cache;
    s.mma = bf16_cache;
    s.rows_blk = s.mma ? (rows <= 8 || f32 ? 8 : 16) : rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : 8;
    // f32 accuracy by TF32 in 64-row blocks, above as many rows as the few-row kernels read the keys for at once or nearly so: f32
    // caches, 8 sequences of 1000 keys, 8 rows 34.5 us (42 wide), 12 rows 42.9 wide (66.2); bf16 caches, which the few-row
    // kernel takes 8 rows a block from the tensor cores, 32 rows 31.8 us (39.1 wide), 64 rows 44 wide (50)
    s.wide = !tc_types && rows > (bf16_cache ? 32 : 8);
    if (s.wide) s.rows_blk = kF32Rows;
    s.pre_wide = !tc_types && !s.wide && all >= 2 * kF32Rows;
    // 16 sequences of 2000 keys: 16 rows 33 us (38 on attn_tc.cu), 24 rows 37.6 there (57)
    s.own_tc = tc_types && rows > 16;
    s.pre_tc = tc_types && all > 16;
    // row tiles of all sequences together: no more than `bound` (the launch covers it), and `tiles` where max_q holds
    auto bound = [&](int64_t rb) { return p.q_start ? (all - p.seqs) / rb + p.seqs : p.seqs * ((rows + rb - 1) / rb); };
    auto tiles = [&](int64_t rb) { return std::max<int64_t>(std::min(bound(rb), p.seqs * ((rows + rb - 1) / rb)), 1); };
    // Blocks of one row tile, two an SM, where no sequence has more and there are more than one an SM: a block's start and end
    // lie behind the other's walk: 24 texts of 128 rows behind 1003 28.8 us (37.8 in blocks of two tiles), of 64 29.2 (36.3), 64 prompts
    // of 120 rows 28.9 (41.3). With fewer blocks their stages of half the size cost more: 64 rows on each of 16 sequences of 2000
    // keys 49 against 35; and so do longer rows, since every tile of keys is read for half as many: 24 texts of 7-150 tokens behind
    // 1003 54.4 against 49.4, of 100-150 60.4 against 53.9, 12 of 7-150 33.8 against 27.4 (48 of them 107.5 both ways), one prompt of
    // 8192 tokens 271 against 234
    s.tc_half = s.own_tc && rows <= 128 && tiles(128) * p.kv_heads > sms;
    // The prefix in front of each text's own keys in the same block, without a join; or apart, for the rows of all texts
    // together, which fill their row tiles: apart if that spares an SM more than ten tiles of 128 keys, or the texts are short.
    // 24 texts behind 1003 rows: 128 rows a text 37.2 us (38.9 apart), 200 rows 54.9 (57.9), 14-300 rows 52 (50.7), 64 rows 36.2
    // apart (41); 64 texts of 14-200 rows behind 4000 161 apart (284), 8 of 60-600 82.7 (84.7)
    s.concat = prefix_len > 0 && s.own_tc && rows > 64 &&
               (tiles(256) - ceil_div(all, 256)) * p.kv_heads * prefix_len <= int64_t(10) * 128 * sms;
    // one row tile a sequence?
    const bool one_tile = !s.own_tc && !s.wide && rows <= s.rows_blk;
    const int64_t resident = !one_tile ? 0
                             : s.mma   ? attn_mma_resident(head_dim, s.rows_blk, dtype)
                                       : with_vec(dtype, head_dim, s.rows_blk, [](auto core) { return rows_resident<decltype(core)>(); });
    const int64_t fit = s.mma || s.rows_blk < 8 ? resident : std::min(resident, sms * 2);  // clusters' blocks
    if (prefix_len > 0 && one_tile) {
        // one launch of clusters that take the prefix too, by the same rule as below: 8 sequences of up to 1000 rows behind 1003
        // 12.6 us (17.7 in launches apart), 14 heads on 2 of 64 7.9 (14.2)
        int c = 8;
        while (c > 2 && (base * c > fit || 32 * c > prefix_len + max_kv)) c /= 2;
        const int64_t cp = std::clamp<int64_t>((c * prefix_len + (prefix_len + max_kv) / 2) / (prefix_len + max_kv), 1, c - 1);
        if (base * c <= fit && prefix_len <= 512 * cp && max_kv <= 512 * (c - cp)) {
            s.frame = kFrameCluster;
            s.cluster = c, s.cluster_pre = int(cp);
            s.own_units = base;
            return s;
        }
    }
    if (prefix_len > 0 && !s.concat) {
        const int rb = s.pre_tc ? (all > 128 && !s.tc_half ? 256 : 128) : s.pre_wide ? kF32Rows : s.rows_blk;
        if (s.pre_tc) s.tc_rows = rb;
        s.pre_tiles = ceil_div(all, rb);
        const int64_t pre = int64_t(p.kv_heads) * s.pre_tiles;
        cut_keys(prefix_len, s.pre_tc ? (pre < sms ? sms / pre : 1) : ceil_div(sms * 4, pre), s.pre_splits, s.pre_chunk);
        s.pre_blocks = pre * s.pre_splits;
    }
    if (s.own_tc) {
        // both row tiles of a block on different rows halve the reads of keys and fill its softmax's gaps, but halve the blocks:
        // one prompt of 300 tokens 12.6 us with 128 rows a block (14.4 with 256), of 1000 20.2 (23.0); 24 texts of 7-150 tokens
        // behind 1003 rows 52 with 256 (63)
        if (s.tc_rows == 0) s.tc_rows = !s.tc_half && tiles(256) * p.kv_heads >= sms / 2 ? 256 : 128;
        s.own_tiles = int(bound(s.tc_rows));
        const int64_t busy = tiles(s.tc_rows) * p.kv_heads;
        cut_keys(max_kv, s.concat ? 1 : busy < sms ? sms / busy : 1, s.own_splits, s.own_chunk);
        s.own_units = int64_t(s.own_tiles) * p.kv_heads * s.own_splits;
    } else if (one_tile && (prefix_len == 0 || s.pre_tc || s.pre_wide) && base * ((int64_t(p.cap) >> 6) + 1) < (int64_t(1) << 31)) {
        // one row tile a sequence: a cluster for each sequence and key/value head where one wave of blocks holds them all
        // with at most 512 keys each, else equal runs of all sequences' tiles: 8 sequences of 1000-2000 keys 12.4 us in clusters
        // (14.1 in runs), 30 of up to 500 5.8 (7.3); one of 8192 keys 13.7 in runs (18.2), of 16384 16.3 (30.6)
        int c = 8;
        while (c > 1 && (base * c > fit || 32 * c > max_kv)) c /= 2;
        if (base * c <= fit && max_kv <= 512 * c) {
            s.frame = kFrameCluster;
            s.cluster = c;
            s.own_units = base;
        } else {
            s.frame = kFrameStream;
            s.stream_shift = head_dim == 64 ? 7 : 6;  // one step of a block's warps
            s.stream_rows = int(p.q_start ? s.rows_blk : rows);
            const int64_t tiles = base * ((max_kv + (1 << s.stream_shift) - 1) >> s.stream_shift);
            s.own_units = tiles < 1 ? 1 : tiles < resident ? tiles : resident;
        }
    } else {
        s.own_tiles = ceil_div(rows > 0 ? rows : 1, s.rows_blk);
        const int64_t own = base * s.own_tiles;
        cut_keys(max_kv, ceil_div(sms * 4, own), s.own_splits, s.own_chunk);
        s.own_units = own * s.own_splits;
    }
    s.slots = s.pre_splits + s.own_splits;
    return s;
}

// The workspace: the slots of every row (where a row has more than one, or its own keys are taken by another frame), then
// the parts of the stream frame. Offsets in bytes; returns the size.
struct Scratch {
    size_t part_ml, stream_o, stream_ml, stream_desc, bytes;
    bool partial;
};
Scratch scratch_of(const PagedArgs &p, const AttnShape &s, int head_dim) {
    Scratch w = {};
    w.partial = s.slots > 1 || (s.pre_splits > 0 && s.own_splits == 0);
    const size_t slots = w.partial ? size_t(p.tokens) * size_t(p.heads) * size_t(s.slots) : 0;
    const bool stream = s.own_splits == 0 && s.frame == kFrameStream;
    const size_t heads = size_t(p.seqs) * size_t(p.kv_heads);  // a sequence's key/value heads
    const size_t parts = stream ? (size_t(s.own_units) * 2 + (s.pre_splits > 0 ? heads : 0)) * size_t(s.rows_blk) : 0;
    w.part_ml = slots * size_t(head_dim) * sizeof(float);
    w.stream_o = (w.part_ml + slots * sizeof(float2) + 255) & ~size_t(255);
    w.stream_ml = w.stream_o + parts * size_t(head_dim) * sizeof(float);
    w.stream_desc = w.stream_ml + parts * sizeof(float2);
    w.bytes = w.stream_desc + (stream ? heads * sizeof(int2) : 0);
    return w;
}

template <typename QT, int HD>
int launch_merge(const AttnArgs &a, cudaStream_t st, const char *name) {
    const int64_t rows = int64_t(a.p.tokens) * a.p.heads;
    launch_k(attn_merge_kernel<QT, HD>, grid_for(rows * 32, 128, 16), 128, 0, st, a);
    return check_launch(name);
}

int attn_run(const vox_cuda_kv_cache *cache, const vox_cuda_kv_batch *batch, const int32_t *prefix_pages, int64_t prefix_len, const void *q,
             int64_t q_stride, void *out, int64_t out_stride, int64_t heads, float scale, int64_t window, int dtype, void *workspace,
             size_t workspace_bytes, size_t *want, void *stream, const char *name) {
    AttnArgs a = {};
    const int rc = paged_args(cache, batch, heads, name, a.p);
    if (rc != VOX_CUDA_OK) return rc;
    VOX_REQUIRE(is_act_dtype(dtype), std::string(name) + ": dtype must be f32 or bf16");
    VOX_REQUIRE(window >= 0 && prefix_len >= 0 && prefix_len < (int64_t(1) << 30), std::string(name) + ": window or prefix_len out of range");
    if (want) *want = 0;
    if (batch->tokens == 0) return VOX_CUDA_OK;
    const int hd = cache->head_dim;
    const int64_t max_q = batch->q_start == nullptr ? a.p.q_per : batch->max_q > 0 && batch->max_q < batch->tokens ? batch->max_q : batch->tokens;
    const int64_t max_kv = batch->max_kv > 0 && batch->max_kv < a.p.cap ? batch->max_kv : a.p.cap;
    const AttnShape s = attn_shape(a.p, hd, dtype, cache->dtype == VOX_CUDA_BF16, max_q, max_kv, prefix_len);
    VOX_REQUIRE(s.own_units * (s.cluster > 1 ? s.cluster : 1) + s.pre_blocks < (int64_t(1) << 31) &&
                    int64_t(s.rows_blk) * a.p.kv_heads * a.p.seqs < (int64_t(1) << 31),
                std::string(name) + ": sizes out of range");
    const Scratch w = scratch_of(a.p, s, hd);
    const size_t need = w.bytes;
    if (want) {
        *want = need;
        return VOX_CUDA_OK;
    }
    const int64_t el = 16 / dtype_size(dtype);
    VOX_REQUIRE(q && out, std::string(name) + ": NULL pointer");
    VOX_REQUIRE(prefix_len == 0 || prefix_pages, std::string(name) + ": NULL prefix_pages");
    VOX_REQUIRE(q_stride >= heads * hd && out_stride >= heads * hd && q_stride % el == 0 && out_stride % el == 0 && aligned16(q) && aligned16(out),
                std::string(name) + ": q and out must be 16-byte aligned, their row strides cover a row in multiples of 16 bytes");
    VOX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0),
                std::string(name) + ": workspace too small or not 256-byte aligned (vox_cuda_attn_workspace)");
    a.q = q, a.out = out, a.q_stride = q_stride, a.out_stride = out_stride;
    a.prefix_pages = prefix_pages, a.prefix_len = int32_t(prefix_len);
    a.window = int32_t(window < (int64_t(1) << 30) ? window : 0);
    a.scale_log2 = scale * 1.4426950408889634f;
    a.gdiv = FastDiv(uint32_t(a.p.group));
    a.own_splits = s.own_splits, a.own_chunk = s.own_chunk, a.own_tiles = s.own_tiles;
    a.pre_splits = s.pre_splits, a.pre_chunk = s.pre_chunk, a.pre_tiles = s.pre_tiles;
    auto div_by = [](int d) { return FastDiv(uint32_t(d > 0 ? d : 1)); };
    a.kvdiv = div_by(a.p.kv_heads), a.otdiv = div_by(a.p.seqs * (s.own_splits > 0 ? s.own_splits : 1)), a.osdiv = div_by(s.own_splits);
    a.ptdiv = div_by(s.pre_tiles), a.srdiv = div_by(s.stream_rows);
    a.splits = s.slots, a.partial = w.partial;
    a.tc_scale = scale == 0.f ? 1.f : fabsf(a.scale_log2);
    a.q_and = scale == 0.f ? 0u : ~0u, a.q_xor = scale < 0.f ? 0x80008000u : 0u;
    a.tc_rows = s.tc_rows, a.tc_half = s.tc_half, a.concat = s.concat;
    a.cluster = s.cluster, a.cluster_pre = s.cluster_pre, a.stream_shift = s.stream_shift, a.stream_rows = s.stream_rows, a.stream_rb = s.rows_blk;
    a.stream_blocks = int32_t(s.frame == kFrameStream ? s.own_units : 0);
    char *scratch = static_cast<char *>(workspace);
    a.part_o = reinterpret_cast<float *>(scratch), a.part_ml = reinterpret_cast<float2 *>(scratch + w.part_ml);
    a.stream_o = reinterpret_cast<float *>(scratch + w.stream_o), a.stream_ml = reinterpret_cast<float2 *>(scratch + w.stream_ml);
    a.stream_desc = reinterpret_cast<int2 *>(scratch + w.stream_desc);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    using bf = __nv_bfloat16;
    const bool qf = dtype == VOX_CUDA_F32;
    int r = VOX_CUDA_OK;
    if (s.pre_blocks > 0 && (s.pre_wide || (s.pre_tc && !s.own_tc))) {  // the prefix in a launch of its own
        a.pre_blocks = int32_t(s.pre_blocks);
        r = s.pre_tc ? attn_tc_launch(a, *cache, s.pre_blocks, st, name) : attn_f32_launch(a, hd, dtype, cache->dtype, s.pre_blocks, st, name);
        if (r != VOX_CUDA_OK) return r;
    }
    a.pre_blocks = s.pre_wide || (s.pre_tc && !s.own_tc) ? 0 : int32_t(s.pre_blocks);
    const int64_t n = a.pre_blocks + s.own_units;
    if (s.own_tc) {
        r = attn_tc_launch(a, *cache, n, st, name);
    } else {
        if (s.wide) {
            r = attn_f32_launch(a, hd, dtype, cache->dtype, n, st, name);
        } else if (s.mma) {
            r = attn_cache_map(*cache, cache->k, 16, a.mk, name);
            if (r == VOX_CUDA_OK) r = attn_cache_map(*cache, cache->v, 16, a.mv, name);
            if (r != VOX_CUDA_OK) return r;
            r = attn_mma_launch(a, hd, s.rows_blk, dtype, s.frame, n, st, name);
        } else {
            r = with_vec(dtype, hd, s.rows_blk, [&](auto core) { return launch_rows<decltype(core)>(a, s.frame, n, st, name); });
        }
        if (s.frame != kFrameGrid) return r;  // joined there
    }
    if (r != VOX_CUDA_OK || !a.partial) return r;
    if (hd == 64) return qf ? launch_merge<float, 64>(a, st, name) : launch_merge<bf, 64>(a, st, name);
    return qf ? launch_merge<float, 128>(a, st, name) : launch_merge<bf, 128>(a, st, name);
}

}  // namespace

int attn_device_error_word(unsigned int **word) { return device_error_word(word); }

}  // namespace voxcuda

using namespace voxcuda;

extern "C" {

int vox_cuda_attn_paged(const vox_cuda_kv_cache *cache, const vox_cuda_kv_batch *batch, const void *q, int64_t q_stride, void *out,
                        int64_t out_stride, int64_t heads, float scale, int64_t window, int dtype, void *workspace, size_t workspace_bytes,
                        void *stream) {
    return attn_run(cache, batch, nullptr, 0, q, q_stride, out, out_stride, heads, scale, window, dtype, workspace, workspace_bytes, nullptr,
                    stream, "vox_cuda_attn_paged");
}

int vox_cuda_attn_prefix(const vox_cuda_kv_cache *cache, const vox_cuda_kv_batch *batch, const int32_t *prefix_pages, int64_t prefix_len,
                         const void *q, int64_t q_stride, void *out, int64_t out_stride, int64_t heads, float scale, int dtype, void *workspace,
                         size_t workspace_bytes, void *stream) {
    return attn_run(cache, batch, prefix_pages, prefix_len, q, q_stride, out, out_stride, heads, scale, 0, dtype, workspace, workspace_bytes,
                    nullptr, stream, "vox_cuda_attn_prefix");
}

int vox_cuda_attn_workspace(const vox_cuda_kv_cache *cache, const vox_cuda_kv_batch *batch, int64_t prefix_len, int64_t heads, int64_t window,
                            int dtype, size_t *bytes) {
    VOX_REQUIRE(bytes != nullptr, "vox_cuda_attn_workspace: bytes is NULL");
    return attn_run(cache, batch, nullptr, prefix_len, nullptr, 0, nullptr, 0, heads, 1.0f, window, dtype, nullptr, 0, bytes, nullptr,
                    "vox_cuda_attn_workspace");
}

}  // extern "C"
