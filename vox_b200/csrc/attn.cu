// Attention over a paged key/value cache: vox_cuda_attn_paged and vox_cuda_attn_prefix, their split of the work, the
// CUDA-core kernel (f32 caches) and the join of split rows.
#include <cmath>

#include "attn.cuh"
#include "sfu.cuh"

namespace voxcuda {
namespace {

constexpr int kVecThreads = 128;
constexpr int kVecWarps = kVecThreads / 32;

template <typename T> struct DtOf;
template <> struct DtOf<float> { static constexpr int v = VOX_CUDA_F32; };
template <> struct DtOf<__nv_bfloat16> { static constexpr int v = VOX_CUDA_BF16; };

__device__ __forceinline__ void store4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void store4(__nv_bfloat16 *p, float4 v) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}
__device__ __forceinline__ float load_f(const float *p) { return *p; }
__device__ __forceinline__ float load_f(const __nv_bfloat16 *p) { return __bfloat162float(*p); }

// softmax(scale q k^T) v on the CUDA cores, f32 throughout: R rows (query heads that share a key/value head, of one or
// more tokens) against the keys of one split. Lane layout: a key's row of HD elements takes LPK lanes of 16 bytes, so a
// warp load brings KPW keys; each group of LPK lanes keeps its own running maximum, sum and output of every row, so the
// loop over the keys has no exchange between groups: per key and row one dot product (a butterfly over the LPK lanes),
// one 2^x, and one multiply-add per element of v. Every warp takes each kVecWarps-th run of KPI keys, U loads of K and U
// of V in flight before the first is used. Groups and warps are joined once, at the end.
template <typename QT, int HD, int R>
__global__ void __launch_bounds__(kVecThreads) attn_vec_kernel(const AttnArgs a) {
    using CT = float;
    constexpr int V = 16 / int(sizeof(CT));     // elements a lane holds of a key
    constexpr int LPK = HD / V, KPW = 32 / LPK; // lanes a key, keys a warp load
    constexpr int U = R <= 2 ? 8 : 4;           // loads of K (and of V) in flight
    constexpr int KPI = KPW * U;                // keys a step; divides or is a multiple of 16
    __shared__ float s_acc[kVecWarps][R][HD];
    __shared__ float2 s_ml[kVecWarps][R];
    pdl_enter();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, grp = lane / LPK, e0 = (lane % LPK) * V;
    const AttnJob j = attn_job(a, blockIdx.x);
    const CT *K = static_cast<const CT *>(a.p.k) + int64_t(j.kvh) * a.p.head_stride + e0;
    const CT *Vp = static_cast<const CT *>(a.p.v) + int64_t(j.kvh) * a.p.head_stride + e0;
    for (int row0 = j.tile * R; row0 < j.rows; row0 += j.tiles * R) {
        float2 q[R][V / 2], acc[R][V / 2];
        float m[R], l[R];
        int hi[R], lo[R];
        int kmin = j.k1, kend = j.k0;
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
            m[r] = -INFINITY, l[r] = 0.f;
            hi[r] = j.causal ? min(j.base + i + 1, j.k1) : j.k1;
            lo[r] = a.window > 0 && j.causal ? max(j.base + i + 1 - a.window, j.k0) : j.k0;
            kmin = min(kmin, lo[r]), kend = max(kend, hi[r]);
        }
        for (int base = (kmin & ~15) + warp * KPI; base < kend; base += kVecWarps * KPI) {
            uint4 kr[U], vr[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int key = base + u * KPW + grp;
                kr[u] = vr[u] = make_uint4(0, 0, 0, 0);  // rows outside the range are never read: zero weight times zero
                if (key >= kmin && key < kend) {
                    const int page = page_checked(a.p, __ldg(j.pages + (key >> a.p.page_shift)));
                    const int64_t off = int64_t(page) * a.p.page_stride + int64_t(key & a.p.page_mask) * a.p.row_stride;
                    kr[u] = ld_stream(K + off);
                    vr[u] = ld_stream(Vp + off);
                }
            }
            float s[U][R];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float2 kf[V / 2];
                unpack2<DtOf<CT>::v>(kr[u], kf);
                const int key = base + u * KPW + grp;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    float2 d = mul2(q[r][0], kf[0]);
#pragma unroll
                    for (int e = 1; e < V / 2; ++e) d = fma2(q[r][e], kf[e], d);
                    float x = d.x + d.y;
#pragma unroll
                    for (int o = LPK / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
                    s[u][r] = key >= lo[r] && key < hi[r] ? x : -INFINITY;
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float mx = m[r];
#pragma unroll
                for (int u = 0; u < U; ++u) mx = fmaxf(mx, s[u][r]);
                const float ms = mx == -INFINITY ? 0.f : mx;  // nothing seen yet: every weight below is 2^-inf = 0
                const float alpha = ex2_approx(m[r] - ms);
                m[r] = mx;
                l[r] *= alpha;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    s[u][r] = ex2_approx(s[u][r] - ms);
                    l[r] += s[u][r];
                }
#pragma unroll
                for (int e = 0; e < V / 2; ++e) acc[r][e] = mul2(acc[r][e], bc2(alpha));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float2 vf[V / 2];
                unpack2<DtOf<CT>::v>(vr[u], vf);
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) acc[r][e] = fma2(vf[e], bc2(s[u][r]), acc[r][e]);
            }
        }
        // the lane groups of a warp, then the warps
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int o = LPK; o < 32; o <<= 1) {
                const float mo = __shfl_xor_sync(0xffffffffu, m[r], o), lo2 = __shfl_xor_sync(0xffffffffu, l[r], o);
                const float mx = fmaxf(m[r], mo), ms = mx == -INFINITY ? 0.f : mx;
                const float wa = ex2_approx(m[r] - ms), wb = ex2_approx(mo - ms);
                m[r] = mx;
                l[r] = l[r] * wa + lo2 * wb;
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    const float2 other = make_float2(__shfl_xor_sync(0xffffffffu, acc[r][e].x, o), __shfl_xor_sync(0xffffffffu, acc[r][e].y, o));
                    acc[r][e] = fma2(acc[r][e], bc2(wa), mul2(other, bc2(wb)));
                }
            }
            if (grp == 0) {
#pragma unroll
                for (int e = 0; e < V / 2; ++e) *reinterpret_cast<float2 *>(&s_acc[warp][r][e0 + 2 * e]) = acc[r][e];
                if (lane == 0) s_ml[warp][r] = make_float2(m[r], l[r]);
            }
        }
        __syncthreads();
        for (int x = threadIdx.x; x < R * (HD / 4); x += kVecThreads) {
            const int r = x / (HD / 4), d = (x % (HD / 4)) * 4;
            if (row0 + r >= j.rows) break;
            float mx = -INFINITY, lt = 0.f;
#pragma unroll
            for (int w = 0; w < kVecWarps; ++w) mx = fmaxf(mx, s_ml[w][r].x);
            const float ms = mx == -INFINITY ? 0.f : mx;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kVecWarps; ++w) {
                const float wt = ex2_approx(s_ml[w][r].x - ms);
                const float4 t = *reinterpret_cast<const float4 *>(&s_acc[w][r][d]);
                lt = fmaf(s_ml[w][r].y, wt, lt);
                o.x = fmaf(t.x, wt, o.x), o.y = fmaf(t.y, wt, o.y), o.z = fmaf(t.z, wt, o.z), o.w = fmaf(t.w, wt, o.w);
            }
            const int i = int(a.gdiv.div(uint32_t(row0 + r))), h = j.kvh * a.p.group + row0 + r - i * a.p.group;
            const int tok = j.tok0 + i;
            if (a.splits == 1) {
                const float inv = lt == 0.f ? 0.f : 1.0f / lt;  // a row that sees no key gives zeros
                store4(static_cast<QT *>(a.out) + int64_t(tok) * a.out_stride + int64_t(h) * HD + d,
                       make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
            } else {
                const int64_t slot = (int64_t(tok) * a.p.heads + h) * a.splits + j.split;
                store4(a.part_o + slot * HD + d, o);
                if (d == 0) a.part_ml[slot] = make_float2(mx, lt);
            }
        }
        __syncthreads();
    }
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
    bool own_tc, pre_tc, concat, mma;  // mma: the rest goes to attn_mma.cu, else to the CUDA cores
    int rows_blk, tc_rows;
    int own_tiles, own_splits, own_chunk;
    int pre_tiles, pre_splits, pre_chunk;
    int64_t own_blocks, pre_blocks;
};

// Keys cut into at most `want` splits of whole 128-key tiles.
void cut_keys(int64_t keys, int64_t want, int &splits, int &chunk) {
    const int64_t tiles = keys > 0 ? (keys + 127) / 128 : 1;
    int64_t n = want < 1 ? 1 : want > tiles ? tiles : want;
    const int64_t per = (tiles + n - 1) / n;
    splits = int((tiles + per - 1) / per);
    chunk = int(per * 128);
}

AttnShape attn_shape(const PagedArgs &p, int64_t max_q, int64_t max_kv, int64_t prefix_len, bool tc_types, bool mma, bool f32) {
    AttnShape s = {};
    const int64_t rows = max_q * p.group, all = int64_t(p.tokens) * p.group, sms = sm_count();
    s.mma = mma;
    s.rows_blk = mma ? (rows <= 8 || f32 ? 8 : 16) : rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : 8;
    s.own_tc = tc_types && rows > 16;
    s.pre_tc = tc_types && all > 16;
    s.concat = prefix_len > 0 && s.own_tc && rows >= 64;
    if (s.own_tc) {
        // row tiles of all sequences together: exact for equal counts, else one more a sequence at most
        auto tiles = [&](int64_t rb) { return p.q_start ? all / rb + p.seqs : p.seqs * ((rows + rb - 1) / rb); };
        s.tc_rows = tiles(256) * p.kv_heads >= sms / 2 ? 256 : 128;
        s.own_tiles = int(tiles(s.tc_rows));
        const int64_t own = int64_t(s.own_tiles) * p.kv_heads;
        cut_keys(max_kv, s.concat ? 1 : own < sms ? sms / own : 1, s.own_splits, s.own_chunk);
        s.own_blocks = own * s.own_splits;
    } else {
        s.own_tiles = ceil_div(rows > 0 ? rows : 1, s.rows_blk);
        const int64_t own = int64_t(p.seqs) * p.kv_heads * s.own_tiles;
        cut_keys(max_kv, ceil_div(sms * 4, own), s.own_splits, s.own_chunk);
        s.own_blocks = own * s.own_splits;
    }
    if (prefix_len > 0 && !s.concat) {
        if (s.pre_tc) s.tc_rows = all > 128 ? 256 : 128;
        s.pre_tiles = ceil_div(all, s.pre_tc ? s.tc_rows : s.rows_blk);
        const int64_t pre = int64_t(p.kv_heads) * s.pre_tiles;
        cut_keys(prefix_len, s.pre_tc ? (pre < sms ? sms / pre : 1) : ceil_div(sms * 4, pre), s.pre_splits, s.pre_chunk);
        s.pre_blocks = pre * s.pre_splits;
    }
    return s;
}

size_t workspace_of(const PagedArgs &p, const AttnShape &s, int head_dim) {
    const int64_t splits = s.own_splits + s.pre_splits;
    if (splits <= 1) return 0;
    const size_t slots = size_t(p.tokens) * size_t(p.heads) * size_t(splits);
    return slots * size_t(head_dim) * sizeof(float) + slots * sizeof(float2);
}

template <typename QT, int HD>
int launch_vec(const AttnArgs &a, const AttnShape &s, int64_t blocks, cudaStream_t st, const char *name) {
    auto kern = s.rows_blk == 1   ? attn_vec_kernel<QT, HD, 1>
                : s.rows_blk == 2 ? attn_vec_kernel<QT, HD, 2>
                : s.rows_blk == 4 ? attn_vec_kernel<QT, HD, 4>
                                  : attn_vec_kernel<QT, HD, 8>;
    launch_k(kern, dim3(unsigned(blocks)), kVecThreads, 0, st, a);
    return check_launch(name);
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
    const std::string nm(name);
    AttnArgs a = {};
    const int rc = paged_args(cache, batch, heads, name, a.p);
    if (rc != VOX_CUDA_OK) return rc;
    VOX_REQUIRE(is_act_dtype(dtype), nm + ": dtype must be f32 or bf16");
    VOX_REQUIRE(window >= 0 && prefix_len >= 0 && prefix_len < (int64_t(1) << 30), nm + ": window or prefix_len out of range");
    if (want) *want = 0;
    if (batch->seqs == 0 || batch->tokens == 0) return VOX_CUDA_OK;
    const int hd = cache->head_dim;
    const int64_t max_q = batch->q_start == nullptr ? a.p.q_per : batch->max_q > 0 && batch->max_q < batch->tokens ? batch->max_q : batch->tokens;
    const int64_t max_kv = batch->max_kv > 0 && batch->max_kv < a.p.cap ? batch->max_kv : a.p.cap;
    const bool tc_types = dtype == VOX_CUDA_BF16 && cache->dtype == VOX_CUDA_BF16;
    const AttnShape s = attn_shape(a.p, max_q, max_kv, prefix_len, tc_types, cache->dtype == VOX_CUDA_BF16, dtype == VOX_CUDA_F32);
    VOX_REQUIRE(s.own_blocks + s.pre_blocks < (int64_t(1) << 31), nm + ": sizes out of range");
    const size_t need = workspace_of(a.p, s, hd);
    if (want) {
        *want = need;
        return VOX_CUDA_OK;
    }
    const int64_t el = 16 / dtype_size(dtype);
    VOX_REQUIRE(q && out, nm + ": NULL pointer");
    VOX_REQUIRE(prefix_len == 0 || prefix_pages, nm + ": NULL prefix_pages");
    VOX_REQUIRE(q_stride >= heads * hd && out_stride >= heads * hd && q_stride % el == 0 && out_stride % el == 0 && aligned16(q) && aligned16(out),
                nm + ": q and out must be 16-byte aligned, their row strides cover a row in multiples of 16 bytes");
    VOX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0),
                nm + ": workspace too small or not 256-byte aligned (vox_cuda_attn_workspace)");
    a.q = q, a.out = out, a.q_stride = q_stride, a.out_stride = out_stride;
    a.prefix_pages = prefix_pages, a.prefix_len = int32_t(prefix_len);
    a.window = int32_t(window < (int64_t(1) << 30) ? window : 0);
    a.scale_log2 = scale * 1.4426950408889634f;
    a.gdiv = FastDiv(uint32_t(a.p.group));
    a.own_splits = s.own_splits, a.own_chunk = s.own_chunk, a.own_tiles = s.own_tiles;
    a.pre_splits = s.pre_splits, a.pre_chunk = s.pre_chunk, a.pre_tiles = s.pre_tiles;
    a.kvdiv = FastDiv(uint32_t(a.p.kv_heads)), a.otdiv = FastDiv(uint32_t(s.own_tiles)), a.osdiv = FastDiv(uint32_t(s.own_splits));
    a.ptdiv = FastDiv(uint32_t(s.pre_tiles > 0 ? s.pre_tiles : 1));
    a.splits = s.own_splits + s.pre_splits;
    a.tc_scale = scale == 0.f ? 1.f : fabsf(a.scale_log2);
    a.q_and = scale == 0.f ? 0u : ~0u, a.q_xor = scale < 0.f ? 0x80008000u : 0u;
    a.tc_rows = s.tc_rows, a.concat = s.concat;
    const size_t slots = size_t(a.p.tokens) * size_t(heads) * size_t(a.splits);
    a.part_o = static_cast<float *>(workspace);
    a.part_ml = reinterpret_cast<float2 *>(static_cast<char *>(workspace) + slots * size_t(hd) * sizeof(float));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    using bf = __nv_bfloat16;
    const bool qf = dtype == VOX_CUDA_F32;
    int r = VOX_CUDA_OK;
    if (s.pre_blocks > 0 && s.pre_tc) {
        a.tc_prefix = 1;
        r = attn_tc_launch(a, *cache, s.pre_blocks, st, name);
        a.tc_prefix = 0;
        if (r != VOX_CUDA_OK) return r;
    }
    if (s.own_tc) {
        r = attn_tc_launch(a, *cache, s.own_blocks, st, name);
    } else {
        a.pre_blocks = s.pre_tc ? 0 : int32_t(s.pre_blocks);
        const int64_t n = a.pre_blocks + s.own_blocks;
        if (s.mma)
            r = attn_mma_launch(a, hd, s.rows_blk, dtype, n, st, name);
        else if (hd == 64)
            r = qf ? launch_vec<float, 64>(a, s, n, st, name) : launch_vec<bf, 64>(a, s, n, st, name);
        else
            r = qf ? launch_vec<float, 128>(a, s, n, st, name) : launch_vec<bf, 128>(a, s, n, st, name);
    }
    if (r != VOX_CUDA_OK || a.splits == 1) return r;
    if (hd == 64) return qf ? launch_merge<float, 64>(a, st, name) : launch_merge<bf, 64>(a, st, name);
    return qf ? launch_merge<float, 128>(a, st, name) : launch_merge<bf, 128>(a, st, name);
}

}  // namespace

int attn_take_device_error(unsigned int *flags) { return take_device_error(flags); }

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
