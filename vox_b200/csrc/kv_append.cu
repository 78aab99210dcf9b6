// vox_cuda_kv_append: the fused projection of a ragged batch of tokens split into q, k and v heads, q and k head-normed
// and rotated at each token's position, K and V written to the pages of the token's sequence.
//
// Per head x of a token at position pos: y = w * (x * 1/sqrt(mean(x^2) + eps)) (q and k, with a norm weight), then for
// p < hd/2 (a, b) = (y[p], y[p + hd/2]) -> (a c - b s, b c + a s) with (c, s) = cs[pos][p], every product rounded by
// itself as the CPU does (kernels.cpp:753-754), so f32 results without a head norm are bit-identical to it. Arithmetic is
// f32 for every type; a bf16 destination is rounded once, at the store.
//
// Bound by HBM at prompts (each projection element is read once and written once, nothing else but a row of the table a
// token) and by latency at single tokens. Layout: a lane holds a 16-byte vector of a head's first half and the one hd/2
// further on, the rotation's partners, so the rotation stays in the lane and a head of width hd takes hd / 2V lanes (V = 4
// f32 or 8 bf16); only the mean square crosses lanes. (One vector a lane, the partner fetched by shuffles: 61 us at 14600
// bf16 tokens of 16 + 8 + 8 heads against 47, 5.3 TB/s, bound by the shuffles.) A warp takes L such pairs of vectors of one token at
// a time. A block takes a run of such items; its tokens' sequences,
// positions and pages (three loads that depend on one another) are looked up once, side by side, while the first items'
// loads fly, and an item's loads are issued before the item ahead of it is worked on.
#include "paged.cuh"

namespace voxcuda {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;

struct AppendArgs {
    PagedArgs p;
    const void *qkv;
    void *q;
    const float *qn, *kn, *cs;
    int64_t qkv_stride, q_stride;  // elements
    int64_t items;                 // tokens * groups of L warp loads
    int32_t cs_rows, units, rounds; // units: heads + 2 kv_heads; rounds: items a warp
    FastDiv gdiv;                  // groups a token
    float eps;
};

template <typename T> struct DtOf;
template <> struct DtOf<float> { static constexpr int v = VOX_CUDA_F32; };
template <> struct DtOf<__nv_bfloat16> { static constexpr int v = VOX_CUDA_BF16; };

// N f32 values -> N elements of T at p (16-byte aligned for N elements of 2 bytes and more).
template <typename T, int N>
__device__ __forceinline__ void store_vals(T *p, const float (&v)[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) reinterpret_cast<float4 *>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else if constexpr (N == 8) {
        *reinterpret_cast<uint4 *>(p) = Vec<VOX_CUDA_BF16>::pack(v);
    } else {
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
    }
}

// Where a token's rows go: its position (-1: it is skipped) and page.
struct TokenAt {
    int pos, page;
};
__device__ __forceinline__ TokenAt token_at(const PagedArgs &p, int t) {
    int b, pos;
    bool ok = true;
    if (p.q_start == nullptr) {
        b = int(p.qdiv.div(uint32_t(t)));
        pos = __ldg(p.kv_len + b) - p.q_per + t - b * p.q_per;
    } else {
        // the last sequence that starts at or before t; empty sequences share their start with the next
        int lo = 0, hi = p.seqs;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (__ldg(p.q_start + mid) <= t) lo = mid + 1;
            else hi = mid;
        }
        b = max(lo - 1, 0);
        const int s0 = __ldg(p.q_start + b), s1 = __ldg(p.q_start + b + 1);
        ok = t >= s0 && t < s1;
        pos = int(int64_t(__ldg(p.kv_len + b)) - s1 + int64_t(t));
    }
    ok = ok && pos >= 0 && pos < p.cap;
    int page = 0;
    if (ok) {
        page = __ldg(p.table + int64_t(b) * p.table_stride + (pos >> p.page_shift));
        ok = uint32_t(page) < uint32_t(p.pages);
    }
    return {ok ? pos : -1, page};
}

constexpr int kRounds = 2;  // items a warp takes, at most

template <typename QT, typename CT, int HD, int L>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(AppendArgs a) {
    constexpr int V = 16 / int(sizeof(QT));  // elements a lane holds of a head
    constexpr int LPH = HD / (2 * V);        // lanes a head
    constexpr int HPW = 32 / LPH;            // heads a warp takes at once
    __shared__ TokenAt at[kWarps * kRounds + 1];
    pdl_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int e0 = (lane % LPH) * V, sub = lane / LPH;
    const uint32_t i0 = blockIdx.x * uint32_t(kWarps * a.rounds), i1 = min(i0 + uint32_t(kWarps * a.rounds), uint32_t(a.items));
    const uint32_t t0 = a.gdiv.div(i0);
    uint4 raw[L][2];
    auto fetch = [&](uint32_t it) {
        const uint32_t t = a.gdiv.div(it);
        const int h0 = int(it - t * a.gdiv.d) * (L * HPW) + sub;
        const QT *src = static_cast<const QT *>(a.qkv) + int64_t(t) * a.qkv_stride + int64_t(h0) * HD + e0;
#pragma unroll
        for (int j = 0; j < L; ++j)
#pragma unroll
            for (int y = 0; y < 2; ++y) raw[j][y] = h0 + j * HPW < a.units ? ld_stream(src + j * HPW * HD + y * (HD / 2)) : make_uint4(0, 0, 0, 0);
    };
    uint32_t it = i0 + warp;
    if (it < i1) fetch(it);
    if (threadIdx.x <= a.gdiv.div(i1 - 1) - t0) {
        TokenAt x = token_at(a.p, int(t0 + threadIdx.x));
        if (x.pos >= a.cs_rows) x.pos = -1;
        if (x.pos < 0) range_error();  // the token is skipped
        at[threadIdx.x] = x;
    }
    __syncthreads();
    for (; it < i1; it += kWarps) {
        const uint32_t t = a.gdiv.div(it);
        const int h0 = int(it - t * a.gdiv.d) * (L * HPW) + sub;
        const TokenAt x_at = at[t - t0];
        uint4 cur[L][2];
#pragma unroll
        for (int j = 0; j < L; ++j) cur[j][0] = raw[j][0], cur[j][1] = raw[j][1];
        if (it + kWarps < i1) fetch(it + kWarps);
        if (x_at.pos < 0) continue;
        float cs[2 * V];
        const float4 *csr = reinterpret_cast<const float4 *>(a.cs + (int64_t(x_at.pos) * (HD / 2) + e0) * 2);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float4 c4 = __ldg(csr + i);
            cs[4 * i] = c4.x, cs[4 * i + 1] = c4.y, cs[4 * i + 2] = c4.z, cs[4 * i + 3] = c4.w;
        }
        const int64_t row = int64_t(x_at.page) * a.p.page_stride + int64_t(x_at.pos & a.p.page_mask) * a.p.row_stride + e0;
        QT *qrow = static_cast<QT *>(a.q) + int64_t(t) * a.q_stride + e0;
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const int h = h0 + j * HPW;
            float x[2][V];
            Vec<DtOf<QT>::v>::unpack(cur[j][0], x[0]);
            Vec<DtOf<QT>::v>::unpack(cur[j][1], x[1]);
            const bool is_q = h < a.p.heads, is_v = h >= a.p.heads + a.p.kv_heads;
            const float *w = is_q ? a.qn : a.kn;
            if (a.qn != nullptr || a.kn != nullptr) {
                float s0 = 0.f, s1 = 0.f;  // the halves first, then across lanes: vox_cuda_qkv_rope's order at f32 heads of 128
#pragma unroll
                for (int e = 0; e < V; ++e) s0 = fmaf(x[0][e], x[0][e], s0), s1 = fmaf(x[1][e], x[1][e], s1);
                float ss = s0 + s1;
#pragma unroll
                for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (w != nullptr && !is_v) {  // hd is a power of two, so ss * (1 / hd) is ss / hd
                    const float inv = rsqrtf(fmaf(ss, 1.0f / float(HD), a.eps));
#pragma unroll
                    for (int y = 0; y < 2; ++y)
#pragma unroll
                        for (int e = 0; e < V; e += 4) {
                            const float4 w4 = __ldg(reinterpret_cast<const float4 *>(w + e0 + y * (HD / 2) + e));
                            x[y][e] = __fmul_rn(w4.x, __fmul_rn(x[y][e], inv)), x[y][e + 1] = __fmul_rn(w4.y, __fmul_rn(x[y][e + 1], inv));
                            x[y][e + 2] = __fmul_rn(w4.z, __fmul_rn(x[y][e + 2], inv)), x[y][e + 3] = __fmul_rn(w4.w, __fmul_rn(x[y][e + 3], inv));
                        }
                }
            }
            if (h >= a.units) continue;
            if (!is_v) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float c = cs[2 * e], s = cs[2 * e + 1], p = x[0][e], q = x[1][e];
                    x[0][e] = __fsub_rn(__fmul_rn(p, c), __fmul_rn(q, s));
                    x[1][e] = __fadd_rn(__fmul_rn(q, c), __fmul_rn(p, s));
                }
            }
            if (is_q) {
                QT *dst = qrow + int64_t(h) * HD;
                store_vals<QT, V>(dst, x[0]);
                store_vals<QT, V>(dst + HD / 2, x[1]);
            } else {
                CT *dst = is_v ? static_cast<CT *>(a.p.v) + row + int64_t(h - a.p.heads - a.p.kv_heads) * a.p.head_stride
                               : static_cast<CT *>(a.p.k) + row + int64_t(h - a.p.heads) * a.p.head_stride;
                store_vals<CT, V>(dst, x[0]);
                store_vals<CT, V>(dst + HD / 2, x[1]);
            }
        }
    }
}

template <typename QT, typename CT, int HD>
int launch_append(AppendArgs &a, cudaStream_t st) {
    constexpr int HPW = 32 / (HD / (32 / int(sizeof(QT))));
    const int loads = (a.units + HPW - 1) / HPW;  // warp steps a token
    // Four pairs of loads an item and two items a warp (47 us at the size above; two pairs and four items 50) where there are
    // warps enough for the device either way, else one of each
    const bool many = int64_t(a.p.tokens) * loads >= int64_t(sm_count()) * 64;
    const int L = many ? 4 : 1, groups = (loads + L - 1) / L;
    a.rounds = many ? kRounds : 1;
    a.items = int64_t(a.p.tokens) * groups;
    a.gdiv = FastDiv(uint32_t(groups));
    auto kern = many ? kv_append_kernel<QT, CT, HD, 4> : kv_append_kernel<QT, CT, HD, 1>;
    const int64_t per = int64_t(kWarps) * a.rounds;
    launch_k(kern, dim3(unsigned((a.items + per - 1) / per)), kThreads, 0, st, a);
    return check_launch("vox_cuda_kv_append");
}

}  // namespace

int paged_args(const vox_cuda_kv_cache *c, const vox_cuda_kv_batch *b, int64_t heads, const char *name, PagedArgs &a) {
    VOX_REQUIRE(c && b, std::string(name) + ": NULL cache or batch");
    VOX_REQUIRE(is_act_dtype(c->dtype), std::string(name) + ": the cache must be f32 or bf16");
    VOX_REQUIRE(c->page_size >= 16 && c->page_size <= (1 << 20) && (c->page_size & (c->page_size - 1)) == 0,
                std::string(name) + ": page_size must be a power of two, 16 to 2^20");
    VOX_REQUIRE(c->pages > 0 && c->kv_heads > 0 && heads > 0 && heads % c->kv_heads == 0 && heads <= 65535,
                std::string(name) + ": bad cache shape (heads must be a multiple of kv_heads)");
    if (c->head_dim != 64 && c->head_dim != 128) return set_error(VOX_CUDA_ERR_UNSUPPORTED, std::string(name) + ": head_dim must be 64 or 128");
    const int64_t el = 16 / dtype_size(c->dtype);
    VOX_REQUIRE(c->page_stride % el == 0 && c->row_stride % el == 0 && c->head_stride % el == 0 && c->page_stride > 0 && c->row_stride > 0 &&
                    c->head_stride > 0,
                std::string(name) + ": cache strides must be positive multiples of 16 bytes");
    VOX_REQUIRE(b->seqs >= 0 && b->tokens >= 0 && b->table_width >= 0 && b->table_stride >= b->table_width && b->max_q >= 0 && b->max_kv >= 0,
                std::string(name) + ": bad batch shape");
    VOX_REQUIRE(b->tokens * heads < (int64_t(1) << 31) && int64_t(b->table_width) * c->page_size <= (int64_t(1) << 30),
                std::string(name) + ": sizes out of range");
    VOX_REQUIRE(b->seqs > 0 || b->tokens == 0, std::string(name) + ": tokens without a sequence");
    if (b->tokens == 0) return VOX_CUDA_OK;
    VOX_REQUIRE(c->k && c->v && (b->page_table || b->table_width == 0) && b->kv_len, std::string(name) + ": NULL pointer");
    VOX_REQUIRE(aligned16(c->k) && aligned16(c->v), std::string(name) + ": the cache must be 16-byte aligned");
    VOX_REQUIRE(b->q_start || b->tokens % b->seqs == 0, std::string(name) + ": without q_start the tokens must be a multiple of seqs");
    a.k = c->k, a.v = c->v, a.table = b->page_table, a.kv_len = b->kv_len, a.q_start = b->q_start;
    a.table_stride = b->table_stride, a.page_stride = c->page_stride, a.row_stride = c->row_stride, a.head_stride = c->head_stride;
    a.page_mask = c->page_size - 1;
    a.page_shift = 0;
    while ((1 << a.page_shift) < c->page_size) ++a.page_shift;
    a.pages = c->pages, a.seqs = b->seqs, a.cap = b->table_width * c->page_size;
    a.tokens = int32_t(b->tokens), a.q_per = int32_t(b->tokens / b->seqs);
    a.heads = int32_t(heads), a.kv_heads = c->kv_heads, a.group = int32_t(heads / c->kv_heads);
    a.qdiv = FastDiv(uint32_t(a.q_per > 0 ? a.q_per : 1));
    return VOX_CUDA_OK;
}

int kv_append_device_error_word(unsigned int **word) { return device_error_word(word); }

}  // namespace voxcuda

using namespace voxcuda;

extern "C" int vox_cuda_kv_append(const vox_cuda_kv_cache *cache, const vox_cuda_kv_batch *batch, const void *qkv, int64_t qkv_stride,
                                  const float *q_norm_w, const float *k_norm_w, const float *cs, int64_t cs_rows, void *q,
                                  int64_t q_stride, int64_t heads, float eps, int dtype, void *stream) {
    AppendArgs a = {};
    const int rc = paged_args(cache, batch, heads, "vox_cuda_kv_append", a.p);
    if (rc != VOX_CUDA_OK) return rc;
    VOX_REQUIRE(is_act_dtype(dtype), "vox_cuda_kv_append: dtype must be f32 or bf16");
    if (batch->tokens == 0) return VOX_CUDA_OK;
    VOX_REQUIRE(qkv && cs && q, "vox_cuda_kv_append: NULL pointer");
    const int hd = cache->head_dim;
    const int64_t el = 16 / dtype_size(dtype), units = heads + 2 * int64_t(cache->kv_heads);
    VOX_REQUIRE(qkv_stride >= units * hd && q_stride >= heads * hd && qkv_stride % el == 0 && q_stride % el == 0,
                "vox_cuda_kv_append: row strides must cover a row and be multiples of 16 bytes");
    VOX_REQUIRE(aligned16(qkv) && aligned16(q) && aligned16(cs) && aligned16(q_norm_w) && aligned16(k_norm_w),
                "vox_cuda_kv_append: tensors must be 16-byte aligned");
    VOX_REQUIRE(cs_rows > 0 && cs_rows < (int64_t(1) << 31) && batch->tokens * units < (int64_t(1) << 31),
                "vox_cuda_kv_append: sizes out of range");
    a.qkv = qkv, a.q = q, a.qn = q_norm_w, a.kn = k_norm_w, a.cs = cs;
    a.qkv_stride = qkv_stride, a.q_stride = q_stride, a.cs_rows = int32_t(cs_rows), a.units = int32_t(units), a.eps = eps;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    using bf = __nv_bfloat16;
    const bool qf = dtype == VOX_CUDA_F32, cf = cache->dtype == VOX_CUDA_F32;
    if (hd == 64)
        return qf ? (cf ? launch_append<float, float, 64>(a, st) : launch_append<float, bf, 64>(a, st))
                  : (cf ? launch_append<bf, float, 64>(a, st) : launch_append<bf, bf, 64>(a, st));
    return qf ? (cf ? launch_append<float, float, 128>(a, st) : launch_append<float, bf, 128>(a, st))
              : (cf ? launch_append<bf, float, 128>(a, st) : launch_append<bf, bf, 128>(a, st));
}
