// vox_cuda_kv_append: the fused projection of a ragged batch of tokens split into q, k and v heads, q and k head-normed
// and rotated at each token's position, K and V written to the pages of the token's sequence.
//
// Per head x of a token at position pos: y = w * (x * 1/sqrt(mean(x^2) + eps)) (q and k, with a norm weight), then for
// p < hd/2 (a, b) = (y[p], y[p + hd/2]) -> (a c - b s, b c + a s) with (c, s) = cs[pos][p], every product rounded by
// itself as the CPU does (kernels.cpp:753-754), so f32 results without a head norm are bit-identical to it. Arithmetic is
// f32 for every type; a bf16 destination is rounded once, at the store.
//
// Bound by HBM at prompts (each projection element is read once and written once, nothing else but a row of the table a
// token) and by latency at single tokens. Layout: a lane holds one 16-byte vector of a head (4 f32 or 8 bf16), so a head
// of width hd takes hd / V lanes and the rotation partner p + hd/2 sits in the lane half of them away: one shuffle, no
// shared memory. A warp takes L such loads of one token, all in flight before the first is used; the token's sequence,
// length and page are looked up while they fly.
#include "paged.cuh"

namespace voxcuda {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct AppendArgs {
    PagedArgs p;
    const void *qkv;
    void *q;
    const float *qn, *kn, *cs;
    int64_t qkv_stride, q_stride;  // elements
    int64_t items;                 // tokens * groups of L warp loads
    int32_t cs_rows, units;        // units: heads + 2 kv_heads
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

template <typename QT, typename CT, int HD, int L>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(AppendArgs a) {
    constexpr int V = 16 / int(sizeof(QT));  // elements a lane holds of a head
    constexpr int LPH = HD / V;              // lanes a head
    constexpr int HPW = 32 / LPH;            // heads a warp load
    pdl_enter();
    const int lane = threadIdx.x & 31;
    const int e0 = (lane % LPH) * V, sub = lane / LPH;
    const bool second = e0 >= HD / 2;  // this lane holds b; its partner holds a
    const int p0 = second ? e0 - HD / 2 : e0;
    const int64_t nw = int64_t(gridDim.x) * kWarps;
    for (int64_t it = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5; it < a.items; it += nw) {
        const uint32_t t = a.gdiv.div(uint32_t(it));
        const int h0 = int(uint32_t(it) - t * a.gdiv.d) * (L * HPW) + sub;
        const QT *src = static_cast<const QT *>(a.qkv) + int64_t(t) * a.qkv_stride + int64_t(h0) * HD + e0;
        uint4 raw[L];
#pragma unroll
        for (int j = 0; j < L; ++j)
            if (h0 + j * HPW < a.units) raw[j] = ld_stream(src + j * HPW * HD);
        // the token's sequence and position
        int b, pos;
        bool ok = true;
        if (a.p.q_start == nullptr) {
            b = int(a.p.qdiv.div(t));
            const int n = __ldg(a.p.kv_len + b);
            pos = n - a.p.q_per + int(t - uint32_t(b) * uint32_t(a.p.q_per));
        } else {
            // the number of sequences that start at or before t, less one; empty sequences share their start with the next
            int c = 0;
            for (int i = lane; i < a.p.seqs; i += 32) c += __ldg(a.p.q_start + i) <= int(t);
            b = __reduce_add_sync(0xffffffffu, c) - 1;
            ok = b >= 0;
            b = max(b, 0);
            const int s0 = __ldg(a.p.q_start + b), s1 = __ldg(a.p.q_start + b + 1), n = __ldg(a.p.kv_len + b);
            ok = ok && int(t) >= s0 && int(t) < s1;
            pos = int(int64_t(n) - s1 + int64_t(t));
        }
        ok = ok && pos >= 0 && pos < a.p.cap && pos < a.cs_rows;
        int page = 0;
        if (ok) {
            page = __ldg(a.p.table + int64_t(b) * a.p.table_stride + (pos >> a.p.page_shift));
            ok = uint32_t(page) < uint32_t(a.p.pages);
        }
        if (!ok) {  // warp-uniform: the token is skipped
            if (lane == 0) range_error();
            continue;
        }
        float cs[2 * V];
        const float4 *csr = reinterpret_cast<const float4 *>(a.cs + (int64_t(pos) * (HD / 2) + p0) * 2);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float4 c4 = __ldg(csr + i);
            cs[4 * i] = c4.x, cs[4 * i + 1] = c4.y, cs[4 * i + 2] = c4.z, cs[4 * i + 3] = c4.w;
        }
        const int64_t row = int64_t(page) * a.p.page_stride + int64_t(pos & a.p.page_mask) * a.p.row_stride + e0;
        QT *qrow = static_cast<QT *>(a.q) + int64_t(t) * a.q_stride + e0;
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const int h = h0 + j * HPW;
            float x[V];
            Vec<DtOf<QT>::v>::unpack(h < a.units ? raw[j] : make_uint4(0, 0, 0, 0), x);
            const bool is_q = h < a.p.heads, is_v = h >= a.p.heads + a.p.kv_heads;
            const float *w = is_q ? a.qn : a.kn;
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (w != nullptr && !is_v) {  // hd is a power of two, so ss * (1 / hd) is ss / hd
                const float inv = rsqrtf(fmaf(ss, 1.0f / float(HD), a.eps));
#pragma unroll
                for (int e = 0; e < V; e += 4) {
                    const float4 w4 = __ldg(reinterpret_cast<const float4 *>(w + e0 + e));
                    x[e] = __fmul_rn(w4.x, __fmul_rn(x[e], inv)), x[e + 1] = __fmul_rn(w4.y, __fmul_rn(x[e + 1], inv));
                    x[e + 2] = __fmul_rn(w4.z, __fmul_rn(x[e + 2], inv)), x[e + 3] = __fmul_rn(w4.w, __fmul_rn(x[e + 3], inv));
                }
            }
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float other = __shfl_xor_sync(0xffffffffu, x[e], LPH / 2);
                const float c = cs[2 * e], s = cs[2 * e + 1];
                o[e] = second ? __fadd_rn(__fmul_rn(x[e], c), __fmul_rn(other, s)) : __fsub_rn(__fmul_rn(x[e], c), __fmul_rn(other, s));
            }
            if (h >= a.units) continue;
            if (is_q)
                store_vals<QT, V>(qrow + int64_t(h) * HD, o);
            else if (!is_v)
                store_vals<CT, V>(static_cast<CT *>(a.p.k) + row + int64_t(h - a.p.heads) * a.p.head_stride, o);
            else
                store_vals<CT, V>(static_cast<CT *>(a.p.v) + row + int64_t(h - a.p.heads - a.p.kv_heads) * a.p.head_stride, x);
        }
    }
}

template <typename QT, typename CT, int HD>
int launch_append(AppendArgs &a, cudaStream_t st) {
    constexpr int HPW = 32 / (HD / (16 / int(sizeof(QT))));
    const int loads = (a.units + HPW - 1) / HPW;  // warp loads a token
    // Four loads in flight a warp where there are warps enough for the device either way, one where there are not
    const bool many = int64_t(a.p.tokens) * loads >= int64_t(sm_count()) * 64;
    const int L = many ? 4 : 1, groups = (loads + L - 1) / L;
    a.items = int64_t(a.p.tokens) * groups;
    a.gdiv = FastDiv(uint32_t(groups));
    auto kern = many ? kv_append_kernel<QT, CT, HD, 4> : kv_append_kernel<QT, CT, HD, 1>;
    launch_k(kern, balanced_grid(a.items, kWarps, resident_blocks((const void *)kern, kThreads, 0)), kThreads, 0, st, a);
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
    VOX_REQUIRE(c->page_stride % el == 0 && c->row_stride % el == 0 && c->head_stride % el == 0 && c->page_stride >= 0 && c->row_stride > 0 &&
                    c->head_stride > 0,
                std::string(name) + ": cache strides must be positive multiples of 16 bytes");
    VOX_REQUIRE(b->seqs >= 0 && b->tokens >= 0 && b->table_width >= 0 && b->table_stride >= b->table_width && b->max_q >= 0 && b->max_kv >= 0,
                std::string(name) + ": bad batch shape");
    VOX_REQUIRE(b->tokens * heads < (int64_t(1) << 31) && int64_t(b->table_width) * c->page_size <= (int64_t(1) << 30),
                std::string(name) + ": sizes out of range");
    if (b->seqs == 0 || b->tokens == 0) return VOX_CUDA_OK;
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

int kv_append_take_device_error(unsigned int *flags) { return take_device_error(flags); }

}  // namespace voxcuda

using namespace voxcuda;

extern "C" int vox_cuda_kv_append(const vox_cuda_kv_cache *cache, const vox_cuda_kv_batch *batch, const void *qkv, int64_t qkv_stride,
                                  const float *q_norm_w, const float *k_norm_w, const float *cs, int64_t cs_rows, void *q,
                                  int64_t q_stride, int64_t heads, float eps, int dtype, void *stream) {
    AppendArgs a = {};
    const int rc = paged_args(cache, batch, heads, "vox_cuda_kv_append", a.p);
    if (rc != VOX_CUDA_OK) return rc;
    VOX_REQUIRE(is_act_dtype(dtype), "vox_cuda_kv_append: dtype must be f32 or bf16");
    if (batch->seqs == 0 || batch->tokens == 0) return VOX_CUDA_OK;
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
