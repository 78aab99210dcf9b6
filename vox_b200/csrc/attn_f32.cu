// The paged attention of many query rows where f32 accuracy is asked for (f32 activations, or an f32 cache): prompts of the
// CPU engine's own precision. Flash attention on the tensor cores in TF32 with operands cut in two, which keeps f32 accuracy:
// x = hi + lo of 11 significant bits each, and x y = hi hi + hi lo + lo hi up to 2^-21 (a bf16 key or value has no lo part:
// two products). A block takes 64 rows (16 a warp) of one key/value head, the heads that share it side by side, and walks the
// keys in tiles of 32 that its four warps share in shared memory (asynchronous copies, two buffers).
//   S = Q K^T, m16n8k8: the summation index may run in any order, so a lane takes 16-byte chunks of Q's and K's rows as they
//   lie and uses their words two by two; P's accumulator layout (a row, keys 2t and 2t + 1) is the next product's operand
//   layout if V's rows are taken in that order, and V's chunks of four elements serve four column tiles, so nothing is
//   shuffled. Each tile's P V is added to the running output by f32 additions (the tensor cores' own accumulation truncates).
// Row strides in shared memory are padded so that the eight lanes of a 16-byte access phase hit different banks.
//
// The tensor cores' truncation bends f32 results, so chains of products stay short and the small lo products, which one
// truncation at the size of the hi sum would swallow, have sums of their own: largest error against 64 bits 5.0e-7 of the
// output's scale, as against 1.1e-6 in one sum (sums in f32 by plain matrix products: 6.3e-7).
// Bound by the issue and latency of the products (three mma of 16 x 8 x 8 a step, and the cutting of operands between), not by
// bytes: 5 ragged prompts of 90-700 tokens, 16 heads of 64, take 113 us where their bytes would need 6 (tensor pipe 48 %, issue
// 36 %). Two blocks an SM: 113 us against 117 with three (64-wide heads). At the 255 registers that this leaves, 64-wide heads
// spill nothing, 128-wide ones on an f32 cache 8 bytes.
#include "attn_rows.cuh"

namespace voxcuda {
namespace {

constexpr int kRows = kF32Rows;
constexpr int kTileKeys = 32;

template <typename CT, int HD> struct Tile {
    static constexpr int kRow = HD * int(sizeof(CT));                     // bytes of a key
    static constexpr int kK = kRow + (sizeof(CT) == 4 ? 64 : 32);         // padded strides
    static constexpr int kV = kRow + 16;
    static constexpr int kBytes = kTileKeys * (kK + kV);
};

// x = hi + lo: hi rounded to TF32's 11 significant bits in the integer unit (the conversion instruction goes through the
// special-function unit, 16 a clock an SM: 144 us against 117 at 5 ragged prompts of 90-700 tokens, 16 heads of 64, same box), lo
// exact in f32; the tensor cores read its first 11 bits, so hi + lo hold x to 2^-21. NaN and infinities pass through hi.
__device__ __forceinline__ void cut(float x, uint32_t &hi, uint32_t &lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ void mma1688(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool in) {  // or zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16u : 0u) : "memory");
}
// Four consecutive elements in shared memory.
__device__ __forceinline__ void load4(uint32_t addr, float (&v)[4], float) {
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void load4(uint32_t addr, float (&v)[4], __nv_bfloat16) {
    uint32_t x, y;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(addr) : "memory");
    v[0] = bf16lo(x), v[1] = bf16hi(x), v[2] = bf16lo(y), v[3] = bf16hi(y);
}
__device__ __forceinline__ float4 load_q4(const float *p) { return as_f4(ld_param(p)); }
__device__ __forceinline__ float4 load_q4(const __nv_bfloat16 *p) {
    const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
    return make_float4(bf16lo(v.x), bf16hi(v.x), bf16lo(v.y), bf16hi(v.y));
}

template <typename QT, typename CT, int HD>
__global__ void __launch_bounds__(kRowsThreads, 2) attn_f32_kernel(const __grid_constant__ AttnArgs a) {
    using T = Tile<CT, HD>;
    constexpr bool CUT = sizeof(CT) == 4;  // keys and values have a lo part
    constexpr int QC = HD / 16;            // chunks of four elements a lane takes of a row of Q and of K
    constexpr int VC = HD / 32;            // of a row of V
    constexpr bool QSMEM = HD == 128;      // Q in shared memory (each lane its own chunks): registers are short
    extern __shared__ __align__(16) uint8_t smem[];
    pdl_enter();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const AttnJob j = attn_job(a, blockIdx.x);
    const CT *K = static_cast<const CT *>(a.p.k) + int64_t(j.kvh) * a.p.head_stride;
    const CT *V = static_cast<const CT *>(a.p.v) + int64_t(j.kvh) * a.p.head_stride;
    const uint32_t base_s = smem_addr(smem);
    float4 *q_s = reinterpret_cast<float4 *>(smem + 2 * T::kBytes) + threadIdx.x;
    for (int row0 = j.tile * kRows; row0 < j.rows; row0 += j.tiles * kRows) {
        const int wr = row0 + 16 * warp;  // the warp's first row
        int hi[2], lo[2];
        float q[QSMEM ? 1 : QC][2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int rr = min(wr + g + 8 * x, j.rows - 1), i = int(a.gdiv.div(uint32_t(rr))), h = j.kvh * a.p.group + rr - i * a.p.group;
            hi[x] = j.causal ? min(j.base + i + 1, j.k1) : j.k1;
            lo[x] = a.window > 0 && j.causal ? max(j.base + i + 1 - a.window, j.k0) : j.k0;
            const QT *src = static_cast<const QT *>(a.q) + int64_t(j.tok0 + i) * a.q_stride + int64_t(h) * HD + t * 4;
#pragma unroll
            for (int c = 0; c < QC; ++c) {
                const float4 v = load_q4(src + 16 * c);
                if constexpr (QSMEM)
                    q_s[(c * 2 + x) * kRowsThreads] = make_float4(v.x * a.scale_log2, v.y * a.scale_log2, v.z * a.scale_log2, v.w * a.scale_log2);
                else
                    q[c][x][0] = v.x * a.scale_log2, q[c][x][1] = v.y * a.scale_log2, q[c][x][2] = v.z * a.scale_log2, q[c][x][3] = v.w * a.scale_log2;
            }
        }
        // keys that some row of the block sees, that some row of the warp sees, and that every row of the warp sees
        int kmin = j.k0, kend = j.k1, whi = wr < j.rows ? j.k1 : j.k0, wlo = j.k0, all_lo = j.k0, all_hi = j.k1;
        if (j.causal) {
            const int i0 = int(a.gdiv.div(uint32_t(row0))), i1 = int(a.gdiv.div(uint32_t(min(row0 + kRows, j.rows) - 1)));
            const int w0 = int(a.gdiv.div(uint32_t(min(wr, j.rows - 1)))), w1 = int(a.gdiv.div(uint32_t(min(wr + 15, j.rows - 1))));
            kend = min(j.base + i1 + 1, j.k1);
            whi = wr < j.rows ? min(j.base + w1 + 1, j.k1) : j.k0;
            all_hi = min(j.base + w0 + 1, j.k1);
            if (a.window > 0) {
                kmin = max(j.base + i0 + 1 - a.window, j.k0);
                wlo = max(j.base + w0 + 1 - a.window, j.k0);
                all_lo = max(j.base + w1 + 1 - a.window, j.k0);
            }
        }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, acc[VC][4][4];
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[c][e][x] = 0.f;
        const int first = kmin & ~(kTileKeys - 1);
        auto issue = [&](int base, int buf) {
            if (base < kend) {
                constexpr int CPR = T::kRow / 16, STEP = kRowsThreads / CPR;  // chunks a row, rows a pass
                const int c = threadIdx.x % CPR;
#pragma unroll
                for (int p = 0; p < kTileKeys / STEP; ++p) {
                    const int r = threadIdx.x / CPR + p * STEP, key = base + r;
                    const bool in = key >= kmin && key < kend;  // rows outside are never read: they may hold anything
                    int64_t off = 0;
                    if (in) {
                        const int page = page_checked(a.p, __ldg(j.pages + (key >> a.p.page_shift)));
                        off = int64_t(page) * a.p.page_stride + int64_t(key & a.p.page_mask) * a.p.row_stride + c * (16 / int(sizeof(CT)));
                    }
                    const uint32_t to = base_s + uint32_t(buf) * T::kBytes;
                    copy16(to + r * T::kK + c * 16, K + off, in);
                    copy16(to + kTileKeys * T::kK + r * T::kV + c * 16, V + off, in);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        issue(first, 0);
        int buf = 0;
        for (int base = first; base < kend; base += kTileKeys, buf ^= 1) {
            issue(base + kTileKeys, buf ^ 1);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncthreads();
            if (base < whi && base + kTileKeys > wlo) {
                const uint32_t tK = base_s + uint32_t(buf) * T::kBytes + g * T::kK + t * (4 * int(sizeof(CT)));
                const uint32_t tV = base_s + uint32_t(buf) * T::kBytes + kTileKeys * T::kK + 2 * t * T::kV + g * (4 * int(sizeof(CT)));
                // key tile n: rows g (registers 0-1) and g + 8, keys 8 n + 2 t, + 1. The lo products have sums of their own: the tensor
                // cores truncate at every step of a chain, which costs nothing at their size and a third of the steps at hi hi's
                float s[4][4], small[4][4];
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) s[n][x] = small[n][x] = 0.f;
#pragma unroll
                for (int c = 0; c < QC; ++c) {
                    float k4[4][4], q0[4], q1[4];
                    if constexpr (QSMEM) {
                        const float4 x0 = q_s[c * 2 * kRowsThreads], x1 = q_s[(c * 2 + 1) * kRowsThreads];
                        q0[0] = x0.x, q0[1] = x0.y, q0[2] = x0.z, q0[3] = x0.w;
                        q1[0] = x1.x, q1[1] = x1.y, q1[2] = x1.z, q1[3] = x1.w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) q0[e] = q[c][0][e], q1[e] = q[c][1][e];
                    }
#pragma unroll
                    for (int n = 0; n < 4; ++n) load4(tK + 8 * n * T::kK + c * (16 * int(sizeof(CT))), k4[n], CT());
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t ah[4], al[4];
                        cut(q0[2 * h], ah[0], al[0]);
                        cut(q1[2 * h], ah[1], al[1]);
                        cut(q0[2 * h + 1], ah[2], al[2]);
                        cut(q1[2 * h + 1], ah[3], al[3]);
                        uint32_t bh[4][2], bl[4][2];
#pragma unroll
                        for (int n = 0; n < 4; ++n)
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                if constexpr (CUT)
                                    cut(k4[n][2 * h + y], bh[n][y], bl[n][y]);
                                else
                                    bh[n][y] = __float_as_uint(k4[n][2 * h + y]);
                            }
#pragma unroll
                        for (int n = 0; n < 4; ++n) mma1688(small[n], al, bh[n][0], bh[n][1]);
                        if constexpr (CUT)
#pragma unroll
                            for (int n = 0; n < 4; ++n) mma1688(small[n], ah, bl[n][0], bl[n][1]);
#pragma unroll
                        for (int n = 0; n < 4; ++n) mma1688(s[n], ah, bh[n][0], bh[n][1]);
                    }
                }
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) s[n][x] += small[n][x];
                if (base < all_lo || base + kTileKeys > all_hi) {
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const int key = base + 8 * n + 2 * t + (x & 1);
                            if (key < lo[x >> 1] || key >= hi[x >> 1]) s[n][x] = -INFINITY;
                        }
                }
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    float mx = m[y];
#pragma unroll
                    for (int n = 0; n < 4; ++n) mx = fmaxf(mx, fmaxf(s[n][2 * y], s[n][2 * y + 1]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float ms = mx == -INFINITY ? 0.f : mx;  // nothing seen yet: every weight below is 2^-inf = 0
                    const float alpha = ex2_approx(m[y] - ms);
                    m[y] = mx;
                    l[y] *= alpha;
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            s[n][2 * y + e] = ex2_approx(s[n][2 * y + e] - ms);
                            l[y] += s[n][2 * y + e];
                        }
                    if (__any_sync(0xffffffffu, alpha != 1.0f))
#pragma unroll
                        for (int c = 0; c < VC; ++c)
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[c][e][2 * y] *= alpha, acc[c][e][2 * y + 1] *= alpha;
                }
                // P as the left operand: slot t = key 2 t, slot t + 4 = key 2 t + 1 of each run of 8
                uint32_t ph[4][4], pl[4][4];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    cut(s[n][0], ph[n][0], pl[n][0]);
                    cut(s[n][2], ph[n][1], pl[n][1]);
                    cut(s[n][1], ph[n][2], pl[n][2]);
                    cut(s[n][3], ph[n][3], pl[n][3]);
                }
#pragma unroll
                for (int c = 0; c < VC; ++c) {
                    float d[4][4], ds[4][4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int x = 0; x < 4; ++x) d[e][x] = ds[e][x] = 0.f;
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        float v0[4], v1[4];
                        load4(tV + 8 * n * T::kV + c * (32 * int(sizeof(CT))), v0, CT());
                        load4(tV + (8 * n + 1) * T::kV + c * (32 * int(sizeof(CT))), v1, CT());
                        uint32_t bh[4][2], bl[4][2];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if constexpr (CUT) {
                                cut(v0[e], bh[e][0], bl[e][0]);
                                cut(v1[e], bh[e][1], bl[e][1]);
                            } else {
                                bh[e][0] = __float_as_uint(v0[e]), bh[e][1] = __float_as_uint(v1[e]);
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) mma1688(ds[e], pl[n], bh[e][0], bh[e][1]);
                        if constexpr (CUT)
#pragma unroll
                            for (int e = 0; e < 4; ++e) mma1688(ds[e], ph[n], bl[e][0], bl[e][1]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) mma1688(d[e], ph[n], bh[e][0], bh[e][1]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int x = 0; x < 4; ++x) acc[c][e][x] += d[e][x] + ds[e][x];
                }
            }
            __syncthreads();  // the buffer is filled again two tiles on
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            l[y] += __shfl_xor_sync(0xffffffffu, l[y], 1);
            l[y] += __shfl_xor_sync(0xffffffffu, l[y], 2);
            const int rr = wr + g + 8 * y;
            if (rr >= j.rows) continue;
            int tok, h;
            row_of(a, j.tok0, j.kvh, rr, tok, h);
            const int64_t slot = (int64_t(tok) * a.p.heads + h) * a.splits + j.split;
            const float inv = a.partial ? 1.0f : l[y] == 0.f ? 0.f : 1.0f / l[y];  // a row that sees no key gives zeros
            // column 2 t + x of column tile (c, e) is element 32 c + 4 (2 t + x) + e
#pragma unroll
            for (int c = 0; c < VC; ++c)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float4 o = make_float4(acc[c][0][2 * y + x] * inv, acc[c][1][2 * y + x] * inv, acc[c][2][2 * y + x] * inv,
                                                 acc[c][3][2 * y + x] * inv);
                    const int d = 32 * c + 4 * (2 * t + x);
                    if (a.partial)
                        store4(a.part_o + slot * HD + d, o);
                    else
                        store4(static_cast<QT *>(a.out) + int64_t(tok) * a.out_stride + int64_t(h) * HD + d, o);
                }
            if (a.partial && t == 0) a.part_ml[slot] = make_float2(m[y], l[y]);
        }
    }
}

template <typename QT, typename CT, int HD>
int launch(const AttnArgs &a, int64_t blocks, cudaStream_t st, const char *name) {
    constexpr size_t smem = 2 * size_t(Tile<CT, HD>::kBytes) + (HD == 128 ? size_t(kRowsThreads) * 16 * 16 : 0);
    auto kern = attn_f32_kernel<QT, CT, HD>;
    if (smem > 48 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess) return check_launch(name);
    launch_k(kern, dim3(unsigned(blocks)), kRowsThreads, smem, st, a);
    return check_launch(name);
}

}  // namespace

int attn_f32_launch(const AttnArgs &a, int head_dim, int dtype, int cache_dtype, int64_t blocks, cudaStream_t st, const char *name) {
    using bf = __nv_bfloat16;
    const bool qf = dtype == VOX_CUDA_F32, cf = cache_dtype == VOX_CUDA_F32;
    if (head_dim == 64)
        return qf ? (cf ? launch<float, float, 64>(a, blocks, st, name) : launch<float, bf, 64>(a, blocks, st, name))
                  : launch<bf, float, 64>(a, blocks, st, name);
    return qf ? (cf ? launch<float, float, 128>(a, blocks, st, name) : launch<float, bf, 128>(a, blocks, st, name))
              : launch<bf, float, 128>(a, blocks, st, name);
}

int attn_f32_device_error_word(unsigned int **word) { return device_error_word(word); }

}  // namespace voxcuda
