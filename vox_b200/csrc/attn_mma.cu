// The paged attention of few query rows on a bf16 cache (single tokens, short continuations): bound by reading K and V
// once, so the products only have to stay out of the way of the loads.
//
// A warp takes 16 keys a step (32 of 64-wide heads) against 8 or 16 rows. One lane has the tensor copy engine bring K and V
// tiles of 16 keys x 128 bytes (a page or part of one) into the warp's own ring of two stages in shared memory, so 8 KB a
// warp (96 KB an SM of three blocks) are in flight at no cost in registers or issue slots; the lanes read 16-byte chunks
// back as operands of mma.m16n8k16. Whole chunks serve as operands because the order of a product's summation index is
// free: S^T = K Q^T sums over the head's elements, so lane (g, t) may supply of key g the 16-byte chunks t, t + 4, .. as they
// lie in memory, if Q's operand takes the same chunks; and O^T = V^T P^T has V's elements as its rows, so lane (g, t) loads
// the chunks g, g + 8 of keys 2t, 2t + 1, 2t + 8, 2t + 9 and pairs two keys' halves with one byte permute. The weights turn
// from S^T's layout (lane: a key, two rows) to P^T's (lane: a row, two keys) by one 8 x 8 transpose in registers. The softmax
// keeps one reference maximum a row for the warp, moved only when a score exceeds it by 8 (base 2), so that the common step
// has one vote and no reduction.
//
// f32 activations keep f32 accuracy on the bf16 tensor cores: q and the weights are each cut into three bf16 parts (8 + 8 +
// 8 significant bits), whose products with the bf16 keys and values are exact and accumulate in f32 in the same registers;
// a step's P V is added to the running output by f32 additions rounded to nearest.
//
// Measured (one token a sequence, 16 query heads on 8 of 128): 16 sequences of 20-32 k keys 238 us, 6.7 TB/s, the rate of a
// plain copy. Shorter calls pay the start of the loads (length scan, page look-up, first copies: some 5 us) and the join (see
// attn_rows.cuh): 96 ragged streams of 14 heads on 2 of 64 take 32.5 us, 33 of 16 on 8 of 128 with f32 activations 41. With
// the chunks loaded from memory into registers instead of copied to a ring, f32 activations 49 us and long bf16 streams
// 250; with three stages, and so fewer blocks an SM, 62 against 46 at the same step.
#include "attn_rows.cuh"
#include "tc.cuh"

namespace voxcuda {
namespace {

// D += A . B, m16n8k16, bf16 operands, f32 accumulator.
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
// (x, y) cut into PIECES bf16 pairs whose sums are x and y (3 pieces: to 24 significant bits).
template <int PIECES>
__device__ __forceinline__ void cut_bf16(float x, float y, uint32_t (&w)[PIECES]) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        w[p] = pack_bf16(x, y);
        x -= bf16lo(w[p]);
        y -= bf16hi(w[p]);
    }
}
__device__ __forceinline__ uint32_t word(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

template <typename QT, int HD_, int NT>
struct MmaCore {
    using Q = QT;
    static constexpr int HD = HD_, RB = 8 * NT;
    static constexpr int kStreamBlocks = NT == 2 || sizeof(QT) == 4 ? 2 : 3;
    static constexpr int kMinBlocks = kStreamBlocks;
    static constexpr int kStages = 2;
    static constexpr uint32_t kBox = 16 * 128;    // bytes of a box: 16 keys x 64 elements
    static constexpr uint32_t kStage = 4 * kBox;  // K and V of a step: 2 halves of 16 keys, or 32 keys of 64-wide heads
    static constexpr size_t kSmem = size_t(kRowsWarps) * kStages * kStage + 1024;

    // The warp's ring and its barriers; parity: bit s = parity of the next phase of stage s.
    struct State {
        uint32_t ring, parity;
        uint64_t *bars;
        uint8_t *base;
    };
    // The warps' results take the place of the rings, which hold nothing any more by then.
    static_assert(size_t(kRowsWarps) * RB * HD_ * 4 <= size_t(kRowsWarps) * kStages * kStage, "results fit the rings");
    static __device__ __forceinline__ float (*acc(State &st))[RB][HD] { return reinterpret_cast<float(*)[RB][HD]>(st.base); }
    static __device__ __forceinline__ void init(State &st) {
        extern __shared__ uint8_t ring_raw[];
        __shared__ uint64_t s_bars[kRowsWarps][kStages];
        const int warp = threadIdx.x >> 5;
        st.base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(ring_raw) + 1023) & ~uintptr_t(1023));
        st.ring = smem_addr(st.base) + uint32_t(warp) * kStages * kStage;
        st.bars = s_bars[warp];
        st.parity = 0;
        if ((threadIdx.x & 31) == 0) {
            for (int s = 0; s < kStages; ++s) mbar_init(&st.bars[s], 1);
            mbar_init_fence();
        }
        __syncwarp();
    }

    template <typename F>
    static __device__ __forceinline__ void run(const AttnArgs &a, const RowsJob &j, float (*s_acc)[RB][HD], float2 (*s_ml)[RB], State &st, F between) {
        constexpr int PIECES = sizeof(QT) == 4 ? 3 : 1;
        constexpr int KT = HD == 128 ? 1 : 2;       // runs of 16 keys a step
        constexpr int KC = HD / 32, VC = HD / 64;   // 16-byte chunks a lane takes of a key of K, of a key of V
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, row0 = j.row0;
        // the keys that some row sees, and those that every row sees: tokens ascend, so the first row sees the earliest keys and
        // the last row the latest
        int kmin = j.k1, kend = j.k0, all_lo = j.k0, all_hi = j.k1;
        {
            const int i0 = int(a.gdiv.div(uint32_t(row0))), i1 = int(a.gdiv.div(uint32_t(min(row0 + RB, j.rows) - 1)));
            if (j.causal) {
                all_hi = min(j.base + i0 + 1, j.k1), kend = min(j.base + i1 + 1, j.k1);
                if (a.window > 0) kmin = max(j.base + i0 + 1 - a.window, j.k0), all_lo = max(j.base + i1 + 1 - a.window, j.k0);
                else kmin = j.k0;
            } else {
                kmin = j.k0, kend = j.k1;
            }
        }
        constexpr int STEP = 16 * KT * kRowsWarps;
        const int first = (kmin & ~15) + warp * 16 * KT;
        // page of the 16 keys from `key` on (they never leave one: pages are 16 rows or more)
        auto page_of = [&](int key) { return key < kend ? __ldg(j.pages + (key >> a.p.page_shift)) : 0; };
        int next[KT];
        // starts the copies of the step at `base` into a stage, then looks up the pages of the step after
        auto issue = [&](int base, int stage) {
            if (base >= kend) return;
            const uint32_t to = st.ring + uint32_t(stage) * kStage;
            uint64_t *bar = &st.bars[stage];
            const int runs = KT == 1 || base + 16 >= kend ? 1 : 2;  // of 16 keys
            if (lane == 0) mbar_arrive_expect_tx(bar, KT == 1 ? kStage : uint32_t(runs) * 2 * kBox);
#pragma unroll
            for (int u = 0; u < KT; ++u) {
                if (u < runs) {
                    const int kb = base + 16 * u, page = page_checked(a.p, next[u]);
                    if (lane == 0) {
#pragma unroll
                        for (int h = 0; h < 2 / KT; ++h) {  // halves of a 128-wide head; x is a multiple of 128 bytes
                            tma_load_4d(to + (u + h) * kBox, &a.mk, 64 * h, j.kvh, kb & a.p.page_mask, page, bar);
                            tma_load_4d(to + (2 + u + h) * kBox, &a.mv, 64 * h, j.kvh, kb & a.p.page_mask, page, bar);
                        }
                    }
                }
                next[u] = page_of(base + STEP + 16 * u);
            }
        };
#pragma unroll
        for (int u = 0; u < KT; ++u) next[u] = page_of(first + 16 * u);
        __syncwarp();
        if (lane == 0) fence_proxy_async();  // the ring was last read by ordinary loads
#pragma unroll
        for (int s = 0; s < kStages - 1; ++s) issue(first + s * STEP, s);
        between();
        // Q^T operand: row g of each n-tile, chunk t + 4 c, words 2 h and 2 h + 1 for the two products of a chunk
        uint32_t q[NT][PIECES][KC][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int rr = row0 + 8 * n + g;
            const int i = int(a.gdiv.div(uint32_t(min(rr, j.rows - 1)))), h = j.kvh * a.p.group + min(rr, j.rows - 1) - i * a.p.group;
            const QT *src = static_cast<const QT *>(a.q) + int64_t(j.tok0 + i) * a.q_stride + int64_t(h) * HD;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                if constexpr (PIECES == 1) {
                    const uint4 v = ld_param(src + (t + 4 * c) * 8);
                    q[n][0][c][0] = v.x, q[n][0][c][1] = v.y, q[n][0][c][2] = v.z, q[n][0][c][3] = v.w;
                } else {
                    const float4 u0 = as_f4(ld_param(src + (t + 4 * c) * 8)), u1 = as_f4(ld_param(src + (t + 4 * c) * 8 + 4));
                    const float f[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t pc[PIECES];
                        cut_bf16<PIECES>(f[2 * w], f[2 * w + 1], pc);
#pragma unroll
                        for (int p = 0; p < PIECES; ++p) q[n][p][c][w] = pc[p];
                    }
                }
            }
        }
        // softmax state of rows 2 t, 2 t + 1 of each n-tile and the keys that they see
        float ref[NT][2], l[NT][2];
        int hi[NT][2], lo[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int rr = min(row0 + 8 * n + 2 * t + e, j.rows - 1), i = int(a.gdiv.div(uint32_t(rr)));
                ref[n][e] = -INFINITY, l[n][e] = 0.f;
                hi[n][e] = j.causal ? min(j.base + i + 1, j.k1) : j.k1;
                lo[n][e] = a.window > 0 && j.causal ? max(j.base + i + 1 - a.window, j.k0) : j.k0;
            }
        float acc[VC][4][NT][4];
#pragma unroll
        for (int i = 0; i < VC; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) acc[i][e][n][x] = 0.f;

        // the ring always starts at stage 0: a run leaves no copy in flight
        int stage = 0;
        for (int base = first; base < kend; base += STEP) {
            if (!wait_soon(&st.bars[stage], (st.parity >> stage) & 1u)) {
                // gave up (the device error flag is set): the copies still in flight land, bounded again, before the ring can be
                // reused or released
                for (int s = 0, k = base; s < kStages && k < kend; ++s, k += STEP) {
                    const int x = (stage + s) % kStages;
                    if (s < kStages - 1) wait_soon(&st.bars[x], (st.parity >> x) & 1u), st.parity ^= 1u << x;
                }
                break;
            }
            st.parity ^= 1u << stage;
            {   // the stage before this one has been read by every lane
                const int free = stage == 0 ? kStages - 1 : stage - 1;
                __syncwarp();
                if (lane == 0) fence_proxy_async();
                issue(base + (kStages - 1) * STEP, free);
            }
            const uint32_t in = st.ring + uint32_t(stage) * kStage;
            stage = stage + 1 == kStages ? 0 : stage + 1;
            // chunk c of row r of a box lies at r * 128 + (c ^ (r % 8)) * 16
            uint4 kr[KT][2][KC];
#pragma unroll
            for (int u = 0; u < KT; ++u)
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int c = 0; c < KC; ++c) kr[u][r][c] = lds16(in + (u + (c >> 1)) * kBox + (g + 8 * r) * 128 + (((t + 4 * (c & 1)) ^ g) << 4));
            // S^T: keys g and g + 8 (registers 0-1, 2-3) of rows 2 t, 2 t + 1
            float s[KT][NT][4];
#pragma unroll
            for (int u = 0; u < KT; ++u)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    // independent chains (a product waits some 35 clocks for the one before it in its chain): one a part of q
                    // and half of a chunk's words, with bf16 q also one a half of the chunks
                    constexpr int CH = PIECES == 1 ? 4 : 2 * PIECES;
                    float d[CH][4];
#pragma unroll
                    for (int y = 0; y < CH; ++y)
#pragma unroll
                        for (int x = 0; x < 4; ++x) d[y][x] = 0.f;
#pragma unroll
                    for (int c = 0; c < KC; ++c)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int p = 0; p < PIECES; ++p)
                                mma16816(d[PIECES == 1 ? 2 * (c & 1) + h : 2 * p + h], word(kr[u][0][c], 2 * h), word(kr[u][1][c], 2 * h),
                                         word(kr[u][0][c], 2 * h + 1), word(kr[u][1][c], 2 * h + 1), q[n][p][c][2 * h], q[n][p][c][2 * h + 1]);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        float sum = d[CH - 2][x] + d[CH - 1][x];  // the small parts first
#pragma unroll
                        for (int y = CH - 4; y >= 0; y -= 2) sum += d[y][x] + d[y + 1][x];
                        s[u][n][x] = sum;
                    }
                }
            const bool mask = base < all_lo || base + 16 * KT > all_hi;
            bool move = false;
#pragma unroll
            for (int u = 0; u < KT; ++u)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        s[u][n][x] *= a.scale_log2;
                        if (mask) {
                            const int key = base + 16 * u + g + 8 * (x >> 1);
                            if (key < lo[n][x & 1] || key >= hi[n][x & 1]) s[u][n][x] = -INFINITY;
                        }
                        move = move || s[u][n][x] > ref[n][x & 1] + 8.0f;  // also a row's first key (ref = -inf)
                    }
            if (__any_sync(0xffffffffu, move)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = -INFINITY;
#pragma unroll
                        for (int u = 0; u < KT; ++u) mx = fmaxf(mx, fmaxf(s[u][n][e], s[u][n][e + 2]));
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                        if (mx > ref[n][e]) {
                            const float alpha = ex2_approx(ref[n][e] - mx);
                            ref[n][e] = mx;
                            l[n][e] *= alpha;
#pragma unroll
                            for (int i = 0; i < VC; ++i)
#pragma unroll
                                for (int f = 0; f < 4; ++f) acc[i][f][n][e] *= alpha, acc[i][f][n][e + 2] *= alpha;
                        }
                    }
            }
            uint32_t pf[KT][NT][PIECES][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float r0 = ref[n][0] == -INFINITY ? 0.f : ref[n][0], r1 = ref[n][1] == -INFINITY ? 0.f : ref[n][1];
#pragma unroll
                for (int u = 0; u < KT; ++u)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float p0 = ex2_approx(s[u][n][2 * x] - r0), p1 = ex2_approx(s[u][n][2 * x + 1] - r1);
                        l[n][0] += p0, l[n][1] += p1;
                        uint32_t w[PIECES];
                        cut_bf16<PIECES>(p0, p1, w);
#pragma unroll
                        for (int p = 0; p < PIECES; ++p) pf[u][n][p][x] = transpose8x8(w[p]);
                    }
            }
            uint4 vr[KT][4][VC];
            const bool cut = base < kmin || base + 16 * KT > kend;  // rows outside the range may hold anything, NaN too
#pragma unroll
            for (int u = 0; u < KT; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = 2 * t + (r & 1) + 8 * (r >> 1), key = base + 16 * u + d;
#pragma unroll
                    for (int c = 0; c < VC; ++c) {
                        vr[u][r][c] = lds16(in + (2 + u + c) * kBox + d * 128 + ((g ^ (d & 7)) << 4));
                        if (cut && (key < kmin || key >= kend)) vr[u][r][c] = make_uint4(0, 0, 0, 0);
                    }
                }
            // O^T += V^T P^T: elements 8 (g + 8 i) + 2 e (registers 0-1) and + 1 (2-3) of rows 2 t, 2 t + 1; the products of all
            // elements are independent chains
            if constexpr (PIECES == 1) {
#pragma unroll
                for (int u = 0; u < KT; ++u)
#pragma unroll
                    for (int i = 0; i < VC; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t w0 = word(vr[u][0][i], e), w1 = word(vr[u][1][i], e), w2 = word(vr[u][2][i], e), w3 = word(vr[u][3][i], e);
#pragma unroll
                            for (int n = 0; n < NT; ++n)
                                mma16816(acc[i][e][n], __byte_perm(w0, w1, 0x5410), __byte_perm(w0, w1, 0x7632), __byte_perm(w2, w3, 0x5410),
                                         __byte_perm(w2, w3, 0x7632), pf[u][n][0][0], pf[u][n][0][1]);
                        }
            } else {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < VC; ++i) {
                        float d[4][4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int x = 0; x < 4; ++x) d[e][x] = 0.f;
#pragma unroll
                        for (int u = 0; u < KT; ++u)
#pragma unroll
                            for (int p = PIECES - 1; p >= 0; --p)
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const uint32_t w0 = word(vr[u][0][i], e), w1 = word(vr[u][1][i], e), w2 = word(vr[u][2][i], e),
                                                   w3 = word(vr[u][3][i], e);
                                    mma16816(d[e], __byte_perm(w0, w1, 0x5410), __byte_perm(w0, w1, 0x7632), __byte_perm(w2, w3, 0x5410),
                                             __byte_perm(w2, w3, 0x7632), pf[u][n][p][0], pf[u][n][p][1]);
                                }
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int x = 0; x < 4; ++x) acc[i][e][n][x] += d[e][x];
                    }
            }
        }
        __syncthreads();  // every warp has read its ring
        // the warps' parts of each row
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], o);
                if (g == 0) s_ml[warp][8 * n + 2 * t + e] = make_float2(ref[n][e], l[n][e]);
#pragma unroll
                for (int i = 0; i < VC; ++i)
#pragma unroll
                    for (int f = 0; f < 4; ++f)
                        *reinterpret_cast<float2 *>(&s_acc[warp][8 * n + 2 * t + e][8 * (g + 8 * i) + 2 * f]) =
                            make_float2(acc[i][f][n][e], acc[i][f][n][e + 2]);
            }
    }
};

template <typename F>
int with_core(int head_dim, int rows_blk, int dtype, F f) {
    using bf = __nv_bfloat16;
    if (dtype == VOX_CUDA_F32) return head_dim == 64 ? f(MmaCore<float, 64, 1>()) : f(MmaCore<float, 128, 1>());
    if (rows_blk > 8) return head_dim == 64 ? f(MmaCore<bf, 64, 2>()) : f(MmaCore<bf, 128, 2>());
    return head_dim == 64 ? f(MmaCore<bf, 64, 1>()) : f(MmaCore<bf, 128, 1>());
}

}  // namespace

int attn_mma_launch(AttnArgs &a, int head_dim, int rows_blk, int dtype, int frame, int64_t units, cudaStream_t st, const char *name) {
    return with_core(head_dim, rows_blk, dtype, [&](auto core) { return launch_rows<decltype(core)>(a, frame, units, st, name); });
}
int attn_mma_resident(int head_dim, int rows_blk, int dtype) {
    return with_core(head_dim, rows_blk, dtype,
                     [](auto core) { return rows_resident<decltype(core)>(); });
}

int attn_mma_device_error_word(unsigned int **word) { return device_error_word(word); }

}  // namespace voxcuda
