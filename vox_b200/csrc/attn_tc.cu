// The paged attention of many query rows on the 5th-generation tensor cores (bf16 activations on a bf16 cache).
//
// A block takes up to two tiles of 128 query rows of one key/value head (row = token * group + query head in the group, so
// the heads that share keys share every tile of K and V) and walks the keys: S = Q K^T (M 128, N 64 keys) and O += P V (M 128,
// N hd, K 64 keys), both accumulated in f32 in tensor memory; P (bf16) overwrites the first half of its S columns, from where
// the second product reads it as its A operand. Every row tile has two S buffers, so the next scores are there when a
// softmax step ends: the products are off its path. TMEM: S of row tile q, buffer b at column 128 q + 64 b; O at 256 + hd q.
//   warps 0-3, 4-7  softmax of row tile 0, 1: thread = row. Online softmax with a lazy reference: the row's reference
//                   maximum moves only when a score exceeds it by 8 (in powers of two: weights stay below 256, far from
//                   any overflow), so O is rescaled in the few steps where it does; exact, since numerator and
//                   denominator always share the reference.
//   warp 8          tensor copies of K and V tiles of 128 keys through a ring of stages, page by page (a box never leaves a
//                   page); rows of V past the last key are zeroed (their weight is 0, and 0 times what lies there may be NaN)
//   warps 9, 10     issue the products of row tile 0, 1: P V of a step, then Q K^T two steps on into the same S buffer
// Tile order in the ring: K0 V0 K1 V1 ... (both row tiles read each). Every wait is bounded.
// QT 1: the same with one row tile, stages of 64 keys and half of the tensor memory, so that two blocks share an SM (many
// short texts; the rule is in attn.cu). Below, roles and columns are QT 2's.
//
// Measured: one prompt of 8192 tokens, 16 query heads on 8 of 128, 237 us in the first 20 ms from idle, at 1965 MHz (1160 TFLOP/s of
// the causal half, 0.70 of the burst rate of a bare product), and 274 us when run on end for two seconds, at 1605 MHz under the
// 1000 W cap (1000 TFLOP/s, 0.72 of the sustained rate); 7 ragged prompts 210 and 239 us (1725 MHz). Bound by the softmax, some 1610 clocks per 64 keys of both row tiles (exponentials, their
// latency, and the tensor-memory loads before them) where the products need half; every block adds some 6 us before its
// first and after its last product. One S buffer a row tile and steps of 128 keys, so that the products stand in the softmax's
// path: 249 us against 210 at 7 ragged prompts, 56 against 50 at 24 texts behind one prefix.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

#include "attn.cuh"
#include "sfu.cuh"
#include "tc.cuh"

namespace voxcuda {
namespace {

constexpr int kStepKeys = 64;
constexpr int tc_keys(int qt) { return 64 * qt; }  // keys a stage
constexpr int tc_threads(int qt) { return 32 * (5 * qt + 1); }
constexpr uint32_t kHalf = 128 * 128;  // bytes of 128 rows of 64 bf16

// Which of eight pairs of weights take ex2_poly. 1, 2, 3 or 4 of them: 230.6, 231.3, 238, 247 us at one prompt of 8192 tokens
// and 68.1, 66.7, 67.4, 69.9 at 4096.
constexpr int POLY = 0x11;

constexpr int tc_stages(int hd) { return hd == 128 ? 4 : 8; }
constexpr size_t tc_smem(int hd, int qt) { return 1024 + size_t(qt) * (hd / 64) * (kHalf + size_t(tc_stages(hd)) * (kHalf / 2)) + 512; }

// The products of one tile, issued by one elected lane of a converged warp in one piece of code (the issuing warp runs once
// a tile between long stretches of softmax code, so its instructions are cold: few of them matter).
// S = Q K^T: HD / 16 steps; both operands K-major, 32 bytes a step, the second 64 elements of Q kHalf bytes on, of K KS 128.
template <int HD, int KS>
__device__ __forceinline__ void umma_qk_warp(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint64_t *bar) {
#define VOX_QK_STEP(QOFF, KOFF, P) "add.s64 a, %1, " QOFF ";\n\tadd.s64 b, %2, " KOFF ";\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, " P ";\n\t"
#define VOX_QK_HEAD "{\n\t.reg .pred e, z, o;\n\t.reg .b64 a, b;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 z, 0, 0;\n\tsetp.eq.b32 o, 0, 0;\n\t"
#define VOX_COMMIT "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%4];\n\t}"
    if constexpr (HD == 128)
        asm volatile(VOX_QK_HEAD VOX_QK_STEP("0", "0", "z") VOX_QK_STEP("2", "2", "o") VOX_QK_STEP("4", "4", "o") VOX_QK_STEP("6", "6", "o")
                         VOX_QK_STEP("1024", "%5", "o") VOX_QK_STEP("1026", "%5+2", "o") VOX_QK_STEP("1028", "%5+4", "o")
                             VOX_QK_STEP("1030", "%5+6", "o") VOX_COMMIT ::"r"(d),
                     "l"(da), "l"(db), "r"(idesc), "r"(smem_addr(bar)), "n"(KS * 8)
                     : "memory");
    else
        asm volatile(VOX_QK_HEAD VOX_QK_STEP("0", "0", "z") VOX_QK_STEP("2", "2", "o") VOX_QK_STEP("4", "4", "o") VOX_QK_STEP("6", "6", "o")
                         VOX_COMMIT ::"r"(d),
                     "l"(da), "l"(db), "r"(idesc), "r"(smem_addr(bar))
                     : "memory");
}
// O (+)= P V over 64 keys, 16 a step: P in TMEM (two bf16 a column: 8 columns a step), V MN-major (2048 bytes a step); acc:
// whether O holds something.
#define VOX_PV_STEP(C, OFF, P) "add.s32 a, %1, " C ";\n\tadd.s64 b, %2, " OFF ";\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, " P ";\n\t"
__device__ __forceinline__ void umma_pv_warp(uint32_t d, uint32_t ta, uint64_t db, uint32_t idesc, uint32_t acc, uint64_t *bar) {
    asm volatile("{\n\t.reg .pred e, p, o;\n\t.reg .b32 a;\n\t.reg .b64 b;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.eq.b32 o, 0, 0;\n\t"
                 VOX_PV_STEP("0", "0", "p") VOX_PV_STEP("8", "128", "o") VOX_PV_STEP("16", "256", "o") VOX_PV_STEP("24", "384", "o")
                 VOX_COMMIT ::"r"(d), "r"(ta), "l"(db), "r"(idesc), "r"(smem_addr(bar)), "r"(acc)
                 : "memory");
}
// 16 consecutive columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float max3(float x, float y, float z) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(x), "f"(y), "f"(z));
    return d;
}
// 2^x for x <= 64 or so on the multiply-add pipe (two elements), beside the 16 results a clock of the special-function unit:
// x = n + f, n the nearest integer (from the low bits of x + 1.5 2^23), 2^f by a cubic whose relative error on
// [-1/2, 1/2] is below 7.5e-5 (a least-maximum fit made for this kernel; the weights are rounded to bf16 next, 2^-8), times 2^n
// built from its exponent bits. n = -127 has the bits of 0, so below -126.5 (masked scores too) it gives exactly 0, as
// ex2_approx does; NaN stays NaN.
__device__ __forceinline__ float2 ex2_poly(float2 x) {
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.x));
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.y));
    const float2 t = add2(x, bc2(12582912.0f));
    const float2 f = add2(x, fma2(t, bc2(-1.0f), bc2(12582912.0f)));
    float2 p = fma2(bc2(0.05517132f), f, bc2(0.24261054f));
    p = fma2(p, f, bc2(0.69326099f));
    p = fma2(p, f, bc2(0.99992811f));
    return mul2(p, make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3F800000u),
                               __uint_as_float((__float_as_uint(t.y) << 23) + 0x3F800000u)));
}
struct TcJob {
    int ok;
    int tok0, rows, row0;  // tokens of the job start at tok0; this block's rows row0 .. of `rows`
    int kvh, split;
    int base, causal;
    int pa0, pa1;          // keys of the shared prefix
    int k0, k1;            // own keys
    const int32_t *pages;  // of the own keys
};

// The job of block `blk`, found by warp 0 (every lane takes part).
__device__ __forceinline__ void tc_job(const AttnArgs &a, uint32_t blk, TcJob &out) {
    const int lane = threadIdx.x & 31;
    TcJob j = {};
    const bool prefix = blk < uint32_t(a.pre_blocks);
    if (!prefix) blk -= uint32_t(a.pre_blocks);
    uint32_t y = a.kvdiv.div(blk);
    j.kvh = int(blk - y * uint32_t(a.p.kv_heads));
    if (prefix) {  // rows of all tokens against a split of the prefix
        const uint32_t s = a.ptdiv.div(y);
        j.row0 = int(y - s * uint32_t(a.pre_tiles)) * a.tc_rows;
        j.rows = a.p.tokens * a.p.group;
        j.split = int(s);
        j.pa0 = min(int(s) * a.pre_chunk, a.prefix_len);
        j.pa1 = int(s) + 1 == a.pre_splits ? a.prefix_len : min(j.pa0 + a.pre_chunk, a.prefix_len);
        j.ok = j.row0 < j.rows;
    } else {
        const uint32_t t0 = a.osdiv.div(y);
        const int s = int(y - t0 * uint32_t(a.own_splits));
        // the list of all sequences' row tiles from its end: within a sequence the last rows, which see most keys, first, but the
        // sequences in descending order whatever their lengths
        int t = a.own_tiles - 1 - int(t0), b = -1, n = 0, tile = 0;
        if (a.p.q_start == nullptr) {
            const int per = (a.p.q_per * a.p.group + a.tc_rows - 1) / a.tc_rows;
            b = t / per;
            tile = t - b * per;
            j.tok0 = b * a.p.q_per, n = a.p.q_per;
        } else {
            for (int c = 0; c < a.p.seqs; c += 32) {
                int tk = 0, m = 0;
                if (c + lane < a.p.seqs) seq_tokens(a.p, c + lane, tk, m);
                const int mine = int((int64_t(m) * a.p.group + a.tc_rows - 1) / a.tc_rows);
                int cum = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, cum, o);
                    if (lane >= o) cum += v;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, cum > t);
                if (hit) {
                    const int l = __ffs(int(hit)) - 1;
                    b = c + l;
                    j.tok0 = __shfl_sync(0xffffffffu, tk, l), n = __shfl_sync(0xffffffffu, m, l);
                    tile = t - __shfl_sync(0xffffffffu, cum - mine, l);
                    break;
                }
                t -= __shfl_sync(0xffffffffu, cum, 31);
            }
        }
        if (b >= 0) {
            const int kv = seq_rows(a.p, b);
            j.rows = n * a.p.group, j.row0 = tile * a.tc_rows;
            j.base = kv - n, j.causal = 1;
            j.split = (a.concat ? 0 : a.pre_splits) + s;
            j.pages = a.p.table + int64_t(b) * a.p.table_stride;
            const int chunk = max(a.own_chunk, ((kv + a.own_splits - 1) / a.own_splits + 127) & ~127);
            j.k0 = int(min(int64_t(s) * chunk, int64_t(kv)));
            j.k1 = int(min(int64_t(j.k0) + chunk, int64_t(kv)));
            if (a.concat) j.pa1 = a.prefix_len;  // the prefix stands in front of the own keys (one split)
            j.ok = j.row0 < j.rows;
        }
    }
    if (lane == 0) out = j;
}

template <int HD, int QT>
__global__ void __launch_bounds__(tc_threads(QT), QT == 1 ? 2 : 1)
    attn_tc_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv) {
    constexpr int NS = tc_stages(HD), H = HD / 64, KS = tc_keys(QT), SPS = KS / kStepKeys;  // SPS: steps a stage
    constexpr int kCopyWarp = 4 * QT, kMmaWarp = kCopyWarp + 1;
    constexpr uint32_t kTile = H * kHalf, kSub = KS * 128, kStage = H * kSub;  // bytes: a Q tile; 64 columns of a stage; a stage
    constexpr uint32_t kIdS = umma_idesc_bf16(128, kStepKeys), kIdO = umma_idesc_bf16(128, HD, true);
    extern __shared__ uint8_t raw[];
    __shared__ TcJob job;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sQ = smem_addr(smem), sKV = sQ + QT * kTile;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + QT * kTile + NS * kStage), *empty = full + NS;
    uint64_t *s_full = empty + NS, *p_full = s_full + 4, *o_done = p_full + 4, *o_full = o_done + 2, *q_full = o_full + 2, *tail = q_full + 2, *drain = tail + 1;
    uint32_t *tslot = reinterpret_cast<uint32_t *>(drain + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_enter();
    if (warp == 0) tc_job(a, blockIdx.x, job);
    if (threadIdx.x == 32) {
        for (int i = 0; i < NS; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], QT);
        for (int i = 0; i < 4; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 4);
        for (int q = 0; q < 2; ++q) mbar_init(&q_full[q], 4), mbar_init(&o_done[q], 1), mbar_init(&o_full[q], 1);
        mbar_init(tail, 1);
        mbar_init(drain, QT);
        mbar_init_fence();
    }
    if (warp == kMmaWarp) tmem_alloc(tslot, 256 * QT);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const TcJob j = job;
    const uint32_t tmem = *tslot;
    if (!j.ok) {
        if (warp == kMmaWarp) tmem_dealloc(tmem, 256 * QT);
        return;
    }
    // key tiles of a stage: nA of the prefix, then the own keys from kb0; hi of a row tile = keys that its last row sees; nt = its
    // steps of 64 keys
    const int nA = (j.pa1 - j.pa0 + KS - 1) / KS;
    int kb0 = j.k0;
    if (a.window > 0 && j.causal) {
        const int first = int(a.gdiv.div(uint32_t(j.row0)));
        kb0 = max(kb0, max(j.base + first + 1 - a.window, 0) & ~(KS - 1));
    }
    int nt[2] = {0, 0}, kend = 0;
#pragma unroll
    for (int q = 0; q < QT; ++q) {
        const int r0 = j.row0 + 128 * q;
        if (r0 < j.rows && 128 * q < a.tc_rows) {
            const int last = int(a.gdiv.div(uint32_t(min(r0 + 127, j.rows - 1))));
            const int hi = j.causal ? min(j.base + last + 1, j.k1) : 0;
            nt[q] = SPS * nA + max(hi - kb0 + kStepKeys - 1, 0) / kStepKeys;
            kend = max(kend, hi);
        }
    }
    const int nmax = (max(nt[0], nt[1]) + SPS - 1) / SPS;
    if (warp < kCopyWarp) {
        // ---------------------------------------------------------------- softmax: thread = row
        {   // the row tile's Q: 16-byte chunks of whole rows, every load in flight before the first is stored, 128-byte
            // swizzle; rows past the end are zero
            const int q = warp >> 2, w = warp & 3;
            const uint32_t tQ = sQ + q * kTile;
            constexpr int CH = HD / 8, RPI = 32 / CH;  // chunks a row, rows a warp step
            uint4 v[32 / RPI];
#pragma unroll
            for (int s = 0; s < 32 / RPI; ++s) {
                const int rr = j.row0 + 128 * q + w * 32 + s * RPI + lane / CH;
                v[s] = make_uint4(0, 0, 0, 0);
                if (rr < j.rows && (q ? nt[1] : nt[0]) > 0) {
                    const int i = int(a.gdiv.div(uint32_t(rr))), h = j.kvh * a.p.group + rr - i * a.p.group;
                    v[s] = ld_param(static_cast<const __nv_bfloat16 *>(a.q) + int64_t(j.tok0 + i) * a.q_stride + int64_t(h) * HD + lane % CH * 8);
                }
            }
#pragma unroll
            for (int s = 0; s < 32 / RPI; ++s) {
                const int r = w * 32 + s * RPI + lane / CH, c = lane % CH;
                const uint32_t dst = tQ + (c >> 3) * kHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"((v[s].x & a.q_and) ^ a.q_xor),
                             "r"((v[s].y & a.q_and) ^ a.q_xor), "r"((v[s].z & a.q_and) ^ a.q_xor), "r"((v[s].w & a.q_and) ^ a.q_xor)
                             : "memory");
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[q]);
        }
        const int q = warp >> 2, row = (warp & 3) * 32 + lane, rr = j.row0 + 128 * q + row;
        const int n = q ? nt[1] : nt[0];
        const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16), tO = lanes + 128 * QT + HD * q;
        const bool live = rr < j.rows && 128 * q < a.tc_rows;
        const int i_tok = int(a.gdiv.div(uint32_t(live ? rr : 0)));
        const int hi_own = live && j.causal ? min(j.base + i_tok + 1, j.k1) : 0;
        const int lo_own = a.window > 0 ? max(j.base + i_tok + 1 - a.window, j.k0) : j.k0;
        float ref = -INFINITY;  // reference maximum (scaled, base 2)
        float2 l2[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        bool ok = true;
#pragma unroll 1
        for (int u = 0; u < n; ++u) {
            const uint32_t tS = lanes + 128 * q + 64 * (u & 1);
            ok = wait_soon(&s_full[2 * q + (u & 1)], uint32_t(u >> 1) & 1u);
            if (!ok) break;
            tc_fence_after();
            uint32_t r[64];
            tmem_ld32(tS, *reinterpret_cast<uint32_t(*)[32]>(r));
            tmem_ld32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(r + 32));
            tmem_wait_ld(*reinterpret_cast<uint32_t(*)[32]>(r));
            tmem_wait_ld(*reinterpret_cast<uint32_t(*)[32]>(r + 32));
            const bool pre = u < SPS * nA;
            const int key0 = pre ? j.pa0 + u * kStepKeys : kb0 + (u - SPS * nA) * kStepKeys;
            const int hi = (pre ? (live ? j.pa1 : 0) : hi_own) - key0, lo = (pre ? j.pa0 : lo_own) - key0;
            if (!__all_sync(0xffffffffu, hi >= kStepKeys && lo <= 0)) {
#pragma unroll
                for (int c = 0; c < kStepKeys; ++c)
                    if (c >= hi || c < lo) r[c] = __float_as_uint(-INFINITY);
            }
            float m4[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) m4[c] = max3(__uint_as_float(r[c]), __uint_as_float(r[c + 4]), __uint_as_float(r[c + 8]));
#pragma unroll
            for (int c = 12; c < 60; c += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e) m4[e] = max3(m4[e], __uint_as_float(r[c + e]), __uint_as_float(r[c + 4 + e]));
#pragma unroll
            for (int e = 0; e < 4; ++e) m4[e] = fmaxf(m4[e], __uint_as_float(r[60 + e]));
            const float mx = fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]) * a.tc_scale;
            const bool move = mx > ref + 8.0f;  // also the first key that the row sees (ref = -inf)
            if (__any_sync(0xffffffffu, move)) {
                const float nref = move ? mx : ref;
                const float alpha = move ? ex2_approx(ref - nref) : 1.0f;
                ref = nref;
#pragma unroll
                for (int e = 0; e < 4; ++e) l2[e] = mul2(l2[e], bc2(alpha));
                if (u > 0) {  // the step before's P V has to be in O first (these scores came behind the one before that)
                    ok = wait_soon(&o_done[q], uint32_t(u - 1) & 1u);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t o[32];
                        tmem_ld32(tO + c, o);
                        tmem_wait_ld(o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tmem_st16(tO + c, *reinterpret_cast<uint32_t(*)[16]>(o));
                        tmem_st16(tO + c + 16, *reinterpret_cast<uint32_t(*)[16]>(o + 16));
                    }
                }
            }
            const float2 sc = bc2(a.tc_scale), nr = bc2(ref == -INFINITY ? 0.f : -ref);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int k = 32 * c + 2 * e;
                    const float2 x = fma2(make_float2(__uint_as_float(r[k]), __uint_as_float(r[k + 1])), sc, nr);
                    // part of the weights on the multiply-add pipe: the special-function unit alone would take all of a step
                    const float2 p = (POLY >> (e & 7)) & 1 ? ex2_poly(x) : make_float2(ex2_approx(x.x), ex2_approx(x.y));
                    l2[e & 3] = add2(l2[e & 3], p);
                    w[e] = pack_bf16(p.x, p.y);
                }
                tmem_st16(tS + 16 * c, w);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[2 * q + (u & 1)]);
        }
        if (n > 0 && ok) {
            ok = wait_soon(&o_full[q], 0);
            tc_fence_after();
        }
        const float2 ls = add2(add2(l2[0], l2[1]), add2(l2[2], l2[3]));
        const float l = ls.x + ls.y;  // of a row that saw no key: exactly 0
        const int h = j.kvh * a.p.group + (live ? rr - i_tok * a.p.group : 0);
        const int64_t tok = j.tok0 + i_tok;
        const int64_t slot = (tok * a.p.heads + h) * a.splits + j.split;
        const float inv = a.partial ? 1.0f : l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;  // NaN stays NaN
        // a warp's 32 rows go through the row tile's Q (its products are complete) so that they are stored in whole runs of a
        // row: 64 columns a pass of the f32 parts, all of a row a pass of the bf16 result (one 16-byte chunk a lane, the
        // chunks of a row swizzled over the banks)
        constexpr int CPR = HD / 8;  // chunks of a row a pass
        const uint32_t stage = sQ + q * kTile + (warp & 3) * (kTile / 4);
        char *dst = a.partial ? reinterpret_cast<char *>(a.part_o + slot * HD)
                              : reinterpret_cast<char *>(static_cast<__nv_bfloat16 *>(a.out) + tok * a.out_stride + int64_t(h) * HD);
        if (!live || !ok) dst = nullptr;
        auto put = [&](int c, uint4 v) {
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * (CPR * 16) + ((c ^ (lane & 7)) << 4)), "r"(v.x), "r"(v.y), "r"(v.z),
                         "r"(v.w)
                         : "memory");
        };
        const int passes = a.partial ? 2 : 1;
#pragma unroll 1
        for (int pass = 0; pass < passes; ++pass) {
            const int cols = a.partial ? HD / 2 : HD;
#pragma unroll 1
            for (int col = 0; col < cols; col += 32) {
                uint32_t o[32];
                if (n > 0 && ok) {
                    tmem_ld32(tO + pass * (HD / 2) + col, o);
                    tmem_wait_ld(o);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0;
                }
                if (a.partial) {
#pragma unroll
                    for (int c = 0; c < 8; ++c) put(col / 4 + c, make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]));
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float f[8];
#pragma unroll
                        for (int u = 0; u < 8; ++u) f[u] = __uint_as_float(o[8 * c + u]) * inv;
                        put(col / 8 + c, Vec<VOX_CUDA_BF16>::pack(f));
                    }
                }
            }
            __syncwarp();
#pragma unroll 4
            for (int x = 0; x < CPR; ++x) {  // CPR lanes a row, 32 / CPR rows a step
                const int r = x * (32 / CPR) + lane / CPR, c = lane % CPR;
                char *to = reinterpret_cast<char *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), r));
                uint4 v;
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                             : "r"(stage + r * (CPR * 16) + ((c ^ (r & 7)) << 4))
                             : "memory");
                if (to != nullptr) *reinterpret_cast<uint4 *>(to + pass * (CPR * 16) + c * 16) = v;
            }
            __syncwarp();
        }
        if (live && ok && a.partial) a.part_ml[slot] = make_float2(ref, l);
    } else if (warp == kCopyWarp) {
        // ---------------------------------------------------------------- copies
        const int pr = min(a.p.page_mask + 1, KS);  // rows a box
        bool ok = true;
        int tails = 0, n = 0;
        for (; n < 2 * nmax && ok; ++n) {
            const int i = n >> 1, s = n % NS;
            const bool is_v = n & 1, pre = i < nA;
            const int key0 = pre ? j.pa0 + i * KS : kb0 + (i - nA) * KS;
            const int valid = min((pre ? j.pa1 : kend) - key0, KS);
            if (n >= NS) ok = wait_soon(&empty[s], uint32_t(n / NS - 1) & 1u);
            if (!ok) break;
            const int boxes = (valid + pr - 1) / pr * H;
            const bool zero = is_v && valid < KS;
            uint64_t *bar = zero ? tail : &full[s];
            const uint32_t st = sKV + s * kStage;
            if (lane == 0) mbar_arrive_expect_tx(bar, uint32_t(boxes * pr) * 128u);
            __syncwarp();
            if (lane < boxes) {
                const int p = lane / H, half = lane % H, key = key0 + p * pr;
                const int page = page_checked(a.p, __ldg((pre ? a.prefix_pages : j.pages) + (key >> a.p.page_shift)));
                tma_load_4d(st + half * kSub + p * pr * 128, is_v ? &mv : &mk, half * 64, j.kvh, key & a.p.page_mask, page, bar);
            }
            if (zero) {
                ok = wait_soon(tail, uint32_t(tails++ & 1));
                for (int x = valid * 8 + lane; x < KS * 8; x += 32)
#pragma unroll
                    for (int half = 0; half < H; ++half)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(st + half * kSub + x * 16), "r"(0) : "memory");
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[s]);
            }
        }
        // every copy issued has landed before the block's shared memory is released
        for (int m = max(n - NS, 0); m < n; ++m) wait_soon(&full[m % NS], uint32_t(m / NS) & 1u);
    } else {
        // ---------------------------------------------------------------- products of row tile q
        const int q = warp - kMmaWarp, n = q ? nt[1] : nt[0];
        bool ok = true;
        auto wait_full = [&](int m) { return wait_soon(&full[m % NS], uint32_t(m / NS) & 1u); };
        constexpr uint32_t kNext = kStage >> 4, kHalfStage = kStepKeys * 128 >> 4;  // a stage, a step's keys on, in descriptor units
        const uint64_t dQ = umma_desc(sQ + q * kTile, 16, 1024), dK = umma_desc(sKV, 16, 1024), dV = umma_desc(sKV, kSub, 1024);
        const uint32_t tS = tmem + 128 * q, tO = tmem + 128 * QT + HD * q;
        auto qk = [&](int u) {  // scores of step u; the last step of a tile gives K back
            const int m = u / SPS * 2, sub = u % SPS;
            if (sub == 0) ok = wait_full(m);
            if (!ok) return;
            tc_fence_after();
            umma_qk_warp<HD, KS>(tS + 64 * (u & 1), dQ, dK + uint32_t(m % NS) * kNext + sub * kHalfStage, kIdS, &s_full[2 * q + (u & 1)]);
            if (sub == SPS - 1 || u + 1 == n) umma_commit_warp(&empty[m % NS]);
        };
        if (n > 0) {
            ok = wait_soon(&q_full[q], 0);
            if (ok) qk(0);
            if (ok && n > 1) qk(1);
        }
#pragma unroll 1
        for (int u = 0; u < n && ok; ++u) {
            const int m = u / SPS * 2 + 1, sub = u % SPS;  // V of the stage
            if (sub == 0) ok = wait_full(m);
            ok = ok && wait_soon(&p_full[2 * q + (u & 1)], uint32_t(u >> 1) & 1u);
            if (!ok) break;
            tc_fence_after();
            umma_pv_warp(tO, tS + 64 * (u & 1), dV + uint32_t(m % NS) * kNext + sub * kHalfStage, kIdO, uint32_t(u > 0), &o_done[q]);
            if (sub == SPS - 1 || u + 1 == n) umma_commit_warp(&empty[m % NS]);
            if (u + 1 == n) umma_commit_warp(&o_full[q]);
            if (u + 2 < n) qk(u + 2);
        }
        // tiles that only the other row tile reads: given back as they come (a stage is free when both warps have said so)
        for (int m = (n + SPS - 1) / SPS * 2; m < 2 * nmax && ok; ++m) {
            ok = wait_full(m);
            if (ok && lane == 0) mbar_arrive(&empty[m % NS]);
        }
        umma_commit_warp(drain);  // every product issued has completed before the tensor memory is released
        __syncwarp();
        wait_soon(drain, 0);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 256 * QT);
    }
}

PFN_cuTensorMapEncodeTiled_v12000 encode() {
    static std::once_flag once;
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
        else
            cudaGetLastError();
    });
    return fn;
}

template <int HD, int QT>
int launch(const AttnArgs &a, const CUtensorMap &mk, const CUtensorMap &mv, int64_t blocks, cudaStream_t st, const char *name) {
    auto kern = attn_tc_kernel<HD, QT>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(tc_smem(HD, QT))) != cudaSuccess) return check_launch(name);
    launch_k(kern, dim3(unsigned(blocks)), tc_threads(QT), tc_smem(HD, QT), st, a, mk, mv);
    return check_launch(name);
}

}  // namespace

int attn_cache_map(const vox_cuda_kv_cache &c, const void *base, int box_rows, CUtensorMap &m, const char *name) {
    auto fn = encode();
    if (!fn) return set_error(VOX_CUDA_ERR_DEVICE, std::string(name) + ": cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[4] = {cuuint64_t(c.head_dim), cuuint64_t(c.kv_heads), cuuint64_t(c.page_size), cuuint64_t(c.pages)};
    // a dimension of one element is never stepped: any stride that the encoder accepts
    const int64_t page = c.pages > 1 ? c.page_stride : c.row_stride * c.page_size, head = c.kv_heads > 1 ? c.head_stride : c.head_dim;
    const cuuint64_t strides[3] = {cuuint64_t(head) * 2, cuuint64_t(c.row_stride) * 2, cuuint64_t(page) * 2};
    const cuuint32_t box[4] = {64, 1, cuuint32_t(box_rows), 1};
    const cuuint32_t es[4] = {1, 1, 1, 1};
    // L2 fetches a head's row at a time: with 256 bytes a 64-wide head's neighbour comes too and some of it is fetched again (96
    // ragged streams of 14 heads on 2: 33.8 us and 161 MB against 32.2 at 146 MB of rows)
    const CUtensorMapL2promotion promotion = c.head_dim == 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B;
    const CUresult r = fn(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(VOX_CUDA_ERR_ARG, std::string(name) + ": cache tensor map rejected (code " + std::to_string(int(r)) + ")");
    return VOX_CUDA_OK;
}

int attn_tc_launch(const AttnArgs &a, const vox_cuda_kv_cache &c, int64_t blocks, cudaStream_t st, const char *name) {
    CUtensorMap mk, mv;
    const int qt = a.tc_half ? 1 : 2, rows = std::min(c.page_size, tc_keys(qt));  // a box never leaves a page
    int rc = attn_cache_map(c, c.k, rows, mk, name);
    if (rc == VOX_CUDA_OK) rc = attn_cache_map(c, c.v, rows, mv, name);
    if (rc != VOX_CUDA_OK) return rc;
    if (c.head_dim == 64) return qt == 1 ? launch<64, 1>(a, mk, mv, blocks, st, name) : launch<64, 2>(a, mk, mv, blocks, st, name);
    return qt == 1 ? launch<128, 1>(a, mk, mv, blocks, st, name) : launch<128, 2>(a, mk, mv, blocks, st, name);
}

int attn_tc_device_error_word(unsigned int **word) { return device_error_word(word); }

}  // namespace voxcuda
