// C++ test of the paged-cache calls of the host seam (include/vox_gpu_cuda.hpp): two sequences append their tokens and attend,
// one call after the other on one stream, checked against a plain computation in double. Built and run by
// tests/test_cpp_paged.py on a GPU machine; prints "OK" and exits 0 when every check holds.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <string>
#include <vector>

#include "vox_gpu_cuda.hpp"

namespace {
int g_fail = 0;
#define CHECK(c)                                                               \
    do {                                                                       \
        if (!(c)) {                                                            \
            ++g_fail;                                                          \
            std::fprintf(stderr, "FAIL %s:%d: %s (%s)\n", __FILE__, __LINE__, #c, vox::gpu_cuda_stats().last_error.c_str()); \
        }                                                                      \
    } while (0)

float noise(uint32_t &s) {  // a small linear congruential generator, in [-1, 1)
    s = s * 1664525u + 1013904223u;
    return float(int32_t(s)) / 2147483648.0f;
}
template <typename T> T *up(const std::vector<T> &v) {
    T *p = static_cast<T *>(vox::gpu_cuda_alloc(v.size() * sizeof(T)));
    CHECK(p && vox::gpu_cuda_upload(p, v.data(), v.size() * sizeof(T)));
    return p;
}
}  // namespace

int main() {
    std::string err;
    if (!vox::gpu_cuda_init(0, err)) {
        std::fprintf(stderr, "%s\n", err.c_str());
        return 1;
    }
    const int H = 4, KV = 2, HD = 64, PAGE = 16, PAGES = 6, T = 5 + 3, U = H + 2 * KV;
    const int lens[2] = {5, 3};
    uint32_t seed = 1;
    std::vector<float> qkv(size_t(T) * U * HD), cs(size_t(32) * HD);
    for (auto &x : qkv) x = noise(seed);
    for (int p = 0; p < 32; ++p)
        for (int i = 0; i < HD / 2; ++i) {
            const double f = p * std::pow(1e4, -2.0 * i / HD);
            cs[(size_t(p) * HD / 2 + i) * 2] = float(std::cos(f)), cs[(size_t(p) * HD / 2 + i) * 2 + 1] = float(std::sin(f));
        }
    const std::vector<int32_t> table = {4, 1}, start = {0, 5, 8}, kv_len = {5, 3}, prefix = {2};
    const size_t cells = size_t(PAGES) * PAGE * KV * HD;
    std::vector<float> zero(cells, 0.f), pk(zero), pv(zero);
    for (size_t i = 0; i < size_t(PAGE) * KV * HD; ++i) pk[size_t(2) * PAGE * KV * HD + i] = noise(seed), pv[size_t(2) * PAGE * KV * HD + i] = noise(seed);
    float *k = up(pk), *v = up(pv), *x = up(qkv), *c = up(cs), *q = up(std::vector<float>(size_t(T) * H * HD)), *o = up(std::vector<float>(size_t(T) * H * HD));
    vox_cuda_kv_cache cache = {k, v, VOX_CUDA_F32, PAGE, PAGES, KV, HD, int64_t(PAGE) * KV * HD, int64_t(KV) * HD, HD};
    vox_cuda_kv_batch batch = {up(table), up(kv_len), up(start), 1, T, 2, 1, 5, 5};
    CHECK(vox::gpu_kv_append(cache, batch, x, nullptr, nullptr, c, 32, q, H, 1e-6f));
    // the rotated heads in double
    auto rot = [&](int t, int h, int pos, int e) {
        const float *p = &qkv[(size_t(t) * U + h) * HD];
        const int i = e % (HD / 2);
        const double a = p[i], b = p[i + HD / 2], co = cs[(size_t(pos) * HD / 2 + i) * 2], si = cs[(size_t(pos) * HD / 2 + i) * 2 + 1];
        return e < HD / 2 ? a * co - b * si : b * co + a * si;
    };
    for (int with = 0; with < 2; ++with) {  // without and with the shared prefix of 10 rows
        const int np = with ? 10 : 0;
        size_t bytes = 0;
        CHECK(vox::gpu_attn_workspace(cache, batch, np, H, 0, VOX_CUDA_F32, &bytes));
        void *ws = bytes ? vox::gpu_cuda_alloc(bytes) : nullptr;
        if (with)
            CHECK(vox::gpu_attn_prefix(cache, batch, up(prefix), np, q, o, H, 0.125f, ws, bytes));
        else
            CHECK(vox::gpu_attn_paged(cache, batch, q, o, H, 0.125f, 0, ws, bytes));
        std::vector<float> got(size_t(T) * H * HD);
        CHECK(vox::gpu_cuda_download(got.data(), o, got.size() * 4) && vox::gpu_cuda_sync());
        double worst = 0;
        for (int b = 0, t0 = 0; b < 2; t0 += lens[b++])
            for (int i = 0; i < lens[b]; ++i)
                for (int h = 0; h < H; ++h) {
                    const int g = h / (H / KV);
                    std::vector<double> w;
                    double sum = 0;
                    for (int j = 0; j < np + i + 1; ++j) {
                        double s = 0;
                        for (int e = 0; e < HD; ++e) {
                            const double key = j < np ? pk[((size_t(2) * PAGE + j) * KV + g) * HD + e] : rot(t0 + j - np, H + g, j - np, e);
                            s += rot(t0 + i, h, i, e) * key;
                        }
                        w.push_back(std::exp(s * 0.125));
                        sum += w.back();
                    }
                    for (int e = 0; e < HD; ++e) {
                        double want = 0;
                        for (int j = 0; j < np + i + 1; ++j)
                            want += w[j] / sum * (j < np ? pv[((size_t(2) * PAGE + j) * KV + g) * HD + e] : qkv[(size_t(t0 + j - np) * U + H + KV + g) * HD + e]);
                        worst = std::fmax(worst, std::fabs(want - got[(size_t(t0 + i) * H + h) * HD + e]));
                    }
                }
        CHECK(worst < 1e-5);  // f32: scores of size 1, 18 keys at most
        vox::gpu_cuda_free(ws);
    }
    // a refusal comes back as false with its message
    cache.page_size = 24;
    CHECK(!vox::gpu_attn_paged(cache, batch, q, o, H, 0.125f, 0, nullptr, 0));
    if (vox::gpu_cuda_stats().last_error.find("page_size") == std::string::npos) ++g_fail;
    if (g_fail == 0) std::printf("OK\n");
    return g_fail != 0;
}
