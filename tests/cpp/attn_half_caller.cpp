// attn_half_caller.cpp - a C++ caller of the attention half of include/fns/kernels.h: two sequences' tokens go through the
// residual add and norm, into the paged 4-bit cache and through attention, and what comes back is checked against plain loops
// in 64 bits over what the cache holds. Built by tests/cpp/Makefile with hipcc; run by tests/test_gpu_attn_half_cpp.py on the
// GPU. Prints "ATTN_HALF_CALLER_OK" and exits 0 when every check passes.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "fns/kernels.h"

namespace {

#define HIPCHK(x)                                                                                       \
    do {                                                                                                \
        hipError_t e_ = (x);                                                                            \
        if (e_ != hipSuccess) {                                                                         \
            std::fprintf(stderr, "HIP error %s at %s:%d\n", hipGetErrorString(e_), __FILE__, __LINE__); \
            std::exit(2);                                                                               \
        }                                                                                               \
    } while (0)

template <class T> T *dev(const std::vector<T> &h) {
    T *d = nullptr;
    HIPCHK(hipMalloc(&d, h.size() * sizeof(T)));
    HIPCHK(hipMemcpy(d, h.data(), h.size() * sizeof(T), hipMemcpyHostToDevice));
    return d;
}
template <class T> std::vector<T> host(const T *d, size_t n) {
    std::vector<T> h(n);
    HIPCHK(hipDeviceSynchronize());
    HIPCHK(hipMemcpy(h.data(), d, n * sizeof(T), hipMemcpyDeviceToHost));
    return h;
}

}  // namespace

int main() {
    constexpr int D = 64, HK = 2, H = 6, PAGE = 16, W = (H + 2 * HK) * D, TOK = 25;
    const std::vector<int32_t> q_start = {0, 20, TOK}, kv_len = {20, 5}, table = {3, 0, 2, 2};  // all tokens are new
    uint64_t seed = 1;
    auto gauss = [&](size_t n) {
        std::vector<float> v(n);
        for (auto &x : v) {
            double s = 0;
            for (int i = 0; i < 12; ++i) seed = seed * 6364136223846793005ull + 1442695040888963407ull, s += (double) (seed >> 11) / 9007199254740992.0;
            x = (float) (s - 6.0);
        }
        return v;
    };
    int bad = 0;
    // a fused projection's rows [q | k | v], their sum with another row and its norm
    const auto x = gauss((size_t) TOK * W), y = gauss((size_t) TOK * W), w = gauss(W);
    float *dx = dev(x), *dy = dev(y), *dw = dev(w), *dn = dev(x);
    uint8_t *xq = dev(std::vector<uint8_t>((size_t) TOK * 2 * W));
    fns::k::add_rms_norm_q8_1(dx, dy, dw, dx, dn, xq, W, 1e-6f, TOK, nullptr);
    const auto sum = host(dx, (size_t) TOK * W), norm = host(dn, (size_t) TOK * W);
    for (int t = 0; t < TOK; ++t) {
        double ss = 0;
        for (int i = 0; i < W; ++i) ss += (double) sum[(size_t) t * W + i] * sum[(size_t) t * W + i];
        for (int i = 0; i < W; ++i) {
            const size_t at = (size_t) t * W + i;
            const double ref = sum[at] * w[i] / std::sqrt(ss / W + 1e-6);
            // sums of 640 squares in 256 lanes and 8 steps, a root, a division and two products: under 32 half steps
            bad += !(sum[at] == x[at] + y[at]) + !(std::fabs(norm[at] - ref) <= std::fabs(ref) * 32 * 5.97e-8);
        }
    }
    // the cache
    const size_t page_bytes = fns_hip_kv_page_bytes(HK, D, PAGE);
    uint8_t *pages = dev(std::vector<uint8_t>(4 * page_bytes, 255));
    const FnsKvCache cache{HK, D, PAGE, 4, pages};
    const FnsKvBatch batch{2, 20, TOK, 20, 2, dev(q_start), dev(kv_len), dev(table)};
    FnsKvAppend app{};
    app.dtype = FNS_TYPE_F32, app.rope = FNS_ROPE_NONE, app.n_head = H;
    float *qr = dev(std::vector<float>((size_t) TOK * H * D));
    app.q = dn, app.k = dn + H * D, app.v = dn + (H + HK) * D, app.q_out = qr;
    app.q_stride = app.k_stride = app.v_stride = W, app.q_out_stride = H * D;
    fns::k::kv_append(cache, batch, app, nullptr);
    float *dk = dev(std::vector<float>((size_t) TOK * HK * D)), *dv = dev(std::vector<float>((size_t) TOK * HK * D));
    fns::k::kv_read(cache, batch, dk, dv, nullptr);
    const auto k = host(dk, (size_t) TOK * HK * D), v = host(dv, (size_t) TOK * HK * D), q = host(qr, (size_t) TOK * H * D);
    for (int t = 0; t < TOK; ++t)
        for (int b = 0; b < 2 * HK * D / 32; ++b) {  // every block within half a step of its scale: 4 to 7 units the largest
            const float *held = (b < HK * D / 32 ? k.data() : v.data()) + (size_t) t * HK * D + b % (HK * D / 32) * 32;
            const float *in = norm.data() + (size_t) t * W + H * D + b * 32;
            float top = 0;
            for (int i = 0; i < 32; ++i) top = std::fmax(top, std::fabs(in[i]));
            for (int i = 0; i < 32; ++i) bad += !(std::fabs(held[i] - in[i]) <= top / 3.5f);  // (the step from 4 to 6, and 7 to 6, is 1 of 3.5)
        }
    // attention
    FnsAttn att{};
    att.dtype = FNS_TYPE_F32, att.n_head = H, att.scale = 0.125f, att.q_stride = att.out_stride = H * D;
    size_t bytes = 0;
    if (fns_hip_attn_workspace(&cache, &batch, &att, &bytes) != 0) return 3;
    float *out = dev(std::vector<float>((size_t) TOK * H * D, 9.0f));
    void *ws = nullptr;
    HIPCHK(hipMalloc(&ws, bytes + 16));
    fns::k::attn(cache, batch, att, qr, out, ws, bytes, nullptr);
    const auto got = host(out, (size_t) TOK * H * D);
    for (int s = 0; s < 2; ++s)
        for (int t = q_start[s]; t < q_start[s + 1]; ++t)
            for (int h = 0; h < H; ++h) {
                const int hk = h / (H / HK), n = t - q_start[s] + 1;
                std::vector<double> p(n);
                double top = -1e300, total = 0, ax = 0, ak = 0, vmax = 0, qmax = 0;
                for (int i = 0; i < D; ++i) qmax = std::fmax(qmax, std::fabs((double) q[((size_t) t * H + h) * D + i]));
                for (int j = 0; j < n; ++j) {
                    double d = 0, a = 0, b = 0;
                    for (int i = 0; i < D; ++i) {
                        const double z = (double) q[((size_t) t * H + h) * D + i] * k[((size_t) (q_start[s] + j) * HK + hk) * D + i];
                        d += z, a += std::fabs(z), b += std::fabs((double) k[((size_t) (q_start[s] + j) * HK + hk) * D + i]);
                        vmax = std::fmax(vmax, std::fabs((double) v[((size_t) (q_start[s] + j) * HK + hk) * D + i]));
                    }
                    p[j] = 0.125 * d, top = std::fmax(top, p[j]), ax = std::fmax(ax, 0.125 * a), ak = std::fmax(ak, 0.125 * b);
                }
                for (auto &z : p) z = std::exp(z - top), total += z;
                for (int i = 0; i < D; ++i) {
                    double ref = 0;
                    for (int j = 0; j < n; ++j) ref += p[j] / total * v[((size_t) (q_start[s] + j) * HK + hk) * D + i];
                    // a score's D + 14 half steps, q within 2^-24 of its row's largest magnitude, p in 22 bits and sums of n
                    // keys and 4 half steps; numerator and denominator; the result's rounding
                    const double tol = 2 * vmax * (ax * (D + 14) * 5.97e-8 + ak * qmax * 5.97e-8 + 4.8e-7 + (n + 4) * 5.97e-8) +
                                       4 * std::fabs(ref) * 5.97e-8;
                    bad += !(std::fabs(got[((size_t) t * H + h) * D + i] - ref) <= tol);
                }
            }
    if (bad) return std::printf("%d values off\n", bad), 1;
    std::printf("ATTN_HALF_CALLER_OK\n");
    return 0;
}
