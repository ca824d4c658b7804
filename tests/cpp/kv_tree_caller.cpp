// kv_tree_caller.cpp - a C++ caller of the trees and bounded caches of include/fns/kernels.h: a prompt, a tree of drafted tokens
// planned, appended by positions of its own and attended to, the weights of the cached positions, the accepted path kept and the
// cache cut; what comes back is checked against plain loops in 64 bits over what the cache holds. Built by tests/cpp/Makefile with
// hipcc; run by tests/test_gpu_kv_tree_cpp.py on the GPU. Prints "KV_TREE_CALLER_OK" and exits 0 when every check passes.
#include <hip/hip_runtime.h>

#include <algorithm>
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

constexpr int D = 64, HK = 2, H = 4, PAGE = 16, PAGES = 4, OLD = 30, NEW = 6, ALL = OLD + NEW, W = (H + 2 * HK) * D;
constexpr double kHalf = 5.97e-8;  // a half step of f32

uint64_t seed = 1;
std::vector<float> gauss(size_t n) {
    std::vector<float> v(n);
    for (auto &x : v) {
        double s = 0;
        for (int i = 0; i < 12; ++i) seed = seed * 6364136223846793005ull + 1442695040888963407ull, s += (double) (seed >> 11) / 9007199254740992.0;
        x = (float) (s - 6.0);
    }
    return v;
}

FnsKvBatch batch(int n, int len, const int32_t *table) {
    return {1, n, n, len, PAGES, dev(std::vector<int32_t>{0, n}), dev(std::vector<int32_t>{len}), table};
}

}  // namespace

int main() {
    const int32_t *table = dev(std::vector<int32_t>{3, 0, 2, 1});
    uint8_t *pages = dev(std::vector<uint8_t>(PAGES * fns_hip_kv_page_bytes(HK, D, PAGE), 255));
    const FnsKvCache cache{HK, D, PAGE, PAGES, pages};
    float *rows = dev(gauss((size_t) ALL * W)), *q_out = dev(std::vector<float>((size_t) NEW * H * D));
    int bad = 0;
    const auto read = [&](int len, std::vector<float> &k, std::vector<float> &v) {  // every position's
        float *dk = dev(std::vector<float>((size_t) len * HK * D)), *dv = dev(std::vector<float>((size_t) len * HK * D));
        fns::k::kv_read(cache, batch(len, len, table), dk, dv, nullptr);
        k = host(dk, (size_t) len * HK * D), v = host(dv, (size_t) len * HK * D);
    };
    // a prompt, then a tree: 0 and 1 follow it, 2 and 3 follow 0, 4 follows 2, 5 is none of it
    std::vector<float> freq(D / 2);
    float magnitude = 0;
    if (fns_hip_rope_scaled(D, 10000.0, 4.0, 16.0, 32.0, 1.0, freq.data(), &magnitude) != 0) return 3;
    bad += !(std::fabs(magnitude - (0.1 * std::log(4.0) + 1.0)) <= magnitude * kHalf);
    FnsKvAppend app{};
    app.dtype = FNS_TYPE_F32, app.rope = FNS_ROPE_NONE;  // (no queries)
    app.k = rows + H * D, app.v = rows + (H + HK) * D, app.k_stride = app.v_stride = app.q_stride = W, app.q_out_stride = H * D;
    fns::k::kv_append(cache, batch(OLD, OLD, table), app, nullptr);
    const FnsKvBatch b = batch(NEW, ALL, table);
    uint64_t *sees = dev(std::vector<uint64_t>(NEW));
    int32_t *pos = dev(std::vector<int32_t>(NEW));
    fns::k::tree_plan(b, dev(std::vector<int32_t>{-1, -1, 0, 0, 2, -2}), nullptr, 1, sees, pos, nullptr);
    const std::vector<uint64_t> bits = {1, 2, 5, 9, 21, 0};
    const std::vector<int32_t> at = {30, 30, 31, 31, 32, 30};
    bad += host(sees, NEW) != bits, bad += host(pos, NEW) != at;
    app.n_head = H, app.rope = FNS_ROPE_HALVES, app.rope_dim = D, app.inv_freq = dev(freq), app.q_out = q_out;
    app.q = rows + (size_t) OLD * W, app.k = rows + (size_t) OLD * W + H * D, app.v = rows + (size_t) OLD * W + (H + HK) * D;
    fns::k::kv_append_at(cache, b, app, pos, magnitude, nullptr);
    const auto in = host(rows, (size_t) ALL * W), q = host(q_out, (size_t) NEW * H * D);
    for (int t = 0; t < NEW; ++t)
        for (int h = 0; h < H; ++h)
            for (int i = 0; i < D / 2; ++i) {
                const float *x = &in[(size_t) (OLD + t) * W + h * D], *y = &q[((size_t) t * H + h) * D];
                const double c = std::cos((double) at[t] * freq[i]), s = std::sin((double) at[t] * freq[i]), m = magnitude;
                // the cosine, the sine, the magnitude on them, two products and their sum: under 8 half steps of either term
                const double tol = 8 * kHalf * m * (std::fabs(x[i]) + std::fabs(x[i + D / 2]));
                bad += !(std::fabs(y[i] - m * (x[i] * c - x[i + D / 2] * s)) <= tol);
                bad += !(std::fabs(y[i + D / 2] - m * (x[i] * s + x[i + D / 2] * c)) <= tol);
            }
    // attention, its denominators, and the weights of what is held
    FnsAttn att{};
    att.dtype = FNS_TYPE_F32, att.n_head = H, att.scale = 0.125f, att.q_stride = att.out_stride = H * D;
    const FnsKvTree tree{sees, 1};
    size_t n1 = 0, n2 = 0;
    if (fns_hip_attn_tree_workspace(&cache, &b, &att, &n1) != 0 || fns_hip_kv_weigh_workspace(&cache, &b, &att, &n2) != 0) return 4;
    void *ws = nullptr;
    HIPCHK(hipMalloc(&ws, std::max(n1, n2) + 16));
    float *out = dev(std::vector<float>((size_t) NEW * H * D, 9.0f)), *lse = dev(std::vector<float>((size_t) NEW * H, 9.0f));
    float *weights = dev(std::vector<float>((size_t) PAGES * HK * PAGE));
    fns::k::attn_tree(cache, b, att, &tree, q_out, out, lse, ws, n1, nullptr);
    fns::k::kv_weigh(cache, b, att, &tree, q_out, lse, nullptr, weights, ws, n2, nullptr);
    std::vector<float> k, v;
    read(ALL, k, v);
    const auto got = host(out, (size_t) NEW * H * D), den = host(lse, (size_t) NEW * H), given = host(weights, (size_t) PAGES * HK * PAGE);
    const auto htable = host(table, PAGES);
    const auto place = [&](int head, int p) { return ((size_t) htable[p / PAGE] * HK + head) * PAGE + p % PAGE; };
    std::vector<double> w((size_t) HK * ALL), wtol((size_t) HK * ALL);
    for (int t = 0; t < NEW; ++t)
        for (int h = 0; h < H; ++h) {
            const int hk = h / (H / HK);
            const float *x = &q[((size_t) t * H + h) * D];
            std::vector<double> p(ALL, -INFINITY);
            double top = -INFINITY, total = 0, off = 0, vmax = 0, qmax = 0;
            for (int i = 0; i < D; ++i) qmax = std::fmax(qmax, std::fabs((double) x[i]));
            for (int j = 0; j < ALL; ++j) {
                if (bits[t] == 0 || (j >= OLD && !(bits[t] >> (j - OLD) & 1))) continue;
                double d = 0, a = 0, s = 0;
                for (int i = 0; i < D; ++i) {
                    const double kk = k[((size_t) j * HK + hk) * D + i];
                    d += x[i] * kk, a += std::fabs(x[i] * kk), s += std::fabs(kk);
                    vmax = std::fmax(vmax, std::fabs((double) v[((size_t) j * HK + hk) * D + i]));
                }
                p[j] = 0.125 * d, top = std::fmax(top, p[j]);
                // a score's D + 14 half steps, and q within 2^-24 of its row's largest magnitude
                off = std::fmax(off, 0.125 * (a * (D + 14) + s * qmax) * kHalf);
            }
            if (bits[t] == 0) {
                bad += !(den[(size_t) t * H + h] == -INFINITY);
                for (int i = 0; i < D; ++i) bad += got[((size_t) t * H + h) * D + i] != 0.0f;
                continue;
            }
            for (auto z : p) total += std::exp(z - top);
            const double ref = top + std::log(total);
            // the scores, p in 22 bits and sums of ALL keys and 4 half steps, the maximum's and the logarithm's, the result's rounding
            const double ltol = off + 4.8e-7 + (ALL + 4) * kHalf + 4 * kHalf * (std::fabs(top) + std::fabs(std::log(total)) + std::fabs(ref));
            bad += !(std::fabs(den[(size_t) t * H + h] - ref) <= ltol);
            for (int j = 0; j < ALL; ++j) {
                const double e = std::exp(p[j] - ref);
                w[(size_t) hk * ALL + j] += e, wtol[(size_t) hk * ALL + j] += 1.01 * e * (off + ltol + 4 * kHalf * std::fabs(ref) + (2 * NEW + 4) * kHalf);
            }
            for (int i = 0; i < D; ++i) {
                double o = 0;
                for (int j = 0; j < ALL; ++j) o += std::exp(p[j] - ref) * v[((size_t) j * HK + hk) * D + i];
                const double tol = 2 * vmax * (off + 4.8e-7 + (ALL + 4) * kHalf) + 4 * std::fabs(o) * kHalf;
                bad += !(std::fabs(got[((size_t) t * H + h) * D + i] - o) <= tol);
            }
        }
    for (int hk = 0; hk < HK; ++hk)
        for (int j = 0; j < ALL; ++j) bad += !(std::fabs(given[place(hk, j)] - w[(size_t) hk * ALL + j]) <= wtol[(size_t) hk * ALL + j]);
    // the path 0, 2, 4 is accepted
    int32_t *new_len = dev(std::vector<int32_t>{0});
    FnsKvKeep keep{dev(std::vector<int32_t>{0, 2, 4}), dev(std::vector<int32_t>{3}), 3, weights, new_len};
    fns::k::kv_keep(cache, b, keep, nullptr);
    constexpr int LEN = OLD + 3;
    bad += host(new_len, 1)[0] != LEN;
    std::vector<float> k2, v2;
    read(LEN, k2, v2);
    const auto kept_w = host(weights, (size_t) PAGES * HK * PAGE);
    const auto source = [&](int p) { return p < OLD ? p : OLD + 2 * (p - OLD); };
    for (int p = 0; p < LEN; ++p)
        for (int hk = 0; hk < HK; ++hk) {
            for (int i = 0; i < D; ++i) {
                const size_t to = ((size_t) p * HK + hk) * D + i, from = ((size_t) source(p) * HK + hk) * D + i;
                bad += k2[to] != k[from], bad += v2[to] != v[from];
            }
            bad += kept_w[place(hk, p)] != given[place(hk, source(p))];
        }
    // and the cache cut to 20 positions a head
    constexpr int BUDGET = 20, FIRST = 2, RECENT = 5;
    const FnsKvBatch whole = batch(1, LEN, table);
    size_t n3 = 9;
    if (fns_hip_kv_evict_workspace(&cache, &whole, &n3) != 0 || n3 != 0) return 5;
    FnsKvEvict cut{};
    cut.budget = BUDGET, cut.first = FIRST, cut.recent = RECENT, cut.weights = cut.weights_out = weights, cut.new_len = new_len;
    cut.kept = dev(std::vector<int32_t>(HK * BUDGET));
    fns::k::kv_evict(cache, whole, cut, nullptr);
    bad += host(new_len, 1)[0] != BUDGET;
    std::vector<float> k3, v3;
    read(BUDGET, k3, v3);
    const auto kept = host(cut.kept, HK * BUDGET);
    const auto cut_w = host(weights, (size_t) PAGES * HK * PAGE);
    for (int hk = 0; hk < HK; ++hk) {
        std::vector<int> order(LEN);
        for (int i = 0; i < LEN; ++i) order[i] = i;
        const auto weight = [&](int p) { return p < FIRST || p >= LEN - RECENT ? INFINITY : kept_w[place(hk, p)]; };
        std::stable_sort(order.begin(), order.end(), [&](int x, int y) { return weight(x) > weight(y); });
        std::sort(order.begin(), order.begin() + BUDGET);
        for (int p = 0; p < BUDGET; ++p) {
            bad += kept[hk * BUDGET + p] != order[p], bad += cut_w[place(hk, p)] != kept_w[place(hk, order[p])];
            for (int i = 0; i < D; ++i) {
                const size_t to = ((size_t) p * HK + hk) * D + i, from = ((size_t) order[p] * HK + hk) * D + i;
                bad += k3[to] != k2[from], bad += v3[to] != v2[from];
            }
        }
    }
    if (bad) return std::printf("%d values off\n", bad), 1;
    std::printf("KV_TREE_CALLER_OK\n");
    return 0;
}
