// kv_weigh.hip - the attention weight that every cached position gets from a batch's new tokens, over the paged 4-bit cache
// (fns_kv.hpp), MI355X gfx950:
//   w[j] = past[j] + sum over the rows (tokens, heads of the group) that see j of exp(x_j - lse),  x_j = scale * q . K_j.
// The product is attention's first one (fns_attn.hpp: K as it is held against the queries' digits, here always as many as f32
// needs) with the operands exchanged: a lane has four rows of one key, and the sum over rows stays in it. Scores start at -lse,
// so that they come as exponents.
#include "fns_attn.hpp"

namespace fns {

namespace {

constexpr int kRowTile = 16;

// Sixteen rows as the product takes them.
template <int D> struct RowImage {
    using Q = QueryShape<D, float>;
    uint2 digit[Q::N][Q::kSteps][64][3];
    int scale[kRowTile];    // block scale of digit 0
    float start[kRowTile];  // -lse in log2 units; -infinity: the row adds nothing
    int from[kRowTile], to[kRowTile], tok[kRowTile];  // Sight
    int any[4];             // the largest `from`, the least `to`, the least `from`, the last position that any row sees
};

struct WeighArgs {
    AttnArgs a;  // cache, batch, q, heads, window, tree
    const float *lse, *past;
    float *weights;
    void *rows;          // RowImage [n_seq * n_kv][row_tiles]
    int64_t row_tiles;
};

template <int D, class T> __global__ __launch_bounds__(64) void k_weigh_rows(WeighArgs x) {
    using Q = QueryShape<D, float>;
    const AttnArgs &a = x.a;
    const int s = blockIdx.x / a.c.n_kv, head = blockIdx.x % a.c.n_kv, lane = threadIdx.x, r = lane % 16, g = lane / 16;
    const SeqRange sr = seq_range(a.b, s);
    const int rows = (int) min((int64_t) sr.n * a.group, (int64_t) INT32_MAX);
    const int64_t row0 = (int64_t) blockIdx.y * kRowTile;
    if (row0 >= rows) return;
    const int row = (int) row0 + r, i = row / a.group, h = head * a.group + row % a.group;
    const NewTokens<true> nt(a, sr);
    Sight<true> see = sight(a, sr, nt, row < rows, i);
    const int64_t tok = sr.q0 + i;
    const float lse = row < rows ? x.lse[tok * a.n_head + h] : INFINITY;
    bool on = fabsf(lse) < INFINITY;
    Digits<D, float> w;
    int scale = query_digits<D, float>(w, (const T *) a.q + tok * a.q_stride + (int64_t) h * D, on, a.scale);
    on = on && scale != 255;
    RowImage<D> &o = ((RowImage<D> *) x.rows)[blockIdx.x * x.row_tiles + blockIdx.y];
#pragma unroll
    for (int n = 0; n < Q::N; ++n)
#pragma unroll
        for (int u = 0; u < Q::kSteps; ++u)
#pragma unroll
            for (int k = 0; k < 3; ++k) o.digit[n][u][lane][k] = on ? make_uint2(w[n][u][2 * k], w[n][u][2 * k + 1]) : make_uint2(0, 0);
    if (!on) see = {-1, INT32_MAX, -1};
    const int last = !on ? -1 : see.tok >= 0 ? sr.len - 1 : see.to;
    int hi = see.from, lo = see.to, least = on ? see.from : INT32_MAX, most = last;
#pragma unroll
    for (int o2 = 1; o2 < 16; o2 *= 2) {
        hi = max(hi, __shfl_xor(hi, o2, 64)), lo = min(lo, __shfl_xor(lo, o2, 64));
        least = min(least, __shfl_xor(least, o2, 64)), most = max(most, __shfl_xor(most, o2, 64));
    }
    if (g == 0) {
        o.scale[r] = on ? scale : 127, o.start[r] = on ? -lse * kLog2e : -INFINITY;
        o.from[r] = see.from, o.to[r] = see.to, o.tok[r] = see.tok;
        if (r == 0) o.any[0] = hi, o.any[1] = lo, o.any[2] = least, o.any[3] = most;
    }
}

template <int SEL> __device__ __forceinline__ f4 row_mfma(i8v q, i8v k, f4 acc, int qsc, int ksc) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(q, k, acc, 2, 4, SEL, qsc, 0, ksc);
}

// A wave: 64 keys, all rows of the sequence.
template <int D> __global__ __launch_bounds__(256) void k_weigh(WeighArgs x) {
    constexpr int KP = kKPieces<D>;
    using Q = QueryShape<D, float>;
    using L = KvParts<D>;
    const AttnArgs &a = x.a;
    const int s = blockIdx.y / a.c.n_kv, head = blockIdx.y % a.c.n_kv, wave = threadIdx.x / 64, lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
    const SeqRange sr = seq_range(a.b, s);
    const int rows = (int) min((int64_t) sr.n * a.group, (int64_t) INT32_MAX);
    if (rows == 0) return;
    // (rows behind max_q tokens have no image)
    const int tiles = (int) min((int64_t) (rows - 1) / kRowTile + 1, x.row_tiles), P = 1 << a.c.shift, first = sr.len - sr.n;
    const int len = (int) min((int64_t) sr.len, a.b.table_stride << a.c.shift);
    const NewTokens<true> nt(a, sr);
    const RowImage<D> *images = (const RowImage<D> *) x.rows + blockIdx.y * x.row_tiles;
    for (int64_t b0 = ((int64_t) blockIdx.x * 4 + wave) * 64; b0 < len; b0 += (int64_t) gridDim.x * 256) {
        const int base = (int) b0;
        i8v k[4][KP];
        int ksc[4][KP];
        bool good[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int pos = base + 16 * t + r, page = pos >= 0 && pos < len ? page_of(a.c, a.b, s, pos) : -1, row = pos & (P - 1);
            const uint8_t *p = a.c.pages + max(page, 0) * a.c.page_bytes + head * kv_head_bytes(D, P);
            int nan = 0;
#pragma unroll
            for (int u = 0; u < KP; ++u) {
                const int block = (D == 64 ? g & 1 : g) + 4 * u;
                u4 v = {};
                int e = 0;
                if (page >= 0) v = *(const u4 *) (p + L::k_row(P, row) + block * 16), e = p[L::k_scale(P, row) + block];
                nan |= e == 255;
                k[t][u] = i8v{(int) v[0], (int) v[1], (int) v[2], (int) v[3], 0, 0, 0, 0};
                ksc[t][u] = e;
            }
            nan |= xor_lane_i<16>(nan);
            nan |= xor_lane_i<32>(nan);
            good[t] = page >= 0 && !nan;
        }
        float sum[4] = {};
        for (int i = 0; i < tiles; ++i) {
            const RowImage<D> &im = images[i];
            if (im.any[3] < base || im.any[2] >= base + 63) continue;
            DigitScales<D, float> qsc;
            qsc.set(im.scale[r]);
            const f4 start = *(const f4 *) (im.start + 4 * g);
            f4 acc[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[t] = start;
#pragma unroll
            for (int n = 0; n < Q::N; ++n)
#pragma unroll
                for (int u = 0; u < Q::kSteps; ++u) {
                    const uint2 *d = im.digit[n][u][lane];
                    const i8v q = {(int) d[0].x, (int) d[0].y, (int) d[1].x, (int) d[1].y, (int) d[2].x, (int) d[2].y, 0, 0};
                    const int w = qsc.w[n / 4];
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        acc[t] = n % 4 == 0 ? row_mfma<0>(q, k[t][u], acc[t], w, ksc[t][u]) : n % 4 == 1 ? row_mfma<1>(q, k[t][u], acc[t], w, ksc[t][u]) :
                                 n % 4 == 2 ? row_mfma<2>(q, k[t][u], acc[t], w, ksc[t][u]) : row_mfma<3>(q, k[t][u], acc[t], w, ksc[t][u]);
                }
            if (im.any[0] >= base || im.any[1] < base + 63) {  // some row does not see all of the keys
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const int row = 4 * g + v;
                    const int from = im.from[row], to = im.to[row], tok = im.tok[row];
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const int pos = base + 16 * t + r, j = pos - first;
                        bool on = pos > from && pos <= to;
                        if (tok >= 0 && j >= 0 && j / 64 < nt.words) on = nt.sees[(int64_t) tok * nt.words + j / 64] >> (j % 64) & 1;
                        acc[t][v] = on ? acc[t][v] : -INFINITY;
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int v = 0; v < 4; ++v) sum[t] += __builtin_amdgcn_exp2f(acc[t][v]);
        }
        float mine = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            float v = sum[t];
            v += xor_lane<16>(v);
            v += xor_lane<32>(v);
            mine = g == t ? (good[t] ? v : 0.0f) : mine;
        }
        const int pos = base + lane, page = pos < len ? page_of(a.c, a.b, s, pos) : -1;
        if (page >= 0) {
            const int64_t at = (((int64_t) page * a.c.n_kv + head) << a.c.shift) + (pos & (P - 1));
            x.weights[at] = (x.past && pos < first ? x.past[at] : 0.0f) + mine;
        }
    }
}

struct WeighPlan {
    int64_t row_tiles;
    size_t bytes;
};
size_t image_bytes(int D) { return D == 64 ? sizeof(RowImage<64>) : D == 128 ? sizeof(RowImage<128>) : sizeof(RowImage<256>); }
WeighPlan weigh_plan(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x) {
    WeighPlan p{};
    const int64_t rows = std::min<int64_t>(b->max_q, b->n_tok) * (x->n_head / c->n_head_kv);
    p.row_tiles = (rows + kRowTile - 1) / kRowTile;
    p.bytes = (size_t) ((int64_t) b->n_seq * c->n_head_kv * p.row_tiles) * image_bytes(c->head_dim);
    return p;
}

int weigh_check(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x) {
    if (!x) return host::set_error(host::ERR_SHAPE, "kv_weigh: null arguments");
    FnsAttn y = *x;
    if (c) y.out_stride = (int64_t) x->n_head * c->head_dim;  // (there is no output)
    return host::attn_check(c, b, &y, "kv_weigh");
}

}  // namespace

namespace impl {

int kv_weigh_workspace(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x, size_t *bytes) {
    FNS_TRY(weigh_check(c, b, x));
    if (!bytes) return host::set_error(host::ERR_SHAPE, "kv_weigh_workspace: null output");
    *bytes = weigh_plan(c, b, x).bytes;
    return host::OK;
}

int kv_weigh(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x, const FnsKvTree *t, const void *q, const float *lse,
             const float *past, float *weights, void *ws, size_t ws_bytes, hipStream_t st) {
    FNS_TRY(weigh_check(c, b, x));
    if (t && (t->words < 1 || t->words > 16)) return host::set_error(host::ERR_SHAPE, "kv_weigh: words must be 1..16 (%d)", t->words);
    if (b->n_seq == 0 || b->n_tok == 0 || b->max_q == 0) return host::OK;
    if (!q || !lse || !weights || (t && !t->sees)) return host::set_error(host::ERR_SHAPE, "kv_weigh: null argument");
    const WeighPlan p = weigh_plan(c, b, x);
    if (p.row_tiles > 65535) return host::set_error(host::ERR_SHAPE, "kv_weigh: %d tokens of a sequence in one call are too many", b->max_q);
    if (!ws || ws_bytes < p.bytes || ((uintptr_t) ws & 15))
        return host::set_error(host::ERR_NOMEM, "kv_weigh: workspace of %zu bytes, %zu needed (16-byte aligned)", ws ? ws_bytes : 0, p.bytes);
    WeighArgs w{};
    w.a.c = host::kv_view(c), w.a.b = host::kv_batch(b), w.a.q = q, w.a.q_stride = x->q_stride, w.a.n_head = x->n_head;
    w.a.group = x->n_head / c->n_head_kv, w.a.window = x->window, w.a.scale = x->scale;
    w.a.sees = t ? t->sees : nullptr, w.a.words = t ? t->words : 0;
    w.lse = lse, w.past = past, w.weights = weights, w.rows = ws, w.row_tiles = p.row_tiles;
    const unsigned heads = (unsigned) (b->n_seq * c->n_head_kv);
    const int64_t blocks = std::max<int64_t>(1, (b->max_kv + 255) / 256);
    const auto go = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        const dim3 rows(heads, (unsigned) p.row_tiles);
        if (x->dtype == FNS_TYPE_F32) hipLaunchKernelGGL((k_weigh_rows<D, float>), rows, dim3(64), 0, st, w);
        else hipLaunchKernelGGL((k_weigh_rows<D, uint16_t>), rows, dim3(64), 0, st, w);
        FNS_TRY(host::check_launch("kv_weigh"));
        hipLaunchKernelGGL((k_weigh<D>), dim3((unsigned) std::min<int64_t>(blocks, 1 << 20), heads), dim3(256), 0, st, w);
        return host::check_launch("kv_weigh");
    };
    if (c->head_dim == 64) return go(std::integral_constant<int, 64>{});
    if (c->head_dim == 128) return go(std::integral_constant<int, 128>{});
    return go(std::integral_constant<int, 256>{});
}

}  // namespace impl

namespace k {
void kv_weigh(const FnsKvCache &cache, const FnsKvBatch &batch, const FnsAttn &x, const FnsKvTree *tree, const void *q,
              const float *lse, const float *past, float *weights, void *ws, size_t ws_bytes, hipStream_t st) {
    host::abort_on_error(impl::kv_weigh(&cache, &batch, &x, tree, q, lse, past, weights, ws, ws_bytes, st), "kv_weigh");
}
}  // namespace k

}  // namespace fns
