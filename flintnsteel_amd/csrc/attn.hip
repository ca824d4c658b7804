// attn.hip - grouped-query attention of a batch's new tokens over the paged 4-bit cache (fns_kv.hpp), MI355X gfx950.
//
//   out[t][h] = sum_j p_j V_j,  p_j = exp(x_j - m) / (sum_j exp(x_j - m) + exp(sink_h - m)),  x_j = scale * q[t][h] . K_j
// over the positions j <= pos(t) (and > pos(t) - window) of the token's sequence, m the largest of x_j and sink_h. A row
// that sees nothing is zero; one that sees a token whose K or V holds a NaN block is NaN.
#include "fns_kv.hpp"

#include "fns/kernels.h"
#include "fns_common.hpp"
#include "fns_host.hpp"
#include "fns_internal.hpp"

namespace fns {

using namespace fns::dev;

namespace {

struct AttnArgs {
    KvView c;
    BatchView b;
    const void *q;
    void *out;
    const float *sinks;
    int64_t q_stride, out_stride;
    int n_head, window;
    float scale;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(uint16_t x) { return __builtin_bit_cast(float, (uint32_t) x << 16); }
__device__ __forceinline__ void put(float *p, float x) { *p = x; }
__device__ __forceinline__ void put(uint16_t *p, float x) {  // bf16: nearest, ties to even; NaN stays NaN
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    *p = (uint16_t) ((u & 0x7fffffffu) > 0x7f800000u ? (u >> 16) | 0x40u : (u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

// One wave per (token, query head): a lane a key for the scores, a lane a byte column (or two) for the values.
template <int D, class T>
__global__ __launch_bounds__(64) void k_attn(AttnArgs a) {
    __shared__ float qs[D], ps[64];
    const int s = blockIdx.z, h = blockIdx.y, i = blockIdx.x, lane = threadIdx.x;
    const SeqRange r = seq_range(a.b, s);
    if (i >= r.n) return;
    const int64_t tok = r.q0 + i;
    const int head = h / (a.n_head / a.c.n_kv), pos = r.len - r.n + i, P = 1 << a.c.shift;
    const int lo = a.window ? max(0, pos - a.window + 1) : 0;
    using L = KvParts<D>;
    constexpr int NC = D / 2;  // byte columns
    for (int d = lane; d < D; d += 64) qs[d] = to_f32(((const T *) a.q)[tok * a.q_stride + (int64_t) h * D + d]) * a.scale;
    __syncthreads();
    float m = a.sinks ? a.sinks[h] : -INFINITY, l = a.sinks ? 1.0f : 0.0f;
    float acc[2][2] = {};
    // positions behind the table have no page; whole tiles, so that no position passes 31 bits
    const int end = (int) min((int64_t) pos + 1, a.b.table_stride << a.c.shift);
    for (int tile = lo / 64; tile < end / 64 + (end % 64 > 0); ++tile) {
        const int base = tile * 64;
        const int key = base + lane, page = key >= lo && key <= pos ? page_of(a.c, a.b, s, key) : -1;
        const uint8_t *src = a.c.pages + (int64_t) max(page, 0) * a.c.page_bytes + head * kv_head_bytes(D, P);
        const int row = key & (P - 1);
        float x = -INFINITY;
        if (page >= 0) {
            x = 0.0f;
            for (int c = 0; c < NC; ++c) {
                const int e = src[L::k_scale(P, row) + c / 16], b = src[L::k_row(P, row) + c];
                x += qs[2 * c] * kv_value(b & 15, e) + qs[2 * c + 1] * kv_value(b >> 4, e);
            }
            for (int c = 0; c < D / 32; ++c)
                if (src[L::v_scale(P, row) + c] == 255) x = __builtin_nanf("");
        }
        const float mt = fmaxf(m, lanes_max<64>(x));
        const float p = page >= 0 ? expf(x - mt) : 0.0f, f = m > -INFINITY ? expf(m - mt) : 0.0f;
        l = l * f + lanes_sum<64>(p);
        m = mt;
        ps[lane] = p;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 2; ++u) acc[u][0] *= f, acc[u][1] *= f;
        for (int j = 0; j < 64; ++j) {
            const int pg = __shfl(page, j);
            if (pg < 0) continue;
            const uint8_t *vs = a.c.pages + (int64_t) pg * a.c.page_bytes + head * kv_head_bytes(D, P);
            const int vr = (base + j) & (P - 1);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int c = lane + 64 * u;
                if (c >= NC) continue;
                const int b = vs[L::v_col(P, c) + vr], e = vs[L::v_scale(P, vr) + c / 16];
                acc[u][0] += ps[j] * kv_value(b & 15, e);
                acc[u][1] += ps[j] * kv_value(b >> 4, e);
            }
        }
        __syncthreads();
    }
    T *o = (T *) a.out + tok * a.out_stride + (int64_t) h * D;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int c = lane + 64 * u;
        if (c >= NC) continue;
        put(o + c / 16 * 32 + c % 16, l == 0.0f ? 0.0f : acc[u][0] / l);
        put(o + c / 16 * 32 + c % 16 + 16, l == 0.0f ? 0.0f : acc[u][1] / l);
    }
}

}  // namespace

namespace impl {

namespace {

int attn_check(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x) {
    FNS_TRY(host::kv_check(c, b, "attn"));
    if (!x) return host::set_error(host::ERR_SHAPE, "attn: null arguments");
    if (x->dtype != FNS_TYPE_F32 && x->dtype != FNS_TYPE_BF16)
        return host::set_error(host::ERR_TYPE, "attn: type %d is not supported (0 f32, 30 bf16)", x->dtype);
    if (x->n_head <= 0 || x->n_head % c->n_head_kv || x->n_head > 65535)
        return host::set_error(host::ERR_SHAPE, "attn: n_head %d is no multiple of n_head_kv %d", x->n_head, c->n_head_kv);
    if (x->window < 0) return host::set_error(host::ERR_SHAPE, "attn: negative window");
    const int64_t w = (int64_t) x->n_head * c->head_dim;
    if (x->q_stride < w || x->out_stride < w) return host::set_error(host::ERR_SHAPE, "attn: a token stride is shorter than a token's heads");
    return host::OK;
}

}  // namespace

int attn_workspace(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x, size_t *bytes) {
    FNS_TRY(attn_check(c, b, x));
    if (!bytes) return host::set_error(host::ERR_SHAPE, "attn_workspace: null output");
    *bytes = 0;
    return host::OK;
}

int attn(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x, const void *q, void *out, void *ws, size_t ws_bytes,
         hipStream_t st) {
    FNS_TRY(attn_check(c, b, x));
    if (b->n_seq == 0 || b->n_tok == 0 || b->max_q == 0) return host::OK;
    if (!q || !out) return host::set_error(host::ERR_SHAPE, "attn: null argument");
    const AttnArgs a{host::kv_view(c), host::kv_batch(b), q, out, x->sinks, x->q_stride, x->out_stride, x->n_head, x->window, x->scale};
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3((unsigned) b->max_q, (unsigned) x->n_head, (unsigned) b->n_seq), dim3(64), 0, st, a);
    };
    const bool f32 = x->dtype == FNS_TYPE_F32;
    if (c->head_dim == 64) f32 ? go(k_attn<64, float>) : go(k_attn<64, uint16_t>);
    else if (c->head_dim == 128) f32 ? go(k_attn<128, float>) : go(k_attn<128, uint16_t>);
    else f32 ? go(k_attn<256, float>) : go(k_attn<256, uint16_t>);
    return host::check_launch("attn");
}

}  // namespace impl

namespace k {
void attn(const FnsKvCache &cache, const FnsKvBatch &batch, const FnsAttn &x, const void *q, void *out, void *ws,
          size_t ws_bytes, hipStream_t st) {
    host::abort_on_error(impl::attn(&cache, &batch, &x, q, out, ws, ws_bytes, st), "attn");
}
}  // namespace k

}  // namespace fns
