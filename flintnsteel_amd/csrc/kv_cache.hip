// kv_cache.hip - filling and reading back the paged 4-bit key/value cache (fns_kv.hpp), for MI355X gfx950.
//
// Append. A token of a batch brings k and v of every kv head (and its queries); its position is the sequence's length
// less the tokens after it. With a rotation, a pair of channels (a, b) of k and q becomes
//   (a cos t - b sin t, a sin t + b cos t),  t = position * inv_freq[i],
// and k and v go into the cache in 4 bits, k from the rotated value before any rounding. The rotation and the block
// arithmetic are done in 64 bits: an f32 angle of a far position is off by its spacing (4e-3 at position 65536), and a
// 4-bit code next to a border would depend on the last bit of a 32-bit rotation. The pass moves the bytes of q, k and
// v and is bound by them (and by its launch for a few tokens), not by this arithmetic.
#include "fns_kv.hpp"

#include <algorithm>

#include "fns/kernels.h"
#include "fns_common.hpp"
#include "fns_host.hpp"
#include "fns_internal.hpp"

namespace fns {

using namespace fns::dev;

namespace {

constexpr int kGroup = 16;  // positions of a workgroup: the V bytes of one column and one 16-position group are 16 bytes

struct AppendArgs {
    KvView c;
    BatchView b;
    const void *k, *v, *q;
    void *q_out;
    const float *inv_freq;
    int64_t k_stride, v_stride, q_stride, qo_stride;
    int rope_dim, n_group;  // n_group: query heads of a kv head (0: no queries)
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(uint16_t x) { return __builtin_bit_cast(float, (uint32_t) x << 16); }

__device__ __forceinline__ uint16_t to_bf16(float x) {  // nearest, ties to even; NaN stays NaN
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t) ((u >> 16) | 0x40u);
    return (uint16_t) ((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ void store8(float *p, const double (&v)[8]) {
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = (float) v[i];
    __builtin_memcpy(p, t, sizeof t);
}
__device__ __forceinline__ void store8(uint16_t *p, const double (&v)[8]) {
    uint16_t t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = to_bf16((float) v[i]);
    __builtin_memcpy(p, t, sizeof t);
}

// Channels ch .. ch + 7 of a head's row, at any alignment of an element: asked for in one place and turned in another, with
// the loads' latency between. Where halves turn against each other, the partners are another lane's of the same row.
template <class T> struct Row8 {
    T x[8];
    __device__ __forceinline__ void load(const T *p) { __builtin_memcpy(x, p, sizeof x); }
};
// After the rotation; cs: the token's (cos, sin) of every pair. All lanes of the row take part.
template <int ROPE, class T>
__device__ __forceinline__ void rotated(const Row8<T> &v, int ch, int rope_dim, const double2 *cs, double (&o)[8]) {
    const bool turns = ch < rope_dim, second = ch >= rope_dim / 2;
    if constexpr (ROPE == FNS_ROPE_PAIRS) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const double2 t = turns ? cs[(ch + i) / 2] : make_double2(1.0, 0.0);
            const double a = to_f32(v.x[i]), b = to_f32(v.x[i + 1]);
            o[i] = turns ? a * t.x - b * t.y : a;
            o[i + 1] = turns ? a * t.y + b * t.x : b;
        }
    } else if constexpr (ROPE == FNS_ROPE_HALVES) {
        const int lane = threadIdx.x % 64, other = 4 * (!turns ? lane : second ? lane - rope_dim / 16 : lane + rope_dim / 16);
        constexpr int N = sizeof(v.x) / 4;
        int w[N];
        T y[8];
        __builtin_memcpy(w, v.x, sizeof w);
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = __builtin_amdgcn_ds_bpermute(other, w[i]);
        __builtin_memcpy(y, w, sizeof w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double2 t = turns ? cs[ch + i - (second ? rope_dim / 2 : 0)] : make_double2(1.0, 0.0);
            const double a = to_f32(v.x[i]), b = to_f32(y[i]);
            o[i] = !turns ? a : second ? b * t.y + a * t.x : a * t.x - b * t.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = to_f32(v.x[i]);
    }
}

// Codes of the eight values of a lane (four lanes of a quad hold a block), 4 bits each; e: the block's scale byte. F is f32
// where the values are (its scaling and comparisons are exact: a magnitude in units of the scale that f32 would round is far
// below the first border), else f64.
template <class F> __device__ __forceinline__ uint32_t hold8(const F (&v)[8], int &e) {
    F amax = 0;
    int bad = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const F a = fabs(v[i]);
        bad |= !(a <= (sizeof(F) == 8 ? (F) 1.7976931348623157e308 : (F) 3.402823466e38f));
        amax = a > amax ? a : amax;
    }
    auto other = [](F x, auto lane) {
        constexpr int O = decltype(lane)::value;
        if constexpr (sizeof(F) == 8) {
            const uint64_t u = __builtin_bit_cast(uint64_t, x);
            const uint32_t lo = (uint32_t) xor_lane_i<O>((int) (uint32_t) u), hi = (uint32_t) xor_lane_i<O>((int) (uint32_t) (u >> 32));
            return __builtin_bit_cast(double, ((uint64_t) hi << 32) | lo);
        } else {
            return xor_lane<O>(x);
        }
    };
    amax = fmax(amax, other(amax, std::integral_constant<int, 1>{}));
    amax = fmax(amax, other(amax, std::integral_constant<int, 2>{}));
    bad |= xor_lane_i<1>(bad);
    bad |= xor_lane_i<2>(bad);
    e = bad ? 255 : kv_scale_of(amax);
    if (bad) return 0;
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= kv_code(v[i], (F) ldexp(fabs(v[i]), 127 - e)) << (4 * i);
    return w;
}

// One workgroup: the new tokens among 16 aligned positions of one sequence, one kv head and its query heads. Rows of 8
// channels a thread: 2 D threads hold the 16 rows of a head. K and V are asked for before the angles are computed, a query
// before the last one is stored, and the queries of the group's tokens are dealt to all threads: in turns by the threads of
// their rows, one token's took as long as everything else (one token, 8 kv heads of 4 queries: 8.0 us, now 5.9; 61 sequences:
// 10.0, now 5.9). Few tokens are bound by what waits for what: the range, the table entry, the row, V's columns through LDS
// (replayed, one token: 4.0 us without queries or rotation; the angles add 0.7, the queries' turn 0.7). Many by the bytes: 4001
// tokens, 168 MB in 34 us (a copy of them: 35; bf16, 86 MB: 34); there it is waves that pay, and a query's loads before the
// angles' arithmetic cost more registers than they hide (38 us).
template <int D, int ROPE, class T>
__global__ __launch_bounds__(2 * D, ROPE == FNS_ROPE_PAIRS ? 6 : 8) void k_kv_append(AppendArgs a) {
    constexpr int NT = 2 * D, NR = D / 8;
    __shared__ double2 cs[ROPE == FNS_ROPE_NONE ? 1 : kGroup * (D / 2)];
    __shared__ __align__(16) uint8_t code[D][kGroup];
    const int s = blockIdx.y / a.c.n_kv, head = blockIdx.y % a.c.n_kv, tid = threadIdx.x;
    const SeqRange r = seq_range(a.b, s);
    const int first = r.len - r.n;                                  // position of the first new token
    const int64_t start = (int64_t) (first & ~(kGroup - 1)) + (int64_t) blockIdx.x * kGroup;
    if (r.n == 0 || start >= r.len) return;
    const int base = (int) start;
    const int lo = max(first, base), hi = r.len - base < kGroup ? r.len : base + kGroup;  // [lo, hi): the tokens of this workgroup
    const int row = tid / NR, ch = tid % NR * 8, pos = base + row;
    const bool have = pos >= lo && pos < hi;
    const int64_t tok = r.q0 + (pos - first);
    const int page = page_of(a.c, a.b, s, base);  // 16 aligned positions lie in one page
    Row8<T> k8 = {}, v8 = {}, q8 = {};
    if (have) {
        k8.load((const T *) a.k + tok * a.k_stride + head * D + ch);
        v8.load((const T *) a.v + tok * a.v_stride + head * D + ch);
    }
    // Item i = row, row + 16, ... of the queries: token lo + i / n_group, head i % n_group of the group. In place too: the
    // threads of a row are lanes of one wave, whose loads all precede the stores they feed.
    const int n_group = a.n_group;
    int qp = hi, qh = 0, dp = 0, dh = 0;
    if (n_group) qp = lo + row / n_group, qh = row % n_group, dp = kGroup / n_group, dh = kGroup % n_group;
    const auto ask = [&] {
        if (qp < hi) q8.load((const T *) a.q + (r.q0 + (qp - first)) * a.q_stride + (int64_t) (head * n_group + qh) * D + ch);
    };
    if constexpr (ROPE != FNS_ROPE_NONE) {
        const int half = a.rope_dim / 2;
        for (int i = tid; i < (hi - lo) * half; i += NT) {
            const int p = lo + i / half, c = i % half;
            // in turns: the product is exact to 53 bits, its whole part leaves no error
            double turns = (double) p * (double) a.inv_freq[c] * 0.15915494309189533577;
            turns -= rint(turns);
            double sn, cn;
            sincospi(2.0 * turns, &sn, &cn);
            cs[(p - base) * (D / 2) + c] = make_double2(cn, sn);
        }
        __syncthreads();
    }
    ask();
    const auto angles = [&](int p) { return cs + (ROPE == FNS_ROPE_NONE ? 0 : (p - base) * (D / 2)); };
    const int P = 1 << a.c.shift;
    uint8_t *dst = a.c.pages + (int64_t) max(page, 0) * a.c.page_bytes + head * kv_head_bytes(D, P);
    using L = KvParts<D>;
    const bool put = have && page >= 0 && pos >= 0;
    int e;
    uint32_t w;
    if constexpr (ROPE == FNS_ROPE_NONE) {
        float k[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) k[i] = to_f32(k8.x[i]);
        w = hold8(k, e);
    } else {
        double k[8] = {};
        if (have) rotated<ROPE>(k8, ch, a.rope_dim, angles(pos), k);
        w = hold8(k, e);
    }
    if (put) {
        *(uint32_t *) (dst + L::k_row(P, pos & (P - 1)) + ch / 2) = w;
        if (ch % 32 == 0) dst[L::k_scale(P, pos & (P - 1)) + ch / 32] = (uint8_t) e;
    }
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(v8.x[i]);
    w = hold8(v, e);
    if (put && ch % 32 == 0) dst[L::v_scale(P, pos & (P - 1)) + ch / 32] = (uint8_t) e;
#pragma unroll
    for (int i = 0; i < 8; ++i) code[ch + i][row] = (uint8_t) ((w >> (4 * i)) & 15u);
    __syncthreads();
    if (page >= 0 && base >= 0) {  // byte column tid / 4, positions 4 (tid % 4) .. + 3
        const int j = tid / 4, p4 = base + tid % 4 * 4;
        const int c0 = j / 16 * 32 + j % 16;
        const uint32_t b = *(const uint32_t *) &code[c0][tid % 4 * 4] | (*(const uint32_t *) &code[c0 + 16][tid % 4 * 4] << 4);
        uint8_t *o = dst + L::v_col(P, j) + (p4 & (P - 1));
        if (p4 >= lo && p4 + 4 <= hi) {
            *(uint32_t *) o = b;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (p4 + i >= lo && p4 + i < hi) o[i] = (uint8_t) (b >> (8 * i));
        }
    }
    while (qp < hi) {
        double q[8];
        rotated<ROPE>(q8, ch, a.rope_dim, angles(qp), q);
        T *out = (T *) a.q_out + (r.q0 + (qp - first)) * a.qo_stride + (int64_t) (head * n_group + qh) * D + ch;
        qp += dp, qh += dh;
        if (qh >= n_group) qh -= n_group, ++qp;
        ask();
        store8(out, q);
    }
}

// Values of the batch's tokens as the cache holds them; NaN where a position has no page. 4001 tokens of 8 heads of 128: 11 us,
// for 33 MB written and 19.5 read; the tokens hold 4.4, but a thread takes its byte out of each of V's columns, whose lines the
// next tokens' workgroups read again. A copy of 37 MB takes 8.
template <int D>
__global__ __launch_bounds__(256) void k_kv_read(KvView c, BatchView b, float *k, float *v) {
    const int s = blockIdx.y / c.n_kv, head = blockIdx.y % c.n_kv;
    const SeqRange r = seq_range(b, s);
    const int P = 1 << c.shift;
    using L = KvParts<D>;
    const int i = blockIdx.x * (256 / (D / 4)) + threadIdx.x / (D / 4), ch = threadIdx.x % (D / 4) * 4;
    if (i >= r.n) return;
    const int pos = r.len - r.n + i, page = page_of(c, b, s, pos);
    float kv[4], vv[4];
    if (page >= 0) {
        const int row = pos & (P - 1);
        const uint8_t *src = c.pages + (int64_t) page * c.page_bytes + head * kv_head_bytes(D, P);
        const int ke = src[L::k_scale(P, row) + ch / 32], ve = src[L::v_scale(P, row) + ch / 32];
        const int kw = src[L::k_row(P, row) + ch / 2] | (src[L::k_row(P, row) + ch / 2 + 1] << 8);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            kv[t] = kv_value((kw >> (4 * t)) & 15, ke);
            const int x = ch % 32 + t;
            vv[t] = kv_value((src[L::v_col(P, ch / 32 * 16 + x % 16) + row] >> (x / 16 * 4)) & 15, ve);
        }
    } else {
#pragma unroll
        for (int t = 0; t < 4; ++t) kv[t] = vv[t] = __builtin_nanf("");
    }
    const int64_t o = ((r.q0 + i) * c.n_kv + head) * D + ch;
    __builtin_memcpy(k + o, kv, sizeof kv);
    __builtin_memcpy(v + o, vv, sizeof vv);
}

}  // namespace

namespace host {

int kv_check(const FnsKvCache *c, const FnsKvBatch *b, const char *what) {
    if (!c || !b) return set_error(ERR_SHAPE, "%s: null cache or batch", what);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return set_error(ERR_SHAPE, "%s: head_dim must be 64, 128 or 256 (%d)", what, c->head_dim);
    if (c->page_size < 16 || c->page_size > 4096 || (c->page_size & (c->page_size - 1)))
        return set_error(ERR_SHAPE, "%s: page_size must be a power of two from 16 to 4096 (%d)", what, c->page_size);
    if (c->n_head_kv <= 0 || c->n_head_kv > 1024 || c->n_pages <= 0 || c->n_pages > INT32_MAX)
        return set_error(ERR_SHAPE, "%s: n_head_kv must be 1..1024 and n_pages 1..2^31-1 (%d, %lld)", what, c->n_head_kv,
                         (long long) c->n_pages);
    if (!c->pages || ((uintptr_t) c->pages & 15)) return set_error(ERR_SHAPE, "%s: pages must be 16-byte aligned device memory", what);
    if (b->n_seq < 0 || b->n_tok < 0 || b->max_q < 0 || b->max_kv < 0 || b->table_stride < 0 || b->n_tok > INT32_MAX ||
        b->max_kv > INT32_MAX || b->table_stride > INT32_MAX)
        return set_error(ERR_SHAPE, "%s: negative or too large batch numbers (n_seq %d n_tok %lld max_q %d)", what, b->n_seq,
                         (long long) b->n_tok, b->max_q);
    if ((int64_t) b->n_seq * c->n_head_kv > 65535)
        return set_error(ERR_SHAPE, "%s: n_seq * n_head_kv must be at most 65535 (%d * %d)", what, b->n_seq, c->n_head_kv);
    if (b->n_seq > 0 && (!b->q_start || !b->kv_len || !b->page_table)) return set_error(ERR_SHAPE, "%s: null batch array", what);
    return OK;
}

}  // namespace host

namespace impl {

size_t kv_page_bytes(int n_head_kv, int head_dim, int page_size) {
    FnsKvCache c{n_head_kv, head_dim, page_size, 1, (void *) 16};
    FnsKvBatch b{};
    if (host::kv_check(&c, &b, "kv_page_bytes") != host::OK) return 0;
    return (size_t) n_head_kv * dev::kv_head_bytes(head_dim, page_size);
}

int kv_append(const FnsKvCache *c, const FnsKvBatch *b, const FnsKvAppend *x, hipStream_t st) {
    FNS_TRY(host::kv_check(c, b, "kv_append"));
    if (!x) return host::set_error(host::ERR_SHAPE, "kv_append: null arguments");
    if (x->dtype != FNS_TYPE_F32 && x->dtype != FNS_TYPE_BF16)
        return host::set_error(host::ERR_TYPE, "kv_append: type %d is not supported (0 f32, 30 bf16)", x->dtype);
    if (x->rope != FNS_ROPE_NONE && x->rope != FNS_ROPE_HALVES && x->rope != FNS_ROPE_PAIRS)
        return host::set_error(host::ERR_SHAPE, "kv_append: unknown rotation %d", x->rope);
    const int D = c->head_dim;
    // a thread rotates 8 channels, and a half's partner channels have to be 8 of the other half
    if (x->rope != FNS_ROPE_NONE && (!x->inv_freq || x->rope_dim <= 0 || x->rope_dim > D || x->rope_dim % 16))
        return host::set_error(host::ERR_SHAPE, "kv_append: a rotation needs inv_freq and a rope_dim that is a multiple of 16 up to head_dim (%d)",
                               x->rope_dim);
    if (x->n_head < 0 || x->n_head % c->n_head_kv)
        return host::set_error(host::ERR_SHAPE, "kv_append: n_head %d is no multiple of n_head_kv %d", x->n_head, c->n_head_kv);
    if (b->n_seq == 0 || b->n_tok == 0 || b->max_q == 0) return host::OK;
    if (!x->k || !x->v || (x->n_head > 0 && (!x->q || !x->q_out))) return host::set_error(host::ERR_SHAPE, "kv_append: null argument");
    const int64_t kvw = (int64_t) c->n_head_kv * D, qw = (int64_t) x->n_head * D;
    if (x->k_stride < kvw || x->v_stride < kvw || (x->n_head > 0 && (x->q_stride < qw || x->q_out_stride < qw)))
        return host::set_error(host::ERR_SHAPE, "kv_append: a token stride is shorter than a token's heads");
    if (x->n_head > 0 && x->q == x->q_out && x->q_stride != x->q_out_stride)
        return host::set_error(host::ERR_SHAPE, "kv_append: queries rotated in place keep their stride");
    AppendArgs a{host::kv_view(c), host::kv_batch(b), x->k, x->v, x->q, x->q_out, x->inv_freq, x->k_stride, x->v_stride,
                 x->q_stride, x->q_out_stride, x->rope_dim, x->n_head / c->n_head_kv};
    // new tokens of a sequence start anywhere in a group
    const int64_t most = std::min<int64_t>(b->max_q, b->n_tok);
    const dim3 grid((unsigned) ((most + kGroup - 2) / kGroup + 1), (unsigned) (b->n_seq * c->n_head_kv));
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(2 * D), 0, st, a); };
    auto by_type = [&](auto dim, auto rope) {
        constexpr int DD = decltype(dim)::value, R = decltype(rope)::value;
        if (x->dtype == FNS_TYPE_F32) go(k_kv_append<DD, R, float>);
        else go(k_kv_append<DD, R, uint16_t>);
    };
    auto by_rope = [&](auto dim) {
        if (x->rope == FNS_ROPE_NONE) by_type(dim, std::integral_constant<int, FNS_ROPE_NONE>{});
        else if (x->rope == FNS_ROPE_HALVES) by_type(dim, std::integral_constant<int, FNS_ROPE_HALVES>{});
        else by_type(dim, std::integral_constant<int, FNS_ROPE_PAIRS>{});
    };
    if (D == 64) by_rope(std::integral_constant<int, 64>{});
    else if (D == 128) by_rope(std::integral_constant<int, 128>{});
    else by_rope(std::integral_constant<int, 256>{});
    return host::check_launch("kv_append");
}

int kv_read(const FnsKvCache *c, const FnsKvBatch *b, float *k, float *v, hipStream_t st) {
    FNS_TRY(host::kv_check(c, b, "kv_read"));
    if (b->n_seq == 0 || b->n_tok == 0 || b->max_q == 0) return host::OK;
    if (!k || !v) return host::set_error(host::ERR_SHAPE, "kv_read: null output");
    const int64_t rows = 256 / (c->head_dim / 4), most = std::min<int64_t>(b->max_q, b->n_tok);
    const dim3 grid((unsigned) ((most + rows - 1) / rows), (unsigned) (b->n_seq * c->n_head_kv));
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, host::kv_view(c), host::kv_batch(b), k, v);
    };
    if (c->head_dim == 64) go(k_kv_read<64>);
    else if (c->head_dim == 128) go(k_kv_read<128>);
    else go(k_kv_read<256>);
    return host::check_launch("kv_read");
}

}  // namespace impl

namespace k {
void kv_append(const FnsKvCache &cache, const FnsKvBatch &batch, const FnsKvAppend &x, hipStream_t st) {
    host::abort_on_error(impl::kv_append(&cache, &batch, &x, st), "kv_append");
}
void kv_read(const FnsKvCache &cache, const FnsKvBatch &batch, float *k, float *v, hipStream_t st) {
    host::abort_on_error(impl::kv_read(&cache, &batch, k, v, st), "kv_read");
}
}  // namespace k

}  // namespace fns
