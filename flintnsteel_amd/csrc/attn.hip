// attn.hip - grouped-query attention of a batch's new tokens over the paged 4-bit cache (fns_kv.hpp), MI355X gfx950.
//
//   out[t][h] = sum_j p_j V_j,  p_j = exp(x_j - m) / (sum_j exp(x_j - m) + exp(sink_h - m)),  x_j = scale * q[t][h] . K_j
// over the positions j <= pos(t) (and > pos(t) - window) of the token's sequence, m the largest of x_j and sink_h. A row
// that sees nothing is zero; one that sees a token whose K or V holds a NaN block is NaN.
#include "fns_kv.hpp"

#include <algorithm>
#include <type_traits>

#include "fns/kernels.h"
#include "fns_common.hpp"
#include "fns_host.hpp"
#include "fns_internal.hpp"

namespace fns {

using namespace fns::dev;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 64;     // keys of a step
constexpr int kHead = 12;     // K and V expand to f16 with their tile's largest block scale at 2^12 (codes to 6: 24576)
constexpr int kBias = 127 + kHead;
// p is carried times 2^8: its low half stays clear of f16's subnormals. Sums are rescaled only where a row's maximum has
// grown by more than 2^7 since the last time, so p stays below 2^15.
constexpr float kPShift = 8.0f, kLazy = 7.0f;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct AttnArgs {
    KvView c;
    BatchView b;
    const void *q;
    void *out;
    const float *sinks;
    float *part;      // [split][n_tok * n_head][D] partial results, each already a weighted mean
    float2 *part_ml;  // [split][n_tok * n_head] their maximum (log2) and sum
    int64_t q_stride, out_stride;
    int n_head, group, window, splits, chunk;
    float scale;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(uint16_t x) { return __builtin_bit_cast(float, (uint32_t) x << 16); }
__device__ __forceinline__ uint16_t to_bf16(float x) {  // nearest, ties to even; NaN stays NaN
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    return (uint16_t) ((u & 0x7fffffffu) > 0x7f800000u ? (u >> 16) | 0x40u : (u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
template <class T> __device__ __forceinline__ void store4(T *p, f4 v) {  // any element alignment
    T t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) t[i] = v[i];
        else t[i] = to_bf16(v[i]);
    }
    __builtin_memcpy(p, t, sizeof t);
}

// A workgroup's rows (row = token of the sequence * group + head of the group) row0 .. row0 + rows - 1, and the tiles of
// keys [t0, t1) that any of them sees.
struct RowTiles {
    int lo, hi;  // positions [lo, hi)
    int t0, t1;
};
__device__ __forceinline__ RowTiles row_tiles(const AttnArgs &a, const SeqRange &r, int row0, int rows) {
    const int i0 = row0 / a.group, i1 = min((row0 + rows - 1) / a.group, r.n - 1);
    const int first = r.len - r.n;
    const int64_t cap = a.b.table_stride << a.c.shift;  // positions behind the table have no page
    RowTiles t;
    t.hi = (int) min((int64_t) first + i1 + 1, cap);
    t.lo = a.window ? max(first + i0 - a.window + 1, 0) : 0;
    t.t0 = t.lo / kTile;
    t.t1 = t.hi > t.lo ? t.hi / kTile + (t.hi % kTile > 0) : t.t0;
    return t;
}
// Tiles of one split: a chunk that the host chose from max_kv, more where the sequence is longer than that.
__device__ __forceinline__ int split_chunk(const AttnArgs &a, const RowTiles &t) {
    return max(a.chunk, (t.t1 - t.t0 + a.splits - 1) / a.splits);
}

// What a wave knows of a tile, a key a lane: which keys are there, which of them hold NaNs, the largest scale bytes.
struct TileInfo {
    uint64_t there, nan;
    int ek, ev;
};
typedef uint16_t us2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_max(uint32_t x, uint32_t y) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, x), __builtin_bit_cast(us2, y)));
}
// The scale bytes of one position's K and V, NB of each.
template <int NB> struct ScaleWords {
    static constexpr int W = (NB + 3) / 4;
    uint32_t k[W], v[W];
};
// ... and the block scales as the f32 operands of the expansion, in the wave's LDS: K [64 in the order of the products'
// rows][NB], V [NB][64 keys]. A block's operand is 2^(e - E + 12) for the tile's (K) or the largest so far (V) scale E; what
// lies 2^36 below that is dropped, which is less than the last bit of any sum it could join.
__device__ __forceinline__ int row_of_key(int key) { return (key >> 2 & 3) * 16 + (key >> 4) * 4 + (key & 3); }
template <int NB>
__device__ __forceinline__ TileInfo tile_scales(ScaleWords<NB> w, bool there, int ev_before, float *ksc, float *vsc) {
    constexpr int W = ScaleWords<NB>::W;
    constexpr uint32_t kEven = 0x00ff00ffu;
    const int lane = threadIdx.x % 64;
    uint32_t e[2][W][2], top[2];  // bytes 0 and 2, 1 and 3 of every word, in halves
    const auto split = [&](int s) {
        top[s] = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const uint32_t x = s ? w.v[i] : w.k[i];
            e[s][i][0] = x & kEven, e[s][i][1] = x >> 8 & kEven;
            top[s] = pk_max(top[s], pk_max(e[s][i][0], e[s][i][1]));
        }
        top[s] = max(top[s] & 0xffffu, top[s] >> 16);
    };
#pragma unroll
    for (int i = 0; i < W; ++i) w.k[i] = there ? w.k[i] : 0, w.v[i] = there ? w.v[i] : 0;
    split(0), split(1);
    TileInfo t;
    t.there = __ballot(there);
    t.nan = __ballot(max(top[0], top[1]) == 255u);
    if (t.nan) {  // rare: their blocks count as zeros, the rows that see them are made NaN
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const uint32_t m = 255u << (8 * b);
                w.k[i] = (w.k[i] & m) == m ? w.k[i] & ~m : w.k[i];
                w.v[i] = (w.v[i] & m) == m ? w.v[i] & ~m : w.v[i];
            }
        split(0), split(1);
    }
    uint32_t both = top[0] << 16 | top[1];
    both = pk_max(both, xor_lane_i<1>(both));
    both = pk_max(both, xor_lane_i<2>(both));
    both = pk_max(both, xor_lane_i<4>(both));
    both = pk_max(both, xor_lane_i<8>(both));
    both = pk_max(both, xor_lane_i<16>(both));
    both = pk_max(both, xor_lane_i<32>(both));
    both = __builtin_amdgcn_readfirstlane(both);
    t.ek = both >> 16;
    t.ev = max((int) (both & 0xffffu), ev_before);
    const auto field = [](uint32_t e, int top) { return __builtin_bit_cast(float, max((int) e + kBias - top, 0) << 23); };
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int i = b / 4, odd = b % 2, sh = b % 4 / 2 * 16;
        ksc[row_of_key(lane) * NB + b] = field(e[0][i][odd] >> sh & 0xffu, t.ek);
        vsc[b * 64 + lane] = field(e[1][i][odd] >> sh & 0xffu, t.ev);
    }
    return t;
}

// Eight consecutive channels of K from their four bytes.
__device__ __forceinline__ h8 expand_k(uint32_t w, float sc) {
    const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 1);
    const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 3);
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// Eight consecutive positions of V from their eight bytes: two channels 16 apart (low and high halves).
__device__ __forceinline__ void expand_v(uint32_t w0, uint32_t w1, const float *sc, h8 &lo, h8 &hi) {
    h2 p[8];
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w0, sc[0], 0), p[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w0, sc[1], 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w0, sc[2], 2), p[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w0, sc[3], 3);
    p[4] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w1, sc[4], 0), p[5] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w1, sc[5], 1);
    p[6] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w1, sc[6], 2), p[7] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w1, sc[7], 3);
    u4 l, h;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = __builtin_bit_cast(uint32_t, p[2 * i]), y = __builtin_bit_cast(uint32_t, p[2 * i + 1]);
        l[i] = __builtin_amdgcn_perm(y, x, 0x05040100u);
        h[i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
    }
    lo = __builtin_bit_cast(h8, l), hi = __builtin_bit_cast(h8, h);
}

// The queries of one column tile (16 rows) as operands of the products: lane (row r = lane % 16, g = lane / 16) holds the
// channels g NB 8 + 8 u .. + 7 of step u, in one (bf16: exact) or two (f32: 22 bits) f16 parts, the row scaled by a power
// of two to a largest magnitude in [2^10, 2^11). Returns what turns a product (of K at its tile's 2^12) into log2 units.
template <int NB, int SPLIT, class T>
__device__ __forceinline__ float load_queries(h8 (&part)[SPLIT][NB], const T *row, bool there, float scale) {
    const int g = threadIdx.x % 64 / 16;
    float v[NB][8], amax = 0.0f;
    bool bad = false;
#pragma unroll
    for (int u = 0; u < NB; ++u) {
        T t[8] = {};
        if (there) __builtin_memcpy(t, row + g * NB * 8 + u * 8, sizeof t);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[u][i] = to_f32(t[i]);
            bad |= !(fabsf(v[u][i]) <= 3.4028234663852886e38f);
            amax = fmaxf(amax, fabsf(v[u][i]));
        }
    }
    amax = fmaxf(amax, xor_lane<16>(amax));
    amax = fmaxf(amax, xor_lane<32>(amax));
    bad |= xor_lane_i<16>(bad);
    bad |= xor_lane_i<32>(bad);
    int k = 0;
    if (amax > 0.0f && !bad) k = ilogbf(amax) + 1;
    k = max(k, -100);
    const float f = bad ? __builtin_nanf("") : ldexpf(scale < 0.0f ? -1.0f : 1.0f, 11 - k);
#pragma unroll
    for (int u = 0; u < NB; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = v[u][i] * f;
            const _Float16 hi = (_Float16) x;
            part[0][u][i] = hi;
            if constexpr (SPLIT == 2) part[1][u][i] = (_Float16) (x - (float) hi);
        }
    return fabsf(scale) * kLog2e * ldexpf(1.0f, k - 11);
}

// A lane's state of one column tile: row r = lane % 16; a lane sums the keys 16 g .. 16 g + 15 of every tile, and holds
// channels 16 dt + 4 g + i of its row in o[dt][i] (in units of 2^(ev - 139)). m: the maximum that p and the sums refer to.
template <int NB> struct RowState {
    f4 o[2 * NB];
    float m, l;
};

// One tile's softmax of a column tile: s (product units) of the lane's 16 keys -> p as operand parts, m and l updated;
// returns what earlier sums have to be multiplied by. see: the lane's keys that its row sees.
template <int SPLIT>
__device__ __forceinline__ float softmax_step(f4 (&s)[4], float mul, uint32_t see, uint32_t nan, float &m, float &l, h8 (&p)[SPLIT][2]) {
    const bool all = __all(see == 0xffffu);
    if (!all) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][i] = see >> (4 * t + i) & 1 ? s[t][i] : -INFINITY;
    }
    float top = fmaxf(s[0][0], s[0][1]);
#pragma unroll
    for (int i = 2; i < 16; i += 2) top = fmaxf(fmaxf(top, s[i / 4][i % 4]), s[i / 4][i % 4 + 1]);
    top = fmaxf(top, xor_lane<16>(top));
    top = fmaxf(top, xor_lane<32>(top));
    const float now = top == -INFINITY ? top : top * mul;
    float keep = 1.0f;
    if (__any(now > m + kLazy)) {
        const float to = fmaxf(m, now);
        keep = __builtin_amdgcn_exp2f(m - (to == -INFINITY ? 0.0f : to));  // (nothing seen so far: no difference of infinities)
        m = to;
    }
    const float add = kPShift - (m == -INFINITY ? 0.0f : m);
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], mul, add));
    if (!all)  // (a scale of zero times -infinity)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][i] = see >> (4 * t + i) & 1 ? s[t][i] : 0.0f;
    if (nan)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][i] = see >> (4 * t + i) & nan >> (4 * t + i) & 1 ? __builtin_nanf("") : s[t][i];
#pragma unroll
    for (int t = 0; t < 4; ++t) sum += (s[t][0] + s[t][1]) + (s[t][2] + s[t][3]);
    l = l * keep + sum;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        u4 w[SPLIT];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = s[2 * v + i / 2][i % 2 * 2], y = s[2 * v + i / 2][i % 2 * 2 + 1];
            if constexpr (SPLIT == 2) {  // toward zero: the second part has the rest
                const h2 hi = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(x, y));
                w[0][i] = __builtin_bit_cast(uint32_t, hi);
                w[1][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x - (float) hi[0], y - (float) hi[1]));
            } else {
                w[0][i] = __builtin_bit_cast(uint32_t, h2{(_Float16) x, (_Float16) y});
            }
        }
#pragma unroll
        for (int h = 0; h < SPLIT; ++h) p[h][v] = __builtin_bit_cast(h8, w[h]);
    }
    return keep;
}

// Bits of the lane's 16 keys (base + 16 g ..) that a row at position pos sees; there: the tile's keys that exist.
__device__ __forceinline__ uint32_t seen(int pos, int window, int base, uint64_t there) {
    const int g = threadIdx.x % 64 / 16;
    const int up = pos - (base + 16 * g);  // the last one
    uint32_t bits = up < 0 ? 0u : up >= 15 ? 0xffffu : (2u << up) - 1u;
    if (window) {
        const int dn = up - window + 1;  // the first one
        bits = dn <= 0 ? bits : dn > 15 ? 0u : bits & (0xffffu << dn);
    }
    return bits & (uint32_t) (there >> (16 * g));
}

// Result of one row's 4 channels or, with splits, its partial.
template <int D, class T>
__device__ __forceinline__ void store_row(const AttnArgs &a, int64_t tok, int h, int split, int ch, f4 v) {
    if (a.splits > 1) *(f4 *) (a.part + ((split * a.b.n_tok + tok) * a.n_head + h) * D + ch) = v;
    else store4((T *) a.out + tok * a.out_stride + (int64_t) h * D + ch, v);
}

// Where a tile's bytes are. With pages of 64 positions or more a tile lies in one page: every address is the tile's (in
// scalar registers) plus an offset that a lane keeps; smaller pages (SMALL) are looked up for every 16 positions.
template <int D, bool SMALL> struct TileReader {
    static constexpr int NB = D / 32, KC = NB * 4;  // KC: code bytes of a lane's channels of one key
    using L = KvParts<D>;
    int P, lane, r, g;
    int64_t head_off;
    const uint8_t *bk, *bv;  // of the lane's K rows (keys 16 (r / 4) ..), and of its own key and V columns (16 g ..)
    int row;                 // of the tile's first position in its page
    bool there;
    __device__ __forceinline__ void page(const AttnArgs &a, int s, int tile, bool in) {
        const int base = tile * kTile;
        row = base & (P - 1);
        if constexpr (SMALL) {
            const int pk = in ? page_of(a.c, a.b, s, base + 16 * (r / 4)) : -1, pv = in ? page_of(a.c, a.b, s, base + 16 * g) : -1;
            bk = a.c.pages + max(pk, 0) * a.c.page_bytes + head_off;
            bv = a.c.pages + max(pv, 0) * a.c.page_bytes + head_off;
            there = pv >= 0;
        } else {
            const int p = in ? __builtin_amdgcn_readfirstlane(page_of(a.c, a.b, s, base)) : -1;
            bk = bv = a.c.pages + max(p, 0) * a.c.page_bytes + head_off;
            there = p >= 0;
        }
    }
    __device__ __forceinline__ void scales(ScaleWords<NB> &w) const {
        const int at = (SMALL ? (row + lane) & (P - 1) : row + lane);
        w = {};
        __builtin_memcpy(w.k, __builtin_assume_aligned(bv + L::k_scale(P, at), NB), NB);
        __builtin_memcpy(w.v, __builtin_assume_aligned(bv + L::v_scale(P, at), NB), NB);
    }
    __device__ __forceinline__ void k(uint32_t (&x)[4][NB]) const {
        const int at = SMALL ? (row + 16 * (r / 4)) & (P - 1) : row + 16 * (r / 4);
        const uint8_t *p = bk + (uint32_t) ((at + r % 4) * (D / 2) + g * KC);
#pragma unroll
        for (int t = 0; t < 4; ++t) __builtin_memcpy(x[t], __builtin_assume_aligned(p + 4 * t * (D / 2), KC < 16 ? KC : 16), KC);
    }
    __device__ __forceinline__ void v(u4 (&x)[NB]) const {
        const int at = SMALL ? (row + 16 * g) & (P - 1) : row + 16 * g;
        const uint8_t *p = bv + (uint32_t) (P * (D / 2) + r * P + at);
#pragma unroll
        for (int j = 0; j < NB; ++j) x[j] = *(const u4 *) (p + (uint32_t) (16 * j * P));
    }
};

// Few rows (decode, verify): the workgroup's waves take tiles of keys in turn and are joined at the end. A wave's tile goes
// from the pages to registers and stays there: S^T = K Q^T with K's rows in an order that leaves every lane with the 16
// consecutive keys 16 g .. 16 g + 15 of its query row, which is where the second product, O^T = V^T P^T, wants P, and where
// V's bytes (16 consecutive positions of a channel pair) are. Bound by the cache's bytes for long contexts and by a few
// dependent loads for short ones. One wave issues a vector instruction about every 5 cycles where the SIMD takes one every
// 2: what pays is waves, so the queries lie in LDS and the next tile's K is asked for when this one's is used up.
template <int D, int CT, bool SMALL, class T>
__global__ __launch_bounds__(256, D == 256 || CT == 2 ? 2 : 4) void k_attn_few(AttnArgs a) {
    constexpr int NB = D / 32, SPLIT = sizeof(T) == 4 ? 2 : 1, NW = 4;
    constexpr int kScale = 2 * 64 * NB, kJoin = NW / 2 * CT * 2 * NB * 256;
    __shared__ __align__(16) float lds[NW * kScale > kJoin ? NW * kScale : kJoin];
    __shared__ __align__(16) h8 qs[CT][SPLIT][NB][64];
    __shared__ float join[NW][2][CT * 16], qmul[CT][16];
    const int s = blockIdx.x / a.c.n_kv, head = blockIdx.x % a.c.n_kv, row0 = blockIdx.y * 16 * CT, split = blockIdx.z;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
    const SeqRange sr = seq_range(a.b, s);
    const int rows = (int) min((int64_t) sr.n * a.group, (int64_t) INT32_MAX);
    if (row0 >= rows) return;
    const RowTiles rt = row_tiles(a, sr, row0, 16 * CT);
    const int chunk = split_chunk(a, rt);
    const int t0 = (int) min((int64_t) rt.t0 + (int64_t) split * chunk, (int64_t) rt.t1);
    const int t1 = min(t0 + chunk, rt.t1);
    if (split > 0 && t0 >= t1) return;  // (split 0 of an empty range writes the zeros)
    const int P = 1 << a.c.shift;

    TileReader<D, SMALL> rd;
    rd.P = P, rd.lane = lane, rd.r = r, rd.g = g, rd.head_off = head * kv_head_bytes(D, P);
    uint32_t kraw[4][NB];
    u4 vraw[NB];
    ScaleWords<NB> sw = {};
    int tile = t0 + wave;
    rd.page(a, s, tile, tile < t1);
    if (tile < t1) rd.scales(sw), rd.k(kraw), rd.v(vraw);

    RowState<NB> st[CT];
    int pos[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int row = row0 + 16 * c + r, i = row / a.group;
        const bool there = row < rows;
        pos[c] = there ? sr.len - sr.n + i : -1;
        if (wave == c) {
            h8 part[SPLIT][NB];
            const float mul = load_queries(part, (const T *) a.q + (sr.q0 + i) * a.q_stride + (int64_t) (head * a.group + row % a.group) * D,
                                           there, a.scale);
#pragma unroll
            for (int h = 0; h < SPLIT; ++h)
#pragma unroll
                for (int u = 0; u < NB; ++u) qs[c][h][u][lane] = part[h][u];
            if (g == 0) qmul[c][r] = mul;
        }
        st[c].m = -INFINITY, st[c].l = 0.0f;
#pragma unroll
        for (int d = 0; d < 2 * NB; ++d) st[c].o[d] = f4{0, 0, 0, 0};
    }
    __syncthreads();
    float mul[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) mul[c] = qmul[c][r];

    float *ksc = lds + wave * kScale, *vsc = ksc + 64 * NB;
    int ev = 1;
    for (; tile < t1; tile += NW) {
        const int base = tile * kTile, key = base + lane;
        const TileInfo ti = tile_scales<NB>(sw, rd.there && key >= rt.lo && key < rt.hi, ev, ksc, vsc);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        f4 sc[CT][4];
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int t = 0; t < 4; ++t) sc[c][t] = f4{0, 0, 0, 0};
        float ks[4][(NB + 3) / 4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int u = 0; u < (NB + 3) / 4; ++u) ks[t][u] = ksc[(16 * t + r) * NB + (g * NB + 4 * u) / 4];
#pragma unroll
        for (int u = 0; u < NB; ++u) {
            h8 q[CT][SPLIT];
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int h = 0; h < SPLIT; ++h) q[c][h] = qs[c][h][u][lane];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const h8 k = expand_k(kraw[t][u], ks[t][u / 4]);
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int h = SPLIT - 1; h >= 0; --h)
                        sc[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[c][h], sc[c][t], 0, 0, 0);
            }
        }
        const bool more = tile + NW < t1;
        rd.page(a, s, tile + NW, more);
        if (more) rd.scales(sw), rd.k(kraw);
        const float back = ldexpf(1.0f, ti.ek - kBias), vkeep = ldexpf(1.0f, max(ev - ti.ev, -126));
        ev = ti.ev;
        h8 p[CT][SPLIT][2];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            const uint32_t see = seen(pos[c], a.window, base, ti.there);
            const uint32_t nan = ti.nan ? (uint32_t) (ti.nan >> (16 * g)) & 0xffffu : 0u;
            const float keep = softmax_step<SPLIT>(sc[c], mul[c] * back, see, nan, st[c].m, st[c].l, p[c]) * vkeep;
            if (__any(keep != 1.0f))
#pragma unroll
                for (int d = 0; d < 2 * NB; ++d) st[c].o[d] *= keep;
        }
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                h8 lo, hi;
                float w[8];
                *(f4 *) w = *(const f4 *) (vsc + j * 64 + 16 * g + 8 * v);
                *(f4 *) (w + 4) = *(const f4 *) (vsc + j * 64 + 16 * g + 8 * v + 4);
                expand_v(vraw[j][2 * v], vraw[j][2 * v + 1], w, lo, hi);
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int h = SPLIT - 1; h >= 0; --h) {
                        st[c].o[2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, p[c][h][v], st[c].o[2 * j], 0, 0, 0);
                        st[c].o[2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, p[c][h][v], st[c].o[2 * j + 1], 0, 0, 0);
                    }
            }
        if (more) rd.v(vraw);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }

    // join the waves: the common maximum and sum of every row, then the sums in a tree over registers of equal layout
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        st[c].l += xor_lane<16>(st[c].l);
        st[c].l += xor_lane<32>(st[c].l);
        if (g == 0) join[wave][0][16 * c + r] = st[c].m, join[wave][1][16 * c + r] = st[c].l;
    }
    __syncthreads();
    float top[CT], sum[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int row = 16 * c + r;
        top[c] = fmaxf(fmaxf(join[0][0][row], join[1][0][row]), fmaxf(join[2][0][row], join[3][0][row]));
        const int h = head * a.group + (row0 + row) % a.group;
        const bool sink = a.splits == 1 && a.sinks && row0 + row < rows;
        const float sk = sink ? a.sinks[h] * kLog2e : -INFINITY;
        const float with = fmaxf(top[c], sk);
        const float off = with == -INFINITY ? 0.0f : with;
        sum[c] = sink ? __builtin_amdgcn_exp2f(sk - off + kPShift) : 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) sum[c] += join[w][1][row] * __builtin_amdgcn_exp2f(join[w][0][row] - off);
        const float f = sum[c] == 0.0f ? 0.0f : ldexpf(__builtin_amdgcn_exp2f(st[c].m - off) / sum[c], ev - kBias);
#pragma unroll
        for (int d = 0; d < 2 * NB; ++d) st[c].o[d] *= f;
    }
#pragma unroll
    for (int half = NW / 2; half >= 1; half /= 2) {
        f4 *x = (f4 *) lds + (wave % half) * CT * 2 * NB * 64 + lane;
        if (wave >= half && wave < 2 * half)
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int d = 0; d < 2 * NB; ++d) x[(c * 2 * NB + d) * 64] = st[c].o[d];
        __syncthreads();
        if (wave < half)
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int d = 0; d < 2 * NB; ++d) st[c].o[d] += x[(c * 2 * NB + d) * 64];
        if (half > 1) __syncthreads();
    }
    if (wave != 0) return;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int row = row0 + 16 * c + r;
        if (row >= rows) continue;
        const int64_t tok = sr.q0 + row / a.group;
        const int h = head * a.group + row % a.group;
#pragma unroll
        for (int d = 0; d < 2 * NB; ++d) store_row<D, T>(a, tok, h, split, 16 * d + 4 * g, st[c].o[d]);
        if (a.splits > 1 && g == 0) a.part_ml[(split * a.b.n_tok + tok) * a.n_head + h] = make_float2(top[c], sum[c]);
    }
}

// The splits of a row into its result: a workgroup a row, its waves the splits in turn (at most 64: one a lane for their
// weights), a lane D / 64 channels.
template <int D, class T>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a, int rows_per_wg) {
    constexpr int C = D / 64, NW = 4;
    __shared__ float part[NW][D], weight[64];
    const int s = blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const SeqRange sr = seq_range(a.b, s);
    const int i = blockIdx.x / a.n_head, h = blockIdx.x % a.n_head;
    if (i >= sr.n) return;
    const int64_t tok = sr.q0 + i, first = tok * a.n_head + h, step = a.b.n_tok * a.n_head;
    const int row = i * a.group + h % a.group, row0 = row / rows_per_wg * rows_per_wg;
    const RowTiles rt = row_tiles(a, sr, row0, rows_per_wg);
    const int chunk = split_chunk(a, rt);
    const int n = max(1, (rt.t1 - rt.t0 + chunk - 1) / max(chunk, 1));  // splits that have tiles (the first one in any case)
    const float sk = a.sinks ? a.sinks[h] * kLog2e : -INFINITY;
    const float2 ml = lane < n ? a.part_ml[lane * step + first] : make_float2(-INFINITY, 0.0f);
    const float top = fmaxf(lanes_max<64>(ml.x), sk);
    const float off = top == -INFINITY ? 0.0f : top;
    const float f = ml.y == 0.0f ? 0.0f : ml.y * __builtin_amdgcn_exp2f(ml.x - off);
    const float sum = lanes_sum<64>(f) + (a.sinks ? __builtin_amdgcn_exp2f(sk - off + kPShift) : 0.0f);
    if (wave == 0) weight[lane] = sum == 0.0f ? 0.0f : f / sum;
    __syncthreads();
    float o[C] = {};
    const float *src = a.part + first * D + lane * C;
#pragma unroll 8
    for (int k = wave; k < n; k += NW) {
        const float wk = weight[k];
        float v[C];
        __builtin_memcpy(v, __builtin_assume_aligned(src + k * step * D, 4 * C), sizeof v);
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] += wk == 0.0f ? 0.0f : wk * v[c];
    }
#pragma unroll
    for (int c = 0; c < C; ++c) part[wave][lane * C + c] = o[c];
    __syncthreads();
    T *out = (T *) a.out + tok * a.out_stride + (int64_t) h * D;
    for (int d = threadIdx.x; d < D; d += 256) {
        const float x = (part[0][d] + part[1][d]) + (part[2][d] + part[3][d]);
        if constexpr (sizeof(T) == 4) out[d] = x;
        else out[d] = to_bf16(x);
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

// How a call is divided: rows of a workgroup, splits of the keys and tiles of a split, by the host's numbers.
struct Plan {
    int rows, row_tiles, splits, chunk;
    size_t ml_off, bytes;
};
Plan attn_plan(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x) {
    Plan p{};
    const int64_t rows = (int64_t) b->max_q * (x->n_head / c->n_head_kv);
    p.rows = rows <= 16 || c->head_dim == 256 ? 16 : 32;
    p.row_tiles = (int) ((rows + p.rows - 1) / p.rows);
    const int64_t wgs = std::max<int64_t>(1, (int64_t) b->n_seq * c->n_head_kv * p.row_tiles);
    const int64_t tiles = std::max<int64_t>(1, (b->max_kv + kTile - 1) / kTile);
    const int64_t want = (2048 + wgs - 1) / wgs, most = (tiles + 3) / 4;
    p.splits = (int) std::max<int64_t>(1, std::min({want, most, (int64_t) 64}));
    p.chunk = (int) ((tiles + p.splits - 1) / p.splits);
    if (p.splits > 1) {
        const size_t n = (size_t) p.splits * b->n_tok * x->n_head;
        p.ml_off = n * c->head_dim * 4;
        p.bytes = p.ml_off + n * 8;
    }
    return p;
}

}  // namespace

int attn_workspace(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x, size_t *bytes) {
    FNS_TRY(attn_check(c, b, x));
    if (!bytes) return host::set_error(host::ERR_SHAPE, "attn_workspace: null output");
    *bytes = attn_plan(c, b, x).bytes;
    return host::OK;
}

int attn(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x, const void *q, void *out, void *ws, size_t ws_bytes,
         hipStream_t st) {
    FNS_TRY(attn_check(c, b, x));
    if (b->n_seq == 0 || b->n_tok == 0 || b->max_q == 0) return host::OK;
    if (!q || !out) return host::set_error(host::ERR_SHAPE, "attn: null argument");
    const Plan p = attn_plan(c, b, x);
    if (p.bytes && (!ws || ws_bytes < p.bytes || ((uintptr_t) ws & 15)))
        return host::set_error(host::ERR_NOMEM, "attn: workspace of %zu bytes, %zu needed (16-byte aligned)", ws ? ws_bytes : 0, p.bytes);
    AttnArgs a{};
    a.c = host::kv_view(c), a.b = host::kv_batch(b);
    a.q = q, a.out = out, a.sinks = x->sinks;
    a.part = (float *) ws, a.part_ml = (float2 *) ((uint8_t *) ws + p.ml_off);
    a.q_stride = x->q_stride, a.out_stride = x->out_stride;
    a.n_head = x->n_head, a.group = x->n_head / c->n_head_kv, a.window = x->window;
    a.splits = p.splits, a.chunk = p.chunk, a.scale = x->scale;
    const dim3 grid((unsigned) (b->n_seq * c->n_head_kv), (unsigned) p.row_tiles, (unsigned) p.splits);
    const bool small = c->page_size < kTile;
    auto few = [&](auto dim, auto ct, auto type) {
        constexpr int D = decltype(dim)::value, CT = decltype(ct)::value;
        if (small) hipLaunchKernelGGL((k_attn_few<D, CT, true, decltype(type)>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((k_attn_few<D, CT, false, decltype(type)>), grid, dim3(256), 0, st, a);
    };
    auto join = [&](auto dim, auto type) {
        const int64_t rows = (int64_t) b->max_q * x->n_head;
        hipLaunchKernelGGL((k_attn_join<decltype(dim)::value, decltype(type)>), dim3((unsigned) rows, (unsigned) b->n_seq),
                           dim3(256), 0, st, a, p.rows);
    };
    auto by_type = [&](auto dim, auto type) {
        constexpr int D = decltype(dim)::value;
        if constexpr (D == 256) few(dim, std::integral_constant<int, 1>{}, type);
        else if (p.rows == 16) few(dim, std::integral_constant<int, 1>{}, type);
        else few(dim, std::integral_constant<int, 2>{}, type);
        FNS_TRY(host::check_launch("attn"));
        if (p.splits > 1) join(dim, type);
        return host::check_launch("attn");
    };
    auto by_dim = [&](auto dim) { return x->dtype == FNS_TYPE_F32 ? by_type(dim, float{}) : by_type(dim, uint16_t{}); };
    if (c->head_dim == 64) return by_dim(std::integral_constant<int, 64>{});
    if (c->head_dim == 128) return by_dim(std::integral_constant<int, 128>{});
    return by_dim(std::integral_constant<int, 256>{});
}

}  // namespace impl

namespace k {
void attn(const FnsKvCache &cache, const FnsKvBatch &batch, const FnsAttn &x, const void *q, void *out, void *ws,
          size_t ws_bytes, hipStream_t st) {
    host::abort_on_error(impl::attn(&cache, &batch, &x, q, out, ws, ws_bytes, st), "attn");
}
}  // namespace k

}  // namespace fns
