// fns_attn.hpp - the kernels of grouped-query attention of a batch's new tokens over the paged 4-bit cache (fns_kv.hpp),
// MI355X gfx950, and their launches; attn.hip and attn_tree.hip make the two sets of them.
//
//   out[t][h] = sum_j p_j V_j,  p_j = exp(x_j - m) / (sum_j exp(x_j - m) + exp(sink_h - m)),  x_j = scale * q[t][h] . K_j
// over the positions j <= pos(t) (and > pos(t) - window) of the token's sequence, m the largest of x_j and sink_h. A row
// that sees nothing is zero; one that sees a token whose K or V holds a NaN block is NaN.
//
// MORE: what a token sees of the batch's new tokens may come as bits (a tree of drafted tokens), and the logarithm of the
// denominator, m + log(sum_j exp(x_j - m) + exp(sink_h - m)), may be an output.
#pragma once

#include "fns_kv.hpp"

#include <algorithm>
#include <type_traits>

#include "fns/kernels.h"
#include "fns_common.hpp"
#include "fns_host.hpp"
#include "fns_internal.hpp"

namespace fns {

namespace host {

// How a call is divided: rows of a workgroup, splits of the keys and tiles of a split, by the host's numbers.
struct AttnPlan {
    int rows, splits, chunk;
    int64_t row_tiles;  // (more than a grid has are refused)
    size_t ml_off, bytes;
};
// (attn.hip) Checks of a call's numbers, its plan, and checks of its pointers against the plan; `what` names the call.
int attn_check(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x, const char *what);
AttnPlan attn_plan(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x);
int attn_check_buffers(const AttnPlan &p, const FnsKvBatch *b, const void *q, const void *out, const void *ws, size_t ws_bytes, const char *what);

}  // namespace host

using namespace fns::dev;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 64;     // keys of a step
constexpr int kFewRows = 64, kManyRows = 128;  // rows that always take the few-row form; rows of a workgroup of the other
constexpr int kFewWaves = 4;  // waves of a workgroup of few rows
constexpr int kHead = 12;     // V expands to f16 with the largest block scale so far, E, at 2^12 (codes to 6: 24576)
constexpr int kBias = 127 + kHead;
constexpr int kBand = 36;     // block scales from E down that f16 holds exactly
// E starts at 2^-17 (V below that is exact too, down to 2^-53), and where it has grown by more than 2^100, sums from before
// may be next to f32's subnormals: a row has at least 2^8 of p, times 2^(12 - 36) of a block, so 2^-16 before the growth.
constexpr int kFloor = 110, kGrown = kFloor + 100;
// A split's mean of V is kept 2^2 down: codes of the largest scale are 1.5 times 2^129, and where such a key weighs little in the
// row it may be all of its split.
constexpr int kPart = 2;
// p is carried times 2^8: its low half stays clear of f16's subnormals. Sums are rescaled only where a row's maximum has
// grown by more than 2^7 since the last time, so p stays below 2^15.
constexpr float kPShift = 8.0f, kLazy = 7.0f;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef int i8v __attribute__((ext_vector_type(8)));

struct AttnArgs {
    KvView c;
    BatchView b;
    const void *q;
    void *out;
    const float *sinks;
    float *part;      // [split][n_tok * n_head][D] partial results, each already a weighted mean, 2^-kPart of it
    float2 *part_ml;  // [split][n_tok * n_head] their maximum (log2) and sum
    int64_t q_stride, out_stride;
    int n_head, group, window, splits, chunk;
    float scale;
    uint8_t *redo;  // many rows: [n_seq * n_kv][row tiles][4 waves], whether some row may have lost something of V
    const uint64_t *sees;  // MORE: [n_tok][words], or null: causal
    float *lse;            // MORE: [n_tok][n_head], or null
    int words;
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

// The position before the first one that a token at pos sees, -1 if that is 0 (pos may be negative, where a sequence has fewer
// positions than new tokens, and a window any width: their difference does not fit 32 bits).
__device__ __forceinline__ int before_window(int pos, int window) {
    return window ? max(max(pos, 0) - window, -1) : -1;
}
// A workgroup's rows (row = token of the sequence * group + head of the group) row0 .. row0 + rows - 1, and the tiles of
// keys [t0, t1) that any of them sees.
struct RowTiles {
    int lo, hi;  // positions [lo, hi)
    int t0, t1;
};
// (of a tree: all that its tokens may see)
template <bool MORE> __device__ __forceinline__ RowTiles row_tiles(const AttnArgs &a, const SeqRange &r, int row0, int rows) {
    const bool tree = MORE && a.sees;
    const int i0 = tree ? 0 : row0 / a.group, i1 = tree ? r.n - 1 : min((row0 + rows - 1) / a.group, r.n - 1);
    const int first = r.len - r.n;
    const int64_t cap = a.b.table_stride << a.c.shift;  // positions behind the table have no page
    RowTiles t;
    t.hi = (int) min((int64_t) first + i1 + 1, cap);
    t.lo = before_window(first + i0, a.window) + 1;
    t.t0 = t.lo / kTile;
    t.t1 = t.hi > t.lo ? t.hi / kTile + (t.hi % kTile > 0) : t.t0;
    return t;
}
// Tiles of one split: as many splits as chunks (the host's number, from max_kv) are needed, of equal lengths; longer ones
// where the sequence is longer than max_kv.
__device__ __forceinline__ int split_chunk(const AttnArgs &a, const RowTiles &t) {
    const int tiles = t.t1 - t.t0;
    const int n = min(max((tiles + a.chunk - 1) / a.chunk, 1), a.splits);
    return max(((tiles + n - 1) / n + kFewWaves - 1) / kFewWaves * kFewWaves, 1);
}

// What a wave knows of a tile, a key a lane: which keys are there, which of them hold NaNs in V; and the wave's V scale.
typedef uint16_t us2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_max(uint32_t x, uint32_t y) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, x), __builtin_bit_cast(us2, y)));
}
// Not zero in the halves of x that are from 1 to bound.
__device__ __forceinline__ uint32_t pk_below(uint32_t x, uint32_t bound) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(__builtin_bit_cast(us2, bound), (us2) (__builtin_bit_cast(us2, x) - (us2) {1, 1})));
}
struct TileInfo {
    uint64_t there, nan;
    int ev;
    bool low;  // there are blocks (of those that the wave expands) that f16 cannot hold beside the largest
};
// The block scales of V as the f32 operands of the expansion, in the wave's LDS, [NB][64 keys]: 2^(e - E + 12), E at least
// every scale so far. Half of 2^(12 - kBand) is the last bit of f16: blocks of E - kBand and below become zeros here and send
// the rows to v_in_bands (they are nothing beside the largest, but there may be rows that do not see the largest). w: the
// scale bytes of the lane's key.
template <int NB> struct ScaleBytes {
    std::conditional_t<NB == 2, uint16_t, uint32_t> w[(NB + 3) / 4];
};
// STEP, first: the blocks first, first + STEP ... only, in rows of their own.
template <int NB, int STEP = 1>
__device__ __forceinline__ TileInfo v_scales(const ScaleBytes<NB> &bytes, bool there, int ev, float *vsc, int first = 0) {
    constexpr int W = (NB + 3) / 4;
    constexpr uint32_t kEven = 0x00ff00ffu;
    const int lane = threadIdx.x % 64;
    uint32_t w[W], top = 0;
    const auto largest = [&] {
        top = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) top = pk_max(top, pk_max(w[i] & kEven, w[i] >> 8 & kEven));
        top = max(top & 0xffffu, top >> 16);
    };
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = there ? bytes.w[i] : 0;
    largest();
    TileInfo t;
    t.there = __ballot(there);
    t.nan = 0;
    t.ev = ev;
    if (__any((int) top > ev)) {
        t.nan = __ballot(top == 255u);
        if (t.nan) {  // rare: their blocks count as zeros, the rows that see them are made NaN
#pragma unroll
            for (int i = 0; i < W; ++i)
#pragma unroll
                for (int b = 0; b < 4; ++b) w[i] = (w[i] >> (8 * b) & 255u) == 255u ? w[i] & ~(255u << (8 * b)) : w[i];
            largest();
        }
        top = max(top, (uint32_t) xor_lane_i<1>(top));
        top = max(top, (uint32_t) xor_lane_i<2>(top));
        top = max(top, (uint32_t) xor_lane_i<4>(top));
        top = max(top, (uint32_t) xor_lane_i<8>(top));
        top = max(top, (uint32_t) xor_lane_i<16>(top));
        top = max(top, (uint32_t) xor_lane_i<32>(top));
        t.ev = max(ev, __builtin_amdgcn_readfirstlane(top));
    }
    const uint32_t bound = (uint32_t) max(t.ev - kBand, 0);
    uint32_t low = 0;
    if constexpr (STEP == 1) {
#pragma unroll
        for (int i = 0; i < W; ++i)  // scales 1 .. bound: less 1, a scale of 0 is the largest
            low |= pk_below(w[i] & kEven, bound * 0x10001u) | pk_below(w[i] >> 8 & kEven, bound * 0x10001u);
    } else {
#pragma unroll
        for (int b = 0; b < NB; ++b)
            if (b % STEP == first) low |= (w[b / 4] >> (b % 4 * 8) & 0xffu) - 1u < bound;
    }
    t.low = __ballot(low != 0) != 0;
    if (t.low) {  // rare
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
            for (int b = 0; b < 4; ++b) w[i] = (w[i] >> (8 * b) & 255u) <= bound ? w[i] & ~(255u << (8 * b)) : w[i];
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
        if (STEP == 1 || b % STEP == first)
            vsc[b / STEP * 64 + lane] = __builtin_bit_cast(float, max((int) (w[b / 4] >> (b % 4 * 8) & 0xffu) + (kBias - t.ev), 0) << 23);
    return t;
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

// The first product takes K as it is held, e2m1 codes and block scales, from the cache to the matrix pipe. Its other operand,
// the queries, is a sum of digits: a row is scaled by a power of two to a largest magnitude in [2, 4) and written as
// d_0 + d_1 + d_2 ..., each the nearest 6-bit e2m3 number, in units of 32^-j, to what the ones before it left (e2m3 has steps
// of at most 1/4 below 4: an eighth is left, 4 units of the next): 5 digits leave 2^-24 of the row's largest element (f32),
// 3 leave 2^-14 (bf16). A product is exact and its sum f32. Operand lane (row r = lane % 16, g = lane / 16) holds the 32
// channels of block g of step u; a head of 64 channels has two blocks, and its lanes g = 2, 3 take the next digit.
template <int D, class T> struct QueryShape {
    static constexpr int kDigits = sizeof(T) == 4 ? 5 : 3;
    static constexpr int kPerStep = D == 64 ? 2 : 1;  // digits of one product
    static constexpr int kSteps = D == 256 ? 2 : 1;   // products of one digit
    static constexpr int N = (kDigits + kPerStep - 1) / kPerStep;
};
typedef uint32_t u6 __attribute__((ext_vector_type(6)));
// MORE: always as many digits as f32 has: a denominator's logarithm is f32, whatever the queries are (3 digits left it 1e-4 off).
// Calls that ask for none pay too: bf16, 32 heads over 8 of 128, without a tree 8 x 30 tokens at 4000 take 43.1 us (36.8 with
// attn's three digits), a prompt of 2801 105 (86), one token at 1500 or 100000 about 1 us more.
template <bool MORE, class T> using DigitType = std::conditional_t<MORE, float, T>;
template <int D, class T> using Digits = u6[QueryShape<D, T>::N][QueryShape<D, T>::kSteps];
// The row is first multiplied by scale * log2(e): scores are log2 units. Returns the block scale of digit 0 (255: the row has a
// NaN or an infinity, and every score is NaN).
// (P: the type whose number of digits it gets.)
template <int D, class P, class T>
__device__ __forceinline__ int query_digits(Digits<D, P> &w, const T *row, bool there, float scale) {
    typedef float v16 __attribute__((ext_vector_type(16)));
    typedef float v32 __attribute__((ext_vector_type(32)));
    using Q = QueryShape<D, P>;
    const int g = threadIdx.x % 64 / 16;
    v16 even[Q::kSteps], odd[Q::kSteps];
    int top = 0;  // bits of the largest magnitude: a NaN's are the largest
#pragma unroll
    for (int u = 0; u < Q::kSteps; ++u) {
        T t[32] = {};
        if (there) __builtin_memcpy(t, row + ((D == 64 ? g & 1 : g) + 4 * u) * 32, sizeof t);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float x = to_f32(t[2 * i]), y = to_f32(t[2 * i + 1]);
            top = max(max(top, __builtin_bit_cast(int, x) & 0x7fffffff), __builtin_bit_cast(int, y) & 0x7fffffff);
            even[u][i] = x, odd[u][i] = y;
        }
    }
    top = max(top, xor_lane_i<16>(top));
    top = max(top, xor_lane_i<32>(top));
    const float in_log2 = scale * kLog2e, amax = __builtin_bit_cast(float, top) * fabsf(in_log2);
    const bool bad = !(amax < INFINITY);
    // (the last digit's scale byte is 125 + k - 25 at least: a smaller row enters with digits of a row at 2^-100)
    const int k = amax < 7.8886090522101181e-31f ? -100 : (int) (__builtin_bit_cast(uint32_t, amax) >> 23) - 126;  // amax < 2^k
    const float f = in_log2 * ldexpf(1.0f, 2 - k);
#pragma unroll
    for (int u = 0; u < Q::kSteps; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) even[u][i] *= f, odd[u][i] *= f;
#pragma unroll
    for (int d = 0; d < Q::N * Q::kPerStep; ++d)
#pragma unroll
        for (int u = 0; u < Q::kSteps; ++u) {
            const float unit = __builtin_bit_cast(float, (uint32_t) (127 - 5 * d) << 23);
            u6 code = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even[u], odd[u], unit);
            // (the conversion writes its result while it still reads its operands, and the compiler lets a result have the
            // registers of operands that end there: these end here)
            asm volatile("" : "+v"(code) : "v"(even[u]), "v"(odd[u]));
            const v32 back = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(code, unit);
#pragma unroll
            for (int i = 0; i < 16; ++i) even[u][i] -= back[2 * i], odd[u][i] -= back[2 * i + 1];
            if constexpr (D == 64) {
                if (d % 2 == 0) w[d / 2][0] = code;
                else
#pragma unroll
                    for (int i = 0; i < 6; ++i) w[d / 2][0][i] = g >= 2 ? code[i] : w[d / 2][0][i];
            } else {
                w[d][u] = code;
            }
        }
    return bad ? 255 : 127 + k - 2;
}

// S^T of 16 keys and 16 query rows: the products of one digit (or pair), of block scale qsc, with every 128 channels.
template <int D> constexpr int kKPieces = D == 256 ? 2 : 1;  // 16-byte pieces of a key that a lane holds
// The digits' block scales, a byte each (the instruction picks one): of the row whose digit 0 has scale qsc0.
template <int D, class T> struct DigitScales {
    static constexpr int W = (QueryShape<D, T>::N + 3) / 4;
    int w[W];
    __device__ __forceinline__ void set(int qsc0) {
        const int first = D == 64 && threadIdx.x % 64 >= 32 ? qsc0 - 5 : qsc0;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            w[i] = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b)
                if (4 * i + b < QueryShape<D, T>::N)
                    w[i] |= (qsc0 == 255 ? 255 : max(first - 5 * QueryShape<D, T>::kPerStep * (4 * i + b), 0)) << (8 * b);
        }
    }
};
template <int SEL> __device__ __forceinline__ f4 score_mfma(i8v a, i8v b, f4 acc, int ksc, int qsc) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 2, 0, ksc, SEL, qsc);
}
template <int D, class T>
__device__ __forceinline__ f4 scores(const u4 (&k)[kKPieces<D>], const int (&ksc)[kKPieces<D>], const u6 (&q)[QueryShape<D, T>::kSteps],
                                     const DigitScales<D, T> &qsc, int n, f4 acc) {
#pragma unroll
    for (int u = 0; u < QueryShape<D, T>::kSteps; ++u) {
        const i8v a = {(int) k[u][0], (int) k[u][1], (int) k[u][2], (int) k[u][3], 0, 0, 0, 0};
        const i8v b = {(int) q[u][0], (int) q[u][1], (int) q[u][2], (int) q[u][3], (int) q[u][4], (int) q[u][5], 0, 0};
        const int w = qsc.w[n / 4];
        acc = n % 4 == 0 ? score_mfma<0>(a, b, acc, ksc[u], w) : n % 4 == 1 ? score_mfma<1>(a, b, acc, ksc[u], w) :
              n % 4 == 2 ? score_mfma<2>(a, b, acc, ksc[u], w) : score_mfma<3>(a, b, acc, ksc[u], w);
    }
    return acc;
}

// A lane's state of one column tile: row r = lane % 16; a lane holds channels 16 dt + 4 g + i of its row in o[dt][i] (in
// units of 2^(ev - 139)). m: the maximum that p and the sums refer to; l: the sum of p, four times the same (a product with
// ones: the matrix pipe has time for it, the vector pipe has none, and p counts as it was rounded).
template <int NB> struct RowState {
    f4 o[2 * NB], l;
    float m;
    __device__ __forceinline__ void reset() {
        m = -INFINITY, l = f4{0, 0, 0, 0};
#pragma unroll
        for (int d = 0; d < 2 * NB; ++d) o[d] = f4{0, 0, 0, 0};
    }
};

// What a tile's scores of a row start from, so that they come as the exponents of p: the row's maximum so far, 2^8 down.
__device__ __forceinline__ float score_origin(float m) { return kPShift - (m == -INFINITY ? 0.0f : m); }

// The positions (from, to] that a row sees; of a row that is not there (its queries are zeros and nothing of it is stored)
// all, so that it never asks for the masked path. Of a tree these are positions before the new tokens, and which of those
// it sees is told by the bits of its token (-1: none).
template <bool MORE> struct Sight {
    int from, to;
};
template <> struct Sight<true> {
    int from, to, tok;
};
// A sequence's new tokens: the position of the first, and a tree's bits of them.
template <bool MORE> struct NewTokens {
    __device__ __forceinline__ NewTokens(const AttnArgs &, const SeqRange &) {}
};
template <> struct NewTokens<true> {
    const uint64_t *sees;
    int first, n, words;
    __device__ __forceinline__ NewTokens(const AttnArgs &a, const SeqRange &r)
        : sees(a.sees ? a.sees + r.q0 * a.words : nullptr), first(r.len - r.n), n(r.n), words(a.words) {}
};
// Of the row of token i of the sequence, if it is there.
template <bool MORE>
__device__ __forceinline__ Sight<MORE> sight(const AttnArgs &a, const SeqRange &r, const NewTokens<MORE> &nt, bool there, int i) {
    const int first = r.len - r.n;
    if constexpr (MORE) {
        if (!there) return {-1, INT32_MAX, -1};
        if (!nt.sees) return {before_window(first + i, a.window), first + i, -1};
        // the window has room for what the bits leave of it; a token that sees no new one, not itself either, sees nothing
        int count = 0;
        for (int w = 0; w < nt.words && 64 * w < nt.n; ++w) {
            const uint64_t bits = nt.sees[(int64_t) i * nt.words + w];
            count += __popcll(nt.n - 64 * w < 64 ? bits & ((1ull << (nt.n - 64 * w)) - 1) : bits);
        }
        if (count == 0) return {-1, -1, -1};
        const int64_t from = a.window ? (int64_t) first + count - a.window - 1 : -1;
        return {(int) min(max(from, (int64_t) -1), (int64_t) first - 1), first - 1, i};
    } else {
        const int pos = first + i;
        return {there ? before_window(pos, a.window) : -1, there ? pos : INT32_MAX};
    }
}
// Bits of the lane's 16 keys (base + 16 g ..) that a row sees; there: the tile's keys that exist.
template <bool MORE>
__device__ __forceinline__ uint32_t seen(const NewTokens<MORE> &nt, const Sight<MORE> &w, int base, uint64_t there) {
    const int g = threadIdx.x % 64 / 16, at = base + 16 * g;
    const int up = w.to - at, dn = w.from + 1 - at;  // the last one, the first one
    uint32_t bits = up < 0 ? 0u : up >= 15 ? 0xffffu : (2u << up) - 1u;
    bits = dn <= 0 ? bits : dn > 15 ? 0u : bits & (0xffffu << dn);
    if constexpr (MORE) {
        const int off = at - nt.first, i = max(off, 0) / 64, sh = max(off, 0) % 64;  // the lane's first key among the new tokens
        if (w.tok >= 0 && off > -16 && i < nt.words) {
            const uint64_t *row = nt.sees + (int64_t) w.tok * nt.words;
            uint64_t m = row[i] >> sh;
            if (sh > 48 && i + 1 < nt.words) m |= row[i + 1] << (64 - sh);
            bits |= (uint32_t) (off < 0 ? m << -off : m) & 0xffffu;
        }
    }
    return bits & (uint32_t) (there >> (16 * g));
}

// One tile's softmax: s (from score_origin) of the lane's 16 keys and CT rows -> p as operand parts, and its sums. Where some
// row does not see every key those become -infinity first; where the maximum has grown, or V's scale (vkeep), m moves and what
// refers to it follows. The common path has one branch around both; inside it they are apart, as the last tile of a row and a
// window's edge need the first alone (five prompts of 1021 tokens with a window of 513: 86 us with both always, 79 apart).
// lx: the lane's own sum of p before it was rounded, where the sum of the rounded one is short of what a logarithm in f32 needs
// (SPLIT = 1: 11 bits, cut toward zero).
template <bool MORE, int NB, int CT, int SPLIT>
__device__ __forceinline__ void softmax_tile(f4 (&s)[CT][4], const NewTokens<MORE> &nt, const Sight<MORE> (&see)[CT], int base, const TileInfo &ti,
                                             float vkeep, RowState<NB> (&st)[CT], h8 (&p)[CT][SPLIT][2], float (&lx)[CT]) {
    const auto largest = [](const f4 (&x)[4]) {
        float top = fmaxf(x[0][0], x[0][1]);
#pragma unroll
        for (int i = 2; i < 16; i += 2) top = fmaxf(fmaxf(top, x[i / 4][i % 4]), x[i / 4][i % 4 + 1]);
        return top;
    };
    // (a lane's own keys will do for the maximum: one that exceeds the row's bound is found by its lane)
    const auto bounded = [&] {
        bool b = vkeep == 1.0f;
#pragma unroll
        for (int c = 0; c < CT; ++c) b = b & (largest(s[c]) <= (st[c].m == -INFINITY ? -INFINITY : kPShift + kLazy));
        return b;
    };
    bool whole = ti.there == ~0ull;
#pragma unroll
    for (int c = 0; c < CT; ++c) whole = whole & (see[c].from < base) & (see[c].to >= base + kTile - 1);
    if (!__all(whole & bounded() & (ti.nan == 0))) {
        if (!__all(whole)) {
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const int bits = (int) seen(nt, see[c], base, ti.there);
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const uint32_t on = (uint32_t) __builtin_amdgcn_sbfe(bits, k, 1);
                    const float x = s[c][k / 4][k % 4];
                    s[c][k / 4][k % 4] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & on) | (0xff800000u & ~on));
                }
            }
        }
        if (ti.nan) {  // a NaN in V is one of the rows that see it
            const uint32_t nan = (uint32_t) (ti.nan >> (16 * (threadIdx.x % 64 / 16)));
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const uint32_t bits = seen(nt, see[c], base, ti.there) & nan;
#pragma unroll
                for (int k = 0; k < 16; ++k) s[c][k / 4][k % 4] = bits >> k & 1 ? __builtin_nanf("") : s[c][k / 4][k % 4];
            }
        }
        if (!__all(bounded())) {
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                float top = largest(s[c]);
                top = fmaxf(top, xor_lane<16>(top));
                top = fmaxf(top, xor_lane<32>(top));
                const float off = st[c].m == -INFINITY ? 0.0f : st[c].m;  // (nothing seen so far: no difference of infinities)
                // (each row by itself: what a row gives does not depend on its neighbours)
                const bool grows = top > (st[c].m == -INFINITY ? -INFINITY : kPShift + kLazy);
                const float to = grows ? top + (off - kPShift) : st[c].m, now = to == -INFINITY ? 0.0f : to;
                const float keep = __builtin_amdgcn_exp2f(st[c].m - now);
#pragma unroll
                for (int t = 0; t < 4; ++t) s[c][t] -= now - off;
                st[c].m = to;
                st[c].l *= keep;
                if constexpr (MORE && SPLIT == 1) lx[c] *= keep;
#pragma unroll
                for (int d = 0; d < 2 * NB; ++d) st[c].o[d] *= keep * vkeep;
            }
        }
    }
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            u4 w[SPLIT];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = __builtin_amdgcn_exp2f(s[c][2 * v + i / 2][i % 2 * 2]), y = __builtin_amdgcn_exp2f(s[c][2 * v + i / 2][i % 2 * 2 + 1]);
                if constexpr (MORE && SPLIT == 1) lx[c] += x + y;
                // toward zero: a second part has the rest, and without one (bf16) the sum of p counts the same values. What is
                // cut, up to 2^-10 of a p, is lost in the output's own rounding: 8 trees of 63 tokens with 64 channels are 1.675e-3
                // (of the norm) from the exact values, 1.659e-3 with f32 all through; a part of them rounds the other way.
                const h2 hi = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(x, y));
                w[0][i] = __builtin_bit_cast(uint32_t, hi);
                if constexpr (SPLIT == 2) {
                    float x1, y1;  // what hi leaves, exactly, without a conversion first (f32, 4096 tokens at 4096: 4% less time)
                    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(x1) : "v"(w[0][i]), "v"(x));
                    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(y1) : "v"(w[0][i]), "v"(y));
                    w[1][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x1, y1));
                }
            }
#pragma unroll
            for (int h = 0; h < SPLIT; ++h) p[c][h][v] = __builtin_bit_cast(h8, w[h]);
        }
    h8 ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = (_Float16) 1.0f;
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int h = SPLIT - 1; h >= 0; --h) st[c].l = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, p[c][h][v], st[c].l, 0, 0, 0);
}

// The natural logarithm of a denominator: sum (2^8 up, as p is) in units of 2^off.
__device__ __forceinline__ float log_of(float off, float sum) {
    return sum == 0.0f ? -INFINITY : (off + (__builtin_amdgcn_logf(sum) - kPShift)) * 0.6931471805599453f;
}

// Result of few rows: 4 channels of one or, with splits, their partial.
template <int D, class T>
__device__ __forceinline__ void store_row(const AttnArgs &a, int64_t tok, int h, int split, int ch, f4 v) {
    if (a.splits > 1) *(f4 *) (a.part + ((split * a.b.n_tok + tok) * a.n_head + h) * D + ch) = v;
    else store4((T *) a.out + tok * a.out_stride + (int64_t) h * D + ch, v);
}

// Where a tile's bytes are. With pages of 64 positions or more a tile lies in one page: every address is the tile's (in
// scalar registers) plus an offset that a lane keeps; smaller pages (SMALL) are looked up for every 16 positions.
template <int D, bool SMALL> struct TileReader {
    static constexpr int NB = D / 32;
    using L = KvParts<D>;
    int P, lane, r, g, last;  // last: the table's last entry
    int64_t head_off;
    const uint8_t *bk, *bv;  // of the lane's K rows (keys 16 (r / 4) ..), and of its own key and V columns (16 g ..)
    int row;                 // of the tile's first position in its page
    bool there;
    int pk, pv;              // table entries of the tile that take() goes to (one of them without SMALL)
    // Asks for a tile's table entries (a tile of the table); take() moves there a step later. Nothing here waits for a load
    // or skips one: a wait would be for every load before it, the next tile's among them.
    __device__ __forceinline__ void ask(const AttnArgs &a, const int32_t *table, int tile) {
        const int at = (tile * kTile) >> a.c.shift;
        if constexpr (SMALL) {
            pk = table[min(at + ((16 * (r / 4)) >> a.c.shift), last)];
            pv = table[min(at + ((16 * g) >> a.c.shift), last)];
        } else {
            pk = pv = table[at];
        }
    }
    __device__ __forceinline__ void take(const AttnArgs &a, int tile) {
        row = (tile * kTile) & (P - 1);
        const auto in = [&](int p) { return p >= 0 && p < a.c.n_pages; };
        if constexpr (SMALL) {
            bk = a.c.pages + (in(pk) ? pk : 0) * a.c.page_bytes + head_off;
            bv = a.c.pages + (in(pv) ? pv : 0) * a.c.page_bytes + head_off;
            there = in(pv);
        } else {
            const int p = __builtin_amdgcn_readfirstlane(pv);
            there = in(p);
            bk = bv = a.c.pages + (there ? p : 0) * a.c.page_bytes + head_off;
        }
    }
    __device__ __forceinline__ void scales(ScaleBytes<NB> &k, ScaleBytes<NB> &v) const {
        const int at = SMALL ? (row + lane) & (P - 1) : row + lane;
        __builtin_memcpy(&k, __builtin_assume_aligned(bv + L::k_scale(P, at), NB), NB);
        __builtin_memcpy(&v, __builtin_assume_aligned(bv + L::v_scale(P, at), NB), NB);
    }
    __device__ __forceinline__ void k(u4 (&x)[4][kKPieces<D>]) const {
        const int at = (SMALL ? (row + 16 * (r / 4)) & (P - 1) : row + 16 * (r / 4)) + r % 4;
        const int block = D == 64 ? g & 1 : g;
        const uint8_t *p = bk + (uint32_t) (at * (D / 2) + block * 16);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int u = 0; u < kKPieces<D>; ++u) x[t][u] = *(const u4 *) (p + 4 * t * (D / 2) + u * 64);
    }
    __device__ __forceinline__ u4 v_block(int j) const {
        const int at = SMALL ? (row + 16 * g) & (P - 1) : row + 16 * g;
        return *(const u4 *) (bv + (uint32_t) (P * (D / 2) + r * P + at) + (uint32_t) (16 * j * P));
    }
    __device__ __forceinline__ void v(u4 (&x)[NB]) const {
        const int at = SMALL ? (row + 16 * g) & (P - 1) : row + 16 * g;
        const uint8_t *p = bv + (uint32_t) (P * (D / 2) + r * P + at);
#pragma unroll
        for (int j = 0; j < NB; ++j) x[j] = *(const u4 *) (p + (uint32_t) (16 * j * P));
    }
};

// The second product of a tile whatever the blocks' sizes: V straight from the cache, in bands of kBand scales, each expanded
// at a scale of its own and added at the row's, E[c] (a lane's, as its row is): the largest that the row has seen so far, of
// kFloor at least. What a row gives depends on no block that it does not see.
template <bool MORE, int D, bool SMALL, int CT, int SPLIT>
__device__ __forceinline__ void v_in_bands(const AttnArgs &a, TileReader<D, SMALL> rd, const int32_t *table, int tile, const TileInfo &ti,
                                           const NewTokens<MORE> &nt, const Sight<MORE> (&see)[CT], const h8 (&p)[CT][SPLIT][2], RowState<D / 32> (&st)[CT], int (&E)[CT]) {
    constexpr int NB = D / 32;
    rd.ask(a, table, tile);
    rd.take(a, tile);
    const int at = SMALL ? (rd.row + 16 * rd.g) & (rd.P - 1) : rd.row + 16 * rd.g, base = tile * kTile;
    const uint32_t keys = (uint32_t) (ti.there >> (16 * rd.g)) & 0xffffu;
    const uint8_t *scale = rd.bv + KvParts<D>::v_scale(rd.P, at);
    int most[CT] = {};
#pragma unroll 1
    for (int i = 0; i < 16; ++i) {
        int e = 0;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int x = scale[i * NB + j];
            e = x == 255 ? e : max(e, x);  // (rows that see a NaN are NaN)
        }
#pragma unroll
        for (int c = 0; c < CT; ++c) most[c] = max(most[c], seen(nt, see[c], base, ti.there) >> i & 1 ? e : 0);
    }
    int from = 0;  // the largest scale that any row sees
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        most[c] = max(most[c], xor_lane_i<16>(most[c]));
        most[c] = max(most[c], xor_lane_i<32>(most[c]));
        const int to = max(E[c], most[c]);
        const float keep = ldexpf(1.0f, E[c] - to);
        E[c] = to;
#pragma unroll
        for (int d = 0; d < 2 * NB; ++d) st[c].o[d] *= keep;
        from = max(from, most[c]);
    }
    from = max(from, xor_lane_i<1>(from));
    from = max(from, xor_lane_i<2>(from));
    from = max(from, xor_lane_i<4>(from));
    from = __builtin_amdgcn_readfirstlane(max(from, xor_lane_i<8>(from)));
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const u4 codes = rd.v_block(j);
#pragma unroll 1
        for (int top = from; top > 0; top -= kBand) {
            float w[16];
            bool any = false;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int e = keys >> i & 1 ? scale[i * NB + j] : 0;
                const bool in = e <= top && e > max(top - kBand, 0);
                any |= in;
                w[i] = in ? __builtin_bit_cast(float, (uint32_t) (e - top + kBias) << 23) : 0.0f;
            }
            if (!__any(any)) continue;
            f4 lo[CT], hi[CT];
#pragma unroll
            for (int c = 0; c < CT; ++c) lo[c] = hi[c] = f4{0, 0, 0, 0};
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                h8 x, y;
                expand_v(codes[2 * v], codes[2 * v + 1], w + 8 * v, x, y);
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int h = SPLIT - 1; h >= 0; --h) {
                        lo[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, p[c][h][v], lo[c], 0, 0, 0);
                        hi[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, p[c][h][v], hi[c], 0, 0, 0);
                    }
            }
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                // (a row that sees nothing of a band more than kBand above its scale has zeros there: any finite unit will do)
                const float unit = ldexpf(1.0f, min(top - E[c], kBand));
                st[c].o[2 * j] += lo[c] * unit, st[c].o[2 * j + 1] += hi[c] * unit;
            }
        }
    }
}

// Few rows (decode, verify): the workgroup's waves take tiles of keys in turn and are joined at the end. A wave's tile goes
// from the pages to registers and stays there: S^T = K Q^T with K's rows in an order that leaves every lane with the 16
// consecutive keys 16 g .. 16 g + 15 of its query row, which is where the second product, O^T = V^T P^T, wants P, and where
// V's bytes (16 consecutive positions of a channel pair) are. Bound by the cache's bytes for one long context (131072 keys of
// 8 heads, bf16: 143 MB in 26 us, 5.5 TB/s; the pages' pattern of loads alone reaches 5.5), by uneven shares for many (48 of
// up to 16000 keys, f32: 272 MB in 59 us, 4.6 TB/s: 920 workgroups have keys and 768 fit at once, so that the busiest place
// does 17 tiles a wave where 10 would be its share; the 260 vector and 56 matrix instructions of a tile, one after another,
// are 26 us), by the start and a few dependent loads for short ones (500 keys: 9 us; 8 sequences of 4096, 4 tokens: two tiles a
// wave, 16 us). What pays is waves, so the queries lie in LDS and the next tile's K is asked for when this one's is used up;
// workgroups of 8 waves, or four waves a SIMD at 128 registers, were slower (48 contexts: 84 and 76 us where this took 74).
// A wave whose blocks of V turn out to be too far apart walks once more, by v_in_bands. REDO: that is known.
template <bool MORE, int D, int CT, bool SMALL, bool REDO, class T>
__device__ __forceinline__ void few_rows(const AttnArgs &a, int row0, int split) {
    constexpr int NB = D / 32, SPLIT = sizeof(T) == 4 ? 2 : 1, NW = kFewWaves;
    constexpr int kScale = 64 * NB + 16 * NB, kJoin = NW / 2 * CT * 2 * NB * 256;
    __shared__ __align__(16) float lds[NW * kScale > kJoin ? NW * kScale : kJoin];
    using Dt = DigitType<MORE, T>;
    using Q = QueryShape<D, Dt>;
    __shared__ __align__(16) uint2 qs[CT][Q::N][Q::kSteps][64][3];
    __shared__ int qscale[CT][16];
    constexpr bool EXACT = MORE && SPLIT == 1;  // the denominator's logarithm takes a sum of its own
    __shared__ float join[NW][EXACT ? 3 : 2][CT * 16];
    const int s = blockIdx.x / a.c.n_kv, head = blockIdx.x % a.c.n_kv;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    int lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
    const SeqRange sr = seq_range(a.b, s);
    const int rows = (int) min((int64_t) sr.n * a.group, (int64_t) INT32_MAX);
    if (row0 >= rows) return;
    const RowTiles rt = row_tiles<MORE>(a, sr, row0, 16 * CT);
    const int chunk = split_chunk(a, rt);
    const int t0 = (int) min((int64_t) rt.t0 + (int64_t) split * chunk, (int64_t) rt.t1);
    const int t1 = min(t0 + chunk, rt.t1);
    if (split > 0 && t0 >= t1) return;  // (split 0 of an empty range writes the zeros)
    const int P = 1 << a.c.shift;

    TileReader<D, SMALL> rd;
    rd.P = P, rd.lane = lane, rd.r = r, rd.g = g, rd.head_off = head * kv_head_bytes(D, P);
    u4 kraw[4][kKPieces<D>], vraw[NB];
    ScaleBytes<NB> swk, swv;  // the scale bytes of the lane's key
    const int32_t *table = a.b.table + s * a.b.table_stride;
    rd.last = (int) a.b.table_stride - 1;
    const auto begin = [&] {
        const int tile = t0 + wave;
        if (tile >= t1) return;
        rd.ask(a, table, tile);
        rd.take(a, tile);
        rd.ask(a, table, min(tile + NW, t1 - 1));
        rd.scales(swk, swv), rd.k(kraw), rd.v(vraw);
    };
    begin();

    if (wave < CT) {  // a wave a column tile
        const int row = row0 + 16 * wave + r, i = row / a.group;
        Digits<D, Dt> w;
        const int scale = query_digits<D, Dt>(w, (const T *) a.q + (sr.q0 + i) * a.q_stride + (int64_t) (head * a.group + row % a.group) * D,
                                             row < rows, a.scale);
#pragma unroll
        for (int n = 0; n < Q::N; ++n)
#pragma unroll
            for (int u = 0; u < Q::kSteps; ++u)
#pragma unroll
                for (int i2 = 0; i2 < 3; ++i2) qs[wave][n][u][lane][i2] = make_uint2(w[n][u][2 * i2], w[n][u][2 * i2 + 1]);
        if (g == 0) qscale[wave][r] = scale;
    }
    RowState<NB> st[CT];
    const NewTokens<MORE> nt(a, sr);
    __shared__ Sight<MORE> sights[MORE ? CT : 1][16];  // (a tree's: the registers are counted, 60 tokens at 100000: 177 -> 169 us)
    Sight<MORE> see[CT];
    float lx[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int row = row0 + 16 * c + r;
        see[c] = sight(a, sr, nt, row < rows, row / a.group);
        if (MORE && wave == 0 && g == 0) sights[MORE ? c : 0][r] = see[c];
    }
    __syncthreads();
    DigitScales<D, Dt> qsc[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) qsc[c].set(qscale[c][r]);

    float *vsc = lds + wave * kScale;
    uint8_t *ksb = (uint8_t *) (vsc + 64 * NB);  // K's scale bytes, [64 keys][NB]
    int ev = kFloor, E[CT];
    // Returns whether some row may have lost something of V; with `all`, none does, and E has the rows' scales.
    const auto walk = [&](auto all) {
        bool low = false;
        ev = kFloor;
#pragma unroll
        for (int c = 0; c < CT; ++c) st[c].reset(), lx[c] = 0.0f;
        for (int tile = t0 + wave; tile < t1; tile += NW) {
            const int base = tile * kTile, key = base + lane;
            *(ScaleBytes<NB> *) (ksb + lane * NB) = swk;
            const TileInfo ti = v_scales<NB>(swv, rd.there && key >= rt.lo && key < rt.hi, ev, vsc);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_sched_barrier(0);
            int ksc[4][kKPieces<D>];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int u = 0; u < kKPieces<D>; ++u) ksc[t][u] = ksb[(16 * (r / 4) + 4 * t + r % 4) * NB + (D == 64 ? g & 1 : g) + 4 * u];
            f4 sc[CT][4];
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int t = 0; t < 4; ++t) sc[c][t] = f4{1, 1, 1, 1} * score_origin(st[c].m);
#pragma unroll
            for (int n = 0; n < Q::N; ++n)  // the largest digit first: the rest adds to small numbers
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    u6 q[Q::kSteps];
#pragma unroll
                    for (int u = 0; u < Q::kSteps; ++u)
#pragma unroll
                        for (int i = 0; i < 3; ++i) {
                            const uint2 w = qs[c][n][u][lane][i];
                            q[u][2 * i] = w.x, q[u][2 * i + 1] = w.y;
                        }
#pragma unroll
                    for (int t = 0; t < 4; ++t) sc[c][t] = scores<D, Dt>(kraw[t], ksc[t], q, qsc[c], n, sc[c][t]);
                }
            // K is used up here, before the next tile's is asked for: the products may not sink below the loads, which would
            // keep both tiles' registers
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int t = 0; t < 4; ++t) asm volatile("" : "+v"(sc[c][t]));
            __builtin_amdgcn_sched_barrier(0);
            // (the last tile is asked for once more behind the end: it is in the cache, and the loop has no branch)
            rd.take(a, min(tile + NW, t1 - 1));
            rd.ask(a, table, min(tile + 2 * NW, t1 - 1));
            rd.scales(swk, swv), rd.k(kraw);
            const float vkeep = all ? 1.0f : ldexpf(1.0f, ev - ti.ev);
            ev = ti.ev;
            h8 p[CT][SPLIT][2];
            if constexpr (MORE)
#pragma unroll
                for (int c = 0; c < CT; ++c) see[c] = sights[c][r];
            softmax_tile<MORE, NB, CT, SPLIT>(sc, nt, see, base, ti, vkeep, st, p, lx);
            if constexpr (all) {
                v_in_bands<MORE, D, SMALL>(a, rd, table, tile, ti, nt, see, p, st, E);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                continue;
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
                    __builtin_amdgcn_sched_barrier(0);  // (one step's operands at a time: the registers are counted)
                }
            low |= ti.low;
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int d = 0; d < 2 * NB; ++d) asm volatile("" : "+v"(st[c].o[d]));  // (and V likewise)
            rd.v(vraw);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        return low || ev > kGrown;
    };
    const bool again = REDO || walk(std::false_type{});
#pragma unroll
    for (int c = 0; c < CT; ++c) E[c] = again ? kFloor : ev;
    if (again) {
        if (!REDO) {
            // (so that nothing of its addresses is kept through the first walk)
            asm volatile("" : "+v"(lane), "+v"(r), "+v"(g));
            rd.lane = lane, rd.r = r, rd.g = g;
            begin();
        }
        walk(std::true_type{});
    }

    // join the waves: the common maximum and sum of every row, then the sums in a tree over registers of equal layout
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        if (g == 0) join[wave][0][16 * c + r] = st[c].m, join[wave][1][16 * c + r] = st[c].l[0];
        if constexpr (EXACT) {
            lx[c] += xor_lane<16>(lx[c]);
            lx[c] += xor_lane<32>(lx[c]);
            if (g == 0) join[wave][EXACT ? 2 : 0][16 * c + r] = lx[c];
        }
    }
    __syncthreads();
    float top[CT], sum[CT], den[CT];  // den: for the logarithm
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int row = 16 * c + r;
        top[c] = join[0][0][row];
#pragma unroll
        for (int w = 1; w < NW; ++w) top[c] = fmaxf(top[c], join[w][0][row]);
        const int h = head * a.group + (row0 + row) % a.group;
        const bool sink = a.splits == 1 && a.sinks && row0 + row < rows;
        const float sk = sink ? a.sinks[h] * kLog2e : -INFINITY;
        const float with = fmaxf(top[c], sk);
        const float off = with == -INFINITY ? 0.0f : with;
        sum[c] = sink ? __builtin_amdgcn_exp2f(sk - off + kPShift) : 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) sum[c] += join[w][1][row] * __builtin_amdgcn_exp2f(join[w][0][row] - off);
        den[c] = sum[c];
        if constexpr (EXACT) {
            den[c] = sink ? __builtin_amdgcn_exp2f(sk - off + kPShift) : 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) den[c] += join[w][2][row] * __builtin_amdgcn_exp2f(join[w][0][row] - off);
        }
        if (MORE && a.splits == 1) den[c] = log_of(off, den[c]);
        const int unit = E[c] - kBias - (a.splits > 1 ? kPart : 0);
        const float f = sum[c] == 0.0f ? 0.0f : ldexpf(__builtin_amdgcn_exp2f(st[c].m - off) / sum[c], unit);
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
        if (a.splits > 1 && g == 0) a.part_ml[(split * a.b.n_tok + tok) * a.n_head + h] = make_float2(top[c], EXACT ? den[c] : sum[c]);
        if (MORE && a.splits == 1 && g == 0 && a.lse) a.lse[tok * a.n_head + h] = den[c];
    }
}
template <bool MORE, int D, int CT, bool SMALL, class T>
__global__ __launch_bounds__(64 * kFewWaves, D == 256 || CT == 2 ? 2 : 3) void k_attn_few(AttnArgs a) {
    few_rows<MORE, D, CT, SMALL, false, T>(a, blockIdx.y * 16 * CT, blockIdx.z);
}
// The rows of k_attn_many's workgroups that have to be done again: none as a rule, which takes 4-5 us with the launch. In one
// workgroup with the pass that found them, their scalars cost the f32 form's loop its registers (29 spilled instead of 9).
template <bool MORE, int D, bool SMALL, class T>
__global__ __launch_bounds__(64 * kFewWaves, 2) void k_attn_redo(AttnArgs a, int row_tiles) {
    for (int tile = blockIdx.y; tile < row_tiles; tile += gridDim.y) {
        if (!((const uint32_t *) a.redo)[(int64_t) blockIdx.x * row_tiles + tile]) continue;
        for (int sub = 0; sub < kManyRows / 16; ++sub) {
            few_rows<MORE, D, 1, SMALL, true, T>(a, tile * kManyRows + 16 * sub, 0);
            __syncthreads();
        }
    }
}

// Many rows (prompts): a workgroup takes 128 rows, 32 a wave, and walks over the keys; its waves expand a tile's V together,
// a tile ahead, into LDS as the second product wants it, [channel][64 keys] (rows 16 bytes apart in banks: a lane's 16-byte
// reads of 16 channels touch every bank once). K needs no expansion: each wave reads its codes, which the workgroup's first
// reader brings into L1, and keeps them in registers with the digits of its queries. A workgroup whose blocks of V turn out to
// be too far apart says so: its rows are then done again by the form of few rows (with low blocks in this loop, 4096 tokens
// at 4096 took 539 us instead of 423).
// 4096 tokens at 4096 keys, 32 heads over 8 of 128, bf16: 395 us, 1.04 PFLOP/s (a library product of 8192^3: 1.22; f32,
// whose five digits and two halves of p are 112 matrix instructions instead of 60: 566 us). A tile
// costs a wave 60 matrix instructions (about 970 cycles) and 147 vector instructions with 32 exponentials (about 890), of
// which two waves a SIMD overlap little: the matrix pipe is busy 38% of the time. More waves do not fit the registers; the
// expansion of V among the first product's instructions, which helps bf16 (by 3%), costs heads of 256 channels 6 to 18%.
__device__ __forceinline__ void tile_barrier() {
    // LDS only: the tiles asked for stay in flight
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
template <bool MORE, int D, bool SMALL, class T>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_attn_many(AttnArgs a) {
    constexpr int NB = D / 32, SPLIT = sizeof(T) == 4 ? 2 : 1, NW = 4, CT = 2;
    constexpr int VS = 64 + 8;             // f16 values between V rows
    constexpr int MB = (NB + NW - 1) / NW; // blocks that a wave expands: wave, wave + 4
    using Dt = DigitType<MORE, T>;
    using Q = QueryShape<D, Dt>;
    __shared__ __align__(16) _Float16 vt[2][D * VS];
    __shared__ __align__(16) float vsc_all[NW][MB * 64];
    __shared__ __align__(16) uint8_t ksb_all[NW][64 * NB];
    __shared__ Sight<MORE> sights[NW][CT][16];  // (the registers are counted)
    const int s = blockIdx.x / a.c.n_kv, head = blockIdx.x % a.c.n_kv;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
    const SeqRange sr = seq_range(a.b, s);
    const int rows = (int) min((int64_t) sr.n * a.group, (int64_t) INT32_MAX);
    // the last rows, which see the most keys, first
    const int row0 = ((int) gridDim.y - 1 - (int) blockIdx.y) * kManyRows;
    uint8_t *redo = a.redo + ((int64_t) blockIdx.x * gridDim.y + row0 / kManyRows) * NW + wave;
    if (row0 >= rows) {
        if (lane == 0) *redo = 0;
        return;
    }
    const RowTiles rt = row_tiles<MORE>(a, sr, row0, kManyRows);
    const NewTokens<MORE> nt(a, sr);
    const int t0 = rt.t0, t1 = rt.t1, P = 1 << a.c.shift, first = sr.len - sr.n;
    float *vsc = vsc_all[wave];
    uint8_t *ksb = ksb_all[wave];

    TileReader<D, SMALL> rd;  // at the next tile, when its K is asked for; then at the one after it, for V
    rd.P = P, rd.lane = lane, rd.r = r, rd.g = g, rd.head_off = head * kv_head_bytes(D, P), rd.last = (int) a.b.table_stride - 1;
    const int32_t *table = a.b.table + s * a.b.table_stride;
    u4 kraw[4][kKPieces<D>], vraw[MB];
    ScaleBytes<NB> swk, swv, unused;
    const auto load_v = [&] {  // the wave's blocks; a wave without one asks for another's
#pragma unroll
        for (int m = 0; m < MB; ++m) vraw[m] = rd.v_block((wave + NW * m) % NB);
    };
    const auto expand = [&](int buf) {
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            const int j = wave + NW * m;
            if (j >= NB) break;
            h8 lo[2], hi[2];
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                float w[8];
                *(f4 *) w = *(const f4 *) (vsc + m * 64 + 16 * g + 8 * v);
                *(f4 *) (w + 4) = *(const f4 *) (vsc + m * 64 + 16 * g + 8 * v + 4);
                expand_v(vraw[m][2 * v], vraw[m][2 * v + 1], w, lo[v], hi[v]);
            }
            h8 *at = (h8 *) (vt[buf] + (32 * j + r) * VS + 16 * g);
            at[0] = lo[0], at[1] = lo[1];
            at += 16 * VS / 8;
            at[0] = hi[0], at[1] = hi[1];
        }
    };
    const auto wave_sync = [] {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    int ev = kFloor;
    int low = 0;
    TileInfo ti{}, next{};
    if (t0 < t1) {
        rd.ask(a, table, t0);
        rd.take(a, t0);
        rd.scales(swk, swv), rd.k(kraw), load_v();
        rd.ask(a, table, min(t0 + 1, t1 - 1));
    }
    Digits<D, Dt> q[CT];
    RowState<NB> st[CT];
    DigitScales<D, Dt> qsc[CT];
    const int w0 = row0 + wave * 32;  // the wave's rows, and the positions that they see at most and at least
    const bool tree = MORE && a.sees;
    const int most = w0 >= rows ? -1 : tree ? sr.len - 1 : first + min(w0 + 31, rows - 1) / a.group;
    const int least = before_window(tree ? first : first + w0 / a.group, a.window) + 1;
    float lx[CT] = {};
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int row = w0 + 16 * c + r, i = row / a.group;
        const bool there = row < rows;
        if (g == 0) sights[wave][c][r] = sight(a, sr, nt, there, i);
        qsc[c].set(query_digits<D, Dt>(q[c], (const T *) a.q + (sr.q0 + i) * a.q_stride + (int64_t) (head * a.group + row % a.group) * D, there, a.scale));
        st[c].reset();
    }
    if (t0 < t1) {
        const int key = t0 * kTile + lane;
        ti = v_scales<NB, NW>(swv, rd.there && key >= rt.lo && key < rt.hi, ev, vsc, wave);
        wave_sync();
        expand(0);
        wave_sync();
        rd.take(a, min(t0 + 1, t1 - 1));
        rd.scales(unused, swv), load_v();
        rd.ask(a, table, min(t0 + 2, t1 - 1));
        tile_barrier();
    }
    for (int tile = t0; tile < t1; ++tile) {
        const int base = tile * kTile, buf = (tile - t0) & 1;
        const bool active = base <= most && base + kTile - 1 >= least;
        f4 sc[CT][4];
        if (active) {
            *(ScaleBytes<NB> *) (ksb + lane * NB) = swk;
            wave_sync();
            int ksc[4][kKPieces<D>];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int u = 0; u < kKPieces<D>; ++u) ksc[t][u] = ksb[(16 * (r / 4) + 4 * t + r % 4) * NB + (D == 64 ? g & 1 : g) + 4 * u];
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int t = 0; t < 4; ++t) sc[c][t] = f4{1, 1, 1, 1} * score_origin(st[c].m);
            __builtin_amdgcn_s_setprio(0);  // (matrix instructions wait for the pipe: the other waves' vector work goes first)
#pragma unroll
            for (int n = 0; n < Q::N; ++n)  // the largest digit first: the rest adds to small numbers
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int t = 0; t < 4; ++t) sc[c][t] = scores<D, Dt>(kraw[t], ksc[t], q[c][n], qsc[c], n, sc[c][t]);
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int t = 0; t < 4; ++t) asm volatile("" : "+v"(sc[c][t]));  // (K is used up before the next one is asked for)
        }
        __builtin_amdgcn_s_setprio(1);
        __builtin_amdgcn_sched_barrier(0);
        rd.scales(swk, unused), rd.k(kraw);
        if (active) {
            const float vkeep = ldexpf(1.0f, ev - ti.ev);
            ev = ti.ev;
            h8 p[CT][SPLIT][2];
            Sight<MORE> see[CT];
#pragma unroll
            for (int c = 0; c < CT; ++c) see[c] = sights[wave][c][r];
            softmax_tile<MORE, NB, CT, SPLIT>(sc, nt, see, base, ti, vkeep, st, p, lx);
            __builtin_amdgcn_s_setprio(0);
            const h8 *at = (const h8 *) (vt[buf] + r * VS + 16 * g);
#pragma unroll
            for (int d = 0; d < 2 * NB; ++d)
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const h8 x = at[d * 16 * VS / 8 + v];
#pragma unroll
                    for (int c = 0; c < CT; ++c)
#pragma unroll
                        for (int h = SPLIT - 1; h >= 0; --h) st[c].o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, p[c][h][v], st[c].o[d], 0, 0, 0);
                    if (SPLIT == 2 && v == 1) __builtin_amdgcn_sched_barrier(0);  // (the registers are counted: no more reads ahead)
                }
        }
        __builtin_amdgcn_s_setprio(1);
        const int after = min(tile + 1, t1 - 1), key = after * kTile + lane;
        next = v_scales<NB, NW>(swv, rd.there && key >= rt.lo && key < rt.hi, ti.ev, vsc, wave);
        wave_sync();
        if (tile + 1 < t1) expand(buf ^ 1);
        wave_sync();
        rd.take(a, min(tile + 2, t1 - 1));
        rd.scales(unused, swv), load_v();
        rd.ask(a, table, min(tile + 3, t1 - 1));
        low |= (int) ti.low;
        ti = next;
        tile_barrier();
    }
    if (lane == 0) *redo = low | (ev > kGrown);
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int row = w0 + 16 * c + r;
        if constexpr (MORE && SPLIT == 1) {
            lx[c] += xor_lane<16>(lx[c]);
            lx[c] += xor_lane<32>(lx[c]);
        }
        if (row >= rows) continue;
        const int64_t tok = sr.q0 + row / a.group;
        const int h = head * a.group + row % a.group;
        float sum = st[c].l[0], off = st[c].m;
        if constexpr (MORE) {
            float den = SPLIT == 1 ? lx[c] : sum, from = off;
            if (a.sinks) {
                const float sk = a.sinks[h] * kLog2e;
                from = fmaxf(off, sk);
                const float o = from == -INFINITY ? 0.0f : from;
                den = den * __builtin_amdgcn_exp2f(off - o) + __builtin_amdgcn_exp2f(sk - o + kPShift);
            }
            if (g == 0 && a.lse) a.lse[tok * a.n_head + h] = log_of(from == -INFINITY ? 0.0f : from, den);
        }
        if (a.sinks) {
            const float sk = a.sinks[h] * kLog2e;
            off = fmaxf(off, sk);
            const float o = off == -INFINITY ? 0.0f : off;
            sum = sum * __builtin_amdgcn_exp2f(st[c].m - o) + __builtin_amdgcn_exp2f(sk - o + kPShift);
        }
        const float o = off == -INFINITY ? 0.0f : off;
        const float f = sum == 0.0f ? 0.0f : ldexpf(__builtin_amdgcn_exp2f(st[c].m - o) / sum, ev - kBias);
#pragma unroll
        for (int d = 0; d < 2 * NB; ++d) store4((T *) a.out + tok * a.out_stride + (int64_t) h * D + 16 * d + 4 * g, st[c].o[d] * f);
    }
}

// The splits of a row into its result, a lane D / 64 channels: a workgroup a row, whose waves take the splits in turn, or
// (WAVE_ROW) a wave a row. At most 64 splits: one a lane for their weights.
template <bool MORE, int D, bool WAVE_ROW, class T>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a, int rows_per_wg) {
    constexpr int C = D / 64, NW = 4;
    __shared__ float part[WAVE_ROW ? 1 : NW][D], weight[NW][64];
    const int s = blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const SeqRange sr = seq_range(a.b, s);
    const int at = WAVE_ROW ? blockIdx.x * NW + wave : blockIdx.x, i = at / a.n_head, h = at % a.n_head;
    if (i >= sr.n) return;  // (the whole workgroup, or a wave that shares nothing)
    const int64_t tok = sr.q0 + i, first = tok * a.n_head + h, step = a.b.n_tok * a.n_head;
    const int row = i * a.group + h % a.group, row0 = row / rows_per_wg * rows_per_wg;
    const RowTiles rt = row_tiles<MORE>(a, sr, row0, rows_per_wg);
    const int chunk = split_chunk(a, rt);
    const int n = max(1, (rt.t1 - rt.t0 + chunk - 1) / chunk);  // splits that have tiles (the first one in any case)
    const float sk = a.sinks ? a.sinks[h] * kLog2e : -INFINITY;
    const float2 ml = lane < n ? a.part_ml[lane * step + first] : make_float2(-INFINITY, 0.0f);
    const float top = fmaxf(lanes_max<64>(ml.x), sk);
    const float off = top == -INFINITY ? 0.0f : top;
    const float f = ml.y == 0.0f ? 0.0f : ml.y * __builtin_amdgcn_exp2f(ml.x - off);
    const float sum = lanes_sum<64>(f) + (a.sinks ? __builtin_amdgcn_exp2f(sk - off + kPShift) : 0.0f);
    weight[wave][lane] = sum == 0.0f ? 0.0f : f / sum;
    if (MORE && a.lse && lane == 0 && (WAVE_ROW || wave == 0)) a.lse[first] = log_of(off, sum);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float o[C] = {};
    const float *src = a.part + first * D + lane * C;
#pragma unroll 8
    for (int k = WAVE_ROW ? 0 : wave; k < n; k += WAVE_ROW ? 1 : NW) {
        const float wk = weight[wave][k];
        float v[C];
        __builtin_memcpy(v, __builtin_assume_aligned(src + k * step * D, 4 * C), sizeof v);
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] += wk == 0.0f ? 0.0f : wk * v[c];
    }
    if constexpr (!WAVE_ROW) {
#pragma unroll
        for (int c = 0; c < C; ++c) part[wave][lane * C + c] = o[c];
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] = (part[0][lane * C + c] + part[1][lane * C + c]) + (part[2][lane * C + c] + part[3][lane * C + c]);
    }
    T t[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        o[c] *= (float) (1 << kPart);
        if constexpr (sizeof(T) == 4) t[c] = o[c];
        else t[c] = to_bf16(o[c]);
    }
    __builtin_memcpy((T *) a.out + tok * a.out_stride + (int64_t) h * D + lane * C, t, sizeof t);
}

AttnArgs attn_args(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x, const host::AttnPlan &p, const void *q, void *out, void *ws) {
    AttnArgs a{};
    a.c = host::kv_view(c), a.b = host::kv_batch(b);
    a.q = q, a.out = out, a.sinks = x->sinks;
    a.part = (float *) ws, a.part_ml = (float2 *) ((uint8_t *) ws + p.ml_off);
    a.q_stride = x->q_stride, a.out_stride = x->out_stride;
    a.n_head = x->n_head, a.group = x->n_head / c->n_head_kv, a.window = x->window;
    a.splits = p.splits, a.chunk = p.chunk, a.scale = x->scale;
    a.redo = (uint8_t *) ws;
    return a;
}

template <bool MORE>
int attn_launch(const AttnArgs &a, const host::AttnPlan &p, const FnsKvCache *c, const FnsKvBatch *b, int dtype, const char *what, hipStream_t st) {
    const int n_seq = b->n_seq, max_q = b->max_q, head_dim = c->head_dim;
    const dim3 grid((unsigned) ((int64_t) n_seq * a.c.n_kv), (unsigned) p.row_tiles, (unsigned) p.splits);
    const bool small = (1 << a.c.shift) < kTile;
    auto few = [&](auto dim, auto ct, auto type) {
        constexpr int D = decltype(dim)::value, CT = decltype(ct)::value;
        if (small) hipLaunchKernelGGL((k_attn_few<MORE, D, CT, true, decltype(type)>), grid, dim3(64 * kFewWaves), 0, st, a);
        else hipLaunchKernelGGL((k_attn_few<MORE, D, CT, false, decltype(type)>), grid, dim3(64 * kFewWaves), 0, st, a);
    };
    auto join = [&](auto dim, auto type) {
        constexpr int D = decltype(dim)::value;
        const int64_t rows = std::min<int64_t>(max_q, a.b.n_tok) * a.n_head;
        // a workgroup a row where there are many splits and all of them are resident at once (64 splits of 32 rows: 5 us); with
        // few splits its start outweighs them (8 of 2048 rows: 6.1 us, a wave each 3.6)
        if (p.splits > 16 && rows * n_seq <= 2048)
            hipLaunchKernelGGL((k_attn_join<MORE, D, false, decltype(type)>), dim3((unsigned) rows, (unsigned) n_seq), dim3(256), 0, st, a, p.rows);
        else
            hipLaunchKernelGGL((k_attn_join<MORE, D, true, decltype(type)>), dim3((unsigned) ((rows + 3) / 4), (unsigned) n_seq), dim3(256), 0, st, a, p.rows);
    };
    auto by_type = [&](auto dim, auto type) {
        constexpr int D = decltype(dim)::value;
        if (p.rows == kManyRows) {
            if (small) hipLaunchKernelGGL((k_attn_many<MORE, D, true, decltype(type)>), grid, dim3(256), 0, st, a);
            else hipLaunchKernelGGL((k_attn_many<MORE, D, false, decltype(type)>), grid, dim3(256), 0, st, a);
            FNS_TRY(host::check_launch(what));
            const dim3 some(grid.x, std::min(grid.y, (512 + grid.x - 1) / grid.x));
            if (small) hipLaunchKernelGGL((k_attn_redo<MORE, D, true, decltype(type)>), some, dim3(64 * kFewWaves), 0, st, a, (int) p.row_tiles);
            else hipLaunchKernelGGL((k_attn_redo<MORE, D, false, decltype(type)>), some, dim3(64 * kFewWaves), 0, st, a, (int) p.row_tiles);
        } else if constexpr (D == 256) few(dim, std::integral_constant<int, 1>{}, type);
        else if (p.rows == 16) few(dim, std::integral_constant<int, 1>{}, type);
        else few(dim, std::integral_constant<int, 2>{}, type);
        FNS_TRY(host::check_launch(what));
        if (p.splits > 1) join(dim, type);
        return host::check_launch(what);
    };
    const auto by_dim = [&](auto dim) { return dtype == FNS_TYPE_F32 ? by_type(dim, float{}) : by_type(dim, uint16_t{}); };
    if (head_dim == 64) return by_dim(std::integral_constant<int, 64>{});
    if (head_dim == 128) return by_dim(std::integral_constant<int, 128>{});
    return by_dim(std::integral_constant<int, 256>{});
}

}  // namespace

}  // namespace fns
