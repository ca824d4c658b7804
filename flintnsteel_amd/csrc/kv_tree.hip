// kv_tree.hip - what changes a paged 4-bit cache (fns_kv.hpp) after its tokens were appended: the bits of a tree of drafted
// tokens, the accepted path made the sequence's own, eviction by accumulated attention weight. For MI355X gfx950.
#include "fns_kv.hpp"

#include <algorithm>
#include <cmath>

#include "fns/kernels.h"
#include "fns_common.hpp"
#include "fns_host.hpp"
#include "fns_internal.hpp"

namespace fns {

using namespace fns::dev;

namespace {

constexpr int kMaxWords = 16, kMaxNew = 64 * kMaxWords;

// A workgroup a sequence, a thread a token: up the parents, which get smaller at every step, once to see that they end at -1
// and how many they are, once to set the bits, a word at a time. Bound by the longest path's LDS reads, one after another (26
// tokens: 2.7 us; 24 sequences of 32: 3.7; 1000 tokens of a tree with two children each 10.9): a tree that is a line is the
// worst there is, with work that grows by its square (lines of 26, 200 and 1000 tokens: 4.5, 22 and 257 us).
__global__ __launch_bounds__(256) void k_tree_plan(BatchView b, const int32_t *parents, const int32_t *base, int words, uint64_t *sees,
                                                   int32_t *pos) {
    __shared__ int up[kMaxNew];
    const int s = blockIdx.x;
    const SeqRange r = seq_range(b, s);
    const int n = min(r.n, 64 * words);
    for (int i = threadIdx.x; i < n; i += 256) {
        const int p = parents[r.q0 + i];
        up[i] = p >= -1 && p < i ? p : -2;
    }
    __syncthreads();
    const int from = base ? base[s] : r.len - r.n;
    for (int i = threadIdx.x; i < n; i += 256) {
        int depth = 0, j = i;
        while (up[j] >= 0) j = up[j], ++depth;
        const bool in = up[j] == -1;
        if (pos) pos[r.q0 + i] = from + (in ? depth : 0);
        uint64_t *row = sees + (r.q0 + i) * words;
        j = in ? i : -1;
        for (int w = words - 1; w >= 0; --w) {
            uint64_t bits = 0;
            while (j >= 64 * w) bits |= 1ull << (j - 64 * w), j = up[j];  // (j < 0 ends it: the words are not below 0)
            row[w] = bits;
        }
    }
}

// A weight as a number whose order is the weights': 0 is no position, the largest one that is kept in any case.
__device__ __forceinline__ uint32_t weight_key(float w) {
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);  // (-0 + 0 is 0)
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xfffffffeu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct EvictArgs {
    KvView c;
    BatchView b;
    const float *w;
    int32_t *kept, *new_len;
    int budget, first, recent;
};

__device__ __forceinline__ int seq_len(const KvView &c, const BatchView &b, int s) {
    return (int) min((int64_t) max(b.kv_len[s], 0), b.table_stride << c.shift);
}

// Inclusive sum over the wave's lanes up to each, by moves within rows of 16 lanes and from the end of rows to later ones.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
    return v;
}

// Which positions a sequence's kv head keeps. The budget-th largest key digit by digit (11, 11, 10 bits), the counts of a
// digit's values in LDS; then the positions in order, those above it and as many equal ones as there is room for.
constexpr int kSel = 1024, kBins = 2048, kSelWaves = kSel / 64;
// Of the counts, in banks beside each other: lanes with the same value wait for each other (many positions may have no weight at
// all: 16 sequences of 20000 without, 36 us and a move; copies in the same bank 48; with weights 27 both).
constexpr int kCopies = 4;
__device__ __forceinline__ int digit_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
__device__ __forceinline__ bool digit_counts(int pass, uint32_t key, uint32_t prefix) {  // whether a key is counted in a pass
    return key != 0 && (pass == 0 || key >> (pass == 1 ? 21 : 10) == prefix);
}
// Keys of positions 4 i .. 4 i + 3 (which lie in one page) of a sequence of n.
__device__ __forceinline__ void weight_keys(const EvictArgs &a, int s, int head, int n, int i, uint32_t (&k)[4]) {
    const int at = (int) (4u * i), page = (uint32_t) at < (uint32_t) n ? page_of(a.c, a.b, s, at) : -1;
    float4 w = {};
    if (page >= 0) w = *(const float4 *) (a.w + (((int64_t) page * a.c.n_kv + head) << a.c.shift) + (at & ((1 << a.c.shift) - 1)));
    const float v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int p = at + j;
        k[j] = page < 0 || p >= n ? 0u : p < a.first || p >= n - a.recent ? 0xffffffffu : weight_key(v[j]);
    }
}
// What the counts of a digit's values say, by a workgroup: the digit of the want-th largest (thread t brings the counts of digits
// 2047 - 2 t and 2046 - 2 t), how many are above it, and how many there are at all.
struct Digit {
    int digit, above, total;
};
__device__ __forceinline__ Digit find_digit(int hi, int lo, int want, bool clip, int *waves, int *found) {
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    int sum = wave_scan(hi + lo), all = 0;
    if (lane == 63) waves[wave] = sum;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelWaves; ++w) {
        const int x = waves[w];
        sum += w < wave ? x : 0, all += x;
    }
    if (clip) want = min(want, all);
    const int above = sum - hi - lo;  // keys of larger digits
    if (want > above && want <= sum) {
        const bool second = want > above + hi;
        found[0] = kBins - 1 - 2 * tid - (second ? 1 : 0);
        found[1] = above + (second ? hi : 0);
    }
    __syncthreads();
    return {found[0], found[1], all};
}
// Keys above the prefix in the low half, equal ones in the high half; and their places, after so many of either.
__device__ __forceinline__ int above_and_equal(const uint32_t (&k)[4], uint32_t prefix) {
    int c = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) c += (k[j] > prefix ? 1 : 0) + (k[j] == prefix ? 1 << 16 : 0);
    return c;
}
__device__ __forceinline__ void put_kept(int32_t *kept, const uint32_t (&k)[4], uint32_t prefix, int want, int quad, int above, int equal) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool is = k[j] == prefix;
        if (k[j] > prefix || (is && equal < want)) kept[above + min(equal, want)] = 4 * quad + j;
        above += k[j] > prefix, equal += is;
    }
}

// Up to 4096 Q positions: a workgroup, of which a thread has its 4 Q keys in registers. Bound by what waits for what: the table,
// the weights, three times counting and the search among 2048 counts, the scan of the kept (4160 positions of 8 heads: 8.2 us,
// 16 sequences of up to 20000: 16.7).
template <int Q> __global__ __launch_bounds__(kSel) void k_kv_select(EvictArgs a) {
    __shared__ __align__(16) int bins[3][kBins][kCopies];
    __shared__ int waves[Q][kSelWaves], found[3][2];
    const int s = blockIdx.x / a.c.n_kv, head = blockIdx.x % a.c.n_kv, tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int n = seq_len(a.c, a.b, s), quads = n / 4 + (n % 4 > 0);
    int32_t *kept = a.kept + (int64_t) blockIdx.x * a.budget;
    uint32_t own[Q][4];
#pragma unroll
    for (int q = 0; q < Q; ++q) weight_keys(a, s, head, n, tid + q * kSel, own[q]);
#pragma unroll
    for (int i = 0; i < 3 * kCopies * kBins / 4 / kSel; ++i) ((int4 *) bins)[tid + i * kSel] = make_int4(0, 0, 0, 0);
    __syncthreads();
    int want = a.budget, keep = 0;
    uint32_t prefix = 0;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
#pragma unroll
        for (int q = 0; q < Q; ++q)
            if (q * kSel < quads)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (digit_counts(pass, own[q][j], prefix))
                        atomicAdd(&bins[pass][(own[q][j] >> digit_shift(pass)) & (pass == 2 ? 1023 : 2047)][lane % kCopies], 1);
        __syncthreads();
        int hi = 0, lo = 0;
#pragma unroll
        for (int i = 0; i < kCopies; i += 4) {
            const int4 x = *(const int4 *) &bins[pass][kBins - 2 - 2 * tid][i], y = *(const int4 *) &bins[pass][kBins - 1 - 2 * tid][i];
            lo += (x.x + x.y) + (x.z + x.w), hi += (y.x + y.y) + (y.z + y.w);
        }
        const Digit d = find_digit(hi, lo, want, pass == 0, waves[0], found[pass]);
        if (pass == 0) keep = want = min(want, d.total);
        if (want > 0) prefix = (prefix << (pass == 2 ? 10 : 11)) | (uint32_t) d.digit, want -= d.above;
    }
    // `want` of the keys equal to `prefix` are kept: the first ones
    if (keep > 0) {
        int before[Q];
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            if (q * kSel >= quads) break;
            const int c = above_and_equal(own[q], prefix), both = wave_scan(c);
            if (lane == 63) waves[q][wave] = both;
            before[q] = both - c;
        }
        __syncthreads();
        int all = 0;  // (at most 32768 of either fit a half)
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            if (q * kSel >= quads) break;
            int at = all + before[q];
#pragma unroll
            for (int w = 0; w < kSelWaves; ++w) {
                const int x = waves[q][w];
                at += w < wave ? x : 0, all += x;
            }
            put_kept(kept, own[q], prefix, want, tid + q * kSel, at & 0xffff, at >> 16);
        }
    }
    for (int i = keep + tid; i < a.budget; i += kSel) kept[i] = -1;
    if (head == 0 && tid == 0) a.new_len[s] = keep;
}

// Longer sequences: chunks of 16384 positions, a workgroup each, which meet between launches: the counts of each digit in memory
// (whole numbers, whose order of adding does not matter), then how many of each chunk are kept. 124729 positions of 2 heads: 38 us in
// six launches, about 115 in one workgroup that reads its weights four times.
constexpr int kChunkQuads = 4, kChunk = 4 * kSel * kChunkQuads;
struct alignas(16) SelectState {  // (counts are read two at a time)
    int bins[3][kBins];
    int want[4], keep;  // want[p]: after p passes
    uint32_t prefix[4];
};
template <int PHASE> __global__ __launch_bounds__(kSel) void k_kv_select_chunks(EvictArgs a, SelectState *states, int32_t *counts, int chunks) {
    __shared__ __align__(16) int bins[kBins][kCopies];
    __shared__ int waves[kChunkQuads][kSelWaves], found[2], sums[2];
    const int s = blockIdx.x / a.c.n_kv, head = blockIdx.x % a.c.n_kv, tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int n = seq_len(a.c, a.b, s), used = n / kChunk + (n % kChunk > 0);
    SelectState &st = states[blockIdx.x];
    if (PHASE == 0) {  // (one workgroup a kv head)
        for (int i = tid; i < 3 * kBins; i += kSel) ((int *) st.bins)[i] = 0;
        if (tid == 0) st.want[0] = a.budget, st.prefix[0] = 0;
        return;
    }
    const bool lead = blockIdx.y == 0;  // (does what is there once, also for a sequence without positions)
    if ((int) blockIdx.y >= used && !lead) return;
    // after PHASE - 1 passes
    int want = st.want[0];
    uint32_t prefix = 0;
    if (PHASE > 1) {
        constexpr int P = PHASE == 5 ? 3 : PHASE - 1;
        if (PHASE < 5) {
            want = st.want[P - 1], prefix = st.prefix[P - 1];
            const int2 two = *(const int2 *) &st.bins[P - 1][kBins - 2 - 2 * tid];
            const Digit d = find_digit(two.y, two.x, want, P == 1, waves[0], found);
            if (P == 1) want = min(want, d.total);
            const int keep = want;
            if (want > 0) prefix = (prefix << (P == 3 ? 10 : 11)) | (uint32_t) d.digit, want -= d.above;
            if (lead && tid == 0) {
                st.want[P] = want, st.prefix[P] = prefix;
                if (P == 1) st.keep = keep;
            }
        } else {
            want = st.want[3], prefix = st.prefix[3];
        }
    }
    int32_t *kept = a.kept + (int64_t) blockIdx.x * a.budget;
    const int keep = PHASE == 5 ? st.keep : 0;
    int above = 0, equal = 0;  // of the chunks before this one
    int done = 0;              // chunks counted in them
    for (int chunk = blockIdx.y; chunk < used; chunk += gridDim.y) {
        uint32_t own[kChunkQuads][4];
#pragma unroll
        for (int q = 0; q < kChunkQuads; ++q) weight_keys(a, s, head, n, chunk * (kChunk / 4) + tid + q * kSel, own[q]);
        if (PHASE <= 3) {
            constexpr int pass = PHASE - 1;
#pragma unroll
            for (int i = 0; i < kCopies * kBins / 4 / kSel; ++i) ((int4 *) bins)[tid + i * kSel] = make_int4(0, 0, 0, 0);
            __syncthreads();
#pragma unroll
            for (int q = 0; q < kChunkQuads; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (digit_counts(pass, own[q][j], prefix))
                        atomicAdd(&bins[(own[q][j] >> digit_shift(pass)) & (pass == 2 ? 1023 : 2047)][lane % kCopies], 1);
            __syncthreads();
            for (int i = tid; i < kBins; i += kSel) {
                int c = 0;
#pragma unroll
                for (int j = 0; j < kCopies; ++j) c += bins[i][j];
                if (c) atomicAdd(&st.bins[pass][i], c);
            }
            __syncthreads();
        } else {
            int before[kChunkQuads];
#pragma unroll
            for (int q = 0; q < kChunkQuads; ++q) {
                const int c = above_and_equal(own[q], prefix), both = wave_scan(c);
                if (lane == 63) waves[q][wave] = both;
                before[q] = both - c;
            }
            __syncthreads();
            int all = 0;
#pragma unroll
            for (int q = 0; q < kChunkQuads; ++q) {
                before[q] += all;
#pragma unroll
                for (int w = 0; w < kSelWaves; ++w) {
                    const int x = waves[q][w];
                    before[q] += w < wave ? x : 0, all += x;
                }
            }
            int32_t *mine = counts + ((int64_t) blockIdx.x * chunks + chunk) * 2;
            if (PHASE == 4) {
                if (tid == 0) mine[0] = all & 0xffff, mine[1] = all >> 16;
            } else if (keep > 0) {
                // what the chunks before have, by the first wave
                if (wave == 0) {
                    int x = 0, y = 0;
                    for (int i = done + lane; i < chunk; i += 64) {
                        const int32_t *c = counts + ((int64_t) blockIdx.x * chunks + i) * 2;
                        x += c[0], y += c[1];
                    }
                    x = lanes_sum_i<64>(x), y = lanes_sum_i<64>(y);
                    if (lane == 0) sums[0] = x, sums[1] = y;
                }
                __syncthreads();
                above += sums[0], equal += sums[1], done = chunk;
#pragma unroll
                for (int q = 0; q < kChunkQuads; ++q)
                    put_kept(kept, own[q], prefix, want, chunk * (kChunk / 4) + tid + q * kSel, above + (before[q] & 0xffff), equal + (before[q] >> 16));
            }
            __syncthreads();
        }
    }
    if (PHASE == 5) {
        const int64_t workers = min((int64_t) max(used, 1), (int64_t) gridDim.y);
        for (int64_t i = keep + (int64_t) blockIdx.y * kSel + tid; i < a.budget; i += workers * kSel) kept[i] = -1;
        if (head == 0 && lead && tid == 0) a.new_len[s] = keep;
    }
}

struct MoveArgs {
    KvView c;
    BatchView b;
    const int32_t *to;  // the table that positions go to
    int64_t to_stride;
    const int32_t *list, *count;  // list[row][list_stride], row: a sequence's kv head, or (NEW) the sequence; count: NEW, per sequence
    int64_t list_stride;
    const float *w;
    float *w_out;
    int32_t *new_len;  // NEW
};

// Where the i-th position of a list comes from and goes to: pages (to = -1: it is not moved) and rows.
struct Place {
    int from, to, row_from, row_to;
};
// Positions list[0], list[1], ... of a sequence's kv head go to positions 0, 1, ... (NEW: both counted from its first new token,
// the list one of the sequence).
template <bool NEW> struct Places {
    const int32_t *list;
    int64_t first;
    int n, fresh;
    __device__ __forceinline__ Places(const MoveArgs &a, int s, int row) : first(0), fresh(0) {
        if constexpr (NEW) {
            const SeqRange r = seq_range(a.b, s);
            first = (int64_t) r.len - r.n, fresh = r.n;
            n = (int) min((int64_t) min(max(a.count[s], 0), r.n), a.list_stride);
            list = a.list + s * a.list_stride;
        } else {
            n = (int) min(a.list_stride, (int64_t) seq_len(a.c, a.b, s));  // (no more are kept)
            list = a.list + row * a.list_stride;
        }
    }
    __device__ __forceinline__ int pick(int64_t i) const { return i < n ? list[i] : -1; }
    __device__ __forceinline__ Place at(const MoveArgs &a, int s, int64_t i, int x) const {  // x = pick(i)
        Place p{-1, -1, 0, 0};
        if (x < 0 || (NEW && x >= fresh)) return p;
        const int64_t src = first + x, dst = first + i;
        if (src == dst && a.to == a.b.table) return p;
        if (src < 0 || dst < 0 || src > INT32_MAX || dst > INT32_MAX) return p;
        const int P = 1 << a.c.shift;
        const int64_t e = dst >> a.c.shift;
        const int q = e < a.to_stride ? a.to[s * a.to_stride + e] : -1;
        p.from = page_of(a.c, a.b, s, (int) src);
        p.to = p.from >= 0 && q >= 0 && q < a.c.n_pages ? q : -1;
        p.row_from = (int) src & (P - 1), p.row_to = (int) dst & (P - 1);
        return p;
    }
};

// In place, any number: a workgroup moves a part of a position (64 bytes of K's codes, 16 byte columns of V, or the scale bytes
// and the weight) for 1024 positions at a time, all of which are read before the first is written, and goes over all of them in
// order: what it writes lies before everything that it has yet to read, since the list ascends (a list of new tokens, which need
// not, has at most 1024). Bound by what waits for what, a step at a time: a step's data, the next one's pages and the list of the
// one after are asked for together (130000 positions of 8 heads cut to 100000: 354 us with the choice, 488 step by step; 9000 of 256
// channels to 8192, 4 sequences of 2 heads: 39 and 106). The bytes alone would be about 49 us of the 354: a head and part is one
// workgroup, 48 of them for 8 heads of 128 on 256 CUs.
constexpr int kMove = 1024;
template <int N, bool NEW, class Pos, class Load, class Store>
__device__ __forceinline__ void walk(const MoveArgs &a, const Places<NEW> &places, int s, Pos pos, Load load, Store store) {
    Place p[N], then[N];
    int x[N];
#pragma unroll
    for (int u = 0; u < N; ++u) p[u] = places.at(a, s, pos(u), places.pick(pos(u)));
#pragma unroll
    for (int u = 0; u < N; ++u) x[u] = places.pick(kMove + pos(u));
    for (int64_t i0 = 0; i0 < places.n; i0 += kMove) {
#pragma unroll
        for (int u = 0; u < N; ++u)
            if (p[u].to >= 0) load(u, p[u]);
#pragma unroll
        for (int u = 0; u < N; ++u) then[u] = places.at(a, s, i0 + kMove + pos(u), x[u]), x[u] = places.pick(i0 + 2 * kMove + pos(u));
        __syncthreads();
#pragma unroll
        for (int u = 0; u < N; ++u) {
            if (p[u].to >= 0) store(u, p[u]);
            p[u] = then[u];
        }
    }
}
template <int D> constexpr int kMoveK = D == 64 ? 2 : 4;             // 16-byte pieces of K of a part
template <int D> constexpr int kMoveParts = D / 32 / kMoveK<D> + 1 + D / 32;
template <int D, bool NEW> __global__ __launch_bounds__(kMove) void k_kv_walk(MoveArgs a) {
    constexpr int NB = D / 32, N = kMoveK<D>, KP = D / 32 / N;
    const int s = blockIdx.x / a.c.n_kv, head = blockIdx.x % a.c.n_kv, part = blockIdx.y, tid = threadIdx.x, P = 1 << a.c.shift;
    const Places<NEW> places(a, s, blockIdx.x);
    if (NEW && head == 0 && part == 0 && tid == 0) a.new_len[s] = (int) max(places.first + places.n, (int64_t) 0);
    using L = KvParts<D>;
    const int64_t head_off = head * kv_head_bytes(D, P);
    const auto at = [&](int page) { return a.c.pages + page * a.c.page_bytes + head_off; };
    const auto one = [&](int) { return tid; };
    if (part < KP) {
        uint4 x[N];
        const int piece = part * N + tid % N;
        walk<N>(a, places, s, [&](int u) { return (u * kMove + tid) / N; },
                [&](int u, const Place &p) { x[u] = *(const uint4 *) (at(p.from) + L::k_row(P, p.row_from) + piece * 16); },
                [&](int u, const Place &p) { *(uint4 *) (at(p.to) + L::k_row(P, p.row_to) + piece * 16) = x[u]; });
    } else if (part == KP) {
        uint8_t k[NB], v[NB];
        float w = 0.0f;
        walk<1>(a, places, s, one,
                [&](int, const Place &p) {
                    __builtin_memcpy(k, __builtin_assume_aligned(at(p.from) + L::k_scale(P, p.row_from), NB), NB);
                    __builtin_memcpy(v, __builtin_assume_aligned(at(p.from) + L::v_scale(P, p.row_from), NB), NB);
                    if (a.w) w = a.w[(((int64_t) p.from * a.c.n_kv + head) << a.c.shift) + p.row_from];
                },
                [&](int, const Place &p) {
                    __builtin_memcpy(__builtin_assume_aligned(at(p.to) + L::k_scale(P, p.row_to), NB), k, NB);
                    __builtin_memcpy(__builtin_assume_aligned(at(p.to) + L::v_scale(P, p.row_to), NB), v, NB);
                    if (a.w) a.w_out[(((int64_t) p.to * a.c.n_kv + head) << a.c.shift) + p.row_to] = w;
                });
    } else {
        const int j = 16 * (part - KP - 1);
        uint8_t x[16];
        walk<1>(a, places, s, one,
                [&](int, const Place &p) {
                    const uint8_t *src = at(p.from) + L::v_col(P, j) + p.row_from;
#pragma unroll
                    for (int u = 0; u < 16; ++u) x[u] = src[(int64_t) u * P];
                },
                [&](int, const Place &p) {
                    uint8_t *dst = at(p.to) + L::v_col(P, j) + p.row_to;
#pragma unroll
                    for (int u = 0; u < 16; ++u) dst[(int64_t) u * P] = x[u];
                });
    }
}

// To other pages, or at most W positions in all: a workgroup W positions of a kv head, whose places are looked up once; all is read
// before anything is written. Few tokens (an accepted path) are bound by what waits for what: the list, the table, the bytes (one
// path of 6: 3.4 us). Kept positions by V's byte columns, of whose lines they are parts: 2048 of each of 16 sequences of up to
// 20000, 8 heads of 128, are 73 MB to move, but take 26.2 us, a copy of 130 MB, since of every line some position is kept.
template <int D, int W, bool NEW> __global__ __launch_bounds__(256) void k_kv_copy(MoveArgs a) {
    constexpr int NB = D / 32, NP = D / 32, KR = (W * NP + 255) / 256, COLS = D / 2 * W / 256;  // a thread's pieces of K, bytes of V
    static_assert(D / 2 * W % 256 == 0 && W <= 64, "columns are dealt out evenly, and scales and weights have a thread each");
    __shared__ Place place[W];
    const int s = blockIdx.x / a.c.n_kv, head = blockIdx.x % a.c.n_kv, tid = threadIdx.x, P = 1 << a.c.shift;
    const Places<NEW> places(a, s, blockIdx.x);
    const int64_t i0 = (int64_t) blockIdx.y * W;
    if (NEW && head == 0 && tid == 0) a.new_len[s] = (int) max(places.first + places.n, (int64_t) 0);
    if (i0 >= places.n) return;
    if (tid < W) place[tid] = places.at(a, s, i0 + tid, places.pick(i0 + tid));
    __syncthreads();
    using L = KvParts<D>;
    const int64_t head_off = head * kv_head_bytes(D, P);
    const auto from = [&](const Place &p) { return a.c.pages + p.from * a.c.page_bytes + head_off; };
    const auto to = [&](const Place &p) { return a.c.pages + p.to * a.c.page_bytes + head_off; };
    uint4 k[KR];
#pragma unroll
    for (int u = 0; u < KR; ++u) {
        const int i = tid + 256 * u;
        if (i < W * NP && place[i / NP].to >= 0) k[u] = *(const uint4 *) (from(place[i / NP]) + L::k_row(P, place[i / NP].row_from) + i % NP * 16);
    }
    const Place own = place[tid % W];  // V, scales and the weight: a thread's position
    uint8_t v[COLS] = {}, e[NB];
    float w = 0.0f;
    const int kind = tid / W, col = kind * COLS;  // its byte columns; the first W threads also K's scales, the next V's, then the weights
    if (own.to >= 0) {
        const uint8_t *src = from(own);
#pragma unroll
        for (int u = 0; u < COLS; ++u) v[u] = src[L::v_col(P, col + u) + own.row_from];
        if (kind < 2)
            __builtin_memcpy(e, __builtin_assume_aligned(src + (kind == 0 ? L::k_scale(P, own.row_from) : L::v_scale(P, own.row_from)), NB), NB);
        else if (kind == 2 && a.w)
            w = a.w[(((int64_t) own.from * a.c.n_kv + head) << a.c.shift) + own.row_from];
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < KR; ++u) {
        const int i = tid + 256 * u;
        if (i < W * NP && place[i / NP].to >= 0) *(uint4 *) (to(place[i / NP]) + L::k_row(P, place[i / NP].row_to) + i % NP * 16) = k[u];
    }
    uint8_t *dst = to(own);
    if constexpr (COLS % 4 == 0 && !NEW) {
        // four lanes have four consecutive positions, aligned: turned, a lane has four positions of a column, one store
        int all = own.to >= 0;
        all &= xor_lane_i<1>(all);
        all &= xor_lane_i<2>(all);
        const uint32_t q = tid % 4, pick = q | (4 + q) << 8;
#pragma unroll
        for (int u = 0; u < COLS; u += 4) {
            const uint32_t x = v[u] | (uint32_t) v[u + 1] << 8 | (uint32_t) v[u + 2] << 16 | (uint32_t) v[u + 3] << 24;
            const uint32_t x0 = __builtin_amdgcn_update_dpp(0, x, 0x00, 0xf, 0xf, false), x1 = __builtin_amdgcn_update_dpp(0, x, 0x55, 0xf, 0xf, false);
            const uint32_t x2 = __builtin_amdgcn_update_dpp(0, x, 0xaa, 0xf, 0xf, false), x3 = __builtin_amdgcn_update_dpp(0, x, 0xff, 0xf, 0xf, false);
            const uint32_t y = __builtin_amdgcn_perm(x1, x0, pick | 0x0c0c0000u) | __builtin_amdgcn_perm(x3, x2, pick << 16 | 0x0c0cu);
            if (all) *(uint32_t *) (dst + L::v_col(P, col + u + (int) q) + (own.row_to & ~3)) = y;
        }
        if (!all && own.to >= 0)
#pragma unroll
            for (int u = 0; u < COLS; ++u) dst[L::v_col(P, col + u) + own.row_to] = v[u];
    } else if (own.to >= 0) {
#pragma unroll
        for (int u = 0; u < COLS; ++u) dst[L::v_col(P, col + u) + own.row_to] = v[u];
    }
    if (own.to >= 0) {
        if (kind < 2)
            __builtin_memcpy(__builtin_assume_aligned(dst + (kind == 0 ? L::k_scale(P, own.row_to) : L::v_scale(P, own.row_to)), NB), e, NB);
        else if (kind == 2 && a.w)
            a.w_out[(((int64_t) own.to * a.c.n_kv + head) << a.c.shift) + own.row_to] = w;
    }
}

template <bool NEW> int move(const MoveArgs &a, int D, int n_seq, const char *what, hipStream_t st) {
    const unsigned heads = (unsigned) (n_seq * a.c.n_kv);
    const auto by_dim = [&](auto dim) {
        constexpr int DD = decltype(dim)::value;
        const auto copy = [&](auto width, unsigned steps) {
            hipLaunchKernelGGL((k_kv_copy<DD, decltype(width)::value, NEW>), dim3(heads, steps), dim3(256), 0, st, a);
        };
        const std::integral_constant<int, 64> most{};
        bool done = false;
        if constexpr (NEW) {
            if ((done = a.list_stride <= 16)) copy(std::integral_constant<int, 16>{}, 1u);
            else if ((done = a.list_stride <= 64)) copy(most, 1u);
        } else if ((done = a.to != a.b.table && a.list_stride <= 64 * 65535)) {
            copy(most, (unsigned) ((a.list_stride + 63) / 64));
        }
        if (!done) hipLaunchKernelGGL((k_kv_walk<DD, NEW>), dim3(heads, kMoveParts<DD>), dim3(kMove), 0, st, a);
        return host::check_launch(what);
    };
    if (D == 64) return by_dim(std::integral_constant<int, 64>{});
    if (D == 128) return by_dim(std::integral_constant<int, 128>{});
    return by_dim(std::integral_constant<int, 256>{});
}

}  // namespace

namespace impl {

int rope_scaled(int rope_dim, double base, double factor, double original, double fast, double slow, float *inv_freq, float *magnitude) {
    if (rope_dim <= 0 || rope_dim % 2 || !inv_freq || !magnitude)
        return host::set_error(host::ERR_SHAPE, "rope_scaled: an even rope_dim and two outputs are needed (%d)", rope_dim);
    if (!(base > 1.0) || !(factor >= 1.0) || !(original >= 1.0) || !(slow > 0.0) || !(fast > slow) || !std::isfinite(base) ||
        !std::isfinite(factor) || !std::isfinite(original) || !std::isfinite(fast))
        return host::set_error(host::ERR_SHAPE, "rope_scaled: base above 1, factor and original of at least 1, fast above slow above 0");
    const double pi = 3.14159265358979323846;
    // the pair (as a real number) that turns `turns` times over the original positions
    const auto at = [&](double turns) { return rope_dim * std::log(original / (turns * 2.0 * pi)) / (2.0 * std::log(base)); };
    // The ramp starts at a pair and, as the published rule has it, ends at an index below rope_dim, which may lie behind the last
    // pair: then none is divided fully. It is empty where the first pair is slow already (all are divided), or the last one fast.
    const double lo = std::max(std::floor(at(fast)), 0.0), hi = std::min(std::ceil(at(slow)), rope_dim - 1.0);
    for (int i = 0; i < rope_dim / 2; ++i) {
        const double f = std::pow(base, -2.0 * i / rope_dim);
        const double slowed = i >= hi ? 1.0 : i <= lo ? 0.0 : (i - lo) / (hi - lo);
        inv_freq[i] = (float) (f * (1.0 - slowed) + f / factor * slowed);
    }
    *magnitude = (float) (0.1 * std::log(factor) + 1.0);
    return host::OK;
}

int tree_plan(const FnsKvBatch *b, const int32_t *parents, const int32_t *base, int words, uint64_t *sees, int32_t *pos, hipStream_t st) {
    // (a batch is checked together with a cache; this call needs none)
    const FnsKvCache none{1, 64, 16, 1, (void *) 16};
    FNS_TRY(host::kv_check(&none, b, "tree_plan"));
    if (words < 1 || words > kMaxWords || b->max_q > 64 * words)
        return host::set_error(host::ERR_SHAPE, "tree_plan: words must be 1..16 and hold max_q tokens (%d for %d)", words, b->max_q);
    if (b->n_seq == 0 || b->n_tok == 0 || b->max_q == 0) return host::OK;
    if (!parents || !sees) return host::set_error(host::ERR_SHAPE, "tree_plan: null argument");
    hipLaunchKernelGGL(k_tree_plan, dim3((unsigned) b->n_seq), dim3(256), 0, st, host::kv_batch(b), parents, base, words, sees, pos);
    return host::check_launch("tree_plan");
}

namespace {

// Positions that a sequence of a call can have at all, by its table (max_kv is no bound), and how they are gone over: the table's
// width decides, not the lengths, so that results hold for any. A wide table costs a short sequence its one launch (4160 positions
// of 8 heads in place: 22.2 us, behind a table of 32768 positions 23.7, of 131072 42.4; 300 positions: 10.1, 11.6, 30.1).
constexpr int64_t kOneSelect = 32 * kSel;
int select_chunks(int64_t room) { return (int) ((std::min<int64_t>(room, INT32_MAX) + kChunk - 1) / kChunk); }

}  // namespace

int kv_evict_workspace(const FnsKvCache *c, const FnsKvBatch *b, size_t *bytes) {
    FNS_TRY(host::kv_check(c, b, "kv_evict"));
    if (!bytes) return host::set_error(host::ERR_SHAPE, "kv_evict_workspace: null output");
    const int64_t room = b->table_stride * c->page_size;
    *bytes = room <= kOneSelect ? 0 : (size_t) b->n_seq * c->n_head_kv * (sizeof(SelectState) + (size_t) select_chunks(room) * 8);
    return host::OK;
}

int kv_evict(const FnsKvCache *c, const FnsKvBatch *b, const FnsKvEvict *x, hipStream_t st) {
    FNS_TRY(host::kv_check(c, b, "kv_evict"));
    if (!x) return host::set_error(host::ERR_SHAPE, "kv_evict: null arguments");
    if (x->budget < 1 || x->budget > (1 << 30) || x->first < 0 || x->recent < 0 || (int64_t) x->first + x->recent > x->budget)
        return host::set_error(host::ERR_SHAPE, "kv_evict: budget must be 1..2^30 and hold first and recent (%d, %d, %d)", x->budget, x->first, x->recent);
    if (x->to_stride < 0 || x->to_stride > INT32_MAX || (x->to_table && x->to_stride == 0))
        return host::set_error(host::ERR_SHAPE, "kv_evict: a table needs its stride");
    if (b->n_seq == 0) return host::OK;
    if (!x->weights || !x->weights_out || !x->kept || !x->new_len || ((uintptr_t) x->weights & 15))
        return host::set_error(host::ERR_SHAPE, "kv_evict: null argument, or weights that are not 16-byte aligned");
    if (x->new_len == b->kv_len) return host::set_error(host::ERR_SHAPE, "kv_evict: new_len must not be kv_len");
    if (x->to_table == b->page_table) return host::set_error(host::ERR_SHAPE, "kv_evict: to_table must not be the batch's (NULL: in place)");
    if (!x->to_table && x->weights_out != x->weights)
        return host::set_error(host::ERR_SHAPE, "kv_evict: in place the weights move in place too");
    size_t need = 0;
    FNS_TRY(kv_evict_workspace(c, b, &need));
    if (need && (!x->workspace || x->workspace_bytes < need || ((uintptr_t) x->workspace & 15)))
        return host::set_error(host::ERR_NOMEM, "kv_evict: workspace of %zu bytes, %zu needed (16-byte aligned)", x->workspace ? x->workspace_bytes : 0, need);
    EvictArgs a{host::kv_view(c), host::kv_batch(b), x->weights, x->kept, x->new_len, x->budget, x->first, x->recent};
    const unsigned heads = (unsigned) (b->n_seq * c->n_head_kv);
    const auto select = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(heads), dim3(kSel), 0, st, a); };
    const int64_t room = b->table_stride * c->page_size;
    if (room <= 4 * kSel) select(k_kv_select<1>);
    else if (room <= 8 * kSel) select(k_kv_select<2>);
    else if (room <= 16 * kSel) select(k_kv_select<4>);
    else if (room <= kOneSelect) select(k_kv_select<8>);
    else {
        const int chunks = select_chunks(room);
        SelectState *states = (SelectState *) x->workspace;
        int32_t *counts = (int32_t *) (states + heads);
        const auto phase = [&](auto kern, unsigned n) { hipLaunchKernelGGL(kern, dim3(heads, n), dim3(kSel), 0, st, a, states, counts, chunks); };
        const unsigned wgs = (unsigned) std::min(chunks, 65535);
        phase(k_kv_select_chunks<0>, 1u);
        phase(k_kv_select_chunks<1>, wgs);
        phase(k_kv_select_chunks<2>, wgs);
        phase(k_kv_select_chunks<3>, wgs);
        phase(k_kv_select_chunks<4>, wgs);
        phase(k_kv_select_chunks<5>, wgs);
    }
    FNS_TRY(host::check_launch("kv_evict"));
    MoveArgs m{a.c, a.b, x->to_table ? x->to_table : b->page_table, x->to_table ? x->to_stride : b->table_stride, x->kept, nullptr,
               x->budget, x->weights, x->weights_out, nullptr};
    return move<false>(m, c->head_dim, b->n_seq, "kv_evict", st);
}

int kv_keep(const FnsKvCache *c, const FnsKvBatch *b, const FnsKvKeep *x, hipStream_t st) {
    FNS_TRY(host::kv_check(c, b, "kv_keep"));
    if (!x) return host::set_error(host::ERR_SHAPE, "kv_keep: null arguments");
    if (x->stride < 1 || x->stride > kMove)
        return host::set_error(host::ERR_SHAPE, "kv_keep: lists of 1..%d new tokens (%lld)", kMove, (long long) x->stride);
    if (b->n_seq == 0) return host::OK;
    if (!x->kept || !x->n_kept || !x->new_len) return host::set_error(host::ERR_SHAPE, "kv_keep: null argument");
    if (x->new_len == b->kv_len || x->new_len == x->n_kept) return host::set_error(host::ERR_SHAPE, "kv_keep: new_len must not be kv_len or n_kept");
    MoveArgs m{host::kv_view(c), host::kv_batch(b), b->page_table, b->table_stride, x->kept, x->n_kept, x->stride, x->weights,
               x->weights, x->new_len};
    return move<true>(m, c->head_dim, b->n_seq, "kv_keep", st);
}

}  // namespace impl

namespace k {
void tree_plan(const FnsKvBatch &batch, const int32_t *parents, const int32_t *base, int words, uint64_t *sees, int32_t *pos, hipStream_t st) {
    host::abort_on_error(impl::tree_plan(&batch, parents, base, words, sees, pos, st), "tree_plan");
}
void kv_evict(const FnsKvCache &cache, const FnsKvBatch &batch, const FnsKvEvict &x, hipStream_t st) {
    host::abort_on_error(impl::kv_evict(&cache, &batch, &x, st), "kv_evict");
}
void kv_keep(const FnsKvCache &cache, const FnsKvBatch &batch, const FnsKvKeep &x, hipStream_t st) {
    host::abort_on_error(impl::kv_keep(&cache, &batch, &x, st), "kv_keep");
}
}  // namespace k

}  // namespace fns
