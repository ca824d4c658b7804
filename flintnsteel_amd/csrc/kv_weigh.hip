// kv_weigh.hip - the attention weight that every cached position gets from a batch's new tokens, over the paged 4-bit cache
// (fns_kv.hpp), MI355X gfx950:
//   w[j] = past[j] + sum over the rows (tokens, heads of the group) that see j of exp(x_j - lse),  x_j = scale * q . K_j.
// The product is attention's first one (fns_attn.hpp: K as it is held against the queries' digits, here always as many as f32
// needs) with the operands exchanged: a lane has four rows of one key, and the sum over rows stays in it. Scores start at -lse,
// so that they come as exponents.
#include "fns_attn.hpp"

#include <cmath>
#include <cstddef>

namespace fns {

namespace {

constexpr int kRowTile = 16;
constexpr int kFewTiles = 4;    // row tiles that a workgroup of few rows holds
constexpr int64_t kMidSteps = 4096;
template <int D> constexpr int kMidPhases = D == 256 ? 2 : 4;
template <int D> constexpr int kMidTiles = D == 256 ? 8 : 16;  // and of sixteen waves, in all of a CU's memory
constexpr int key_tiles(int D) { return D == 256 ? 4 : 8; }     // 16-key tiles of a wave of many rows (the registers are counted)
constexpr int key_block(int D) { return 4 * 16 * key_tiles(D); }  // keys of its workgroup

// Sixteen rows as the product takes them.
template <int D> struct RowImage {
    using Q = QueryShape<D, float>;
    uint4 low[Q::N][Q::kSteps][64];   // a lane's 32 digits: 16 bytes,
    uint2 high[Q::N][Q::kSteps][64];  // and 8
    static constexpr int kHalves = D == 64 ? 2 : 1;  // (of 64 channels lanes below 32 and the others have different digits)
    int scale[DigitScales<D, float>::W][kHalves][kRowTile];  // block scales of the digits
    float start[kRowTile];  // -lse in log2 units; -infinity: the row adds nothing
    int from[kRowTile], to[kRowTile], tok[kRowTile];  // Sight
    int any[4];             // the largest `from`, the least `to`, the least `from`, the last position that any row sees
};

struct WeighArgs {
    AttnArgs a;  // cache, batch, q, heads, window, tree
    const float *lse, *past;
    float *weights;
    void *rows;         // many rows: RowImage [n_seq * n_kv][row_tiles]
    int64_t row_tiles;
    int32_t *plan;      // [n_seq * n_kv][blocks + 1] the (block, row tile) steps before a block
    float *part;        // [n_seq * n_kv][shares][2][block] sums over some of a block's rows
    int blocks, shares, block;  // blocks of keys by the host's number; workgroups of a kv head; key_block
};

// The image of rows row0 .. row0 + 15 of a sequence's kv head, by a wave.
template <int D, class T>
__device__ __forceinline__ void make_image(const WeighArgs &x, const SeqRange &sr, const NewTokens<true> &nt, int head, int rows, int row0, RowImage<D> &o) {
    using Q = QueryShape<D, float>;
    const AttnArgs &a = x.a;
    const int lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
    const int row = row0 + r, i = row / a.group, h = head * a.group + row % a.group;
    const bool there = row0 < rows && r < rows - row0;
    Sight<true> see = sight(a, sr, nt, there, i);
    const int64_t tok = sr.q0 + i;
    const float lse = there ? x.lse[tok * a.n_head + h] : INFINITY;
    bool on = fabsf(lse) < INFINITY;
    Digits<D, float> w;
    const int scale = query_digits<D, float>(w, (const T *) a.q + tok * a.q_stride + (int64_t) h * D, on, a.scale);
    on = on && scale != 255 && (!nt.sees || see.tok >= 0);  // (a token without bits sees nothing)
#pragma unroll
    for (int n = 0; n < Q::N; ++n)
#pragma unroll
        for (int u = 0; u < Q::kSteps; ++u) {
            const u6 d = w[n][u];
            o.low[n][u][lane] = on ? make_uint4(d[0], d[1], d[2], d[3]) : make_uint4(0, 0, 0, 0);
            o.high[n][u][lane] = on ? make_uint2(d[4], d[5]) : make_uint2(0, 0);
        }
    if (!on) see = {-1, INT32_MAX, -1};
    int hi = see.from, lo = see.to, least = on ? see.from : INT32_MAX, most = !on ? -1 : see.tok >= 0 ? sr.len - 1 : see.to;
    const auto join = [&](auto lane_bit) {
        constexpr int O = decltype(lane_bit)::value;
        hi = max(hi, xor_lane_i<O>(hi)), lo = min(lo, xor_lane_i<O>(lo));
        least = min(least, xor_lane_i<O>(least)), most = max(most, xor_lane_i<O>(most));
    };
    join(std::integral_constant<int, 1>{}), join(std::integral_constant<int, 2>{});
    join(std::integral_constant<int, 4>{}), join(std::integral_constant<int, 8>{});
    DigitScales<D, float> qsc;
    qsc.set(on ? scale : 127);
    if (g % 2 == 0 && g / 2 < RowImage<D>::kHalves)
#pragma unroll
        for (int i = 0; i < qsc.W; ++i) o.scale[i][g / 2][r] = qsc.w[i];
    if (g == 0) {
        o.start[r] = on ? -lse * kLog2e : -INFINITY;
        o.from[r] = see.from, o.to[r] = see.to, o.tok[r] = see.tok;
        if (r == 0) o.any[0] = hi, o.any[1] = lo, o.any[2] = least, o.any[3] = most;
    }
}

template <int SEL> __device__ __forceinline__ f4 row_mfma(i8v q, i8v k, f4 acc, int qsc, int ksc) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(q, k, acc, 2, 4, SEL, qsc, 0, ksc);
}

// A wave's keys: KT tiles of 16, lane (r, g): the 16-byte pieces of key 16 t + r that the product wants there.
template <int D, int KT> struct Keys {
    u4 k[KT][kKPieces<D>];
    int scale[KT][kKPieces<D>];
    // page: of key base + 16 t + r, -1 where there is none
    __device__ __forceinline__ void load(const WeighArgs &x, int head, int base, int t, int page) {
        using L = KvParts<D>;
        const int lane = threadIdx.x % 64, r = lane % 16, g = lane / 16, P = 1 << x.a.c.shift, row = (base + 16 * t + r) & (P - 1);
        const uint8_t *p = x.a.c.pages + max(page, 0) * x.a.c.page_bytes + head * kv_head_bytes(D, P);
#pragma unroll
        for (int u = 0; u < kKPieces<D>; ++u) {
            const int block = (D == 64 ? g & 1 : g) + 4 * u;
            k[t][u] = *(const u4 *) (p + L::k_row(P, row) + block * 16);
            scale[t][u] = p[L::k_scale(P, row) + block];
        }
    }
    __device__ __forceinline__ void wait() {  // (what is used here has arrived)
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int u = 0; u < kKPieces<D>; ++u) asm volatile("" : "+v"(k[t][u]), "+v"(scale[t][u]));
    }
    __device__ __forceinline__ bool nan(int t) const {  // of key 16 t + r
        int bad = 0;
#pragma unroll
        for (int u = 0; u < kKPieces<D>; ++u) bad |= scale[t][u] == 255;
        bad |= xor_lane_i<16>(bad);
        bad |= xor_lane_i<32>(bad);
        return bad;
    }
};

// Bits off .. off + 63 of a token's: what it sees of the new tokens from the off-th on.
__device__ __forceinline__ uint64_t new_bits(const NewTokens<true> &nt, int tok, int off) {
    if (off <= -64 || off >= 64 * nt.words) return 0;
    const uint64_t *row = nt.sees + (int64_t) tok * nt.words;
    const int i = off >> 6, sh = off & 63;
    const uint64_t lo = i >= 0 ? row[i] : 0, hi = sh && i + 1 < nt.words ? row[i + 1] : 0;
    return (lo >> sh) | (sh ? hi << (64 - sh) : 0);
}

// The rows of an image against 64 keys (tiles T0 .. T0 + 3 of a wave's, from base on), a lane's key being base + 16 t + r and its
// rows 4 g .. 4 g + 3: exponents of what they add, in two steps.
template <int D> struct RowDigits {
    using Q = QueryShape<D, float>;
    i8v q[Q::N][Q::kSteps];
    int scale[DigitScales<D, float>::W];
    f4 start;
    // (offsets in 32 bits that a lane keeps, from an image's place in scalar registers)
    __device__ __forceinline__ void read(const RowImage<D> &im) {
        using I = RowImage<D>;
        const uint32_t lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
        const char *p = (const char *) &im;
        const uint32_t at_low = lane * 16, at_high = lane * 8 + (uint32_t) offsetof(I, high);
        const uint32_t at_scale = (I::kHalves == 2 ? g / 2 * kRowTile + r : r) * 4 + (uint32_t) offsetof(I, scale);
#pragma unroll
        for (int n = 0; n < Q::N; ++n)
#pragma unroll
            for (int u = 0; u < Q::kSteps; ++u) {
                const u4 lo = *(const u4 *) (p + (at_low + (n * Q::kSteps + u) * 1024));
                const uint2 hi = *(const uint2 *) (p + (at_high + (n * Q::kSteps + u) * 512));
                q[n][u] = i8v{(int) lo[0], (int) lo[1], (int) lo[2], (int) lo[3], (int) hi.x, (int) hi.y, 0, 0};
            }
#pragma unroll
        for (int i = 0; i < DigitScales<D, float>::W; ++i) scale[i] = *(const int *) (p + (at_scale + i * I::kHalves * kRowTile * 4));
        start = *(const f4 *) (p + (g * 16 + (uint32_t) offsetof(I, start)));
    }
};
template <int T0, int D, int KT>
__device__ __forceinline__ void products(const RowDigits<D> &rows, const Keys<D, KT> &keys, f4 (&acc)[4]) {
    using Q = QueryShape<D, float>;
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] = rows.start;
#pragma unroll
    for (int n = 0; n < Q::N; ++n)  // the largest digit first: the rest adds to small numbers
#pragma unroll
        for (int u = 0; u < Q::kSteps; ++u)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const u4 x = keys.k[T0 + t][u];
                const i8v k = {(int) x[0], (int) x[1], (int) x[2], (int) x[3], 0, 0, 0, 0}, q = rows.q[n][u];
                const int e = keys.scale[T0 + t][u], w = rows.scale[n / 4];
                acc[t] = n % 4 == 0 ? row_mfma<0>(q, k, acc[t], w, e) : n % 4 == 1 ? row_mfma<1>(q, k, acc[t], w, e) :
                         n % 4 == 2 ? row_mfma<2>(q, k, acc[t], w, e) : row_mfma<3>(q, k, acc[t], w, e);
            }
}
// TREE: of a tree (causal rows need no look at its bits, whose loads would be waited for with all the others).
template <bool TREE, int D>
__device__ __forceinline__ void hide(const RowImage<D> &im, const NewTokens<true> &nt, int base, f4 (&acc)[4]) {
    const int r = threadIdx.x % 16, g = threadIdx.x % 64 / 16;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        const int from = im.from[4 * g + v], to = im.to[4 * g + v];
        uint64_t bits = 0;
        if (TREE && nt.sees) {
            const int tok = im.tok[4 * g + v];
            bits = tok >= 0 ? new_bits(nt, tok, base - nt.first) : 0;
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int pos = base + 16 * t + r;
            const bool on = (pos > from && pos <= to) || (TREE && (bits >> (16 * t + r) & 1));
            acc[t][v] = on ? acc[t][v] : -INFINITY;
        }
    }
}
__device__ __forceinline__ void add_exps(const f4 (&acc)[4], float *sum) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int v = 0; v < 4; ++v) sum[t] += __builtin_amdgcn_exp2f(acc[t][v]);
}
// (nothing of the image is seen of the 64 keys from base on)
template <int D> __device__ __forceinline__ bool unseen(const RowImage<D> &im, int base, int keys) {
    return im.any[3] < base || im.any[2] >= base + keys - 1;
}

// The sums of 64 keys (tiles t0 .. t0 + 3), one a lane; good: whether key 16 t + r takes any.
template <int KT> __device__ __forceinline__ float one_a_lane(const float (&sum)[KT], const bool (&good)[KT], int t0) {
    float mine = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        float v = good[t0 + t] ? sum[t0 + t] : 0.0f;
        v += xor_lane<16>(v);
        v += xor_lane<32>(v);
        mine = (int) threadIdx.x % 64 / 16 == t ? v : mine;
    }
    return mine;
}
__device__ __forceinline__ int64_t weight_at(const WeighArgs &x, int head, int page, int pos) {
    return (((int64_t) page * x.a.c.n_kv + head) << x.a.c.shift) + (pos & ((1 << x.a.c.shift) - 1));
}
__device__ __forceinline__ float past_weight(const WeighArgs &x, int head, int page, int pos, int first) {
    return page >= 0 && x.past && pos < first ? x.past[weight_at(x, head, page, pos)] : 0.0f;
}
__device__ __forceinline__ void put_weight(const WeighArgs &x, int head, int page, int pos, int first, float sum) {
    if (page >= 0) x.weights[weight_at(x, head, page, pos)] = past_weight(x, head, page, pos, first) + sum;
}
__device__ __forceinline__ int key_len(const AttnArgs &a, const SeqRange &sr) {  // positions behind the table have no page
    return (int) min((int64_t) sr.len, a.b.table_stride << a.c.shift);
}

// The row tiles [t0, t1) of `tiles` that see any of the keys base .. base + keys - 1 (of a tree: all; with a window every step then
// is a masked one, 300 tokens of a tree at 100000: 476 us without, 710 with a window of 512).
struct TileRange {
    int t0, t1;
};
template <bool TREE> __device__ __forceinline__ TileRange tiles_seeing(const AttnArgs &a, int first, int tiles, int64_t base, int keys) {
    TileRange t{0, tiles};
    if (!TREE) {
        const int64_t row0 = max(base - first, (int64_t) 0) * a.group;
        t.t0 = (int) min(row0 / kRowTile, (int64_t) tiles);
        if (a.window) {
            const int64_t row1 = (base + keys - 1 + a.window - first) * a.group;  // (the token at pos sees from pos - window + 1 on)
            t.t1 = (int) max((int64_t) t.t0, min((int64_t) tiles, max(row1, (int64_t) 0) / kRowTile + 1));
        }
    }
    return t;
}
// Row tiles that have images, and the blocks of keys of a sequence by the host's number.
__device__ __forceinline__ int image_tiles(const WeighArgs &x, const SeqRange &sr) {
    const int64_t rows = min((int64_t) sr.n * x.a.group, (int64_t) INT32_MAX);
    return (int) min((rows + kRowTile - 1) / kRowTile, x.row_tiles);
}
__device__ __forceinline__ int planned_blocks(const WeighArgs &x, int len) { return (int) min(((int64_t) len + x.block - 1) / x.block, (int64_t) x.blocks); }

// Few rows (decode, verify): their images are made by every workgroup, whose waves take 64 keys in turn, the next ones' K
// asked for before this one's products. Bound by what waits for what where there is little (one token at 1500 keys, 8 heads of 128:
// 6.4 us: the range, the table and q, K, the store), by K's and the weights' bytes where there is much (24 at up to 16000, 8
// heads, bf16: 77 MB in 25.5 us, 3.0 TB/s, since some 2100 workgroups each make the images and then pass over one to a few steps; a
// copy of them 16.6). K is asked for before it is known whether a row sees it: a window saves the products, not the bytes (one
// token at 100000: 18.7 us, with a window of 512 16.7). PH > 1 (up to sixteen tiles of rows): PH waves have the same keys
// and every PH-th tile each, and the first adds up what they found.
template <int D, int RT, int PH, class T> __global__ __launch_bounds__(256 * PH, D < 256 ? 4 : 2) void k_weigh_few(WeighArgs x) {
    const AttnArgs &a = x.a;
    __shared__ __align__(16) RowImage<D> im[RT];
    __shared__ float found[PH > 1 ? PH - 1 : 1][256];
    const int s = blockIdx.y / a.c.n_kv, head = blockIdx.y % a.c.n_kv, lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), phase = wave / 4, keys_of = wave % 4;
    const SeqRange sr = seq_range(a.b, s);
    const int rows = (int) min((int64_t) sr.n * a.group, x.row_tiles * kRowTile), tiles = PH > 1 ? (rows - 1) / kRowTile + 1 : RT;
    const int len = key_len(a, sr), first = sr.len - sr.n, step = (int) gridDim.x * 256;
    if (rows == 0 || (int) blockIdx.x * 256 >= len) return;
    const NewTokens<true> nt(a, sr);
    Keys<D, 4> keys, next;
    int page = -1, after = -1;  // of the lane's own key, of these 64 and of the next
    float past = 0.0f, coming = 0.0f;
    const auto ask = [&](int64_t base) { return base + lane < len ? page_of(a.c, a.b, s, (int) base + lane) : -1; };
    const auto load = [&](Keys<D, 4> &k, int base, int own) {
#pragma unroll
        for (int t = 0; t < 4; ++t) k.load(x, head, base, t, __builtin_amdgcn_readlane(own, 16 * t));  // 16 aligned positions lie in one page
    };
    const auto before = [&](int base, int own) { return phase == 0 ? past_weight(x, head, own, base + lane, first) : 0.0f; };
    int64_t b0 = (int64_t) blockIdx.x * 256 + keys_of * 64;
    if (b0 < len) {
        page = ask(b0);
        load(keys, (int) b0, page);
        past = before((int) b0, page);
        after = ask(b0 + step);
    }
    for (int t = wave; t < tiles; t += 4 * PH) make_image<D, T>(x, sr, nt, head, rows, t * kRowTile, im[t]);
    __syncthreads();
    for (; PH > 1 ? b0 - keys_of * 64 < len : b0 < len; b0 += step) {  // (PH > 1: of the whole workgroup)
        const int base = (int) b0;
        if (b0 + step < len) {
            load(next, base + step, after);
            coming = before(base + step, after);
        }
        const int then = ask(b0 + 2 * (int64_t) step);
        float sum[4] = {};
        if (PH == 1 || b0 < len) {
#pragma unroll 1
            for (int t = phase; t < tiles; t += PH) {
                if (unseen(im[t], base, 64)) continue;
                RowDigits<D> rows_;
                f4 acc[4];
                rows_.read(im[t]);
                products<0>(rows_, keys, acc);
                if (!(im[t].any[0] < base && im[t].any[1] >= base + 63)) hide<true>(im[t], nt, base, acc);  // (some row does not see all)
                add_exps(acc, sum);
            }
        }
        bool good[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) good[t] = !keys.nan(t);
        float sums = one_a_lane(sum, good, 0);
        if (PH > 1) {
            if (phase > 0) found[phase - 1][keys_of * 64 + lane] = sums;
            __syncthreads();
            if (phase == 0)
#pragma unroll
                for (int i = 0; i < PH - 1; ++i) sums += found[i][keys_of * 64 + lane];
            __syncthreads();
        }
        if (phase == 0 && page >= 0) x.weights[weight_at(x, head, page, base + lane)] = past + sums;
        keys = next, page = after, after = then, past = coming;
    }
}

// `all` steps dealt to n workgroups: the first ones get one more where they do not come out even.
struct Shares {
    int each, more;
    __device__ __forceinline__ Shares(int all, int n) : each(all / n), more(all % n) {}
    __device__ __forceinline__ int from(int share) const { return share * each + min(share, more); }
    __device__ __forceinline__ int of(int step) const {  // (there is one: all > 0)
        const int larger = more * (each + 1);
        return step < larger ? step / (each + 1) : more + (step - larger) / max(each, 1);
    }
};

// The images of many rows; the first wave of a kv head also counts the steps of its blocks of keys. Bound by the bytes: 2801 tokens
// of 32 heads of 128, f32: 46 MB of q and as many of images in 16.7 us, 5.5 TB/s.
template <int D, class T> __global__ __launch_bounds__(64) void k_weigh_rows(WeighArgs x) {
    const AttnArgs &a = x.a;
    const int s = blockIdx.x / a.c.n_kv, head = blockIdx.x % a.c.n_kv, lane = threadIdx.x;
    const SeqRange sr = seq_range(a.b, s);
    const int rows = (int) min((int64_t) sr.n * a.group, (int64_t) INT32_MAX);
    if (blockIdx.y == 0) {
        const int blocks = planned_blocks(x, key_len(a, sr)), tiles = image_tiles(x, sr), first = sr.len - sr.n;
        int32_t *plan = x.plan + (int64_t) blockIdx.x * (x.blocks + 1), before = 0;  // (weigh_plan sees that all steps fit)
        for (int i0 = 0; i0 < blocks; i0 += 64) {
            const int i = i0 + lane;
            int n = 0;
            if (i < blocks) {
                const int64_t base = (int64_t) i * x.block;
                const TileRange t = a.sees ? tiles_seeing<true>(a, first, tiles, base, x.block) : tiles_seeing<false>(a, first, tiles, base, x.block);
                n = t.t1 - t.t0;
            }
            int sum = n;
#pragma unroll
            for (int o = 1; o < 64; o *= 2) {
                const int u = __shfl_up(sum, o, 64);
                sum += lane >= o ? u : 0;
            }
            if (i < blocks) plan[i] = before + sum - n;
            before += __shfl(sum, 63, 64);
        }
        if (lane == 0) plan[blocks] = before;
    }
    const int64_t row0 = (int64_t) blockIdx.y * kRowTile;
    if (row0 >= rows) return;
    const NewTokens<true> nt(a, sr);
    make_image<D, T>(x, sr, nt, head, rows, (int) row0, ((RowImage<D> *) x.rows)[blockIdx.x * x.row_tiles + blockIdx.y]);
}

// Many rows (prompts, large trees): a workgroup takes 512 keys at a time (256 of 256 channels), a quarter a wave and in its
// registers, and walks over the images of the rows, each wave by itself, the next image on its way to registers meanwhile (its
// four readers find it in L1). Products of 64 keys go with the exponentials of the 64 before: both pipes work for one wave. The
// steps of a kv head (a block of keys and an image) are counted and dealt out evenly, so a workgroup may begin and end inside a
// block; what it has of a block that others share goes to `part`. Heads are the grid's first dimension: workgroups of one go to
// one XCD (where their number is a multiple of 8), whose L2 then holds its images. 2801 tokens of 32 heads over 8 of 128: 60 us,
// 126 million products of 128 in five digits. The matrix pipe is busy 34% of the time, vector instructions take 47% (an exponential
// is four issue slots): two waves a SIMD, which is what the registers of 128 keys and two images allow. Three waves of 64 keys took 75.
template <bool TREE, int D> __global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_weigh_many(WeighArgs x) {
    constexpr int KT = key_tiles(D), kBlock = key_block(D);
    const AttnArgs &a = x.a;
    const int s = blockIdx.x / a.c.n_kv, head = blockIdx.x % a.c.n_kv, share = blockIdx.y, lane = threadIdx.x % 64, r = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const SeqRange sr = seq_range(a.b, s);
    if (sr.n == 0) return;
    const int tiles = image_tiles(x, sr), first = sr.len - sr.n, len = key_len(a, sr), blocks = planned_blocks(x, len);
    const NewTokens<true> nt(a, sr);
    const RowImage<D> *images = (const RowImage<D> *) x.rows + blockIdx.x * x.row_tiles;
    const int32_t *plan = x.plan + (int64_t) blockIdx.x * (x.blocks + 1);
    const Shares sh(plan[blocks], x.shares);
    const int from = sh.from(share), to = sh.from(share + 1);
    int block = -1;  // the first one with a step of this share: the last that begins at `from` or before
    for (int i = 0; i < blocks; i += 64) block += __popcll(__ballot(i + lane < blocks && plan[i + lane] <= from));
    int at = from;
    // then blocks behind the host's number (a sequence longer than it says), each whole
    for (int64_t extra = (int64_t) x.blocks + share; at < to || extra * kBlock < len;) {
        const bool planned = at < to;
        const int64_t b0 = planned ? (int64_t) block * kBlock : extra * kBlock;
        TileRange tr = tiles_seeing<TREE>(a, first, tiles, b0, kBlock);
        bool whole = true, begins = true;
        if (planned) {
            const int p0 = plan[block], p1 = plan[block + 1], e = min(to, p1);
            whole = at == p0 && e == p1, begins = at == p0;
            const int t0 = tr.t0 + (at - p0);
            tr.t1 = tr.t0 + (e - p0), tr.t0 = t0;
            at = e;
            ++block;
        } else {
            extra += x.shares;
        }
        // of them, those that see any of the wave's keys
        const int base = (int) b0 + wave * 16 * KT;
        const TileRange own = tiles_seeing<TREE>(a, first, tiles, base, 16 * KT);
        const int t0 = max(tr.t0, own.t0), t1 = base < 0 || base >= len ? 0 : min(tr.t1, own.t1);
        Keys<D, KT> keys;
        bool good[KT] = {};
        float sum[KT] = {};
        if (t0 < t1) {
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const int pos = base + 16 * t + r;
                keys.load(x, head, base, t, pos >= 0 && pos < len ? page_of(a.c, a.b, s, pos) : -1);
            }
            // Rows from c0 to c1 see all of the keys: no masks there.
            int c0 = t0, c1 = t1;
            if (TREE) {
                if (a.window || base + 16 * KT > first) c0 = t1;
            } else {
                const int64_t past_last = ((int64_t) base + 16 * KT - 1 - first) * a.group;  // the first row at the last key
                c0 = (int) min(max((int64_t) t0, (past_last + kRowTile - 1) / kRowTile), (int64_t) t1);
                if (a.window) {
                    const int64_t below = ((int64_t) base + a.window - first) * a.group;  // the first row that does not see the first key
                    c1 = (int) min(max(below / kRowTile, (int64_t) c0), (int64_t) t1);
                }
            }
            // Causal rows see the key at pos from row (pos - first) * group on, with a window up to row (pos + window - first) * group.
            int lo[KT], hi[KT];
            if (!TREE && (t0 < c0 || c1 < t1)) {
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    const int64_t row = ((int64_t) base + 16 * t + r - first) * a.group;
                    lo[t] = (int) min(max(row, (int64_t) 0), (int64_t) INT32_MAX);
                    hi[t] = a.window ? (int) min(max(row + (int64_t) a.window * a.group, (int64_t) 0), (int64_t) INT32_MAX) : INT32_MAX;
                }
            }
#pragma unroll
            for (int t = 0; t < KT; ++t) good[t] = !keys.nan(t);
            keys.wait();  // (here, or every step would wait for what it has asked for)
            const auto walk = [&](int i0, int i1, auto masked) {
                constexpr bool MASK = decltype(masked)::value;
                if (i0 >= i1) return;
                RowDigits<D> now, next;
                now.read(images[i0]);
                f4 acc[2][4];
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[1][t] = f4{1, 1, 1, 1} * -INFINITY;
                const auto begin = [](f4 (&x)[4]) {  // (the exponentials stay below here)
#pragma unroll
                    for (int t = 0; t < 4; ++t) asm volatile("" : "+v"(x[t]));
                };
                const auto end = [](float *x) {  // (and above here)
#pragma unroll
                    for (int t = 0; t < 4; ++t) asm volatile("" : "+v"(x[t]));
                };
                const auto mix = [&] {  // some instructions of the matrix pipe, then an exponential in their shadow
                    if (MASK) return;
                    constexpr int M = QueryShape<D, float>::N * QueryShape<D, float>::kSteps;  // of four exponentials
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x8, (M + 3) / 4, 0);
                        __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x2, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x8, (M + 1) / 4, 0);
                        __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x2, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x8, (M + 2) / 4, 0);
                        __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x2, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x8, M / 4, 0);
                        __builtin_amdgcn_sched_group_barrier(0x2, 1, 0);
                    }
                };
                const auto cut = [&](int i, int h, f4 (&x)[4]) {
                    if constexpr (MASK && TREE) {
                        hide<TREE>(images[i], nt, base + 64 * h, x);
                    } else if constexpr (MASK) {
#pragma unroll
                        for (int t = 0; t < 4; ++t)
#pragma unroll
                            for (int v = 0; v < 4; ++v) {
                                const int row = i * kRowTile + 4 * (lane / 16) + v;
                                x[t][v] = row >= lo[4 * h + t] && row < hi[4 * h + t] ? x[t][v] : -INFINITY;
                            }
                    }
                };
                const auto turn = [&](int i, RowDigits<D> &rows_, RowDigits<D> &then, auto which) {
                    constexpr int W = decltype(which)::value;
                    then.read(images[min(i + 1, i1 - 1)]);  // (no branch: it would be waited for)
                    if constexpr (KT == 8) {
                        begin(acc[1]);
                        products<0>(rows_, keys, acc[0]);
                        add_exps(acc[1], sum + 4);
                        mix();
                        end(sum + 4);
                        cut(i, 0, acc[0]);
                        begin(acc[0]);
                        products<4>(rows_, keys, acc[1]);
                        add_exps(acc[0], sum);
                        mix();
                        end(sum);
                        cut(i, 1, acc[1]);
                    } else {
                        begin(acc[W ^ 1]);
                        products<0>(rows_, keys, acc[W]);
                        add_exps(acc[W ^ 1], sum);
                        mix();
                        end(sum);
                        cut(i, 0, acc[W]);
                    }
                };
#pragma unroll 1
                for (int i = i0;;) {  // (the way back is from the second turn alone: what is on its way is then known)
                    turn(i, now, next, std::integral_constant<int, 0>{});
                    if (++i >= i1) break;
                    turn(i, next, now, std::integral_constant<int, 1>{});
                    if (++i >= i1) break;
                }
                add_exps(acc[KT == 8 || (i1 - i0) % 2 == 0], sum + KT - 4);
            };
            walk(t0, c0, std::true_type{});
            walk(c0, c1, std::false_type{});
            if (a.window) walk(c1, t1, std::true_type{});
        }
#pragma unroll
        for (int t = 0; t < KT; t += 4) {
            const int pos = base + 16 * t + lane;
            const float mine = one_a_lane(sum, good, t);
            if (whole) put_weight(x, head, pos >= 0 && pos < len ? page_of(a.c, a.b, s, pos) : -1, pos, first, mine);
            else x.part[(((int64_t) blockIdx.x * x.shares + share) * 2 + begins) * kBlock + wave * 16 * KT + 16 * t + lane] = mine;
        }
    }
}

// The sums of blocks that workgroups share, or that no row sees, in the rows' order (2801 tokens: 4.7 us, a launch and two loads).
__global__ __launch_bounds__(256) void k_weigh_join(WeighArgs x) {
    const AttnArgs &a = x.a;
    const int s = blockIdx.x / a.c.n_kv, head = blockIdx.x % a.c.n_kv, in = blockIdx.y % (x.block / 256) * 256 + threadIdx.x;
    const SeqRange sr = seq_range(a.b, s);
    const int len = key_len(a, sr), block = blockIdx.y / (x.block / 256), blocks = planned_blocks(x, len);
    const int64_t pos = (int64_t) block * x.block + in;
    if (sr.n == 0 || block >= blocks || pos >= len) return;
    const int32_t *plan = x.plan + (int64_t) blockIdx.x * (x.blocks + 1);
    const int p0 = plan[block], p1 = plan[block + 1];
    float sum = 0.0f;
    if (p0 < p1) {
        const Shares sh(plan[blocks], x.shares);
        const int w0 = sh.of(p0), w1 = sh.of(p1 - 1);
        if (w0 == w1) return;  // (written by that workgroup)
        const float *part = x.part + (int64_t) blockIdx.x * x.shares * 2 * x.block + in;
        sum = part[(w0 * 2 + 1) * x.block];
#pragma unroll 8
        for (int w = w0 + 1; w <= w1; ++w) sum += part[w * 2 * x.block];
    }
    put_weight(x, head, page_of(a.c, a.b, s, (int) pos), (int) pos, sr.len - sr.n, sum);
}

struct WeighPlan {
    int few;  // row tiles that a workgroup of few rows holds (1, 2, 4 or more), or 0
    int64_t row_tiles, blocks, shares;
    int block;
    size_t plan_off, part_off, bytes;
};
size_t image_bytes(int D) { return D == 64 ? sizeof(RowImage<64>) : D == 128 ? sizeof(RowImage<128>) : sizeof(RowImage<256>); }
WeighPlan weigh_plan(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x) {
    WeighPlan p{};
    const auto per = [](int64_t n, int64_t d) { return (n + d - 1) / d; };
    const int64_t rows = std::min<int64_t>(b->max_q, b->n_tok) * (x->n_head / c->n_head_kv), heads = std::max<int64_t>(1, (int64_t) b->n_seq * c->n_head_kv);
    p.row_tiles = per(rows, kRowTile);
    const int64_t steps = per(std::max<int64_t>(b->max_kv, 1), 256);
    // Up to 64 rows take the form of few rows; up to 256 (128 of 256 channels) too, in workgroups of sixteen waves (eight), unless
    // there is so much to do that the many-row form's cheaper steps outweigh its two more launches (a tree of 20 tokens, 8 heads
    // over 2 of 128, at 400 keys: 9.8 us against 25.9 in three launches; 4 sequences of 62 tokens at 56000: 59 against 81; 24 of 32
    // tokens at 16000, 64 heads over 8: 208 against 174, but 256 channels 211 against 252).
    const int mid = c->head_dim == 256 ? kMidTiles<256> : kMidTiles<128>;
    const bool middle = p.row_tiles > kFewTiles && p.row_tiles <= mid && (c->head_dim == 256 || heads * steps <= kMidSteps);
    if (p.row_tiles <= kFewTiles || middle) {
        p.few = p.row_tiles <= 1 ? 1 : p.row_tiles == 2 ? 2 : middle ? mid : 4;
        // Workgroups of 256 keys at a time: of one sequence as many as run at once, of unequal ones twice that (one of 131072, f32:
        // 19.4 us with 1024, 21.4 with 2048; 24 of up to 16000, bf16: 27.4 and 25.1).
        p.blocks = std::min(steps, per(middle ? 256 : b->n_seq == 1 ? 1024 : 2048, heads));
        return p;
    }
    p.block = key_block(c->head_dim);
    // Blocks that are planned: what the join's grid has, and their steps are counted in 32 bits (65535 tiles of the 32767 blocks of
    // 512 keys fit; of 256 keys there may be 65535). Those behind are gone over whole.
    p.blocks = std::min<int64_t>(per(std::max<int64_t>(b->max_kv, 1), p.block), 65535 / (p.block / 256));
    p.blocks = std::max<int64_t>(1, std::min(p.blocks, INT32_MAX / p.row_tiles));
    // Workgroups of a kv head: as many as there are places for all heads' at once (two a CU; one of 256 channels), or, of many
    // heads, which may be of unequal sequences, so many that the longest, or the last round, does not run on alone; no more than
    // give a share of four steps (24 sequences of up to 9000 keys, 64 tokens, 8 heads: 144 us against 229 in one round; 4 of 205
    // tokens at 20000, 4 heads: 83 against 71).
    const int64_t places = c->head_dim == 256 ? 256 : 512;
    p.shares = heads <= places / (b->n_seq == 1 ? 2 : 16) ? places / heads : per(4 * places, heads);
    p.shares = std::max<int64_t>(1, std::min(p.shares, p.row_tiles * p.blocks / 4));
    const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    p.plan_off = up((size_t) (heads * p.row_tiles) * image_bytes(c->head_dim));
    p.part_off = p.plan_off + up((size_t) (heads * (p.blocks + 1)) * 4);
    p.bytes = p.part_off + (size_t) (heads * p.shares) * 2 * p.block * 4;
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
    if (p.bytes && (!ws || ws_bytes < p.bytes || ((uintptr_t) ws & 15)))
        return host::set_error(host::ERR_NOMEM, "kv_weigh: workspace of %zu bytes, %zu needed (16-byte aligned)", ws ? ws_bytes : 0, p.bytes);
    WeighArgs w{};
    w.a.c = host::kv_view(c), w.a.b = host::kv_batch(b), w.a.q = q, w.a.q_stride = x->q_stride, w.a.n_head = x->n_head;
    w.a.group = x->n_head / c->n_head_kv, w.a.window = x->window, w.a.scale = x->scale;
    w.a.sees = t ? t->sees : nullptr, w.a.words = t ? t->words : 0;
    w.lse = lse, w.past = past, w.weights = weights, w.rows = ws, w.row_tiles = p.row_tiles;
    w.plan = (int32_t *) ((uint8_t *) ws + p.plan_off), w.part = (float *) ((uint8_t *) ws + p.part_off);
    w.blocks = (int) p.blocks, w.shares = (int) p.shares, w.block = p.block;
    const unsigned heads = (unsigned) (b->n_seq * c->n_head_kv), blocks = (unsigned) p.blocks;
    const auto by_type = [&](auto dim, auto type) {
        constexpr int D = decltype(dim)::value;
        using T = decltype(type);
        const auto few = [&](auto kern, unsigned waves) { hipLaunchKernelGGL(kern, dim3(blocks, heads), dim3(64 * waves), 0, st, w); };
        if (p.few == 1) few(k_weigh_few<D, 1, 1, T>, 4);
        else if (p.few == 2) few(k_weigh_few<D, 2, 1, T>, 4);
        else if (p.few == kFewTiles) few(k_weigh_few<D, kFewTiles, 1, T>, 4);
        else if (p.few) few(k_weigh_few<D, kMidTiles<D>, kMidPhases<D>, T>, 4 * kMidPhases<D>);
        if (p.few) return host::check_launch("kv_weigh");
        hipLaunchKernelGGL((k_weigh_rows<D, T>), dim3(heads, (unsigned) p.row_tiles), dim3(64), 0, st, w);
        FNS_TRY(host::check_launch("kv_weigh"));
        const auto many = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(heads, (unsigned) p.shares), dim3(256), 0, st, w); };
        if (t) many(k_weigh_many<true, D>);
        else many(k_weigh_many<false, D>);
        FNS_TRY(host::check_launch("kv_weigh"));
        hipLaunchKernelGGL(k_weigh_join, dim3(heads, blocks * (p.block / 256)), dim3(256), 0, st, w);
        return host::check_launch("kv_weigh");
    };
    const auto by_dim = [&](auto dim) { return x->dtype == FNS_TYPE_F32 ? by_type(dim, float{}) : by_type(dim, uint16_t{}); };
    if (c->head_dim == 64) return by_dim(std::integral_constant<int, 64>{});
    if (c->head_dim == 128) return by_dim(std::integral_constant<int, 128>{});
    return by_dim(std::integral_constant<int, 256>{});
}

}  // namespace impl

namespace k {
void kv_weigh(const FnsKvCache &cache, const FnsKvBatch &batch, const FnsAttn &x, const FnsKvTree *tree, const void *q,
              const float *lse, const float *past, float *weights, void *ws, size_t ws_bytes, hipStream_t st) {
    host::abort_on_error(impl::kv_weigh(&cache, &batch, &x, tree, q, lse, past, weights, ws, ws_bytes, st), "kv_weigh");
}
}  // namespace k

}  // namespace fns
