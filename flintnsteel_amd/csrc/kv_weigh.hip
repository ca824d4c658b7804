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
constexpr int kFewTiles = 4;    // row tiles that a workgroup of few rows holds
constexpr int kKeyTiles = 8;    // 16-key tiles of a wave of many rows
constexpr int kBlock = 4 * 16 * kKeyTiles;  // keys of its workgroup

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
    float *part;        // many rows in parts: [n_seq * n_kv][parts][blocks * kBlock] their sums
    int64_t row_tiles;
    int parts, blocks;
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
    on = on && scale != 255;
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

// What 16 rows add to KT tiles of keys from base on: a lane's key is base + 16 t + r, its rows 4 g .. 4 g + 3.
// TREE: of a tree (causal rows need no look at its bits, whose loads would be waited for with all the others).
template <bool TREE, int D, int KT>
__device__ __forceinline__ void add_rows(const RowImage<D> &im, const NewTokens<true> &nt, const Keys<D, KT> &keys, int base, float (&sum)[KT]) {
    using Q = QueryShape<D, float>;
    const int lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
    if (im.any[3] < base || im.any[2] >= base + 16 * KT - 1) return;
    int qsc[DigitScales<D, float>::W];
#pragma unroll
    for (int i = 0; i < DigitScales<D, float>::W; ++i) qsc[i] = im.scale[i][RowImage<D>::kHalves == 2 ? g / 2 : 0][r];
    const f4 start = *(const f4 *) (im.start + 4 * g);
    f4 acc[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) acc[t] = start;
#pragma unroll
    for (int n = 0; n < Q::N; ++n)  // the largest digit first: the rest adds to small numbers
#pragma unroll
        for (int u = 0; u < Q::kSteps; ++u) {
            const uint4 lo = im.low[n][u][lane];
            const uint2 hi = im.high[n][u][lane];
            const i8v q = {(int) lo.x, (int) lo.y, (int) lo.z, (int) lo.w, (int) hi.x, (int) hi.y, 0, 0};
            const int w = qsc[n / 4];
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const i8v k = {(int) keys.k[t][u][0], (int) keys.k[t][u][1], (int) keys.k[t][u][2], (int) keys.k[t][u][3], 0, 0, 0, 0};
                const int e = keys.scale[t][u];
                acc[t] = n % 4 == 0 ? row_mfma<0>(q, k, acc[t], w, e) : n % 4 == 1 ? row_mfma<1>(q, k, acc[t], w, e) :
                         n % 4 == 2 ? row_mfma<2>(q, k, acc[t], w, e) : row_mfma<3>(q, k, acc[t], w, e);
            }
        }
    if (im.any[0] >= base || im.any[1] < base + 16 * KT - 1) {  // some row does not see all of the keys
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int from = im.from[4 * g + v], to = im.to[4 * g + v];
            uint64_t bits[KT / 4] = {};
            if (TREE && nt.sees) {
                const int tok = im.tok[4 * g + v];
#pragma unroll
                for (int i = 0; i < KT / 4; ++i) bits[i] = tok >= 0 ? new_bits(nt, tok, base + 64 * i - nt.first) : 0;
            }
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const int pos = base + 16 * t + r;
                const bool on = (pos > from && pos <= to) || (bits[t / 4] >> (16 * (t % 4) + r) & 1);
                acc[t][v] = on ? acc[t][v] : -INFINITY;
            }
        }
    }
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int v = 0; v < 4; ++v) sum[t] += __builtin_amdgcn_exp2f(acc[t][v]);
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

// Few rows (decode, verify): their images are made by every workgroup, whose waves take 64 keys in turn, the next ones' K
// asked for before this one's products.
template <int D, int RT, class T> __global__ __launch_bounds__(256) void k_weigh_few(WeighArgs x) {
    const AttnArgs &a = x.a;
    __shared__ __align__(16) RowImage<D> im[RT];
    const int s = blockIdx.y / a.c.n_kv, head = blockIdx.y % a.c.n_kv, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const SeqRange sr = seq_range(a.b, s);
    const int rows = (int) min((int64_t) sr.n * a.group, (int64_t) RT * kRowTile);
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
    int64_t b0 = (int64_t) blockIdx.x * 256 + wave * 64;
    if (b0 < len) {
        page = ask(b0);
        load(keys, (int) b0, page);
        past = past_weight(x, head, page, (int) b0 + lane, first);
        after = ask(b0 + step);
    }
    for (int t = wave; t < RT; t += 4) make_image<D, T>(x, sr, nt, head, rows, t * kRowTile, im[t]);
    __syncthreads();
    for (; b0 < len; b0 += step) {
        const int base = (int) b0;
        const bool more = b0 + step < len;
        if (more) {
            load(next, base + step, after);
            coming = past_weight(x, head, after, base + step + lane, first);
        }
        const int then = ask(b0 + 2 * (int64_t) step);
        float sum[4] = {};
        bool good[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) good[t] = !keys.nan(t);
#pragma unroll 1
        for (int t = 0; t < RT; ++t) add_rows<true, D, 4>(im[t], nt, keys, base, sum);
        const float sums = one_a_lane(sum, good, 0);
        if (page >= 0) x.weights[weight_at(x, head, page, base + lane)] = past + sums;
        keys = next, page = after, after = then, past = coming;
    }
}

template <int D, class T> __global__ __launch_bounds__(64) void k_weigh_rows(WeighArgs x) {
    const AttnArgs &a = x.a;
    const int s = blockIdx.x / a.c.n_kv, head = blockIdx.x % a.c.n_kv;
    const SeqRange sr = seq_range(a.b, s);
    const int rows = (int) min((int64_t) sr.n * a.group, (int64_t) INT32_MAX);
    const int64_t row0 = (int64_t) blockIdx.y * kRowTile;
    if (row0 >= rows) return;
    const NewTokens<true> nt(a, sr);
    make_image<D, T>(x, sr, nt, head, rows, (int) row0, ((RowImage<D> *) x.rows)[blockIdx.x * x.row_tiles + blockIdx.y]);
}

// Many rows (prompts, large trees): a workgroup takes 512 keys, 128 a wave and in its registers, and walks over the images of a
// part of the rows, which come through LDS, the next two on their way to registers meanwhile. Heads are the grid's first
// dimension: workgroups of one go to one XCD (where their number is a multiple of 8), whose L2 then holds its images.
template <bool TREE, int D> __global__ __launch_bounds__(256, 2) void k_weigh_many(WeighArgs x) {
    constexpr int KT = kKeyTiles, PIECES = sizeof(RowImage<D>) / 16, PER = (PIECES + 255) / 256;
    static_assert(sizeof(RowImage<D>) % 16 == 0, "images are copied in pieces of 16 bytes");
    const AttnArgs &a = x.a;
    __shared__ __align__(16) RowImage<D> im[2];
    const int s = blockIdx.x / a.c.n_kv, head = blockIdx.x % a.c.n_kv, part = blockIdx.z, tid = threadIdx.x, lane = tid % 64, r = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const SeqRange sr = seq_range(a.b, s);
    const int rows = (int) min((int64_t) sr.n * a.group, (int64_t) INT32_MAX);
    if (rows == 0) return;
    const int tiles = (int) min((int64_t) (rows - 1) / kRowTile + 1, x.row_tiles);  // (rows behind max_q tokens have no image)
    const int first = sr.len - sr.n, len = key_len(a, sr);
    const NewTokens<true> nt(a, sr);
    const RowImage<D> *images = (const RowImage<D> *) x.rows + blockIdx.x * x.row_tiles;
    for (int64_t b0 = (int64_t) blockIdx.y * kBlock; b0 < len; b0 += (int64_t) gridDim.y * kBlock) {
        const bool apart = x.parts > 1 && b0 < (int64_t) x.blocks * kBlock;  // (longer than the host's number: the first part does all)
        if (!apart && part > 0) break;
        // the row tiles of this part that see any of these keys
        int t0 = apart ? (int) ((int64_t) tiles * part / x.parts) : 0, t1 = apart ? (int) ((int64_t) tiles * (part + 1) / x.parts) : tiles;
        if (!TREE) {
            const int64_t row0 = max(b0 - first, (int64_t) 0) * a.group;
            t0 = (int) max((int64_t) t0, row0 / kRowTile);
            if (a.window) {
                const int64_t row1 = (b0 + kBlock - 1 + a.window - first) * a.group;  // (the token at pos sees from pos - window + 1 on)
                t1 = (int) min((int64_t) t1, max(row1, (int64_t) 0) / kRowTile + 1);
            }
        }
        const int base = (int) b0 + wave * 16 * KT;
        Keys<D, KT> keys;
        bool good[KT];
        float sum[KT] = {};
        u4 stage[2][PER];
        const auto fetch = [&](int t, u4 (&to)[PER]) {
#pragma unroll
            for (int p = 0; p < PER; ++p)
                to[p] = ((const u4 *) (images + t))[min(tid + 256 * p, PIECES - 1)];
        };
        if (t0 < t1) {
            fetch(t0, stage[0]);
            fetch(min(t0 + 1, t1 - 1), stage[1]);
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const int pos = base + 16 * t + r;
                keys.load(x, head, base, t, pos >= 0 && pos < len ? page_of(a.c, a.b, s, pos) : -1);
            }
#pragma unroll
            for (int t = 0; t < KT; ++t) good[t] = !keys.nan(t);
            keys.wait();  // (here, or every step would wait for its own fetch)
            const auto turn = [&](int i, auto which) {
                constexpr int W = decltype(which)::value;
                u4 *to = (u4 *) &im[W];
#pragma unroll
                for (int p = 0; p < PER; ++p)
                    if (tid + 256 * p < PIECES) to[tid + 256 * p] = stage[W][p];
                fetch(min(i + 2, t1 - 1), stage[W]);  // (no branch: it would be waited for)
                tile_barrier();
                add_rows<TREE, D, KT>(im[W], nt, keys, base, sum);
            };
            for (int i = t0;;) {  // (the way back is from the second turn alone: what is on its way is then known, and not waited for)
                turn(i, std::integral_constant<int, 0>{});
                if (++i >= t1) break;
                turn(i, std::integral_constant<int, 1>{});
                if (++i >= t1) break;
            }
            tile_barrier();  // (the next block writes the images again)
        }
#pragma unroll
        for (int t = 0; t < KT; t += 4) {
            const int pos = base + 16 * t + lane;
            const float mine = t0 < t1 ? one_a_lane(sum, good, t) : 0.0f;
            if (apart) x.part[((int64_t) blockIdx.x * x.parts + part) * x.blocks * kBlock + pos] = mine;
            else put_weight(x, head, pos >= 0 && pos < len ? page_of(a.c, a.b, s, pos) : -1, pos, first, mine);
        }
    }
}

// The parts of a key's sum, in order.
__global__ __launch_bounds__(256) void k_weigh_join(WeighArgs x) {
    const AttnArgs &a = x.a;
    const int s = blockIdx.x / a.c.n_kv, head = blockIdx.x % a.c.n_kv, pos = blockIdx.y * 256 + threadIdx.x;
    const SeqRange sr = seq_range(a.b, s);
    if (sr.n == 0 || pos >= key_len(a, sr)) return;
    const int64_t step = (int64_t) x.blocks * kBlock;
    const float *p = x.part + blockIdx.x * x.parts * step + pos;
    float sum = 0.0f;
#pragma unroll 8
    for (int i = 0; i < x.parts; ++i) sum += p[i * step];
    put_weight(x, head, page_of(a.c, a.b, s, pos), pos, sr.len - sr.n, sum);
}

struct WeighPlan {
    int few;  // row tiles of the form of few rows (1, 2 or 4), or 0
    int64_t row_tiles, blocks, parts;
    size_t part_off, bytes;
};
size_t image_bytes(int D) { return D == 64 ? sizeof(RowImage<64>) : D == 128 ? sizeof(RowImage<128>) : sizeof(RowImage<256>); }
WeighPlan weigh_plan(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x) {
    WeighPlan p{};
    const auto per = [](int64_t n, int64_t d) { return (n + d - 1) / d; };
    const int64_t rows = std::min<int64_t>(b->max_q, b->n_tok) * (x->n_head / c->n_head_kv), heads = std::max<int64_t>(1, (int64_t) b->n_seq * c->n_head_kv);
    p.row_tiles = per(rows, kRowTile);
    if (p.row_tiles <= kFewTiles) {
        p.few = p.row_tiles <= 1 ? 1 : p.row_tiles == 2 ? 2 : 4;
        // workgroups of 256 keys at a time; no more than some 2048 of them
        p.blocks = std::min(per(std::max<int64_t>(b->max_kv, 1), 256), per(2048, heads));
        return p;
    }
    p.blocks = std::min<int64_t>(per(std::max<int64_t>(b->max_kv, 1), kBlock), 65535 / (kBlock / 256));
    p.parts = std::max<int64_t>(1, std::min(std::min<int64_t>(per(1024, heads * p.blocks), p.row_tiles / 8), (int64_t) 64));
    p.part_off = (size_t) (heads * p.row_tiles) * image_bytes(c->head_dim);
    p.bytes = p.part_off + (p.parts > 1 ? (size_t) (heads * p.parts * p.blocks) * kBlock * 4 : 0);
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
    w.part = (float *) ((uint8_t *) ws + p.part_off), w.parts = (int) p.parts, w.blocks = (int) p.blocks;
    const unsigned heads = (unsigned) (b->n_seq * c->n_head_kv), blocks = (unsigned) p.blocks;
    const auto by_type = [&](auto dim, auto type) {
        constexpr int D = decltype(dim)::value;
        using T = decltype(type);
        const auto few = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(blocks, heads), dim3(256), 0, st, w); };
        if (p.few == 1) few(k_weigh_few<D, 1, T>);
        else if (p.few == 2) few(k_weigh_few<D, 2, T>);
        else if (p.few) few(k_weigh_few<D, 4, T>);
        if (p.few) return host::check_launch("kv_weigh");
        hipLaunchKernelGGL((k_weigh_rows<D, T>), dim3(heads, (unsigned) p.row_tiles), dim3(64), 0, st, w);
        FNS_TRY(host::check_launch("kv_weigh"));
        const auto many = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(heads, blocks, (unsigned) p.parts), dim3(256), 0, st, w); };
        if (t) many(k_weigh_many<true, D>);
        else many(k_weigh_many<false, D>);
        FNS_TRY(host::check_launch("kv_weigh"));
        if (p.parts > 1) hipLaunchKernelGGL(k_weigh_join, dim3(heads, blocks * (kBlock / 256)), dim3(256), 0, st, w);
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
