// attn_tree.hip - attention of a tree of drafted tokens over the paged 4-bit cache, and the logarithms of the softmax's
// denominators: the kernels of fns_attn.hpp with what a token sees of its sequence's new tokens given as bits. Below the new
// tokens a tile of keys is a causal one; the one or two tiles that hold them take the masked path, whose bits come from the
// token's words. What a call costs beside attn's is that every row tile of a sequence walks over all of its new tokens.
// 60 tokens of 32 heads over 8 of 128 at 100000 positions, f32: 167 us, 590 TFLOP/s of plain products (five digits and two halves of
// p make 15 matrix instructions of 256 scores, 47 vector ones); vector instructions take 59% of the time, the matrix pipe is busy
// 49%, two waves a SIMD. 26 tokens of 32 heads at 726: 12.4 us, a start, a walk of twelve tiles and the join of the waves.
#include "fns_attn.hpp"

namespace fns {

namespace {

// Into how many splits the tiles of a call's workgroups go (of sequences of one length): the least of what they are expected to take. Workgroups run in
// rounds of `places` a CU; with k of them on a CU a tile takes 1.5 + k units (of 0.1 to 0.25 us: 64 channels, 32 rows, 184 workgroups
// over 40000 positions 235 us, twice as many 167), a round's starts and joins in LDS 25, the join of splits 30 and its bytes, a unit
// 400000. So that neither a few workgroups are left for a round of their own (90 tokens of 64 heads over 8 of 64 at 40000: 184 us in
// three splits, which are 552 workgroups for 512 places, 144 in five) nor half the places stay empty (146 of 32 over 4 of 256 at
// 14320: 195 us whole, 160 in three; 33 of 16 over 2 of 256 at 60000: 102 in 16, 544 workgroups, 80 in 15).
int64_t splits_of(int64_t wgs, int64_t tiles, int places, int64_t row_bytes) {
    const auto per = [](int64_t n, int64_t d) { return (n + d - 1) / d; };
    int64_t best = 1, least = INT64_MAX;
    for (int64_t s = 1; s <= 64 && (s == 1 || s * 4 < tiles + 4); ++s) {
        const int64_t full = wgs * s / (256 * places), rest = wgs * s % (256 * places), rounds = full + (rest > 0 ? 1 : 0);
        const int64_t units2 = per(tiles, s) * (full * (3 + 2 * places) + (rest ? 3 + 2 * per(rest, 256) : 0)) + 50 * rounds +
                               (s > 1 ? 60 + s * row_bytes / 200000 : 0);  // (in halves)
        if (units2 < least) least = units2, best = s;
    }
    return best;
}

// How a tree's call is divided: attn's form, but that of few rows otherwise than for causal rows, since a tree's rows all walk over
// the same tiles. Sixteen rows a workgroup, until their steps (of 64 keys) are so many that reading K and V half as often
// is ahead of having twice the workgroups (26 tokens of 4 heads over 726 positions: 12.6 us against 16.7 with 32; 60 tokens
// over 100000: 194 against 167; 32 tokens of 8 heads over 24 contexts of up to 2900: both 49). Splits as above, but
// long contexts of unequal sequences in pieces of 40 tiles up to 1024 workgroups, so that the longest do not run on alone (16 of up
// to 9000 positions, 24 tokens of 32 heads over 8 of 128: 64 us in three, 130 whole; 8 of up to 4200, 63 tokens: 63 whole, 75 in
// two).
host::AttnPlan division(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x) {
    host::AttnPlan p = host::attn_plan(c, b, x);
    if (p.rows == kManyRows) return p;
    const auto per = [](int64_t n, int64_t d) { return (n + d - 1) / d; };
    const int64_t rows = std::min<int64_t>(b->max_q, b->n_tok) * (x->n_head / c->n_head_kv), heads = (int64_t) b->n_seq * c->n_head_kv;
    const int64_t tiles = std::max<int64_t>(1, (b->max_kv + kTile - 1) / kTile);
    p.rows = c->head_dim == 256 || rows <= 16 || heads * per(rows, 16) * tiles < 100000 ? 16 : 32;
    p.row_tiles = per(rows, p.rows);
    const int64_t wgs = std::max<int64_t>(1, heads * p.row_tiles);
    const int places = c->head_dim == 256 || p.rows == 32 ? 2 : 3;  // (by the registers)
    int64_t splits = splits_of(wgs, tiles, places, (int64_t) b->n_tok * x->n_head * c->head_dim * 8);
    if (b->n_seq > 1 && wgs >= 256) splits = std::max(splits, std::min(tiles / 40, per(1024, wgs)));
    p.splits = (int) splits;
    p.chunk = (int) per(tiles, p.splits);
    const size_t n = p.splits > 1 ? (size_t) p.splits * b->n_tok * x->n_head : 0;
    p.ml_off = n * c->head_dim * 4;
    p.bytes = std::max(p.bytes, p.ml_off + n * 8);  // (one size, with a tree or without)
    return p;
}

}  // namespace

namespace impl {

int attn_tree_workspace(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x, size_t *bytes) {
    FNS_TRY(host::attn_check(c, b, x, "attn_tree"));
    if (!bytes) return host::set_error(host::ERR_SHAPE, "attn_tree_workspace: null output");
    *bytes = division(c, b, x).bytes;
    return host::OK;
}

int attn_tree(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x, const FnsKvTree *t, const void *q, void *out, float *lse,
              void *ws, size_t ws_bytes, hipStream_t st) {
    FNS_TRY(host::attn_check(c, b, x, "attn_tree"));
    if (t && (t->words < 1 || t->words > 16)) return host::set_error(host::ERR_SHAPE, "attn_tree: words must be 1..16 (%d)", t->words);
    if (b->n_seq == 0 || b->n_tok == 0 || b->max_q == 0) return host::OK;
    if (t && !t->sees) return host::set_error(host::ERR_SHAPE, "attn_tree: a tree without bits");
    const host::AttnPlan p = t ? division(c, b, x) : host::attn_plan(c, b, x);
    FNS_TRY(host::attn_check_buffers(p, b, q, out, ws, ws_bytes, "attn_tree"));
    AttnArgs a = attn_args(c, b, x, p, q, out, ws);
    a.sees = t ? t->sees : nullptr, a.words = t ? t->words : 0, a.lse = lse;
    return attn_launch<true>(a, p, c, b, x->dtype, "attn_tree", st);
}

}  // namespace impl

namespace k {
void attn_tree(const FnsKvCache &cache, const FnsKvBatch &batch, const FnsAttn &x, const FnsKvTree *tree, const void *q, void *out,
               float *lse, void *ws, size_t ws_bytes, hipStream_t st) {
    host::abort_on_error(impl::attn_tree(&cache, &batch, &x, tree, q, out, lse, ws, ws_bytes, st), "attn_tree");
}
}  // namespace k

}  // namespace fns
