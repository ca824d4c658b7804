// attn.hip - grouped-query attention of a batch's new tokens over the paged 4-bit cache: how a call is checked and divided, and
// the launches (the kernels are fns_attn.hpp's).
#include "fns_attn.hpp"

namespace fns {

namespace host {

int attn_check(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x, const char *what) {
    FNS_TRY(kv_check(c, b, what));
    if (!x) return set_error(ERR_SHAPE, "%s: null arguments", what);
    if (x->dtype != FNS_TYPE_F32 && x->dtype != FNS_TYPE_BF16)
        return set_error(ERR_TYPE, "%s: type %d is not supported (0 f32, 30 bf16)", what, x->dtype);
    if (x->n_head <= 0 || x->n_head % c->n_head_kv || x->n_head > 65535)
        return set_error(ERR_SHAPE, "%s: n_head %d is no multiple of n_head_kv %d", what, x->n_head, c->n_head_kv);
    if (x->window < 0) return set_error(ERR_SHAPE, "%s: negative window", what);
    const int64_t w = (int64_t) x->n_head * c->head_dim;
    if (x->q_stride < w || x->out_stride < w) return set_error(ERR_SHAPE, "%s: a token stride is shorter than a token's heads", what);
    return OK;
}

AttnPlan attn_plan(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x) {
    AttnPlan p{};
    const int64_t rows = std::min<int64_t>(b->max_q, b->n_tok) * (x->n_head / c->n_head_kv);  // of a sequence and kv head
    const auto per = [](int64_t n, int64_t d) { return (n + d - 1) / d; };
    // The form of few rows reads K and V once for 32 rows instead of 128, but has more workgroups. It is ahead up to 64 rows
    // (64 sequences of 600 keys, 64 rows of 8 heads: 45 us against 51; 128 rows: 79 against 60), and wherever the other form
    // leaves CUs idle: less than two workgroups a CU of it (256 tokens behind 1024 keys, 1024 rows of 8 heads: 26 us against
    // 34 with 64 workgroups; 1024 tokens: 68 against 95 with 256; 2048 tokens: 145 against the few-row form's 168 with 512).
    const int64_t heads = (int64_t) b->n_seq * c->n_head_kv;
    const bool many = rows > kFewRows && heads * per(rows, kManyRows) >= 512;
    p.rows = many ? kManyRows : rows <= 16 || c->head_dim == 256 ? 16 : 32;
    p.row_tiles = per(rows, p.rows);
    const int64_t wgs = std::max<int64_t>(1, heads * p.row_tiles);
    const int64_t tiles = std::max<int64_t>(1, (b->max_kv + kTile - 1) / kTile);
    // A split costs its join and a second start, 4-6 us, about what 11 tiles cost a workgroup; what it saves is the tiles' time
    // on the CUs that have nothing. So, where that outweighs it, splits until 512 workgroups (131072 keys of 8 heads: 32 us
    // with 512, 37 with 256), of four tiles (one a wave) at least: 24 sequences of 1500 keys, 8 heads: 20.5 us whole, 24.5 in
    // three; 8 of 2048: 16.8 in eight, 21.6 whole; 500 keys: 9.2 whole, 10.9 in two. Beyond that, pieces of 40 tiles, up to
    // 2304, so that the longest of unequal sequences does not run on alone (48 of up to 16000 keys: 74 us with 2304, 94 with
    // 512).
    int64_t splits = 1;
    if (!many) splits = std::max(tiles * (256 - wgs) > 11 * 256 ? std::min(per(512, wgs), per(tiles, 4)) : 1, std::min(tiles / 40, per(2304, wgs)));
    p.splits = (int) std::max<int64_t>(1, std::min<int64_t>(splits, 64));
    p.chunk = (int) per(tiles, p.splits);
    if (p.splits > 1) {
        const size_t n = (size_t) p.splits * b->n_tok * x->n_head;
        p.ml_off = n * c->head_dim * 4;
        p.bytes = p.ml_off + n * 8;
    }
    if (many) p.bytes = (size_t) (heads * p.row_tiles) * 4;  // a byte a wave: whether the rows are to be done again
    return p;
}

int attn_check_buffers(const AttnPlan &p, const FnsKvBatch *b, const void *q, const void *out, const void *ws, size_t ws_bytes, const char *what) {
    if (!q || !out) return set_error(ERR_SHAPE, "%s: null argument", what);
    if (q == out) return set_error(ERR_SHAPE, "%s: q and out must not overlap", what);
    if (p.row_tiles > 65535)
        return set_error(ERR_SHAPE, "%s: %lld tokens of a sequence in one call are too many", what, (long long) std::min<int64_t>(b->max_q, b->n_tok));
    if (p.bytes && (!ws || ws_bytes < p.bytes || ((uintptr_t) ws & 15)))
        return set_error(ERR_NOMEM, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", what, ws ? ws_bytes : 0, p.bytes);
    return OK;
}

}  // namespace host

namespace impl {

int attn_workspace(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x, size_t *bytes) {
    FNS_TRY(host::attn_check(c, b, x, "attn"));
    if (!bytes) return host::set_error(host::ERR_SHAPE, "attn_workspace: null output");
    *bytes = host::attn_plan(c, b, x).bytes;
    return host::OK;
}

int attn(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x, const void *q, void *out, void *ws, size_t ws_bytes,
         hipStream_t st) {
    FNS_TRY(host::attn_check(c, b, x, "attn"));
    if (b->n_seq == 0 || b->n_tok == 0 || b->max_q == 0) return host::OK;
    const host::AttnPlan p = host::attn_plan(c, b, x);
    FNS_TRY(host::attn_check_buffers(p, b, q, out, ws, ws_bytes, "attn"));
    return attn_launch<false>(attn_args(c, b, x, p, q, out, ws), p, c, b, x->dtype, "attn", st);
}

}  // namespace impl

namespace k {
void attn(const FnsKvCache &cache, const FnsKvBatch &batch, const FnsAttn &x, const void *q, void *out, void *ws,
          size_t ws_bytes, hipStream_t st) {
    host::abort_on_error(impl::attn(&cache, &batch, &x, q, out, ws, ws_bytes, st), "attn");
}
}  // namespace k

}  // namespace fns
