// attn_tree.hip - attention of a tree of drafted tokens over the paged 4-bit cache, and the logarithms of the softmax's
// denominators: the kernels of fns_attn.hpp with what a token sees of its sequence's new tokens given as bits. Below the new
// tokens a tile of keys is a causal one; the one or two tiles that hold them take the masked path, whose bits come from the
// token's words. What a call costs beside attn's is that every row tile of a sequence walks over all of its new tokens.
#include "fns_attn.hpp"

namespace fns {

namespace impl {

int attn_tree(const FnsKvCache *c, const FnsKvBatch *b, const FnsAttn *x, const FnsKvTree *t, const void *q, void *out, float *lse,
              void *ws, size_t ws_bytes, hipStream_t st) {
    FNS_TRY(host::attn_check(c, b, x, "attn_tree"));
    if (t && (t->words < 1 || t->words > 16)) return host::set_error(host::ERR_SHAPE, "attn_tree: words must be 1..16 (%d)", t->words);
    if (b->n_seq == 0 || b->n_tok == 0 || b->max_q == 0) return host::OK;
    if (t && !t->sees) return host::set_error(host::ERR_SHAPE, "attn_tree: a tree without bits");
    const host::AttnPlan p = host::attn_plan(c, b, x);
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
