// fns_kv.hpp - the paged 4-bit key/value cache: its layout, the description of a batch over it, and the arithmetic of
// its blocks, shared by the kernels that fill it (kv_cache.hip) and the attention that reads it (attn.hip).
//
// A block is 32 channels of one token's K or V (of one kv head): 4-bit codes c and one byte e, value(c) * 2^(e - 127),
// value = +-{0, .5, 1, 1.5, 2, 3, 4, 6} (e2m1) - the elements and scales of the published microscaling formats, which
// gfx950 expands two codes at a time, scale included, exactly. e is the least with max |block| <= 7 * 2^(e - 127) (at
// least 1, 0 for a block of zeros): what lies in (6, 7] units rounds to 6, nothing is clipped further. Against the
// power of two of floor(log2 max) - 2, whose largest codes clip from 8 to 6: rms error of normal values 0.112 for
// 0.115, uniform ones 0.099 for 0.144. Codes round to nearest, ties to the even code. A block that holds a NaN or an
// infinity has e = 255 and stands for NaNs.
//
// A page holds page_size positions (a power of two, at least 16) of every kv head; the part of one kv head is
//   K codes [page_size][D / 2]    byte b of a row: channel 2 b in the low half, 2 b + 1 in the high half
//   V codes [D / 2][page_size]    byte column j = 16 i + r, r < 16: channels 32 i + r (low) and 32 i + 16 + r (high)
//   K scales [page_size][D / 32] | V scales [page_size][D / 32]
// so that 16 consecutive positions of a V channel pair are 16 bytes: the matrix products of attention contract K over
// channels and V over positions, and either operand is then a plain 16-byte load.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "fns_hip.h"

namespace fns::dev {

struct KvView {
    uint8_t *pages;
    int64_t n_pages, page_bytes;
    int n_kv, shift;  // page_size = 1 << shift
};
struct BatchView {
    const int32_t *q_start, *kv_len, *table;
    int64_t n_tok, table_stride;
};

__host__ __device__ constexpr int64_t kv_head_bytes(int D, int P) { return (int64_t) P * (D + D / 16); }

// The tokens [q0, q0 + n) of a sequence and its length; n = 0 where q_start is no range of the batch's tokens.
struct SeqRange {
    int64_t q0;
    int n, len;
};
__device__ __forceinline__ SeqRange seq_range(const BatchView &b, int s) {
    const int64_t a = b.q_start[s], e = b.q_start[s + 1];
    SeqRange r;
    r.q0 = a;
    r.len = max(b.kv_len[s], 0);
    r.n = a >= 0 && e > a && e <= b.n_tok ? (int) (e - a) : 0;
    return r;
}

// Page of a position of sequence s, or -1: outside the table, or no page of the cache.
__device__ __forceinline__ int page_of(const KvView &c, const BatchView &b, int s, int pos) {
    const int64_t i = pos >> c.shift;
    if (pos < 0 || i >= b.table_stride) return -1;
    const int p = b.table[s * b.table_stride + i];
    return p >= 0 && p < c.n_pages ? p : -1;
}

// Parts of one kv head's share of a page (base: its first byte).
template <int D> struct KvParts {
    static constexpr int NB = D / 32;
    static __device__ __forceinline__ int64_t k_row(int P, int row) { return (int64_t) row * (D / 2); }
    static __device__ __forceinline__ int64_t v_col(int P, int j) { return (int64_t) P * (D / 2) + (int64_t) j * P; }
    static __device__ __forceinline__ int64_t k_scale(int P, int row) { return (int64_t) P * D + row * NB; }
    static __device__ __forceinline__ int64_t v_scale(int P, int row) { return (int64_t) P * (D + NB) + row * NB; }
};

// value(code) * 2^(e - 127) in f32; a 255 scale gives NaN.
__device__ __forceinline__ float kv_value(int code, int e) {
    constexpr uint64_t kTwice = 0x0C08060403020100ull;  // 2 * {0, .5, 1, 1.5, 2, 3, 4, 6}, a byte each
    const float v = 0.5f * (float) (int) ((kTwice >> (8 * (code & 7))) & 0xff);
    const float r = ldexpf(code & 8 ? -v : v, e - 127);
    return e == 255 ? __builtin_nanf("") : r;
}

// Scale byte of a block whose largest magnitude is amax (finite): the rule above.
template <class F> __device__ __forceinline__ int kv_scale_of(F amax) {
    if (amax == 0) return 0;
    int k;
    const F m = frexp(amax, &k);  // amax = m 2^k, m in [.5, 1)
    return min(max(k + 124 + (m > (F) 0.875 ? 1 : 0), 1), 254);
}
// Code of a value x, of which a = |x| in units of the block's scale.
template <class F> __device__ __forceinline__ uint32_t kv_code(F x, F a) {
    const uint32_t c = (uint32_t) (a > (F) 0.25) + (a >= (F) 0.75) + (a > (F) 1.25) + (a >= (F) 1.75) + (a > (F) 2.5) + (a >= (F) 3.5) +
                       (a > (F) 5);
    return c | (x < 0 ? 8u : 0u);
}

}  // namespace fns::dev

namespace fns::host {

// Checks of a cache and a batch over it (kv_cache.hip); `what` names the call.
int kv_check(const FnsKvCache *c, const FnsKvBatch *b, const char *what);
inline dev::KvView kv_view(const FnsKvCache *c) {
    int shift = 0;
    while ((1 << shift) < c->page_size) ++shift;
    return {(uint8_t *) c->pages, c->n_pages, c->n_head_kv * dev::kv_head_bytes(c->head_dim, c->page_size), c->n_head_kv, shift};
}
inline dev::BatchView kv_batch(const FnsKvBatch *b) {
    return {b->q_start, b->kv_len, b->page_table, b->n_tok, b->table_stride};
}

}  // namespace fns::host
