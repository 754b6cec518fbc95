/*
 * circatt_b200_tokens.h -- C ABI of the operators on token sequences: rotary positions, attention with a sliding
 * window and first tokens that stay visible, and the same attention over a paged cache.
 *
 * They have no counterpart in CirculantAttention.jl: its windows wrap around and are centred, which suits signals and
 * images.  A token stream has an end, is often read in one direction, and is served token by token from a cache.  The
 * conventions are those of circatt_b200.h (device pointers of the caller, a stream, an int status, no allocation, no
 * synchronisation); the differences are stated here.
 *
 *  - Dense tensors are (D, heads, N, B) arrays in Julia's notation with any strides, as long as the features are
 *    contiguous: element (f, h, t, b) sits at f + head*h + token*t + batch*b.  Addresses and strides are multiples of
 *    16 bytes.  Packed tokens of several sequences are (D, heads, T): `batch` is then unused.
 *  - A cache is (D, page, heads, pages): element (f, o, h, p) at f + token*o + head*h + page*p, the same rules.
 *  - dtype: CA_F32, CA_BF16 or CA_F16.  Sums, statistics and angles are held in 32 bits or more.
 *  - heads_q is a multiple of heads_kv; query head h reads key head h / (heads_q / heads_kv).
 */
#ifndef CIRCATT_B200_TOKENS_H
#define CIRCATT_B200_TOKENS_H
#include <stddef.h>
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

enum { CA_F16 = 3 };   /* element type of these operators, next to CA_F32 and CA_BF16 */
#define CA_MAX_AXES 4

/* Strides in elements. */
typedef struct ca_seq_view {
    void* data;
    int64_t head, token, batch;
} ca_seq_view;

typedef struct ca_page_view {
    void* data;
    int64_t token, head, page;
} ca_page_view;

/* The sequences of a batch in a paged cache.  Sequence s has the packed tokens starts[s] .. starts[s+1]-1, the last ones
 * of the lengths[s] tokens that its pages hold, and token j lives at offset j % page of page table[j / page + width*s].
 * An entry outside 0 .. pages-1 is a page that is gone: its tokens are not visible and nothing is stored there.  Packed tokens
 * before starts[0] and from starts[sequences] on belong to no sequence: attention gives zeros for them, and the cache write
 * leaves them out. */
typedef struct ca_pages {
    const int32_t* table;     /* (width, sequences) */
    const int32_t* starts;    /* (sequences + 1) */
    const int32_t* lengths;   /* (sequences) */
    int32_t width, page, pages, sequences;
} ca_pages;

/* ---------------------------------------------------------------- rotary positions
 * Pair p of a head's features is turned by the angle 2 pi * position * turns[p] / 2^64, the position being that of the
 * pair's axis: the first sections[0] pairs turn with axis 0, the next sections[1] with axis 1, and so on.  `turns` are
 * 64-bit two's complement fractions of a turn, so that the product with an integer position is exact modulo one turn at
 * any distance.  Pairs are (2p, 2p+1) with `interleaved`, else (p, p + pairs); features from 2*pairs on pass unchanged.
 * `inverse` turns back: the gradient of the rotation.  positions: (axes, N, B) with strides. */
typedef struct ca_rotary_desc {
    int32_t dtype, dim, pairs, interleaved, inverse;
    int32_t axes, sections[CA_MAX_AXES];
    int32_t tokens, batch;
    const int32_t* positions;
    int64_t axis_stride, token_stride, batch_stride;
    const int64_t* turns;
} ca_rotary_desc;

/* Up to two tensors (q and k) of the same tokens in one launch; x2 may be NULL. */
int ca_rotary(const ca_rotary_desc* d, const ca_seq_view* x1, const ca_seq_view* y1, int32_t heads1,
              const ca_seq_view* x2, const ca_seq_view* y2, int32_t heads2, void* stream);

/* The serving form: q is turned into q_out, k is turned and stored into the cache, v is stored as it is.  d->tokens
 * packed tokens, d->batch = 1. */
int ca_rotary_append(const ca_rotary_desc* d, const ca_seq_view* q, const ca_seq_view* q_out, int32_t heads_q,
                     const ca_seq_view* k, const ca_seq_view* v, int32_t heads_kv,
                     const ca_page_view* k_pages, const ca_page_view* v_pages, const ca_pages* pages, void* stream);

/* ---------------------------------------------------------------- attention with a window and first tokens
 * Key j is visible to query i when both are below the sequence's length, j <= i + right, and j >= i - left or
 * j < sinks; left < 0: no left end.  y = softmax over the visible keys of scale * q.k, times v; a query that sees
 * nothing gives zeros.  What invisible keys hold beyond the length, or in pages that no query of the call sees, has no
 * effect, NaN and infinities included. */
typedef struct ca_seq_desc {
    int32_t dtype, dim, heads_q, heads_kv;
    int32_t tokens, batch;              /* N and B; packed tokens and 1 over a paged cache */
    int32_t left, right, sinks;
    float scale;
} ca_seq_desc;

/* lengths: B int32, or NULL for N each.  lse (nullable): heads_q*N*B floats, the logarithm to base 2 of each row's sum
 * (-inf: the row sees nothing), group member fastest, then token, key head, batch: what the backward needs.
 * y_rest (nullable): what rounding took from y, in the same type.  The backward subtracts dy.y from each dy.v; with y
 * alone, gradients of short windows in 16-bit types come out up to half as wrong again as their own rounding makes them
 * (2.7e-3 against 1.7e-3 of the norm in bfloat16). */
int ca_window_fwd(const ca_seq_desc* d, const ca_seq_view* q, const ca_seq_view* k, const ca_seq_view* v,
                  const int32_t* lengths, const ca_seq_view* y, const ca_seq_view* y_rest, float* lse, void* stream);

/* Gradients of the above for the cotangent dy.  Deterministic: no atomics.  The workspace is 16-byte aligned. */
size_t ca_window_bwd_workspace(const ca_seq_desc* d);
int ca_window_bwd(const ca_seq_desc* d, const ca_seq_view* q, const ca_seq_view* k, const ca_seq_view* v,
                  const ca_seq_view* y, const ca_seq_view* y_rest, const ca_seq_view* dy, const int32_t* lengths, const float* lse,
                  const ca_seq_view* dq, const ca_seq_view* dk, const ca_seq_view* dv, void* workspace, void* stream);

/* A chunk of new tokens, whose keys are already stored, over a paged cache; right is 0. */
int ca_paged_window(const ca_seq_desc* d, const ca_seq_view* q, const ca_page_view* k_pages, const ca_page_view* v_pages,
                    const ca_pages* pages, const ca_seq_view* y, void* stream);

#ifdef __cplusplus
}
#endif
#endif
