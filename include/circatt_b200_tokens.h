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

/* ---------------------------------------------------------------- the same with other scores and masks
 * Scores are cap * tanh(scale * q.k / cap) where there is a cap, less slopes[query head] * |i - j| where there are slopes.
 *
 * spans (dense calls): what each token sees, made once a batch by ca_token_spans for the calls of all layers.  With spans the
 * key j is visible to the query i when both are below the sequence's length, they are of one document, j >= i - left (or
 * left < 0), and j <= i or both are of one group; right and sinks are 0.
 *
 * prefix (calls over a cache): prefix[s] tokens of sequence s are visible to all of its tokens, whether they come later or
 * not, as far as the window's left end leaves them. */
typedef struct ca_seq_form {
    float cap;                /* 0: scores as they are; up to 2^100 */
    const float* slopes;      /* heads_q, nullable */
    const int32_t* spans;     /* (4, N, B), 16-byte aligned, nullable */
    const int32_t* prefix;    /* (sequences), nullable */
} ca_seq_form;

/* From the number of each token's document and group to spans.  A document is a run of equal numbers that are not negative,
 * negative numbers are padding, which sees nothing and is seen by nothing; a group is a run of equal positive numbers within a
 * document.  documents, groups (nullable): (N, B); spans: (4, N, B), for each token the first one that it sees, the first one
 * that sees it, the last one that it sees, the last one that sees it. */
int ca_token_spans(const int32_t* documents, const int32_t* groups, int32_t tokens, int32_t batch, int32_t* spans, void* stream);

int ca_window_form_fwd(const ca_seq_desc* d, const ca_seq_form* form, const ca_seq_view* q, const ca_seq_view* k, const ca_seq_view* v,
                       const int32_t* lengths, const ca_seq_view* y, const ca_seq_view* y_rest, float* lse, void* stream);
/* Takes a workspace of ca_window_bwd_workspace(d) bytes.  There is no gradient of the slopes. */
int ca_window_form_bwd(const ca_seq_desc* d, const ca_seq_form* form, const ca_seq_view* q, const ca_seq_view* k, const ca_seq_view* v,
                       const ca_seq_view* y, const ca_seq_view* y_rest, const ca_seq_view* dy, const int32_t* lengths, const float* lse,
                       const ca_seq_view* dq, const ca_seq_view* dk, const ca_seq_view* dv, void* workspace, void* stream);
int ca_paged_window_form(const ca_seq_desc* d, const ca_seq_form* form, const ca_seq_view* q, const ca_page_view* k_pages,
                         const ca_page_view* v_pages, const ca_pages* pages, const ca_seq_view* y, void* stream);

/* ---------------------------------------------------------------- the pages of a cache
 * A state: the table, for each page the number of table entries that hold it (refs; a page is free if that is not above 0), and
 * the tokens of each sequence.  The operators read one and write the next into other memory; all of it is on the device and
 * nothing waits for the host.  Pages are taken from the lowest number on, for sequences and places in their order.  At most 2^30
 * sequences and pages. */
typedef struct ca_table {
    const int32_t* table;     /* (width, sequences) */
    const int32_t* refs;      /* (pages) */
    const int32_t* lengths;   /* (sequences); ca_compact_pages does not read it */
    int32_t width, sequences, page, pages;
} ca_table;

/* The keys or the values of one layer, of any type; strides in bytes.  One row is a token's features of one head. */
typedef struct ca_pool {
    void* data;
    int64_t token, head, page;
    int32_t row, tokens, heads;
} ca_pool;

size_t ca_pages_workspace(const ca_table* t);

/* Before a call's new tokens are stored: lengths[s] counts the starts[s+1] - starts[s] new tokens of sequence s with it.  Pages
 * that neither they nor later tokens see (a window of `left`, negative: no left end; the first `sinks` tokens), and those
 * behind the length, are given back, all of them where the length is 0; places of new tokens without a page get one.  *missing:
 * places of the table that got none.  Tokens beyond the table's width have no place: they are not stored and not counted there.
 *
 * A place that has a page keeps it, however many entries hold that page.  A sequence that has become shorter so that it ends within a
 * page of others (ca_fork_pages shares full ones) would therefore write its next tokens into theirs: fork it before they come, with
 * its parent going on, and the copy has a last page of its own. */
int ca_advance_pages(const ca_table* t, const int32_t* starts, int32_t left, int32_t sinks, int32_t* table, int32_t* refs, int32_t* missing,
                     void* workspace, void* stream);

/* Sequence s continues as a copy of sequence parents[s] as it was before the call; itself: it stays as it is; no sequence: it
 * becomes empty.  Pages are shared, but for the partly filled last one: the parent keeps it if it goes on, else the first that
 * continues it, and the others get copies in all pools.  *missing: copies that found no free page; their place has no page. */
int ca_fork_pages(const ca_table* t, const int32_t* parents, const ca_pool* pools, int32_t npools, int32_t* table, int32_t* refs,
                  int32_t* lengths, int32_t* missing, void* workspace, void* stream);

/* Moves the pages in use to the lowest numbers; *live: how many there are.  Entries of pages that are not in use become -1. */
int ca_compact_pages(const ca_table* t, const ca_pool* pools, int32_t npools, int32_t* table, int32_t* refs, int32_t* live,
                     void* workspace, void* stream);

#ifdef __cplusplus
}
#endif
#endif
