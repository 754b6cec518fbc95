"""Operators on token sequences, next to the circulant attention of signals and images.

Circulant windows wrap around and are centred.  A token stream has an end, is mostly read in one direction and is served
token by token, so it needs windows that do not wrap, a few first tokens that stay visible when they have left the window,
positions (a window alone does not know where a token is), and a cache:

* `rotary` turns q and k by their positions, on one axis or several (time, height, width); differentiable;
* `window_attention` is attention with such a window, forward and backward;
* `rotary_append_` and `paged_window_attention` are the same two for serving: a chunk of new tokens per sequence (one when
  decoding), whose keys and values live in a paged cache;
* `token_spans` makes the document and prefix masks of a batch for `window_attention`;
* `advance_pages`, `fork_pages` and `compact_pages` keep the pages of such a cache.

Tensors are Julia-shaped like those of the rest of the package, but features come first, not the image: `(D, heads, N, B)`,
packed tokens of several sequences `(D, heads, T)`, a cache `(D, page, heads, pages)`; a tensor of the circulant operators has
to be transposed.  Column-major storage is what `jl` makes; any other strides are taken as they are when the features are
contiguous and the rest is 16-byte aligned, else the tensor is copied.  Float32, BFloat16 and Float16; q may have a multiple of
the heads of k and v.  Everything runs on torch's current stream."""
from __future__ import annotations

import math

import torch

from ._lib import host


def rotary_turns(pairs, base=10000.0, sections=None, device="cuda"):
    """Turns per position of each pair of features, as 64-bit fractions of a turn (Int64, for `rotary`).

    Pair p turns by base^(-p / pairs) radians per position: one ladder of frequencies over all axes.  With `sections`
    each axis gets a ladder of its own, base^(-i / n) for the i-th of its n pairs."""
    if pairs < 1:
        raise AssertionError(f"pairs ({pairs}) must be positive")
    if sections is not None and sum(sections) != pairs:
        raise AssertionError(f"the sections {tuple(sections)} do not hold {pairs} pairs")
    ladders = [pairs] if sections is None else list(sections)
    fixed = [round(float(base) ** (-i / n) / (2 * math.pi) * 2.0 ** 64) % (1 << 64) for n in ladders for i in range(n)]
    return torch.tensor([f - (1 << 64) if f >= (1 << 63) else f for f in fixed], dtype=torch.int64, device=device)


def _sections(sections, turns):
    return [int(n) for n in sections] if sections is not None else [turns.numel()]


def rotary(x, positions, turns, sections=None, interleaved=False):
    """Rotary positions: pair p of each head is turned by `positions * turns[p]`; differentiable in `x`.

    x: `(D, heads, N, B)` or `(D, heads, T)`, or a tuple (q, k) of two such tensors that differ in their heads, which take
    one launch.  positions: Int32 `(axes, N, B)`, or `(axes, N)` for the whole batch.  The first `sections[0]` pairs turn
    with axis 0, the next `sections[1]` with axis 1, and so on (up to four axes; default: all with the only axis).  Pairs are
    features (2p, 2p+1) when `interleaved`, else (p, p + pairs); features from 2 * pairs on pass unchanged.  Angles are
    exact modulo one turn at any position."""
    if isinstance(x, (tuple, list)):
        if len(x) != 2:
            raise TypeError(f"x is one tensor or two (q, k), got {len(x)}")
        return host.rotary(x[0], x[1], positions, turns, _sections(sections, turns), bool(interleaved))
    return host.rotary(x, None, positions, turns, _sections(sections, turns), bool(interleaved))[0]


def rotary_append_(q, k, v, k_pages, v_pages, table, starts, lengths, positions, turns, sections=None, interleaved=False):
    """The serving form of `rotary`: returns the turned q, and stores the turned k and v as it is into the cache.

    q, k, v: packed tokens `(D, heads, T)`; tokens `starts[s]` to `starts[s+1] - 1` are the last ones of the `lengths[s]`
    tokens that sequence s has with them.  Token j of the sequence lives at offset `j % page` of page
    `table[j // page, s]` of `k_pages` and `v_pages`, `(D, page, heads, pages)` with pages of a multiple of 16 tokens; where
    the table has no valid page nothing is stored.  positions: `(axes, T)`.  Tokens of no sequence, before `starts[0]` and
    from `starts[S]` on (a call of fixed size that is not full), are turned in q and not stored.  No gradients."""
    return host.rotary_append(q, k, v, k_pages, v_pages, table, starts, lengths, positions, turns, _sections(sections, turns),
                              bool(interleaved))


def _left(left):
    if left is None:
        return -1
    if left < 0:
        raise AssertionError(f"left ({left}) must not be negative: None is a window without a left end")
    return int(left)


def token_spans(documents, groups=None):
    """Document and prefix masks for `window_attention`: which tokens each token sees, from numbers that say what it belongs to.

    documents: Int32 `(N, B)` or `(N,)`.  A document is a run of equal numbers; tokens see their own document only.  Negative
    numbers are padding, which sees nothing and is seen by nothing.  groups: the same size; a group is a run of equal positive
    numbers within a document, whose tokens see each other both ways (the prefix of a prompt, a picture between text, a whole
    document); all others see up to themselves.  The result, Int32 `(4, N, B)`, serves the calls of all layers on this batch."""
    return host.token_spans(documents, groups)


def window_attention(q, k, v, left, right=0, sinks=0, lengths=None, scale=None, cap=None, slopes=None, spans=None):
    """y_i = sum_j softmax_j(score_ij) v_j over the tokens j that token i sees: those from i - left to i + right, and the first
    `sinks` ones as long as they are not later than i + right.  Differentiable in q, k, v; deterministic.

    q `(D, heads, N, B)`, k and v `(D, heads', N, B)` with heads a multiple of heads'; D a multiple of 8 up to 128.
    left=None: no left end.  lengths: Int32 `(B,)`, the tokens that exist in each sequence (what lies behind them has no
    effect, whatever it holds; y and the gradients are zero there).

    The score is scale * q_i . k_j, scale 1/sqrt(D) by default.  cap: it becomes cap * tanh(score / cap), cap up to 2^100.
    slopes: Float32 `(heads,)`, slopes[head] * |i - j| is taken from it after the cap; no gradient.  spans: what `token_spans`
    says of the tokens' documents and groups takes the place of `right` and `sinks`, which are 0 then: token i sees those of its
    document from i - left to i or, if that is further, to the end of its group.

    Infinities and NaN in keys or values that no token sees have no effect.  Where some token sees them, neighbours that do
    not may get NaN too: their weight is zero, and zero times infinity is not a number."""
    return host.window_attention(q, k, v, _left(left), int(right), int(sinks), lengths, scale, cap, slopes, spans)


def paged_window_attention(q, k_pages, v_pages, table, starts, lengths, left=None, sinks=0, scale=None, cap=None, slopes=None,
                           prefix=None):
    """`window_attention` (right = 0) of a chunk of new tokens for each sequence over a paged cache that holds their keys
    and values already (see `rotary_append_` for the layout).  Returns y `(D, heads, T)`.

    cap, slopes: as there.  prefix: Int32 `(S,)`, the first prefix[s] tokens of sequence s are visible to all of its tokens,
    later ones among them, as far as the window's left end leaves them and the cache holds them.

    Tokens that no new token sees are not read, so the pages behind the window may be freed: any page number, -1 among
    them, may stand in their place in the table.  A missing page (-1) inside the window is skipped.  No gradients."""
    return host.paged_window_attention(q, k_pages, v_pages, table, starts, lengths, _left(left), int(sinks), scale, cap, slopes,
                                       prefix)


def advance_pages(table, refs, starts, lengths, page, left=None, sinks=0):
    """The pages of a serving step, before `rotary_append_` stores its new tokens.  Returns the next (table, refs, missing).

    table, starts, lengths: as for `paged_window_attention`, with the new tokens counted.  refs: Int32 `(pages,)`, how many
    table entries hold each page; a page is free where that is not above 0.  Pages that neither the new nor later tokens see
    through a window of `left` and `sinks`, and those behind a sequence's length, go back: all of them where the length is 0 (a
    sequence that has ended).  Places of new tokens without a page get the lowest free ones, sequence by sequence, pages of
    this call among them.  missing: Int32 `(1,)`, places that got none; tokens there are not stored, and neither are those beyond
    the table's width, which have no place to count: the table has to be wide enough for the lengths.

    A place that has a page keeps it.  After `fork_pages` full pages belong to several sequences: one that is then made shorter, to
    end within such a page, would write its next tokens into the others' page.  Fork it once more before they come, with its
    parent going on as it is: the copy's last page is its own.

    Like the other operators on pages it gives a new state and leaves the old one as it is, and nothing waits for the host; a
    captured step copies the new table and refs over the old ones at its end."""
    return host.advance_pages(table, refs, starts, lengths, int(page), _left(left), int(sinks))


def fork_pages(pools, table, refs, lengths, parents):
    """Sequences that continue as copies of others: answers to one prompt, beams.  Returns the next (table, refs, lengths,
    missing) and copies pages in `pools`, in place.

    parents: Int32 `(S,)`; sequence s continues sequence parents[s] as it was before the call.  Its own number: it stays as it
    is.  A number that is no sequence, -1: it becomes empty, and its pages go back.  pools: the `(D, page, heads, pages)`
    tensors of all layers, keys and values, of any types.  Full pages are shared; the partly filled last one stays with the
    parent if it goes on, else with the first that continues it, and the others get copies in the lowest free pages.  missing:
    Int32 `(1,)`, copies that found none; the place is then -1 and its tokens are not visible."""
    return host.fork_pages(list(pools), table, refs, lengths, parents)


def compact_pages(pools, table, refs):
    """Moves the pages in use to the lowest numbers, in order, so that the rest of the cache can be given up or cut off.  Returns
    the next (table, refs, live), live Int32 `(1,)` the pages in use; `pools` are changed in place.  Pages that lie low enough
    already stay.  A table entry whose page has no count becomes -1."""
    return host.compact_pages(list(pools), table, refs)
