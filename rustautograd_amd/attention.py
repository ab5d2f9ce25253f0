"""Attention whose scores are capped, fall with distance or are closed by documents and prefixes, and
its form over a paged cache. Each is one operation of the engine with kernels of its own; contexts
may be long, since no score is kept. The reference has no counterpart.

Values are float32 or float64, one dtype a call; documents, prefixes, lengths, tables and positions
are int32. Heads have at most 256 values, of float64 on the device at most 128.
"""

import math

from .ops import _as_index
from .sequence import _present, _with_results
from .tensor import error

# The operand and variant flags of include/rg_plan.h.
_JOINED, _SLOPES, _DOCUMENTS, _PREFIX, _LENGTHS, _CAUSAL = 1, 2, 4, 8, 16, 32


def _parts(q, k, v, heads):
    """(operands, (heads, key heads), head, flags) of queries, keys and values, or of all in one."""
    if q.ndim != 4 or (k is not None and k.ndim != 4):
        raise error("SHAPE_MISMATCH", {"input_shapes": [list(x.shape) for x in (q, k) if x is not None]}, "heads_must_be_batch_length_heads_head")
    if (k is None) != (v is None):
        raise error("INVALID_ARGUMENT", {"k": k is not None, "v": v is not None}, "k_and_v_go_together")
    if k is None:
        if heads is None:
            raise error("INVALID_ARGUMENT", {"heads": None}, "heads_of_q_and_of_k_must_be_given_for_a_joined_operand")
        pair = tuple(int(n) for n in heads)
        if len(pair) != 2 or min(pair) < 1:
            raise error("INVALID_ARGUMENT", {"heads": list(pair)}, "heads_must_be_two_positive_counts")
        return (q,), pair, _JOINED
    if heads is not None:
        raise error("INVALID_ARGUMENT", {"heads": list(heads)}, "heads_are_given_for_a_joined_operand_only")
    return (q, k, v), (q.shape[2], k.shape[2]), 0


def _attrs(q, pair, scale, cap, flags):
    if cap is not None and not cap > 0:
        raise error("INVALID_ARGUMENT", {"cap": cap}, "cap_must_be_positive")
    return {"flags": flags, "heads": list(pair), "scale": 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale),
            "cap": 0.0 if cap is None else float(cap)}


def attention(q, k=None, v=None, heads=None, causal=True, scale=None, cap=None, slopes=None, documents=None, prefix=None, lengths=None):
    """Self-attention of `q` (batch, length, heads, head) over `k` and `v` (batch, length, key heads,
    head), where each key head serves heads / key heads neighbouring heads of q. Without `k` and `v`,
    `q` is (batch, length, heads + 2 * key heads, head), the heads of q, k and v one after the other
    as one projection makes them, and `heads` the pair (heads, key heads).

    A score is `scale` q.k, 1 / sqrt(head) by default; with `cap`, cap * tanh(score / cap); with
    `slopes` (heads,), lowered by slope * |i - j|. Query i sees key j if j <= i (any j if not
    `causal`), or j < `prefix` (batch,); if both are of the same document of `documents` (batch,
    length), of which a negative one is none; and if both are before `lengths` (batch,). A query that
    sees nothing gives 0. Infinities and NaN reach what sees them and nothing else; what lies past the
    lengths or in no document is not looked at. Differentiable in q, k, v and the slopes, once."""
    operands, pair, flags = _parts(q, k, v, heads)
    index = [x if x is None else _as_index(x) for x in (documents, prefix, lengths)]
    values, mask = _present(operands, (slopes, *index), (_SLOPES, _DOCUMENTS, _PREFIX, _LENGTHS))
    return _with_results("attention", values, _attrs(q, pair, scale, cap, flags | mask | (_CAUSAL if causal else 0)), 1)[0]


def paged_attention(q, k=None, v=None, *, cache, table, first, lengths=None, heads=None, scale=None, cap=None, slopes=None):
    """Attention of new tokens over a paged cache, for single tokens and for chunks of a prompt:
    returns `(y, cache)`, the cache with the new tokens' keys and values in it. `q`, `k` and `v`, or
    `q` alone with `heads`, are those of `attention`, of the new tokens.

    `cache` is a pair of pages (pages, page, key heads, head), of keys and of values; `table` (batch,
    n) names the pages of each sequence, position p lying in row p % page of page table[b, p //
    page]; `first` (batch,) is the number of positions that sequence b already has. Its new tokens
    stand at first, first + 1, ...; each sees every position before it and itself, with `scale`, `cap`
    and `slopes` as in `attention`. With `lengths` (batch,), only the first lengths[b] of the new
    tokens are there: for the others y is 0 and nothing is written.

    A table's entry that is no page, or a position past the table, has no row: nothing is read or
    written there. The rows before `first` are read as they were, and of two sequences that write one
    row the later one's stays. A step loop that carries the cache in its state, and uses it nowhere
    else, writes the rows into it in place. Not differentiable."""
    operands, pair, flags = _parts(q, k, v, heads)
    pages = tuple(cache)
    if len(pages) != 2:
        raise error("INVALID_ARGUMENT", {"cache": len(pages)}, "cache_must_be_the_pages_of_k_and_of_v")
    if lengths is not None:
        lengths = _as_index(lengths)
    values, mask = _present((*operands, *pages, _as_index(table), _as_index(first)), (slopes, lengths), (_SLOPES, _LENGTHS))
    y, keys, held = _with_results("paged_attention", values, _attrs(q, pair, scale, cap, flags | mask), 3)
    return y, (keys, held)
