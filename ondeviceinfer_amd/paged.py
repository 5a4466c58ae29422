"""Operators over a paged fp16 key/value cache: many sequences of different
lengths in one call.

The reference's cache holds one contiguous tensor per layer and one length for
the whole batch (``ondeviceinfer/cache.py:22-92``), and its rotation, cache
update and attention work on such batches (``layers.py:64-80``,
``attention.py:35-85``).  Here the keys and values of a layer lie in a pool of
pages ``[pages, kv_heads, page_size, 128]``, a sequence is a row of page
numbers, and one call serves single tokens, chunks of prompts and trees of
drafted tokens side by side.
"""
from __future__ import annotations

from typing import NamedTuple

from torch import Tensor

from . import _native


class PagedBatch(NamedTuple):
    """Which tokens of a call belong to which sequence, and where its pages are.

    ``page_table`` int32 ``[sequences, pages]``: position ``i`` of sequence
    ``b`` is row ``i % page_size`` of page ``page_table[b, i // page_size]``
    (entries behind its length are never read); ``query_starts`` int32
    ``[sequences + 1]``: tokens ``query_starts[b] .. query_starts[b + 1] - 1``
    are the newest of sequence ``b``; ``seq_lens`` int32 ``[sequences]``: its
    positions, those tokens included.  All on the device, read there."""

    page_table: Tensor
    query_starts: Tensor
    seq_lens: Tensor


def paged_append(qkv: Tensor, key_pages: Tensor, value_pages: Tensor, batch: PagedBatch, *, q_heads: int,
                 q_norm: Tensor | None, k_norm: Tensor | None, eps: float, cos_table: Tensor, sin_table: Tensor,
                 positions: Tensor | None = None, out: Tensor | None = None) -> Tensor:
    """Per-head q/k RMSNorm and rotation of the fused q|k|v rows ``[tokens,
    (q_heads + 2 kv_heads) * 128]``; k and v land in their sequences' pages,
    the queries come back as ``[tokens, q_heads, 128]``.

    ``q_norm`` / ``k_norm`` may be None (no norm).  A token is rotated by row
    ``positions[token]`` of the tables, its index in the sequence by default.
    A token without a page or a table row gets NaN queries and writes nothing;
    rows behind the last sequence keep what ``out`` held."""
    return _native.paged_append(qkv, q_heads, q_norm, k_norm, eps, cos_table, sin_table, key_pages, value_pages,
                                batch.page_table, batch.query_starts, batch.seq_lens, positions, out)


def paged_attention(query: Tensor, key_pages: Tensor, value_pages: Tensor, batch: PagedBatch, *, scale: float,
                    tree_mask: Tensor | None = None, out: Tensor | None = None,
                    workspace: Tensor | None = None) -> Tensor:
    """Grouped-query attention of ``[tokens, q_heads, 128]`` queries over the
    pages of their sequences, which hold the new tokens' keys already
    (``paged_append``).

    Without ``tree_mask`` every token attends its sequence up to itself.  With
    it (int64 ``[tokens]``) the new tokens of a sequence, at most 64, are
    drafted ones: each attends everything before them, and of them those whose
    bit is set in its mask (its own bit included).  A token that attends
    nothing gets zeros, one that attends a position without a page NaN; rows
    behind the last sequence keep what ``out`` held."""
    return _native.paged_attention(query, key_pages, value_pages, batch.page_table, batch.query_starts, batch.seq_lens,
                                   scale, tree_mask, out, workspace)
