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

from dataclasses import dataclass
from typing import NamedTuple, Sequence

import torch
from torch import Tensor

from . import _native

MAX_TREE_TOKENS = 64   # drafted tokens of one sequence in one step: one bit of the mask each


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
    of two that name the same row of a page the elements of either are left;
    rows behind the last sequence keep what ``out`` held.  ``out`` must not
    overlap ``qkv``."""
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
    behind the last sequence keep what ``out`` held.  ``out`` may be ``query``
    itself and must not overlap it otherwise."""
    return _native.paged_attention(query, key_pages, value_pages, batch.page_table, batch.query_starts, batch.seq_lens,
                                   scale, tree_mask, out, workspace)


def tree_layout(parents: Sequence[int]) -> tuple[list[int], list[int]]:
    """``(masks, depths)`` of a tree of drafted tokens: token ``i`` follows token
    ``parents[i] < i``, or the cached tokens where that is -1.  A mask has the
    bits of the token's ancestors and its own; the depth of a token that follows
    the cached ones is 0."""
    if len(parents) > MAX_TREE_TOKENS:
        raise ValueError(f'at most {MAX_TREE_TOKENS} drafted tokens per sequence, got {len(parents)}')
    masks, depths = [], []
    for i, parent in enumerate(parents):
        if not -1 <= parent < i:
            raise ValueError(f'parent of token {i} must be -1 or an earlier token, got {parent}')
        masks.append((masks[parent] if parent >= 0 else 0) | (1 << i))
        depths.append(depths[parent] + 1 if parent >= 0 else 0)
    return masks, depths


class PagedKVCache:
    """The keys and values of all layers in one pool of pages,
    ``[2, layers, pages, kv_heads, page_size, head_dim]`` (K then V), shared by
    any number of sequences.

    A sequence is an integer handed out by ``add``; its pages are taken from
    the pool as it grows and given back by ``truncate`` and ``free``.  The
    bookkeeping is the host's; a step's ``PagedBatch`` carries it to the
    device."""

    def __init__(self, *, num_layers: int, num_pages: int, num_key_value_heads: int, head_dim: int,
                 device: torch.device | str, dtype: torch.dtype = torch.float16, page_size: int = 16) -> None:
        if num_pages <= 0:
            raise ValueError(f'num_pages must be positive, got {num_pages}')
        if page_size <= 0 or page_size % 16:
            raise ValueError(f'page_size must be a positive multiple of 16, got {page_size}')
        self.page_size, self.num_pages, self.device = page_size, num_pages, torch.device(device)
        self._block = torch.empty((2, num_layers, num_pages, num_key_value_heads, page_size, head_dim), device=device,
                                  dtype=dtype)
        self.key_pages = list(self._block[0].unbind(0))
        self.value_pages = list(self._block[1].unbind(0))
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}
        self._lengths: dict[int, int] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def storage_bytes(self) -> int:
        return self._block.numel() * self._block.element_size()

    def add(self) -> int:
        """A new, empty sequence."""
        seq = self._next
        self._next += 1
        self._pages[seq], self._lengths[seq] = [], 0
        return seq

    def length(self, seq: int) -> int:
        return self._lengths[seq]

    def free(self, seq: int) -> None:
        """Forget a sequence; its pages go back to the pool."""
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._lengths[seq]

    def truncate(self, seq: int, length: int) -> None:
        """Forget a sequence's positions from ``length`` on."""
        if not 0 <= length <= self._lengths[seq]:
            raise ValueError(f'sequence {seq} has {self._lengths[seq]} positions, cannot keep {length}')
        pages = self._pages[seq]
        while len(pages) * self.page_size >= length + self.page_size:
            self._free.append(pages.pop())
        self._lengths[seq] = length

    def extend(self, sequences: Sequence[int], counts: Sequence[int]) -> PagedBatch:
        """Room for ``counts[i]`` new tokens of ``sequences[i]``, and the batch
        that a step over them takes.  Nothing has changed if it raises (too few
        pages in the pool, no memory for the batch)."""
        if len(sequences) != len(counts) or len(set(sequences)) != len(sequences):
            raise ValueError('a step takes each of its sequences once, with a count each')
        if any(n < 0 for n in counts):
            raise ValueError('counts must not be negative')
        lens = [self._lengths[s] + n for s, n in zip(sequences, counts)]
        want = [-(-n // self.page_size) - len(self._pages[s]) for s, n in zip(sequences, lens)]
        if sum(want) > len(self._free):
            raise ValueError(f'KV cache capacity exceeded: {sum(want)} more pages needed, {len(self._free)} free')
        spare = reversed(self._free)
        more = [[next(spare) for _ in range(n)] for n in want]
        rows = [self._pages[s] + pages for s, pages in zip(sequences, more)]
        width = max([1, *map(len, rows)])
        rows = [row + [-1] * (width - len(row)) for row in rows]
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        # One copy to the device for all three.
        flat = torch.tensor([x for row in rows for x in row] + starts + lens, dtype=torch.int32).to(self.device)
        for s, pages, n in zip(sequences, more, lens):
            self._pages[s].extend(pages)
            self._lengths[s] = n
        del self._free[len(self._free) - sum(want):]
        table = len(rows) * width
        return PagedBatch(flat[:table].view(len(rows), width), flat[table:table + len(starts)],
                          flat[table + len(starts):])

    def keep(self, seq: int, start: int, accepted: Sequence[int]) -> None:
        """Of the tokens from position ``start`` on (a step's drafted ones) keep
        those ``accepted`` (indices from ``start``, ascending), moved up to
        follow it without gaps, in all layers; forget the others."""
        length = self._lengths[seq]
        if any(b <= a for a, b in zip(accepted, accepted[1:])):
            raise ValueError('accepted tokens must be in ascending order')
        if not 0 <= start <= length or (accepted and not (0 <= accepted[0] and start + accepted[-1] < length)):
            raise ValueError(f'accepted tokens must lie in the positions {start} .. {length - 1} of sequence {seq}')
        pages, size = self._pages[seq], self.page_size
        moves = [(start + j, start + i) for i, j in enumerate(accepted) if i != j]
        if moves:
            index = torch.tensor([(pages[a // size], a % size, pages[b // size], b % size) for a, b in moves]).to(
                self.device)
            from_page, from_row, to_page, to_row = index.unbind(1)
            # The rows are read before any is written.
            self._block[:, :, to_page, :, to_row] = self._block[:, :, from_page, :, from_row]
        self.truncate(seq, start + len(accepted))


@dataclass
class PagedStep:
    """One forward step over a paged cache: the new tokens of its sequences,
    handed to the decoder layers in the place of a cache."""

    cache: PagedKVCache
    batch: PagedBatch
    cos_table: Tensor
    sin_table: Tensor
    scale: float
    positions: Tensor | None = None
    tree_mask: Tensor | None = None

    def attend(self, layer_idx: int, qkv: Tensor, q_heads: int, q_norm: Tensor | None, k_norm: Tensor | None,
               eps: float) -> Tensor:
        """``[tokens, q_heads, head_dim]`` attention output of the fused
        projection's rows, their keys and values appended to the layer's pages."""
        keys, values = self.cache.key_pages[layer_idx], self.cache.value_pages[layer_idx]
        query = paged_append(qkv, keys, values, self.batch, q_heads=q_heads, q_norm=q_norm, k_norm=k_norm, eps=eps,
                             cos_table=self.cos_table, sin_table=self.sin_table, positions=self.positions)
        return paged_attention(query, keys, values, self.batch, scale=self.scale, tree_mask=self.tree_mask)
