"""The paged-cache operators (paged.paged_append, paged.paged_attention) against
their formulas in 64 bits on the CPU: ragged batches, page sizes and head
groups, trees of drafted tokens, rows that attend nothing, pages that do not
exist, padding, strided pools, captured replays."""
import math
import random

import pytest
import torch

from ondeviceinfer_amd.layers import RotaryEmbedding
from ondeviceinfer_amd.paged import PagedBatch, paged_append, paged_attention

pytestmark = pytest.mark.gpu
D = 128
HALF_ULP = 2.0 ** -11          # fp16: a rounding's largest relative error
TINY = 2.0 ** -25              # ... and its largest absolute one among the subnormals


class Pool:
    """Pages in random order; every row that belongs to no sequence holds NaN."""

    def __init__(self, new, past, *, hq, hkv, page, seed, interleaved=False, extra_width=1, pad=0):
        gen = torch.Generator().manual_seed(seed)
        self.new, self.past, self.hq, self.hkv, self.page = new, past, hq, hkv, page
        lens = [n + p for n, p in zip(new, past)]
        used = [(max(n, 0) + page - 1) // page for n in lens]
        pages = sum(used) + 2
        order = torch.randperm(pages, generator=gen).tolist()
        width = max(used) + extra_width
        self.table = torch.full((len(new), width), -7, dtype=torch.int32)
        shape = (pages, 2, hkv, page, D) if interleaved else (2, pages, hkv, page, D)
        block = torch.full(shape, float('nan'), dtype=torch.float16)
        self.k, self.v = (block[:, 0], block[:, 1]) if interleaved else (block[0], block[1])
        at = 0
        for b, n in enumerate(lens):
            for e in range(used[b]):
                self.table[b, e] = order[at]
                at += 1
                rows = min(page, n - e * page)
                for t in (self.k, self.v):
                    t[order[at - 1], :, :rows] = torch.randn(hkv, rows, D, generator=gen).half()
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.starts, self.tokens, self.pad = starts, starts[-1], pad
        self.lens = lens
        self.gen = gen
        self.block = block

    def rand(self, *shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=self.gen)).half()

    def to(self, gpu):
        block = self.block.to(gpu)
        k, v = (block[:, 0], block[:, 1]) if self.k.stride(0) != self.hkv * self.page * D else (block[0], block[1])
        return k, v, PagedBatch(self.table.to(gpu), torch.tensor(self.starts, dtype=torch.int32, device=gpu),
                                torch.tensor(self.lens, dtype=torch.int32, device=gpu))

    def rows(self, b, t):
        """[length, hkv, D] of sequence b from the pool ``t``."""
        out = []
        for i in range(max(self.lens[b], 0)):
            out.append(t[self.table[b, i // self.page].item(), :, i % self.page])
        return torch.stack(out) if out else torch.zeros(0, self.hkv, D, dtype=t.dtype)


def tree_masks(new, rng):
    masks = []
    for count in new:
        rows = []
        for i in range(count):
            rows.append((1 << i) | (rows[rng.randrange(max(0, i - 5), i)] if i else 0))
        masks += rows
    return masks


def signed(m):
    return m - (1 << 64) if m >> 63 else m


def expected_attention(pool, query, scale, masks=None):
    """(out, tolerance) in float64.  The probabilities' rounding moves a result
    by at most 2^-11 sum p|v| (and 2^-25 per key, in units of the row's largest
    probability, where they are subnormal), the result's own rounding by 2^-11
    |o|; the 32-bit scores add, to first order, 130 2^-24 scale sum|q||k| to a
    probability's exponent (128 products and their sum, twice the weight's
    share: numerator and denominator), below a tenth of the first term here."""
    out = torch.zeros(pool.tokens + pool.pad, pool.hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    group = pool.hq // pool.hkv
    for b, (n, p) in enumerate(zip(pool.new, pool.past)):
        if n == 0:
            continue
        k, v = pool.rows(b, pool.k).double(), pool.rows(b, pool.v).double()
        for i in range(n):
            t = pool.starts[b] + i
            if masks is None:
                seen = list(range(max(p + i + 1, 0)))
            else:
                seen = list(range(max(p, 0))) + [p + j for j in range(n) if (masks[t] >> j) & 1 and p + j >= 0]
            if not seen:
                continue
            ks, vs = k[seen], v[seen]
            q = query[t].double().view(pool.hkv, group, D)
            s = torch.einsum('hgd,khd->hgk', q, ks) * scale
            w = torch.exp(s - s.amax(-1, keepdim=True))
            l = w.sum(-1, keepdim=True)
            o = torch.einsum('hgk,khd->hgd', w / l, vs)
            a = torch.einsum('hgk,khd->hgd', w / l, vs.abs())
            size = torch.einsum('hgd,khd->hgk', q.abs(), ks.abs()).amax(-1, keepdim=True) * scale
            bound = (a * (HALF_ULP + 2 * 130 * 2.0 ** -24 * size) + len(seen) * TINY * vs.abs().amax() / l
                     + o.abs() * HALF_ULP + TINY)
            out[t], tol[t] = o.reshape(pool.hq, D), bound.reshape(pool.hq, D)
    return out, tol


def check(got, want, tol):
    got = got.double().cpu()
    assert not torch.isnan(got).any()
    worst = ((got - want).abs() / tol.clamp(min=1e-30)).where(got != want, torch.zeros_like(got)).max().item()
    print(f'worst error / tolerance: {worst:.3f}', flush=True)
    assert worst <= 1.0


BATCHES = {
    # name: (new, past, hq, hkv, page)
    'one-token': ([1], [0], 4, 2, 16),
    'one-behind-15': ([1], [15], 4, 2, 16),
    'one-behind-16': ([1], [16], 4, 2, 16),
    'decode': ([1, 1, 1, 1, 1], [0, 31, 32, 700, 133], 10, 2, 32),
    'decode-long': ([1, 1], [2500, 3], 16, 2, 16),
    'decode-page-64': ([1] * 3, [64 * 33, 64 * 16 - 1, 900], 5, 1, 64),
    'group-16': ([1, 3], [40, 90], 16, 1, 48),
    'group-1': ([2, 1], [17, 300], 3, 3, 16),
    'sits-out': ([1, 0, 1, 0], [50, 20, 0, 7], 8, 2, 16),
    'chunk': ([37, 5], [0, 100], 8, 2, 16),
    'chunk-wide': ([150, 1, 64], [77, 600, 1], 10, 2, 32),
    'chunk-page-128': ([90], [200], 4, 1, 128),
    'seventy': ([1] * 70, [(37 * b) % 200 for b in range(70)], 4, 2, 16),
}


@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('name', list(BATCHES))
def test_causal_attention(gpu, name, interleaved):
    new, past, hq, hkv, page = BATCHES[name]
    print(name, interleaved, flush=True)
    pool = Pool(new, past, hq=hq, hkv=hkv, page=page, seed=len(name), interleaved=interleaved, pad=3)
    query = pool.rand(pool.tokens + pool.pad, hq, D, scale=1.5)
    scale = 1.0 / math.sqrt(D)
    want, tol = expected_attention(pool, query, scale)
    k, v, batch = pool.to(gpu)
    out = torch.full((pool.tokens + pool.pad, hq, D), 7.0, dtype=torch.float16, device=gpu)
    got = paged_attention(query.to(gpu), k, v, batch, scale=scale, out=out)
    assert got is out
    torch.cuda.synchronize()
    assert (out[pool.tokens:] == 7.0).all()          # padding behind the last sequence: left as it was
    check(out[:pool.tokens], want[:pool.tokens], tol[:pool.tokens])


TREES = {
    'one': ([1], [0], 4, 2, 16),
    'seven': ([7], [700], 10, 2, 16),
    'sixty-four': ([64, 1, 33], [100, 45, 0], 8, 2, 32),
    'long': ([12, 64], [2600, 1500], 5, 1, 16),
}


@pytest.mark.parametrize('name', list(TREES))
def test_tree_attention(gpu, name):
    new, past, hq, hkv, page = TREES[name]
    print(name, flush=True)
    pool = Pool(new, past, hq=hq, hkv=hkv, page=page, seed=3)
    masks = tree_masks(new, random.Random(9))
    query = pool.rand(pool.tokens, hq, D, scale=1.5)
    scale = 1.0 / math.sqrt(D)
    want, tol = expected_attention(pool, query, scale, masks)
    k, v, batch = pool.to(gpu)
    mask = torch.tensor([signed(m) for m in masks], dtype=torch.int64, device=gpu)
    got = paged_attention(query.to(gpu), k, v, batch, scale=scale, tree_mask=mask)
    check(got, want, tol)


def test_as_many_sequences_as_a_call_takes(gpu):
    """65536 sequences of one new token each over one shared page, 1 to 16 positions; then an append
    whose last 16 tokens are one sequence's, the others alone in theirs."""
    n = 65536
    gen = torch.Generator().manual_seed(31)
    k, v = torch.randn(2, 1, 1, 16, D, generator=gen).half().unbind(0)
    query = torch.randn(n, 1, D, generator=gen).half()
    length = torch.arange(n) % 16 + 1
    batch = PagedBatch(*(t.to(torch.int32).to(gpu) for t in (torch.zeros(n, 1), torch.arange(n + 1), length)))
    got = paged_attention(query.to(gpu), k.to(gpu), v.to(gpu), batch, scale=0.1)
    scores = query[:, 0].double() @ k[0, 0].double().t() * 0.1
    p = torch.softmax(scores.masked_fill(torch.arange(16) >= length[:, None], float('-inf')), dim=1)
    want = p @ v[0, 0].double()
    # As for the other tests: the probabilities' rounding, their sum's and the result's, 16 scores of a size below 16.
    tol = (p @ v[0, 0].double().abs()) * (HALF_ULP + 2 * 130 * 2.0 ** -24 * 16) + 2 * want.abs() * HALF_ULP + TINY
    check(got[:, 0], want, tol)
    cos, sin = tables(16)
    qkv = torch.randn(n, 3 * D, generator=gen).half().to(gpu)
    starts = torch.full((n + 1,), n, dtype=torch.int32, device=gpu)     # n - 15 and on: no tokens
    starts[:n - 15] = torch.arange(n - 15, device=gpu)
    lens = torch.full((n,), 1, dtype=torch.int32, device=gpu)
    lens[n - 16] = 16
    pages = torch.zeros(2, 1, 1, 16, D, dtype=torch.float16, device=gpu)
    paged_append(qkv, pages[0], pages[1], PagedBatch(batch.page_table, starts, lens), q_heads=1, q_norm=None, k_norm=None,
                 eps=1e-6, cos_table=cos.to(gpu), sin_table=sin.to(gpu))
    assert torch.equal(pages[1, 0, 0, 1:], qkv[n - 15:, 2 * D:])


WIDE = {
    'page-1024': ([1, 3, 70], [1500, 1021, 1000], 4, 2, 1024),
    'page-4112': ([1, 2], [4111, 10], 4, 2, 4112),
    'group-16-large-tiles': ([37, 1, 20], [60, 300, 0], 16, 1, 16),
    'group-7': ([60, 9], [45, 333], 14, 2, 16),
}


@pytest.mark.parametrize('name', list(WIDE))
def test_long_pages_and_wide_groups(gpu, name):
    new, past, hq, hkv, page = WIDE[name]
    print(name, flush=True)
    pool = Pool(new, past, hq=hq, hkv=hkv, page=page, seed=len(name))
    query = pool.rand(pool.tokens, hq, D, scale=1.5)
    scale = 1.0 / math.sqrt(D)
    want, tol = expected_attention(pool, query, scale)
    k, v, batch = pool.to(gpu)
    check(paged_attention(query.to(gpu), k, v, batch, scale=scale), want, tol)


@pytest.mark.parametrize('name', ['decode', 'decode-long', 'chunk-wide'])
def test_queries_may_be_overwritten(gpu, name):
    new, past, hq, hkv, page = BATCHES[name]
    pool = Pool(new, past, hq=hq, hkv=hkv, page=page, seed=4)
    k, v, batch = pool.to(gpu)
    query = pool.rand(pool.tokens, hq, D).to(gpu)
    want = paged_attention(query, k, v, batch, scale=0.1)
    assert paged_attention(query, k, v, batch, scale=0.1, out=query) is query
    assert torch.equal(query, want)


LONG = {
    # name: (new, past, hq, hkv, page, tree): what of the kernels' loops it reaches that shorter sequences do not
    'more-chunks-than-lanes': ([1], [9000], 2, 1, 16, False),             # small tiles: 71 chunks, 64 of them at once
    'more-chunks-than-half-a-wave': ([64], [9001], 1, 1, 32, True),       # large tiles: 36 chunks, 32 at once
    'many-chunks-of-a-prompt': ([300, 70], [8700, 8300], 1, 1, 16, False),
    'unsplit-tokens': ([1] * 1100, [4600 if b in (3, 600) else b % 37 for b in range(1100)], 3, 3, 16, False),
    'unsplit-chunks': ([129] * 8, [1300 if b == 5 else 3 * b for b in range(8)], 64, 64, 16, False),
}


@pytest.mark.parametrize('name', list(LONG))
def test_long_sequences(gpu, name):
    """Merges of more chunks than a wave or half of one holds, and the page numbers of a wave's or a tile's keys looked
    up a second time (more than 1024 keys in one chunk: where the call's tiles fill the machine nothing is split)."""
    new, past, hq, hkv, page, tree = LONG[name]
    print(name, flush=True)
    pool = Pool(new, past, hq=hq, hkv=hkv, page=page, seed=len(name))
    masks = tree_masks(new, random.Random(17)) if tree else None
    query = pool.rand(pool.tokens, hq, D, scale=1.5)
    scale = 1.0 / math.sqrt(D)
    want, tol = expected_attention(pool, query, scale, masks)
    k, v, batch = pool.to(gpu)
    mask = None if masks is None else torch.tensor([signed(m) for m in masks], dtype=torch.int64, device=gpu)
    check(paged_attention(query.to(gpu), k, v, batch, scale=scale, tree_mask=mask), want, tol)


def test_rows_that_attend_nothing_are_zero(gpu):
    """An empty mask in front of an empty cache, and lengths shorter than the new tokens."""
    pool = Pool([3, 2], [0, 40], hq=4, hkv=2, page=16, seed=1)
    masks = [0b001, 0, 0b101, 0, 0b11]       # token 1: nothing; token 3: only the cached ones
    query = pool.rand(5, 4, D)
    want, tol = expected_attention(pool, query, 0.1, masks)
    k, v, batch = pool.to(gpu)
    got = paged_attention(query.to(gpu), k, v, batch, scale=0.1,
                          tree_mask=torch.tensor(masks, dtype=torch.int64, device=gpu))
    assert (got[1] == 0).all()
    check(got, want, tol)
    # Sequence 0 has two positions for its three new tokens: the first token lies before the first position.
    pool = Pool([3, 2], [-1, 40], hq=4, hkv=2, page=16, seed=2)
    query = pool.rand(5, 4, D)
    want, tol = expected_attention(pool, query, 0.1)
    k, v, batch = pool.to(gpu)
    got = paged_attention(query.to(gpu), k, v, batch, scale=0.1)
    assert (got[0] == 0).all()
    check(got, want, tol)


def test_positions_without_a_page_give_nan(gpu):
    """A page number outside the pool, or a length past the table: NaN for the tokens that attend it and no others."""
    pool = Pool([1, 1, 1, 2], [40, 100, 300, 30], hq=4, hkv=2, page=16, seed=5, extra_width=0)
    query = pool.rand(5, 4, D)
    want, tol = expected_attention(pool, query, 0.1)
    k, v, batch = pool.to(gpu)
    pages = k.shape[0]
    table = batch.page_table.clone()
    table[0, 1] = pages                     # one past the pool
    table[1, 6] = -1                        # the last page, position 96 ..
    table[3, 1] = 1 << 30                   # positions 16 .. 31 of the two-token sequence
    lens = batch.seq_lens.clone()
    lens[2] = 2 ** 31 - 1                   # far past the table's width
    got = paged_attention(query.to(gpu), k, v, PagedBatch(table, batch.query_starts, lens), scale=0.1)
    for t in (0, 1, 2, 3, 4):
        assert torch.isnan(got[t]).all(), t
    # The same entries one position behind what is attended are never read.
    table = batch.page_table.clone()
    table = torch.cat((table, torch.full((4, 2), 1 << 30, dtype=torch.int32, device=gpu)), dim=1).contiguous()
    check(paged_attention(query.to(gpu), k, v, PagedBatch(table, batch.query_starts, batch.seq_lens), scale=0.1), want, tol)


@pytest.mark.parametrize('tree', [False, True])
@pytest.mark.parametrize('count', [6, 60])          # small tiles, large tiles
@pytest.mark.parametrize('what', [float('nan'), float('inf'), -float('inf')])
def test_what_is_not_attended_has_no_influence(gpu, what, count, tree):
    """Infinite and NaN keys and values of a later token, or of another branch, beside rows that do not attend it."""
    pool = Pool([count, 1], [75, 40], hq=8, hkv=2, page=16, seed=count)
    query = pool.rand(count + 1, 8, D)
    masks = [(1 << i) | ((1 << min(i, 4)) - 1) for i in range(count)] + [1] if tree else None   # 0 .. 3, then leaves
    want, tol = expected_attention(pool, query, 0.1, masks)
    clean = [t for t in range(count + 1) if t == count or (t != 5 if tree else t < 5)]
    for at, page_row in ((5, 80),):                       # token 5 of sequence 0 is its position 80
        slot = pool.table[0, page_row // 16].item()
        pool.v[slot, 1, page_row % 16, 17] = what
        pool.k[slot, 0, page_row % 16, 3] = what
        pool.v[slot, 0, page_row % 16, 100] = what
    k, v, batch = pool.to(gpu)
    mask = None if masks is None else torch.tensor([signed(m) for m in masks], dtype=torch.int64, device=gpu)
    got = paged_attention(query.to(gpu), k, v, batch, scale=0.1, tree_mask=mask)
    check(got[clean], want[clean], tol[clean])
    attended = [5] if tree else list(range(5, count))
    assert not torch.isfinite(got[attended][:, 4:, 17]).any() and not torch.isfinite(got[attended][:, :4, 100]).any()


def test_large_tiles_with_bad_pages_and_empty_rows(gpu):
    """As the single tokens': a page outside the pool, a length past the table, lengths below the new tokens."""
    new, past = [60, 50, 40, 45], [40, 100, 30, -44]
    pool = Pool(new, past, hq=8, hkv=2, page=16, seed=9, extra_width=0)
    query = pool.rand(195, 8, D)
    want, tol = expected_attention(pool, query, 0.1)
    k, v, batch = pool.to(gpu)
    table, lens = batch.page_table.clone(), batch.seq_lens.clone()
    table[0, 4] = k.shape[0] + 5            # positions 64 .. 79 of 100: tokens 24 .. of sequence 0
    table[1, 2] = -3                        # cached positions
    lens[2] = 16 * table.shape[1] + 20      # the last 20 of 40 tokens lie past the table
    got = paged_attention(query.to(gpu), k, v, PagedBatch(table, batch.query_starts, lens), scale=0.1)
    assert torch.isnan(got[24:60]).all() and torch.isnan(got[60:110]).all() and torch.isnan(got[110 + 20:150]).all()
    check(got[:24], want[:24], tol[:24])
    assert (got[150:194] == 0).all()        # 45 new tokens, one position
    check(got[150:], want[150:], tol[150:])


@pytest.mark.parametrize('past', [37, 2500])            # one chunk, several
@pytest.mark.parametrize('count', [1, 40])             # small tiles, large tiles
def test_large_scores(gpu, count, past):
    """Keys c u and queries a u of one direction u of +-1, a and c of eleven bits: scores up to 2^36 whose
    products with the scale are rounded by many octaves, keys that are alike having the same score.  A row's largest
    key is ahead of the next by far, so it has all the weight, or half of it where two are alike.  The result is that
    key's value, or the mean of two, with one rounding."""
    pool = Pool([count], [past], hq=4, hkv=2, page=16, seed=count)
    gen, length = pool.gen, count + past
    u = torch.randint(2, (D,), generator=gen).float() * 2 - 1
    odd = lambda *shape: 1 + torch.randint(1024, shape, generator=gen).float() / 1024  # noqa: E731
    size = odd(length) * 2.0 ** torch.randint(0, 11, (length,), generator=gen).float()
    for i, top in ((3, 12), (past // 2, 13), (past // 2 + 1, 13), (past - 1, 14)):
        size[i] = 1397 / 1024 * 2.0 ** top
    for i in range(length):
        slot = pool.table[0, i // 16].item()
        pool.k[slot, :, i % 16] = (size[i] * u).half()
    query = (u * odd(count, 4, 1) * 2.0 ** torch.randint(8, 15, (count, 4, 1), generator=gen).float()).half()
    k, v, batch = pool.to(gpu)
    values = pool.rows(0, pool.v).double()
    for scale in (1.0 / math.sqrt(D), 1.0, 100.0, 2.0 ** -18, 2.0 ** -20):
        want = values[past - 1].repeat_interleave(2, dim=0)
        got = paged_attention(query.to(gpu), k, v, batch, scale=scale).double().cpu()
        assert torch.equal(got, want.expand(count, 4, D))
        # One position less than cached: the last token sees the two that are alike at the most.
        near = batch._replace(seq_lens=batch.seq_lens - count - 1)
        got = paged_attention(query.to(gpu), k, v, near, scale=scale)[-1].double().cpu()
        want = ((values[past // 2] + values[past // 2 + 1]) / 2).repeat_interleave(2, dim=0)
        assert ((got - want).abs() <= want.abs() * HALF_ULP + TINY).all()


@pytest.mark.parametrize('octaves', [20, 24.5, 26.3, 28])
@pytest.mark.parametrize('count', [1, 64])             # small tiles, large tiles
def test_many_small_probabilities_beside_a_large_one(gpu, count, octaves):
    """One key draws a query, 9000 others lie 20 to 28 octaves below: nothing each, and below fp16's subnormals as
    fractions of the largest, but all there is of the result where the one key's value is 0."""
    pool = Pool([count], [9000], hq=2, hkv=1, page=16, seed=count)
    u = torch.randint(2, (D,), generator=pool.gen).float() * 2 - 1
    scale = 1.0 / math.sqrt(D)
    sink = (u * (octaves * math.log(2.0) / (D * scale))).half()
    for i in range(9000 + count):
        slot = pool.table[0, i // 16].item()
        pool.k[slot, 0, i % 16] = sink if i == 4321 else 0.0
        pool.v[slot, 0, i % 16] = 0.0 if i == 4321 else 1000.0 + 100.0 * pool.v[slot, 0, i % 16]
    query = u.half().expand(count, 2, D).contiguous()
    want, _ = expected_attention(pool, query, scale)
    # The weights and their sum are of probabilities rounded by 2^-11 of each, or by 2^-36 of the largest, which is
    # nearly all of the sum; the result is rounded once.  All terms are positive.
    tol = want * 3 * HALF_ULP + TINY + 9100 * 2.0 ** -36 * 1500.0
    k, v, batch = pool.to(gpu)
    check(paged_attention(query.to(gpu), k, v, batch, scale=scale), want, tol)


@pytest.mark.parametrize('count', [1, 40])
def test_pages_beyond_32_bit_offsets(gpu, count):
    """Pages 2^30 elements apart: the last one starts 6 GiB into the pool."""
    pool = Pool([count], [50 - count], hq=4, hkv=2, page=16, seed=14)
    block = torch.empty(3 * 2 ** 30 + 2 * 2 * 16 * D, dtype=torch.float16, device=gpu)
    k = block.as_strided((4, 2, 16, D), (2 ** 30, 16 * D, D, 1))
    v = block.as_strided((4, 2, 16, D), (2 ** 30, 16 * D, D, 1), 2 * 16 * D)
    table = torch.tensor([[3, 1, 2, 0]], dtype=torch.int32)
    for e in range(4):
        k[table[0, e]], v[table[0, e]] = pool.k[pool.table[0, e]].to(gpu), pool.v[pool.table[0, e]].to(gpu)
    _, _, batch = pool.to(gpu)
    batch = batch._replace(page_table=table.to(gpu))
    query = pool.rand(count, 4, D)
    want, tol = expected_attention(pool, query, 0.1)
    check(paged_attention(query.to(gpu), k, v, batch, scale=0.1), want, tol)
    cos, sin = tables()
    qkv = pool.rand(count, 8 * D).to(gpu)
    near_k, near_v, near = pool.to(gpu)
    args = dict(q_heads=4, q_norm=None, k_norm=None, eps=1e-6, cos_table=cos.to(gpu), sin_table=sin.to(gpu))
    q = paged_append(qkv, k, v, batch, **args)
    assert torch.equal(q, paged_append(qkv, near_k, near_v, near, **args))
    for e in range(4):
        for far, close in ((k, near_k), (v, near_v)):
            assert torch.equal(far[table[0, e]].view(torch.int16), close[pool.table[0, e]].view(torch.int16))


def test_starts_out_of_order_touch_only_their_sequence(gpu):
    pool = Pool([2, 3, 1], [20, 30, 40], hq=4, hkv=2, page=16, seed=6)
    query = pool.rand(6, 4, D)
    want, tol = expected_attention(pool, query, 0.1)
    k, v, batch = pool.to(gpu)
    out = torch.full((6, 4, D), 7.0, dtype=torch.float16, device=gpu)
    starts = torch.tensor([0, 2, 500, 500], dtype=torch.int32, device=gpu)     # sequences 1 and 2: past the tokens
    paged_attention(query.to(gpu), k, v, PagedBatch(batch.page_table, starts, batch.seq_lens), scale=0.1, out=out)
    assert (out[2:] == 7.0).all()
    check(out[:2], want[:2], tol[:2])


def test_more_than_64_drafted_tokens_give_nan(gpu):
    pool = Pool([65, 2], [10, 5], hq=4, hkv=2, page=16, seed=8)
    query = pool.rand(67, 4, D)
    k, v, batch = pool.to(gpu)
    mask = torch.full((67,), 3, dtype=torch.int64, device=gpu)
    got = paged_attention(query.to(gpu), k, v, batch, scale=0.1, tree_mask=mask)
    assert torch.isnan(got[:65]).all() and not torch.isnan(got[65:]).any()


# ----------------------------------------------------------------------------- append

def tables(positions=400):
    cos, sin = RotaryEmbedding(D).table(positions, 'cpu')
    return cos, sin


def expected_rows(x, weight, cos, sin, eps):
    """[heads, D] rows of one token in float64 (before the rounding)."""
    u = x.double()
    if weight is not None:
        u = u / torch.sqrt((u * u).mean(-1, keepdim=True) + eps) * weight.double()
    turned = torch.cat((-u[:, 64:], u[:, :64]), dim=-1)
    return u * cos.double() + turned * sin.double()


@pytest.mark.parametrize('norm', [True, False])
@pytest.mark.parametrize('name', ['one-token', 'decode', 'sits-out', 'chunk', 'group-1', 'seventy'])
def test_append(gpu, name, norm):
    new, past, hq, hkv, page = BATCHES[name]
    past = [min(p, 300) for p in past]
    print(name, norm, flush=True)
    pool = Pool(new, past, hq=hq, hkv=hkv, page=page, seed=11, interleaved=len(name) % 2 == 0, pad=2)
    cos, sin = tables()
    qkv = pool.rand(pool.tokens + 2, (hq + 2 * hkv) * D, scale=2.0)
    qn, kn = (1 + 0.3 * pool.rand(D).float()).half(), (1 + 0.3 * pool.rand(D).float()).half()
    if not norm:
        qn = kn = None
    k, v, batch = pool.to(gpu)
    k0, v0 = k.clone(), v.clone()
    out = torch.full((pool.tokens + 2, hq, D), 7.0, dtype=torch.float16, device=gpu)
    up = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    paged_append(qkv.to(gpu), k, v, batch, q_heads=hq, q_norm=up(qn), k_norm=up(kn), eps=1e-6, cos_table=up(cos),
                 sin_table=up(sin), out=out)
    torch.cuda.synchronize()
    assert (out[pool.tokens:] == 7.0).all()
    want_k, want_v = k0.cpu(), v0.cpu()
    got_k, got_v, got_q = k.cpu(), v.cpu(), out.cpu()
    for b, (n, p) in enumerate(zip(new, past)):
        for i in range(n):
            t, at = pool.starts[b] + i, p + i
            x = qkv[t].view(hq + 2 * hkv, D)
            slot = pool.table[b, at // page].item()
            want_v[slot, :, at % page] = x[hq + hkv:]
            for got, heads, w in ((got_q[t], x[:hq], qn), (got_k[slot, :, at % page], x[hq:hq + hkv], kn)):
                want = expected_rows(heads, w, cos[at], sin[at], 1e-6)
                # One rounding of the result; in 32 bits each of the two products carries the norm's few roundings
                # (sum of squares, reciprocal root, two products: below 16 half-ulps of 2^-24 together).
                size = expected_rows(heads.abs(), w, cos[at].abs(), sin[at].abs(), 1e-6).abs() + want.abs()
                tol = want.abs() * HALF_ULP + TINY + 16 * 2.0 ** -24 * 3 * size
                big = torch.cat((heads[:, 64:], heads[:, :64]), dim=-1).abs().double() * 3 + heads.abs().double() * 3
                tol = tol + 16 * 2.0 ** -24 * big
                assert ((got.double() - want).abs() <= tol).all()
            want_k[slot, :, at % page] = got_k[slot, :, at % page]
    # Nothing but the new tokens' rows changed.
    assert torch.equal(got_k.view(torch.int16), want_k.view(torch.int16))
    assert torch.equal(got_v.view(torch.int16), want_v.view(torch.int16))


def test_append_refuses_tokens_without_a_place(gpu):
    """No page, a page outside the pool, an index past the table, a position past the tables: NaN queries, no write."""
    pool = Pool([1, 1, 1, 1, 2], [20, 20, 20, 390, 20], hq=4, hkv=2, page=16, seed=12, extra_width=0)
    cos, sin = tables(388)
    qkv = pool.rand(6, 8 * D)
    k, v, batch = pool.to(gpu)
    table, lens = batch.page_table.clone(), batch.seq_lens.clone()
    table[0, 1] = -1
    table[1, 1] = k.shape[0]
    lens[2] = 16 * table.shape[1] + 1
    lens[4] = 1                       # two new tokens, one position: the first has index -1
    k0, v0 = k.clone(), v.clone()
    got = paged_append(qkv.to(gpu), k, v, PagedBatch(table, batch.query_starts, lens), q_heads=4, q_norm=None,
                       k_norm=None, eps=1e-6, cos_table=cos.to(gpu), sin_table=sin.to(gpu))
    torch.cuda.synchronize()
    assert torch.isnan(got[:5]).all() and not torch.isnan(got[5]).any()
    page = table[4, 0].item()
    k0[page, :, 0], v0[page, :, 0] = k[page, :, 0], v[page, :, 0]
    assert torch.equal(k.view(torch.int16), k0.view(torch.int16))
    assert torch.equal(v.view(torch.int16), v0.view(torch.int16))


def test_append_takes_given_positions(gpu):
    pool = Pool([4], [30], hq=2, hkv=1, page=16, seed=13)
    cos, sin = tables()
    qkv = pool.rand(4, 4 * D)
    k, v, batch = pool.to(gpu)
    positions = torch.tensor([30, 31, 31, 32], dtype=torch.int32, device=gpu)
    got = paged_append(qkv.to(gpu), k, v, batch, q_heads=2, q_norm=None, k_norm=None, eps=1e-6,
                       cos_table=cos.to(gpu), sin_table=sin.to(gpu), positions=positions).cpu()
    for t, at in enumerate((30, 31, 31, 32)):
        want = expected_rows(qkv[t].view(4, D)[:2], None, cos[at], sin[at], 1e-6)
        assert (got[t].double() - want).abs().max() <= want.abs().max() * HALF_ULP + 1e-5


# ----------------------------------------------------------------------------- graphs, streams

def decode_inputs(pool, seed):
    gen = torch.Generator().manual_seed(seed)
    return (2 * torch.randn(pool.tokens, (pool.hq + 2 * pool.hkv) * D, generator=gen)).half()


def decode_step(qkv, k, v, batch, cos, sin, hq, scale):
    q = paged_append(qkv, k, v, batch, q_heads=hq, q_norm=None, k_norm=None, eps=1e-6, cos_table=cos, sin_table=sin)
    return q, paged_attention(q, k, v, batch, scale=scale)


@pytest.mark.parametrize('long', [False, True])
def test_captured_steps_follow_the_lengths(gpu, long):
    """One graph of a decode step, replayed while the sequences grow (by the graph itself): every replay equals the
    eager step on a copy; two graphs of the same shapes replayed in turn on two streams do not disturb each other."""
    past = [2000, 40, 700] if long else [20, 40, 7]
    scale = 1.0 / math.sqrt(D)
    cos, sin = (t.to(gpu) for t in tables(4096))

    def world(seed):
        pool = Pool([1, 1, 1], [p + 8 for p in past], hq=10, hkv=2, page=16, seed=seed)
        k, v, batch = pool.to(gpu)
        k.nan_to_num_(0.5)
        v.nan_to_num_(0.5)
        batch.seq_lens.copy_(torch.tensor([p + 1 for p in past], dtype=torch.int32))
        return pool, k, v, batch, torch.zeros(3, 14 * D, dtype=torch.float16, device=gpu)

    worlds = [world(1), world(2)]
    graphs = []
    for pool, k, v, batch, qkv in worlds:
        decode_step(qkv, k, v, batch, cos, sin, 10, scale)        # before the capture, on the same rows
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = decode_step(qkv, k, v, batch, cos, sin, 10, scale)
            batch.seq_lens.add_(1)
        batch.seq_lens.copy_(torch.tensor([p + 1 for p in past], dtype=torch.int32))
        graphs.append((graph, outs))
    eager = [(k.clone(), v.clone(), PagedBatch(*(t.clone() for t in batch))) for _, k, v, batch, _ in worlds]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(5):
        want = []
        for w, (pool, k, v, batch, qkv) in enumerate(worlds):
            x = decode_inputs(pool, 10 * turn + w).to(gpu)
            qkv.copy_(x)
            ek, ev, eb = eager[w]
            want.append(decode_step(x, ek, ev, eb, cos, sin, 10, scale))
            eb.seq_lens.add_(1)
        torch.cuda.synchronize()
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for w, (_, outs) in enumerate(graphs):
            for got, ref in zip(outs, want[w]):
                assert torch.equal(got, ref), (turn, w)
            assert torch.equal(worlds[w][1], eager[w][0]) and torch.equal(worlds[w][2], eager[w][1])


def test_calls_on_two_streams_at_once(gpu):
    """The same shapes on two streams without a workspace of one's own: each call has its own partials."""
    worlds = []
    for seed in (3, 4):
        pool = Pool([1] * 4, [1500, 900, 2200, 30], hq=10, hkv=2, page=16, seed=seed)
        k, v, batch = pool.to(gpu)
        worlds.append((pool.rand(4, 10, D).to(gpu), k, v, batch))
    want = [paged_attention(q, k, v, b, scale=0.1).clone() for q, k, v, b in worlds]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, (q, k, v, b) in enumerate(worlds):
            with torch.cuda.stream(streams[i]):
                got[i].append(paged_attention(q, k, v, b, scale=0.1))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_refusals(gpu):
    pool = Pool([1, 1], [20, 30], hq=4, hkv=2, page=16, seed=5)
    k, v, batch = pool.to(gpu)
    q = pool.rand(2, 4, D).to(gpu)
    bad = [
        (TypeError, dict(query=q.float())), (ValueError, dict(query=q[0])), (ValueError, dict(query=q[:, :, :64])),
        (ValueError, dict(query=q.transpose(0, 1))), (TypeError, dict(key_pages=k.float())),
        (ValueError, dict(value_pages=v[:-1])), (ValueError, dict(key_pages=k.transpose(1, 2))),
        (ValueError, dict(key_pages=k[:1].expand(k.shape))), (ValueError, dict(scale=0.0)),
        (ValueError, dict(scale=float('nan'))), (TypeError, dict(tree_mask=torch.zeros(2, device=gpu))),
        (ValueError, dict(tree_mask=torch.zeros(3, dtype=torch.int64, device=gpu))),
        (ValueError, dict(out=torch.empty(2, 4, 64, dtype=torch.float16, device=gpu))),
        (TypeError, dict(batch=batch._replace(page_table=batch.page_table.long()))),
        (ValueError, dict(batch=batch._replace(page_table=batch.page_table[:1]))),
        (ValueError, dict(batch=batch._replace(query_starts=batch.query_starts[:2]))),
        (ValueError, dict(batch=batch._replace(seq_lens=batch.seq_lens.cpu()))),
    ]
    good = dict(query=q, key_pages=k, value_pages=v, batch=batch, scale=0.1)
    for error, change in bad:
        with pytest.raises(error):
            paged_attention(**{**good, **change})
    long = batch._replace(page_table=torch.zeros(2, 300, dtype=torch.int32, device=gpu))
    with pytest.raises(ValueError, match='workspace'):
        paged_attention(**{**good, 'batch': long}, workspace=torch.empty(16, dtype=torch.uint8, device=gpu))
    assert paged_attention(**{**good, 'query': q[:0], 'batch': batch._replace(query_starts=batch.query_starts * 0)}).shape == (0, 4, D)
