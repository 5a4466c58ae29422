"""The paged cache's bookkeeping, the layout of drafted trees, and what the
paged and sampling entry points refuse before any GPU work (CPU only)."""
import ctypes
import random

import pytest
import torch

from ondeviceinfer_amd import _native
from ondeviceinfer_amd.paged import PagedBatch, PagedKVCache, paged_append, paged_attention, tree_layout
from ondeviceinfer_amd.sampling import sample_tokens


def cache(pages=12, size=16, layers=2, heads=2, dim=8):
    return PagedKVCache(num_layers=layers, num_pages=pages, page_size=size, num_key_value_heads=heads, head_dim=dim,
                        device='cpu', dtype=torch.float32)


def test_extend_hands_out_pages_and_describes_the_step():
    c = cache()
    a, b = c.add(), c.add()
    batch = c.extend([a, b], [17, 3])
    assert c.length(a) == 17 and c.length(b) == 3 and c.free_pages == 9
    assert batch.query_starts.tolist() == [0, 17, 20] and batch.seq_lens.tolist() == [17, 3]
    assert batch.page_table.shape == (2, 2) and batch.page_table[1, 1] == -1
    used = batch.page_table[batch.page_table >= 0].tolist()
    assert len(set(used)) == 3
    again = c.extend([b, a], [1, 0])
    assert again.query_starts.tolist() == [0, 1, 1] and again.seq_lens.tolist() == [4, 17]
    assert again.page_table[0, 0] == batch.page_table[1, 0]
    assert all(t.dtype == torch.int32 and t.is_contiguous() for t in again)


def test_a_step_that_does_not_fit_changes_nothing():
    c = cache(pages=3)
    a, b = c.add(), c.add()
    c.extend([a], [16])
    with pytest.raises(ValueError, match='capacity'):
        c.extend([a, b], [17, 17])
    assert c.free_pages == 2 and c.length(a) == 16 and c.length(b) == 0
    with pytest.raises(ValueError):
        c.extend([a, a], [1, 1])
    with pytest.raises(ValueError):
        c.extend([a], [-1])


def test_a_step_whose_batch_cannot_be_made_changes_nothing():
    c = cache(pages=6)
    a, b = c.add(), c.add()
    first = c.extend([a], [20]).page_table.tolist()
    c.device = 'nowhere'
    with pytest.raises(RuntimeError):
        c.extend([a, b], [20, 5])
    assert c.free_pages == 4 and c.length(a) == 20 and c.length(b) == 0
    c.device = torch.device('cpu')
    batch = c.extend([b, a], [5, 20])
    assert batch.page_table[1, :2].tolist() == first[0]
    assert len(set(batch.page_table[batch.page_table >= 0].tolist())) == 4 and c.free_pages == 2


def test_pages_come_back():
    c = cache(pages=6)
    a = c.add()
    c.extend([a], [50])                 # four pages
    c.truncate(a, 33)                   # three
    assert c.free_pages == 3 and c.length(a) == 33
    c.truncate(a, 32)
    assert c.free_pages == 4
    c.truncate(a, 0)
    assert c.free_pages == 6
    with pytest.raises(ValueError):
        c.truncate(a, 1)
    c.extend([a], [96])
    c.free(a)
    assert c.free_pages == 6
    with pytest.raises(KeyError):
        c.length(a)


def test_many_random_steps_never_share_a_page():
    rng = random.Random(3)
    c = cache(pages=40)
    live = []
    for _ in range(300):
        what = rng.random()
        if what < 0.2 or not live:
            live.append(c.add())
        elif what < 0.3:
            c.free(live.pop(rng.randrange(len(live))))
        elif what < 0.5:
            s = rng.choice(live)
            c.truncate(s, rng.randrange(c.length(s) + 1))
        else:
            some = rng.sample(live, rng.randrange(1, len(live) + 1))
            try:
                c.extend(some, [rng.randrange(0, 40) for _ in some])
            except ValueError:
                pass
        held = [p for s in live for p in c._pages[s]]
        assert len(held) == len(set(held)) == 40 - c.free_pages
        assert all(len(c._pages[s]) == -(-c.length(s) // 16) for s in live)


def rows_of(c, seq, layer, which):
    pool = (c.key_pages if which == 0 else c.value_pages)[layer]
    return torch.stack([pool[c._pages[seq][i // 16], :, i % 16] for i in range(c.length(seq))])


def test_keep_moves_the_accepted_tokens_up():
    c = cache()
    seq, other = c.add(), c.add()
    c.extend([seq, other], [14, 20])
    c.extend([seq], [9])                # drafted positions 14 .. 22, over a page's end
    c._block.copy_(torch.randn_like(c._block))
    before = [[rows_of(c, seq, i, w) for w in (0, 1)] for i in range(2)]
    untouched = [rows_of(c, other, i, w) for i in range(2) for w in (0, 1)]
    c.keep(seq, 14, [0, 3, 4, 8])
    assert c.length(seq) == 18
    for layer in range(2):
        for which in (0, 1):
            got = rows_of(c, seq, layer, which)
            assert torch.equal(got[:14], before[layer][which][:14])
            assert torch.equal(got[14:], before[layer][which][[14, 17, 18, 22]])
    assert all(torch.equal(x, y) for x, y in zip(untouched, [rows_of(c, other, i, w) for i in range(2) for w in (0, 1)]))
    c.keep(seq, 14, [])
    assert c.length(seq) == 14
    with pytest.raises(ValueError):
        c.keep(seq, 10, [2, 1])
    with pytest.raises(ValueError):
        c.keep(seq, 10, [4])
    with pytest.raises(ValueError):
        c.keep(seq, 10, [-1])


def test_tree_layout():
    masks, depths = tree_layout([-1, 0, 0, 1, -1, 3])
    assert masks == [0b1, 0b11, 0b101, 0b1011, 0b10000, 0b101011] and depths == [0, 1, 1, 2, 0, 3]
    assert tree_layout([]) == ([], [])
    for bad in ([0], [-1, 1], [-1, -2], [-1] * 65):
        with pytest.raises(ValueError):
            tree_layout(bad)


def status(name, *args):
    return getattr(_native.load(), name)(*args)


def test_workspace_sizes_and_shapes_are_checked_on_the_host():
    b = ctypes.c_size_t()
    size = lambda *a: status('wq_paged_attention_workspace_size', *a, ctypes.byref(b))  # noqa: E731
    assert size(1, 1, 40, 8, 128, 257, 16) == _native.WQ_OK and b.value > 0
    assert size(1, 1, 40, 8, 128, 4, 16) == _native.WQ_OK and b.value == 0        # 64 positions: one workgroup's
    assert size(0, 0, 40, 8, 128, 4, 16) == _native.WQ_OK and b.value == 0
    assert size(1, 1, 40, 8, 64, 4, 16) == _native.WQ_ERR_UNSUPPORTED             # head_dim
    assert size(1, 1, 34, 2, 128, 4, 16) == _native.WQ_ERR_UNSUPPORTED            # 17 heads per kv head
    assert size(1, 1, 40, 7, 128, 4, 16) == _native.WQ_ERR_INVALID_ARGUMENT
    assert size(1, 1, 40, 8, 128, 4, 24) == _native.WQ_ERR_INVALID_ARGUMENT       # page_size
    assert size(1, 1, 40, 8, 128, 1 << 28, 16) == _native.WQ_ERR_INVALID_ARGUMENT # positions past 2^30
    assert size(-1, 1, 40, 8, 128, 4, 16) == _native.WQ_ERR_INVALID_ARGUMENT
    assert size(1, 65537, 40, 8, 128, 4, 16) == _native.WQ_ERR_INVALID_ARGUMENT
    assert status('wq_paged_attention_workspace_size', 1, 1, 8, 8, 128, 4, 16, None) == _native.WQ_ERR_INVALID_ARGUMENT
    size = lambda *a: status('wq_sample_workspace_size', *a, ctypes.byref(b))  # noqa: E731
    assert size(1, 151936) == _native.WQ_OK and b.value > 0
    assert size(0, 10) == _native.WQ_OK and b.value == 0
    for bad in ((65536, 10), (1, 0), (1, (1 << 30) + 1), (-1, 10)):
        assert size(*bad) == _native.WQ_ERR_INVALID_ARGUMENT


def attention_args(**change):
    page = 2 * 16 * 128
    a = dict(q=16, tokens=1, hq=4, hkv=2, d=128, k=16, ks=page, v=16, vs=page, pages=4, size=16, table=16, width=4,
             starts=16, lens=16, seqs=1, mask=None, scale=0.1, out=16, ws=None, wsb=0, stream=None)
    a.update(change)
    return tuple(a.values())


@pytest.mark.parametrize('change,code', [
    (dict(q=None), _native.WQ_ERR_INVALID_ARGUMENT), (dict(q=8), _native.WQ_ERR_INVALID_ARGUMENT),
    (dict(scale=0.0), _native.WQ_ERR_INVALID_ARGUMENT), (dict(scale=float('nan')), _native.WQ_ERR_INVALID_ARGUMENT),
    (dict(scale=float('inf')), _native.WQ_ERR_INVALID_ARGUMENT), (dict(ks=4000), _native.WQ_ERR_INVALID_ARGUMENT),
    (dict(vs=4100), _native.WQ_ERR_INVALID_ARGUMENT), (dict(pages=0), _native.WQ_ERR_INVALID_ARGUMENT),
    (dict(mask=20), _native.WQ_ERR_INVALID_ARGUMENT), (dict(starts=18), _native.WQ_ERR_INVALID_ARGUMENT),
    (dict(tokens=1 << 24), _native.WQ_ERR_INVALID_ARGUMENT), (dict(width=200), _native.WQ_ERR_WORKSPACE),
    (dict(hq=3), _native.WQ_ERR_INVALID_ARGUMENT), (dict(tokens=0), _native.WQ_OK), (dict(seqs=0), _native.WQ_OK)])
def test_attention_refuses_before_any_launch(change, code):
    assert status('wq_paged_attention', *attention_args(**change)) == code


def append_args(**change):
    page = 2 * 16 * 128
    a = dict(qkv=16, tokens=1, hq=4, hkv=2, d=128, qn=None, kn=None, eps=1e-6, cos=16, sin=16, rows=10, pos=None,
             table=16, width=4, starts=16, lens=16, seqs=1, k=16, ks=page, v=16, vs=page, pages=4, size=16, out=16,
             stream=None)
    a.update(change)
    return tuple(a.values())


@pytest.mark.parametrize('change,code', [
    (dict(qkv=None), _native.WQ_ERR_INVALID_ARGUMENT), (dict(out=24), _native.WQ_ERR_INVALID_ARGUMENT),
    (dict(rows=0), _native.WQ_ERR_INVALID_ARGUMENT), (dict(d=64), _native.WQ_ERR_UNSUPPORTED),
    (dict(hkv=0), _native.WQ_ERR_INVALID_ARGUMENT), (dict(pos=18), _native.WQ_ERR_INVALID_ARGUMENT),
    (dict(size=0), _native.WQ_ERR_INVALID_ARGUMENT), (dict(tokens=0), _native.WQ_OK)])
def test_append_refuses_before_any_launch(change, code):
    assert status('wq_paged_append', *append_args(**change)) == code


@pytest.mark.parametrize('out,code', [
    (1 << 20, _native.WQ_ERR_INVALID_ARGUMENT),                           # the projection itself
    ((1 << 20) + 3 * 8 * 256 - 16, _native.WQ_ERR_INVALID_ARGUMENT),      # its last 16 bytes
    ((1 << 20) - 3 * 4 * 256 + 16, _native.WQ_ERR_INVALID_ARGUMENT)])     # its first 16 bytes
def test_append_refuses_queries_over_the_projection(out, code):
    """A token's queries would land on rows that another token's workgroup has not read."""
    assert status('wq_paged_append', *append_args(qkv=1 << 20, tokens=3, out=out)) == code


@pytest.mark.parametrize('out,code', [
    ((1 << 20) + 256, _native.WQ_ERR_INVALID_ARGUMENT),                  # a head further
    ((1 << 20) - 3 * 4 * 256 + 16, _native.WQ_ERR_INVALID_ARGUMENT),     # its first 16 bytes
    ((1 << 20) + 3 * 4 * 256, _native.WQ_ERR_WORKSPACE),                 # behind it: refused for the missing workspace
    (1 << 20, _native.WQ_ERR_WORKSPACE)])                                # the queries themselves
def test_attention_refuses_outputs_over_other_queries(out, code):
    assert status('wq_paged_attention', *attention_args(q=1 << 20, tokens=3, out=out, width=200)) == code


def sample_args(**change):
    a = dict(logits=16, kind=0, rows=2, vocab=100, stride=100, u=16, t=None, ta=1.0, k=None, ka=0, p=None, pa=1.0,
             m=None, ma=0.0, out=16, ws=16, wsb=1 << 30, stream=None)
    a.update(change)
    return tuple(a.values())


@pytest.mark.parametrize('change,code', [
    (dict(logits=None), _native.WQ_ERR_INVALID_ARGUMENT), (dict(kind=2), _native.WQ_ERR_INVALID_ARGUMENT),
    (dict(stride=99), _native.WQ_ERR_INVALID_ARGUMENT), (dict(logits=18, kind=1), _native.WQ_ERR_INVALID_ARGUMENT),
    (dict(ws=None), _native.WQ_ERR_WORKSPACE), (dict(wsb=8), _native.WQ_ERR_WORKSPACE),
    (dict(ws=20), _native.WQ_ERR_WORKSPACE), (dict(out=20), _native.WQ_ERR_INVALID_ARGUMENT),
    (dict(u=None), _native.WQ_ERR_INVALID_ARGUMENT), (dict(rows=0), _native.WQ_OK)])
def test_sampling_refuses_before_any_launch(change, code):
    assert status('wq_sample', *sample_args(**change)) == code


def test_a_workspace_counts_the_memory_it_spans():
    """An expanded tensor has elements without memory of their own."""
    assert _native._scratch(torch.empty(6, 4, dtype=torch.float32))[1] == 96
    for bad in (torch.empty(1, dtype=torch.uint8).expand(1 << 20), torch.empty(64, dtype=torch.uint8)[::2]):
        with pytest.raises(ValueError, match='contiguous'):
            _native._scratch(bad)


def test_cpu_tensors_are_refused():
    c = cache(dim=128)
    seq = c.add()
    batch = c.extend([seq], [1])
    q = torch.zeros(1, 4, 128, dtype=torch.float16)
    k = c.key_pages[0].half()
    with pytest.raises(ValueError, match='GPU'):
        paged_attention(q, k, k, batch, scale=0.1)
    with pytest.raises(ValueError, match='GPU'):
        paged_append(torch.zeros(1, 1024, dtype=torch.float16), k, k, PagedBatch(*batch), q_heads=4, q_norm=None,
                     k_norm=None, eps=1e-6, cos_table=q[0], sin_table=q[0])
    with pytest.raises(ValueError, match='GPU'):
        sample_tokens(torch.zeros(1, 4), torch.zeros(1))
