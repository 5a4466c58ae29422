"""Many sequences through the quantized model over the paged cache: ragged
prompts and decode steps against the oracle's forward, trees of drafted tokens
against the same tokens one after another, sampled generation."""
import numpy as np
import pytest
import torch

from oracle import qdq, qwen3
from ondeviceinfer_amd.generation import sample_generate
from test_gpu_qwen3 import TinyCfg, build, numpy_model

pytestmark = pytest.mark.gpu


def close(got, want, what):
    """The bar of the reference's own harness (cosine, relative L2) and the framework's for the largest error.  The
    paged path rounds the rotated queries and keys once where the oracle rounds every step, so the mean error, of
    the size of one fp16 rounding, has no bar of its own."""
    m = qdq.parity_metrics(got.float().cpu().numpy(), np.asarray(want).astype(np.float32))
    assert m['finite'] and m['cosine'] >= 0.9999 and m['relative_l2'] <= 0.02 and \
        m['max_abs'] <= 1e-2 * m['ref_inf'], (what, m)


@pytest.fixture(scope='module')
def tiny(gpu):
    np_model = numpy_model(TinyCfg)
    model, backend = build(np_model, TinyCfg)
    return np_model, model


def ids(rng, n):
    return rng.integers(0, TinyCfg.vocab_size, n)


def test_ragged_prompts_chunks_and_decode_steps_match_the_oracle(tiny):
    np_model, model = tiny
    rng = np.random.default_rng(1)
    cache = model.make_paged_cache(num_pages=64, page_size=16)
    oracle = {}

    def step(seqs, tokens, **kw):
        out = model.forward_paged(torch.from_numpy(np.concatenate(tokens)), cache, seqs, [len(t) for t in tokens], **kw)
        rows = [qwen3.forward(t, np_model, TinyCfg, oracle[s]) for s, t in zip(seqs, tokens)]
        want = np.concatenate(rows) if kw.get('all_logits') else np.stack([r[-1] for r in rows])
        assert out.logits.shape == want.shape
        for i in range(len(want)):
            close(out.logits[i], want[i], (seqs, i))

    a, b, c = (cache.add() for _ in range(3))
    for s in (a, b, c):
        oracle[s] = qwen3.KVCacheOracle(TinyCfg.num_hidden_layers)
    print('prompts', flush=True)
    step([a, b], [ids(rng, 61), ids(rng, 7)], all_logits=True)
    print('a chunk beside single tokens and a new prompt', flush=True)
    step([b, c, a], [ids(rng, 1), ids(rng, 40), ids(rng, 30)])
    for i in range(3):
        print('decode', i, flush=True)
        step([a, b, c], [ids(rng, 1) for _ in range(3)])
    assert [cache.length(s) for s in (a, b, c)] == [94, 11, 43]
    cache.free(b)
    d = cache.add()
    oracle[d] = qwen3.KVCacheOracle(TinyCfg.num_hidden_layers)
    step([d, c], [ids(rng, 20), ids(rng, 1)])     # d takes over b's pages


def test_drafted_trees_match_their_branches(tiny):
    """Every token of a tree sees what it would have seen as the end of its branch; after the rejected ones are
    dropped the sequences go on as if only the accepted ones had been there."""
    np_model, model = tiny
    rng = np.random.default_rng(2)
    cache = model.make_paged_cache(num_pages=64)
    prompts = [ids(rng, 30), ids(rng, 45)]
    seqs = [cache.add(), cache.add()]
    model.forward_paged(torch.from_numpy(np.concatenate(prompts)), cache, seqs, [30, 45])
    parents = [[-1, 0, 0, 1, 2, 4, -1], [-1, 0, 1]]
    drafted = [ids(rng, 7), ids(rng, 3)]
    out = model.forward_paged(torch.from_numpy(np.concatenate(drafted)), cache, seqs, [7, 3], tree_parents=parents,
                              all_logits=True)
    row = 0
    for prompt, parent, tokens in zip(prompts, parents, drafted):
        for i in range(len(parent)):
            branch, j = [], i
            while j >= 0:
                branch.insert(0, tokens[j])
                j = parent[j]
            want = qwen3.forward(np.concatenate([prompt, branch]), np_model, TinyCfg)[-1]
            close(out.logits[row], want, ('tree', i))
            row += 1
    cache.keep(seqs[0], 30, [0, 2, 4])
    cache.keep(seqs[1], 45, [])
    more = [ids(rng, 2), ids(rng, 1)]
    out = model.forward_paged(torch.from_numpy(np.concatenate(more)), cache, seqs, [2, 1])
    for i, tokens in enumerate((np.concatenate([prompts[0], drafted[0][[0, 2, 4]], more[0]]),
                                np.concatenate([prompts[1], more[1]]))):
        close(out.logits[i], qwen3.forward(tokens, np_model, TinyCfg)[-1], ('after', i))


def test_a_step_without_room_leaves_the_sequences_as_they_were(tiny):
    _, model = tiny
    cache = model.make_paged_cache(num_pages=3)
    seq = cache.add()
    model.forward_paged(torch.arange(20), cache, [seq], [20])
    with pytest.raises(ValueError, match='capacity'):
        model.forward_paged(torch.arange(40), cache, [seq], [40])
    with pytest.raises(ValueError):
        model.forward_paged(torch.arange(4), cache, [seq], [3])
    with pytest.raises(ValueError):
        model.forward_paged(torch.arange(2), cache, [seq], [2], tree_parents=[[-1, 5]])
    assert cache.length(seq) == 20 and cache.free_pages == 1


def test_a_step_that_fails_at_the_lm_head_has_not_happened(tiny, monkeypatch):
    _, model = tiny
    cache = model.make_paged_cache(num_pages=8)
    seqs = [cache.add(), cache.add()]
    tokens = torch.arange(40)
    model.forward_paged(tokens[:25], cache, seqs, [20, 5])
    free = cache.free_pages

    def no_memory(hidden_states):
        raise torch.OutOfMemoryError('no memory for the logits')

    with monkeypatch.context() as patch:
        patch.setattr(model, '_logits', no_memory)
        for kw in (dict(), dict(all_logits=True)):
            with pytest.raises(torch.OutOfMemoryError):
                model.forward_paged(tokens[25:40], cache, seqs, [13, 2], **kw)
            assert [cache.length(s) for s in seqs] == [20, 5] and cache.free_pages == free
    got = model.forward_paged(tokens[25:40], cache, seqs, [13, 2]).logits
    other = model.make_paged_cache(num_pages=8)
    again = [other.add(), other.add()]
    model.forward_paged(tokens[:25], other, again, [20, 5])
    assert torch.equal(got, model.forward_paged(tokens[25:40], other, again, [13, 2]).logits)


def test_sampled_generation(tiny):
    np_model, model = tiny
    rng = np.random.default_rng(3)
    prompts = [ids(rng, n).tolist() for n in (9, 33, 1, 18)]
    cache = model.make_paged_cache(num_pages=48)

    def run(**kw):
        out = sample_generate(model, prompts, max_new_tokens=8, cache=cache,
                              generator=torch.Generator(device='cuda').manual_seed(5), **kw)
        assert cache.free_pages == 48
        return out

    greedy = run(temperature=0.0)
    for prompt, new in zip(prompts, greedy):
        assert len(new) == 8
        logits = qwen3.forward(np.array(prompt + new[:-1]), np_model, TinyCfg)[len(prompt) - 1:].astype(np.float32)
        top2 = np.sort(logits, axis=-1)[:, -2:]
        decisive = (top2[:, 1] - top2[:, 0]) > 2e-2 * np.abs(logits).max()
        assert np.array_equal(np.argmax(logits, -1)[decisive], np.array(new)[decisive])
    first = run(temperature=0.8, top_k=50, top_p=0.9)
    assert first == run(temperature=0.8, top_k=50, top_p=0.9) and first != greedy
    per_prompt = run(temperature=torch.tensor([0.0, 0.8, 0.8, 0.0], device='cuda'), top_k=50, top_p=0.9)
    assert per_prompt[0][0] == greedy[0][0] and per_prompt[3][0] == greedy[3][0]
    assert per_prompt[1][0] == first[1][0]
    # Ends with the token that is named, which is kept; the others go on.
    eos = greedy[1][2]
    ended = run(temperature=0.0, eos_token_id=eos)
    for new, whole in zip(ended, greedy):
        assert new[-1] == eos or len(new) == 8
        assert eos not in new[:-1]
    assert ended[1][-1] == eos and len(ended[1]) == greedy[1].index(eos) + 1
    with pytest.raises(ValueError):
        sample_generate(model, [[]], max_new_tokens=2, cache=cache)
