"""sampling.sample_tokens against its definition in 64 bits on the CPU, token
for token: types, odd vocabularies and strides, ties, every filter alone and
together, infinities, rows without a distribution, scalars and per-row
settings, captured replays."""
import math

import numpy as np
import pytest
import torch

from ondeviceinfer_amd.sampling import sample_tokens

pytestmark = pytest.mark.gpu


def definition(row, u, temperature, top_k, top_p, min_p):
    """The token of one row, from the definition (numpy float64)."""
    values = row.astype(np.float64) + 0.0
    if np.isnan(values).any() or not (values > -np.inf).any():
        return -1
    order = np.lexsort((np.arange(values.size), -values))
    if temperature == 0.0:
        return int(order[0])
    top = values[order[0]]
    with np.errstate(invalid='ignore'):
        z = np.where(values == top, 0.0, (values - top) / float(np.float32(temperature)))[order]
    if top_k > 0:
        order, z = order[:top_k], z[:top_k]
    w = np.exp(z)
    if top_p < 1.0:
        goal = float(np.float32(top_p)) * w.sum()
        n = max(1, int((np.cumsum(w) - w < goal).sum()))
        order, z, w = order[:n], z[:n], w[:n]
    if min_p > 0.0:
        keep = z >= math.log(np.float32(min_p))
        keep[0] = True
        order, w = order[keep], w[keep]
    by_index = np.argsort(order)
    order, w = order[by_index], w[by_index]
    run = np.cumsum(w)
    hit = (run > float(np.float32(u)) * run[-1]) & (w > 0)
    return int(order[np.argmax(hit)] if hit.any() else order[np.nonzero(w)[0][-1]])


def settings(rows, kind, rng):
    out = []
    for _ in range(rows):
        m = rng.choice(['both', 'top_k', 'top_p', 'min_p', 'none', 'greedy', 'all']) if kind == 'mixed' else kind
        out.append((0.0 if m == 'greedy' else round(rng.uniform(0.3, 1.6), 3),
                    int(rng.integers(1, 200)) if m in ('both', 'top_k', 'all') else 0,
                    round(rng.uniform(0.1, 0.99), 3) if m in ('both', 'top_p', 'all') else 1.0,
                    round(rng.uniform(0.001, 0.3), 4) if m in ('min_p', 'all') else 0.0))
    return out


def run(gpu, logits, u, asks, **kw):
    t, k, p, m = zip(*asks)
    f = lambda x: torch.tensor(x, dtype=torch.float32, device=gpu)  # noqa: E731
    return sample_tokens(logits, u.to(gpu), temperature=f(t), top_k=torch.tensor(k, dtype=torch.int32, device=gpu),
                         top_p=f(p), min_p=f(m), **kw)


def compare(got, logits, u, asks):
    got = got.cpu().tolist()
    rows = logits.cpu().float().numpy()
    want = [definition(rows[r], u[r].item(), *asks[r]) for r in range(len(asks))]
    assert got == want, [(r, g, w, asks[r]) for r, (g, w) in enumerate(zip(got, want)) if g != w]


@pytest.mark.parametrize('kind', ['none', 'top_k', 'top_p', 'min_p', 'both', 'mixed'])
@pytest.mark.parametrize('dtype', [torch.float16, torch.float32])
@pytest.mark.parametrize('rows,vocab', [(3, 1), (5, 7), (4, 1000), (9, 4097), (40, 12289), (2, 151936)])
def test_tokens_follow_the_definition(gpu, rows, vocab, dtype, kind):
    print(rows, vocab, dtype, kind, flush=True)
    gen = torch.Generator().manual_seed(vocab + rows)
    rng = np.random.default_rng(vocab)
    logits = torch.randn(rows, vocab, generator=gen) * 2.5
    logits[:, torch.randint(vocab, (20,), generator=gen)] += 9.0
    logits = logits.to(dtype)
    u = torch.rand(rows, generator=gen)
    asks = settings(rows, kind, rng)
    compare(run(gpu, logits.to(gpu), u, asks), logits, u, asks)


@pytest.mark.parametrize('step', [0.25, 2.0, 1000.0])
def test_ties_go_to_the_lowest_index(gpu, step):
    """Few distinct values, so that every cut ends among equal ones; step 1000: all equal."""
    gen = torch.Generator().manual_seed(1)
    rng = np.random.default_rng(2)
    logits = (torch.round(torch.randn(30, 9000, generator=gen) / step) * step).half()
    u = torch.rand(30, generator=gen)
    for kind in ('top_k', 'top_p', 'both', 'all'):
        asks = settings(30, kind, rng)
        compare(run(gpu, logits.to(gpu), u, asks), logits, u, asks)


def test_equal_values_are_cut_exactly(gpu):
    """4096 equal weights, half of the mass: the first 2048 tokens and no others."""
    logits = torch.zeros(4, 4096)
    logits[:, 1::2] = -0.0                     # equal to +0
    u = torch.tensor([0.0, 0.5, 1.0 - 2.0 ** -24, 1023 / 2048])
    got = sample_tokens(logits.to(gpu), u.to(gpu), top_p=0.5)
    assert got.tolist() == [0, 1024, 2047, 1023]
    got = sample_tokens(logits.to(gpu), u.to(gpu), top_k=8)
    assert got.tolist() == [0, 4, 7, 3]


@pytest.mark.parametrize('value', [0.75, 1.0, 3.0, -4.0, 0.1])
@pytest.mark.parametrize('vocab', [4096, 16384])
def test_draws_on_the_border_between_equal_tokens(gpu, vocab, value):
    """vocab equal weights w, u = k / vocab: token k.  The sums of the weights are rounded, at most vocab 2^-53 of the
    whole and so far below one w each way: the target may fall on the other side of token k's border, but no further."""
    print(vocab, value, flush=True)
    k = torch.arange(0, vocab, 8 if vocab == 4096 else 32)
    k = torch.cat((k, k + 1, torch.arange(1023, vocab, 1024)))
    u = k.float() / vocab
    for dtype in (torch.float16, torch.float32):
        logits = torch.full((1, vocab), value, dtype=dtype, device=gpu)
        many = sample_tokens(logits.expand(k.numel(), vocab).contiguous(), u.to(gpu)).cpu()   # a wave per part
        assert ((many - k).abs() <= 1).all(), (k[(many - k).abs() > 1][:5], many[(many - k).abs() > 1][:5])
        few = torch.cat([sample_tokens(logits, u[i:i + 1].to(gpu)) for i in range(0, k.numel(), 7)]).cpu()
        assert ((few - k[::7]).abs() <= 1).all(), (k[::7][(few - k[::7]).abs() > 1][:5], few[(few - k[::7]).abs() > 1][:5])


@pytest.mark.parametrize('value', [0.75, 1.0, 3.0, -4.0, 0.1, -0.3, 700.0])
@pytest.mark.parametrize('temperature', [1.0, 0.7, 50.0])
def test_equal_logits_are_drawn_and_cut_exactly(gpu, temperature, value):
    """The largest weighs exactly 1, so rows of equal logits of any value have exact sums: u = k / 8192 draws token k,
    top_p = 1/2 keeps 4096 of them, top_p = 3/4 of 4096 kept by top-k 3072; behind far smaller ones too."""
    print(value, temperature, flush=True)
    n = 8192
    k = torch.cat((torch.arange(0, n, 64), torch.arange(1023, n, 1024)))
    u = (k.float() / n).to(gpu)
    rows = k.numel()
    for dtype in (torch.float16, torch.float32):
        logits = torch.full((rows, n), value, dtype=dtype, device=gpu)
        one = logits[:1]
        assert torch.equal(sample_tokens(logits, u, temperature=temperature).cpu(), k)
        assert torch.equal(sample_tokens(logits, u, temperature=temperature, top_p=0.5).cpu(), k // 2)
        assert torch.equal(sample_tokens(logits, u, temperature=temperature, top_p=0.75, top_k=4096).cpu(), 3 * k // 8)
        few = torch.cat([sample_tokens(one, u[i:i + 1], temperature=temperature, top_p=0.5) for i in range(0, rows, 9)])
        assert torch.equal(few.cpu(), k[::9] // 2)
        wide = torch.full((rows, 4 * n), -60000.0, dtype=dtype, device=gpu)
        wide[:, 2::4] = value
        assert torch.equal(sample_tokens(wide, u, temperature=temperature).cpu(), 4 * k + 2)
        assert torch.equal(sample_tokens(wide, u, temperature=temperature, top_p=0.5).cpu(), 4 * (k // 2) + 2)


def test_flat_and_peaked_rows(gpu):
    """Large and small temperatures: nearly all tokens in one octave of weights, or one token with all of it."""
    gen = torch.Generator().manual_seed(4)
    logits = torch.randn(12, 30000, generator=gen)
    u = torch.rand(12, generator=gen)
    for temperature in (1e-6, 0.01, 50.0, 1e6):
        for top_k, top_p, min_p in ((0, 1.0, 0.0), (500, 1.0, 0.0), (0, 0.6, 0.0), (700, 0.3, 0.5), (0, 0.95, 0.99)):
            asks = [(temperature, top_k, top_p, min_p)] * 12
            compare(run(gpu, logits.to(gpu), u, asks), logits, u, asks)
            half = logits.half()
            compare(run(gpu, half.to(gpu), u, asks), half, u, asks)


@pytest.mark.parametrize('kind', ['none', 'top_k', 'top_p', 'min_p', 'both'])
def test_logits_just_below_zero(gpu, kind):
    """Scaled logits y in (-2^-54, 0): y + 1 rounds to 1, so the fraction above floor(y) = -1 is a whole octave.  Tiny
    values and subnormals beside ordinary ones, among themselves, and ordinary ones at a temperature of 1e20."""
    print(kind, flush=True)
    gen = torch.Generator().manual_seed(21)
    tiny = torch.tensor([-1e-20, -3e-17, -1e-45, -1e-39, 0.0, 1e-45, 1e-20, -1e-30])
    logits = tiny[torch.randint(8, (12, 6000), generator=gen)]
    logits[:4, ::3] = torch.randn(4, 2000, generator=gen) * 2.0
    logits[4:8] = torch.randn(4, 6000, generator=gen)
    u = torch.rand(12, generator=gen)
    asks = settings(12, kind, np.random.default_rng(21))
    asks[4:8] = [(1e20, k, p, m) for _, k, p, m in asks[4:8]]
    compare(run(gpu, logits.to(gpu), u, asks), logits, u, asks)
    one = logits[8:]     # few rows: four waves per part
    for r in range(4):
        compare(run(gpu, one[r:r + 1].to(gpu), u[8 + r:9 + r], asks[8 + r:9 + r]), one[r:r + 1], u[8 + r:9 + r],
                asks[8 + r:9 + r])


def test_masked_and_infinite_logits(gpu):
    inf = float('inf')
    logits = torch.randn(8, 5000, generator=torch.Generator().manual_seed(5))
    logits[0, :4990] = -inf                    # a grammar that allows ten tokens
    logits[1] = -inf
    logits[2, 17] = float('nan')
    logits[3, [5, 4000]] = inf                 # they share the whole weight
    logits[4] = torch.finfo(torch.float32).min
    logits[4, 77] = 1.0
    logits[5] = torch.finfo(torch.float32).min     # all at the type's lowest value: equal
    logits[6, 1:] = -inf
    u = torch.tensor([0.3, 0.3, 0.3, 0.7, 0.5, 0.25, 0.99, 0.1])
    for asks in ([(1.0, 0, 1.0, 0.0)] * 8, [(0.7, 20, 0.9, 0.0)] * 8, [(0.0, 0, 1.0, 0.0)] * 8, [(1.0, 0, 0.5, 0.2)] * 8):
        got = run(gpu, logits.to(gpu), u, asks)
        compare(got, logits, u, asks)
        assert got[1] == -1 and got[2] == -1 and got[4] == 77 and got[6] == 0


@pytest.mark.parametrize('kind', ['none', 'top_k', 'top_p', 'min_p', 'both', 'all'])
@pytest.mark.parametrize('dtype', [torch.float16, torch.float32])
@pytest.mark.parametrize('rows,vocab,share', [(2, 60, 0.1), (3, 5000, 0.0), (40, 5000, 0.01), (200, 30000, 0.9)])
def test_infinite_logits_with_every_filter(gpu, rows, vocab, share, dtype, kind):
    """+inf in one token (share 0) up to most of a row: the bins above theirs hold no value at all.  fp16 logits overflow to
    it."""
    print(rows, vocab, share, dtype, kind, flush=True)
    gen = torch.Generator().manual_seed(rows + vocab)
    logits = torch.randn(rows, vocab, generator=gen) * 3.0
    logits[torch.rand(rows, vocab, generator=gen) < share] = float('inf')
    logits[torch.arange(rows), torch.randint(vocab, (rows,), generator=gen)] = 1e6 if dtype == torch.float16 else float('inf')
    logits[:, ::7] = -float('inf')
    logits[:, -1] = float('inf')
    logits = logits.to(dtype)
    u = torch.rand(rows, generator=gen)
    asks = settings(rows, kind, np.random.default_rng(rows))
    compare(run(gpu, logits.to(gpu), u, asks), logits, u, asks)


@pytest.mark.parametrize('dtype', [torch.float16, torch.float32])
@pytest.mark.parametrize('rows,vocab', [(2, 3000), (24, 3000), (6, 60000)])
def test_zero_draws_the_first_token_that_stays(gpu, rows, vocab, dtype):
    """u = 0: the first kept token with any weight in 64 bits, were it 2^-1000 beside the largest."""
    print(rows, vocab, dtype, flush=True)
    gen = torch.Generator().manual_seed(vocab)
    logits = (torch.randn(rows, vocab, generator=gen) * torch.linspace(2.0, 60.0, rows)[:, None]).to(dtype)
    u = torch.zeros(rows)
    for top_k in (0, 10, 300, 2000):
        asks = [((1.0, 0.4)[r % 2], top_k, 1.0, 0.0) for r in range(rows)]
        compare(run(gpu, logits.to(gpu), u, asks), logits, u, asks)


def test_settings_without_a_meaning_give_minus_one(gpu):
    nan, inf = float('nan'), float('inf')
    logits = torch.randn(8, 300, generator=torch.Generator().manual_seed(6)).to(gpu)
    u = torch.tensor([0.5] * 7 + [nan], device=gpu)
    f = lambda *x: torch.tensor(x, dtype=torch.float32, device=gpu)  # noqa: E731
    got = sample_tokens(logits, u, temperature=f(-1.0, nan, inf, 1, 1, 1, 1, 1), top_p=f(1, 1, 1, nan, 1, 0.0, -3.0, 1),
                        min_p=f(0, 0, 0, 0, nan, 0, 0, 0)).tolist()
    assert got[:5] == [-1] * 5 and got[7] == -1
    assert got[5:7] == logits.argmax(dim=1).tolist()[5:7]       # top_p of nothing: the first always stays
    got = sample_tokens(logits, u, top_k=-4, min_p=2.0).tolist()
    assert got[:7] == logits.argmax(dim=1).tolist()[:7] and got[7] == -1


def test_greedy_is_the_argmax(gpu):
    logits = torch.randn(6, 151936, generator=torch.Generator().manual_seed(7)).half().to(gpu)
    logits[:, [40, 90000]] = 30.0
    assert sample_tokens(logits, torch.rand(6, device=gpu), temperature=0.0).tolist() == [40] * 6


@pytest.mark.parametrize('dtype', [torch.float16, torch.float32])
def test_strided_and_misaligned_rows(gpu, dtype):
    gen = torch.Generator().manual_seed(8)
    rng = np.random.default_rng(9)
    block = torch.randn(6, 3, 5003, generator=gen).to(dtype)
    u = torch.rand(6, generator=gen)
    for offset in (0, 1, 3):
        rows = block.to(gpu)[:, -1, offset:]
        asks = settings(6, 'mixed', rng)
        compare(run(gpu, rows, u, asks), block[:, -1, offset:], u, asks)


def test_many_rows_and_an_output_of_ones_own(gpu):
    gen = torch.Generator().manual_seed(10)
    rng = np.random.default_rng(11)
    logits = (torch.randn(1500, 700, generator=gen) * 3).half()
    u = torch.rand(1500, generator=gen)
    asks = settings(1500, 'mixed', rng)
    out = torch.full((1500,), -5, dtype=torch.int64, device=gpu)
    got = run(gpu, logits.to(gpu), u, asks, out=out)
    assert got is out
    compare(got, logits, u, asks)
    assert sample_tokens(logits[:0].to(gpu), u[:0].to(gpu)).shape == (0,)


def test_captured_replays_follow_their_inputs(gpu):
    gen = torch.Generator().manual_seed(12)
    rng = np.random.default_rng(13)
    logits = torch.zeros(16, 20000, dtype=torch.float16, device=gpu)
    u = torch.zeros(16, device=gpu)
    asks = settings(16, 'mixed', rng)
    run(gpu, logits, u, asks)
    t, k, p, m = zip(*asks)
    f = lambda x: torch.tensor(x, dtype=torch.float32, device=gpu)  # noqa: E731
    args = dict(temperature=f(t), top_k=torch.tensor(k, dtype=torch.int32, device=gpu), top_p=f(p), min_p=f(m))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sample_tokens(logits, u, **args)
    for _ in range(4):
        new = (torch.randn(16, 20000, generator=gen) * 3).half()
        numbers = torch.rand(16, generator=gen)
        logits.copy_(new)
        u.copy_(numbers)
        graph.replay()
        torch.cuda.synchronize()
        compare(got, new, numbers, asks)


@pytest.mark.parametrize('kind', ['none', 'top_k', 'top_p', 'min_p', 'both'])
def test_cuts_in_more_tokens_than_a_list_holds(gpu, kind):
    """260 rows share 64 MiB of lists: 32263 tokens each, of 40000 that all lie within a step or two."""
    print(kind, flush=True)
    gen = torch.Generator().manual_seed(260)
    logits = (torch.randn(260, 40000, generator=gen) * 0.01).half()
    u = torch.rand(260, generator=gen)
    asks = settings(260, kind, np.random.default_rng(260))
    compare(run(gpu, logits.to(gpu), u, asks), logits, u, asks)


@pytest.mark.parametrize('dtype', [torch.float16, torch.float32])
@pytest.mark.parametrize('rows,vocab', [(8, 16000), (8, 40000), (70, 151936)])
def test_top_k_far_below_a_peak(gpu, rows, vocab, dtype):
    """One token 3 to 60 logits above the others: top-k ends in a bin of most of the vocabulary, top-p in one of few."""
    print(rows, vocab, dtype, flush=True)
    gen = torch.Generator().manual_seed(rows + vocab)
    logits = torch.randn(rows, vocab, generator=gen) * 2.0
    lift = torch.tensor([3.0, 12.0, 30.0, 60.0])[torch.arange(rows) % 4]
    logits[torch.arange(rows), torch.randint(vocab, (rows,), generator=gen)] = logits.amax(dim=1) + lift
    logits = logits.to(dtype)
    u = torch.rand(rows, generator=gen)
    u[::3] = 1.0 - 2.0 ** -24   # the last of what stays
    asks = [((0.5, 1.0, 2.0)[r % 3], (94, 700, 5000)[r % 3], (1.0, 0.729, 0.9999)[r // 2 % 3], (0.0, 1e-9)[r % 2])
            for r in range(rows)]
    compare(run(gpu, logits.to(gpu), u, asks), logits, u, asks)


@pytest.mark.parametrize('dtype', [torch.float16, torch.float32])
@pytest.mark.parametrize('vocab', [9000, 30000])
def test_top_p_behind_a_top_k_that_ends_in_a_full_bin(gpu, vocab, dtype):
    """Flat rows: top-k ends in a bin of more tokens than are put in order at once, whose step it is found in, and the
    search for top-p's end follows in the same row, in the same bin or another."""
    print(vocab, dtype, flush=True)
    gen = torch.Generator().manual_seed(vocab)
    rows = 96
    logits = torch.randn(rows, vocab, generator=gen).to(dtype)
    u = torch.rand(rows, generator=gen)
    asks = [((0.5, 1.0, 3.0, 20.0)[r % 4], (700, 2500, 6000)[r // 4 % 3], (0.5, 0.9, 0.999)[r // 12 % 3], 0.0)
            for r in range(rows)]
    compare(run(gpu, logits.to(gpu), u, asks), logits, u, asks)


def test_as_many_tokens_as_a_row_may_have(gpu):
    """2^30 equal logits: every sum is exact, u = j / 2^24 draws token 64 j."""
    j = torch.tensor([0, 1, 16383, 8388608, 16777215])
    logits = torch.full((1, 1 << 30), 0.5, dtype=torch.float16, device=gpu)
    u = (j.float() / 2 ** 24).to(gpu)
    got = torch.cat([sample_tokens(logits, u[i:i + 1]) for i in range(len(j))])
    assert torch.equal(got.cpu(), 64 * j)
    row = logits[:, :1 << 24]
    got = torch.cat([sample_tokens(row, u[i:i + 1], min_p=0.5) for i in range(len(j))])
    assert torch.equal(got.cpu(), j)


def test_as_many_rows_as_a_call_takes(gpu):
    rows = 65535
    u = torch.rand(rows, generator=torch.Generator().manual_seed(22)).to(gpu)
    logits = torch.zeros(rows, 17, device=gpu)
    logits[:, 16] = -float('inf')
    assert torch.equal(sample_tokens(logits, u), (u * 16).long())
    assert torch.equal(sample_tokens(logits, u, top_k=8), (u * 8).long())
    assert torch.equal(sample_tokens(logits, u, top_p=0.25), (u * 4).long())


def test_a_temperature_beyond_fp32_is_refused(gpu):
    logits, u = torch.tensor([[0.0, 1.0]], device=gpu), torch.zeros(1, device=gpu)
    with pytest.raises(ValueError, match='temperature'):
        sample_tokens(logits, u, temperature=1e39)
    assert sample_tokens(logits, u, temperature=3e38).tolist() == [0]      # both weigh 1


def test_a_workspace_without_memory_of_its_own_is_refused(gpu):
    with pytest.raises(ValueError, match='contiguous'):
        sample_tokens(torch.zeros(4, 10, device=gpu), torch.zeros(4, device=gpu),
                      workspace=torch.empty(1, dtype=torch.uint8, device=gpu).expand(1 << 20))


def test_refusals(gpu):
    logits, u = torch.zeros(4, 10, device=gpu), torch.zeros(4, device=gpu)
    with pytest.raises(TypeError):
        sample_tokens(logits.double(), u)
    with pytest.raises(TypeError):
        sample_tokens(logits.bfloat16(), u)
    with pytest.raises(ValueError):
        sample_tokens(logits[0], u)
    with pytest.raises(ValueError):
        sample_tokens(logits.t().contiguous().t(), u)
    with pytest.raises(ValueError):
        sample_tokens(logits[:1].expand(4, 10), u)
    with pytest.raises(ValueError):
        sample_tokens(logits, u[:3])
    with pytest.raises(TypeError):
        sample_tokens(logits, u.double())
    with pytest.raises(TypeError):
        sample_tokens(logits, u, top_k=torch.zeros(4, dtype=torch.int64, device=gpu))
    with pytest.raises(ValueError):
        sample_tokens(logits, u, temperature=-1.0)
    with pytest.raises(ValueError):
        sample_tokens(logits, u, top_p=float('nan'))
    with pytest.raises(ValueError):
        sample_tokens(logits, u.cpu())
    with pytest.raises(ValueError):
        sample_tokens(logits, u, workspace=torch.empty(8, dtype=torch.uint8, device=gpu))
