"""Performance cases of the operators that serve many sequences at once from a paged key/value cache.

A case is a dict of plain values; ``kind`` says which public entry point it calls:

* ``append``: ``paged.paged_append`` takes the fused q|k|v projection of every new token, applies the per-head q/k
  RMSNorm and the position rotation, writes k and v into the sequences' pages and returns q;
* ``attend``: ``paged.paged_attention``, causal grouped-query attention of every new token over its sequence's pages:
  single tokens (``new`` = 1) and chunks of prompts;
* ``tree``: the same entry point for drafted tokens that form a tree behind the cached ones;
* ``sample``: ``sampling.sample_tokens`` draws one token per row of logits from given uniform numbers, after
  temperature, top-k, top-p and min-p.

Every attention has 128-wide heads, as the decoder's; 40 / 8 heads and 151936 tokens are those of the 14B
configuration (``config.QWEN3_14B``), the other sizes are generic.  ``own`` chooses between the operators' plain form
and the framework's kernels.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = 'cuda:0'
D = 128
EPS = 1e-6
VOCAB = 151936
POSITIONS = 40960          # rows of the cos / sin tables
MOST_PAIRS = 45e6          # (query, key) pairs per head of the largest drawn chunk
MOST_CACHED = 420_000      # cached tokens of the largest drawn batch


def listed() -> list[dict]:
    return [
        # One token of one sequence: nothing but latency, launch and host work.
        {'name': 'append-b1', 'kind': 'append', 'q_heads': 40, 'kv_heads': 8, 'page': 16, 'batch': 1, 'new': 1,
         'past': 700, 'mix': 0, 'pad': 0},
        # Chunks of five prompts prefilled together, 4100 tokens at most: the largest append.
        {'name': 'append-chunks', 'kind': 'append', 'q_heads': 40, 'kv_heads': 8, 'page': 32, 'batch': 5, 'new': 2050,
         'past': 3000, 'mix': 1, 'pad': 3},
        # The headline benchmark's decode: one token behind a 4096-token prompt.
        {'name': 'attend-b1-past4100', 'kind': 'attend', 'q_heads': 40, 'kv_heads': 8, 'page': 16, 'batch': 1,
         'new': 1, 'past': 4100, 'mix': 0, 'pad': 0},
        # A decode batch of 24 chats of very different lengths.
        {'name': 'attend-b24', 'kind': 'attend', 'q_heads': 40, 'kv_heads': 8, 'page': 32, 'batch': 24, 'new': 1,
         'past': 4100, 'mix': 2, 'pad': 0},
        # A decode batch of 64 long documents: all of it cache bandwidth, the largest read.
        {'name': 'attend-b64-long', 'kind': 'attend', 'q_heads': 64, 'kv_heads': 8, 'page': 64, 'batch': 64, 'new': 1,
         'past': 12000, 'mix': 3, 'pad': 0},
        # A whole 4096-token prompt: the largest product.
        {'name': 'attend-prompt-4096', 'kind': 'attend', 'q_heads': 40, 'kv_heads': 8, 'page': 16, 'batch': 1,
         'new': 4096, 'past': 0, 'mix': 0, 'pad': 0},
        # Ragged chunks of six prompts behind what each has cached already.
        {'name': 'attend-chunks', 'kind': 'attend', 'q_heads': 32, 'kv_heads': 4, 'page': 16, 'batch': 6, 'new': 700,
         'past': 2500, 'mix': 4, 'pad': 2},
        # Seven drafted tokens of one sequence verified at once.
        {'name': 'tree-b1-n7', 'kind': 'tree', 'q_heads': 40, 'kv_heads': 8, 'page': 16, 'batch': 1, 'new': 7,
         'past': 4100, 'mix': 0, 'pad': 0},
        # Wide trees of a batch of twelve.
        {'name': 'tree-b12-n61', 'kind': 'tree', 'q_heads': 40, 'kv_heads': 8, 'page': 32, 'batch': 12, 'new': 61,
         'past': 7000, 'mix': 5, 'pad': 0},
        # One token of one chat: top-k and top-p over the whole vocabulary.
        {'name': 'sample-b1', 'kind': 'sample', 'dtype': 'fp16', 'rows': 1, 'vocab': VOCAB, 'mode': 'both', 'mix': 0},
        # A decode batch of 64 whose requests each bring their own settings.
        {'name': 'sample-b64', 'kind': 'sample', 'dtype': 'fp16', 'rows': 64, 'vocab': VOCAB, 'mode': 'mixed',
         'mix': 1},
        # 32-bit logits (after a caller's own penalties) over an odd vocabulary: temperature and min-p.
        {'name': 'sample-b24-fp32', 'kind': 'sample', 'dtype': 'fp32', 'rows': 24, 'vocab': 50257, 'mode': 'min_p',
         'mix': 2},
    ]


def _log(rng, lo: float, hi: float) -> int:
    return max(int(lo), min(int(hi), round(lo * (hi / lo) ** rng.random())))


def draw(rng) -> dict:
    pick = rng.random()
    mix = rng.randrange(1 << 30)
    if pick < 0.25:
        return {'kind': 'sample', 'dtype': rng.choice(('fp16', 'fp32')), 'rows': _log(rng, 1, 64),
                'vocab': _log(rng, 1000, VOCAB), 'mode': rng.choice(('both', 'mixed', 'min_p', 'top_k', 'top_p', 'none')),
                'mix': mix}
    heads, kv = rng.choice(((40, 8), (40, 8), (64, 8), (32, 4), (32, 8), (16, 8), (4, 2), (14, 2), (8, 8)))
    case = {'q_heads': heads, 'kv_heads': kv, 'page': rng.choice((16, 32, 64, 128)), 'mix': mix,
            'pad': rng.choice((0, 0, 0, 5))}
    if pick < 0.4:
        batch = _log(rng, 1, 64)
        return {'kind': 'append', **case, 'batch': batch, 'new': _log(rng, 1, max(1, 4096 // batch)),
                'past': _log(rng, 1, 8000)}
    if pick < 0.65:      # single tokens
        batch = _log(rng, 1, 64)
        past = min(_log(rng, 30, 16000), MOST_CACHED // batch)
        return {'kind': 'attend', **case, 'batch': batch, 'new': 1, 'past': past}
    if pick < 0.85:      # chunks of prompts
        batch = _log(rng, 1, 8)
        new = _log(rng, 2, 2048 // batch)
        past = min(_log(rng, 1, 8000), int(MOST_PAIRS / 8 / (batch * new)))
        return {'kind': 'attend', **case, 'batch': batch, 'new': new, 'past': past}
    batch = _log(rng, 1, 16)
    past = min(_log(rng, 20, 8000), MOST_CACHED // 8 // batch)
    return {'kind': 'tree', **case, 'batch': batch, 'new': rng.randrange(2, 65), 'past': past}


# ----------------------------------------------------------------------------- inputs

def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """New and cached tokens of every sequence: ``new`` and ``past`` are the longest, the first sequence has them."""
    rng = random.Random(case['mix'])
    new, past = [], []
    for b in range(case['batch']):
        if b == 0:
            new.append(case['new'])
            past.append(case['past'])
        elif case['kind'] != 'tree' and case['new'] > 1 and rng.random() < 0.1:
            new.append(0)                                          # a sequence that sits this step out
            past.append(rng.randrange(0, case['past'] + 1))
        else:
            new.append(case['new'] if case['new'] == 1 else rng.randrange(1, case['new'] + 1))
            past.append(rng.randrange(0, case['past'] + 1) if rng.random() < 0.5
                        else rng.randrange(3 * case['past'] // 4, case['past'] + 1))
    return new, past


def _tree_masks(new: list[int], mix: int) -> list[int]:
    """For each drafted token the bits of its ancestors and itself."""
    rng = random.Random(mix + 1)
    masks = []
    for count in new:
        rows = []
        for i in range(count):
            rows.append((1 << i) | (rows[rng.randrange(max(0, i - 6), i)] if i else 0))
        masks += rows
    return [m - (1 << 64) if m >> 63 else m for m in masks]


def _depths(masks: list[int]) -> list[int]:
    return [bin(m & ((1 << 64) - 1)).count('1') - 1 for m in masks]


def _params(case: dict) -> dict[str, list]:
    rng = random.Random(case['mix'] + 7)
    rows, mode = case['rows'], case['mode']
    out = {'temperature': [], 'top_k': [], 'top_p': [], 'min_p': []}
    for _ in range(rows):
        m = rng.choice(('both', 'min_p', 'top_k', 'top_p', 'none', 'greedy')) if mode == 'mixed' else mode
        out['temperature'].append(0.0 if m == 'greedy' else round(rng.uniform(0.5, 1.3), 3))
        out['top_k'].append(rng.randrange(10, 100) if m in ('both', 'top_k') else 0)
        out['top_p'].append(round(rng.uniform(0.7, 0.97), 3) if m in ('both', 'top_p') else 1.0)
        out['min_p'].append(round(rng.uniform(0.02, 0.1), 3) if m == 'min_p' else 0.0)
    return out


def _rope_tables() -> tuple[torch.Tensor, torch.Tensor]:
    inv = 1.0 / (1_000_000.0 ** (torch.arange(0, D, 2, dtype=torch.float64) / D))
    ang = torch.arange(POSITIONS, dtype=torch.float64).unsqueeze(1) * inv
    ang = torch.cat((ang, ang), dim=1)
    return ang.cos().half().to(DEVICE), ang.sin().half().to(DEVICE)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    if case['kind'] == 'sample':
        rows, vocab = case['rows'], case['vocab']
        # A body of improbable tokens and a few dozen candidates that stand out.
        logits = torch.randn(rows, vocab, generator=gen, device=DEVICE) * 2.2 - 1.0
        n_out = min(60, vocab)
        where = torch.randint(vocab, (rows, n_out), generator=gen, device=DEVICE)
        boost = torch.rand(rows, n_out, generator=gen, device=DEVICE) * 14.0
        logits = logits.scatter_add(1, where, boost)
        state = {'case': case, 'logits': logits.half() if case['dtype'] == 'fp16' else logits,
                 'uniform': torch.rand(rows, generator=gen, device=DEVICE)}
        for key, values in _params(case).items():
            state[key] = torch.tensor(values, device=DEVICE, dtype=torch.int32 if key == 'top_k' else torch.float32)
        return state
    hq, hkv, page, batch = case['q_heads'], case['kv_heads'], case['page'], case['batch']
    new, past = _lengths(case)
    lens = [n + p for n, p in zip(new, past)]
    tokens = sum(new)
    width = max((n + page - 1) // page for n in lens) + 2
    used = [(n + page - 1) // page for n in lens]
    pages = sum(used) + 3
    # Pages in the order a pool that has been in use for a while hands them out.
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((batch, width), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state = {'case': case, 'new': new, 'past': past, 'starts': starts, 'tokens': tokens, 'page_table': table,
             'query_starts': torch.tensor(starts, dtype=torch.int32, device=DEVICE),
             'seq_lens': torch.tensor(lens, dtype=torch.int32, device=DEVICE)}
    shape = (pages, hkv, page, D)
    rows = tokens + case['pad']
    state['key_pages'] = torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float16)
    state['value_pages'] = torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float16)
    state['out'] = torch.zeros(rows, hq, D, device=DEVICE, dtype=torch.float16)
    if case['kind'] == 'append':
        state['qkv'] = torch.randn(rows, (hq + 2 * hkv) * D, generator=gen, device=DEVICE).half()
        for key in ('q_norm', 'k_norm'):
            state[key] = (1.0 + 0.2 * torch.randn(D, generator=gen, device=DEVICE)).half()
        state['cos'], state['sin'] = _rope_tables()
        return state
    # Normalized queries against keys of unit variance; a few keys of every sequence draw most of the attention.
    state['query'] = (1.5 * torch.randn(rows, hq, D, generator=gen, device=DEVICE)).half()
    state['scale'] = 1.0 / math.sqrt(D)
    # What lies behind a sequence's last token in its last page is whatever was there before.
    for b, n in enumerate(lens):
        if n % page:
            for name in ('key_pages', 'value_pages'):
                state[name][table[b, n // page].long(), :, n % page:] = float('nan')
    if case['kind'] == 'tree':
        state['masks'] = _tree_masks(new, case['mix'])
        state['tree_mask'] = torch.tensor(state['masks'] + [0] * case['pad'], dtype=torch.int64, device=DEVICE)
    return state


# ----------------------------------------------------------------------------- the framework's operators

def _own(state: dict):
    from ondeviceinfer_amd.paged import PagedBatch, paged_append, paged_attention
    from ondeviceinfer_amd.sampling import sample_tokens
    case = state['case']
    if case['kind'] == 'sample':
        return sample_tokens(state['logits'], state['uniform'], temperature=state['temperature'],
                             top_k=state['top_k'], top_p=state['top_p'], min_p=state['min_p'])
    batch = PagedBatch(state['page_table'], state['query_starts'], state['seq_lens'])
    if case['kind'] == 'append':
        q = paged_append(state['qkv'], state['key_pages'], state['value_pages'], batch, q_heads=case['q_heads'],
                         q_norm=state['q_norm'], k_norm=state['k_norm'], eps=EPS, cos_table=state['cos'],
                         sin_table=state['sin'], out=state['out'])
        return q, state['key_pages'], state['value_pages']
    return paged_attention(state['query'], state['key_pages'], state['value_pages'], batch, scale=state['scale'],
                           tree_mask=state.get('tree_mask'), out=state['out'])


# ----------------------------------------------------------------------------- the plain forms

def _plain_append(state: dict):
    case = state['case']
    hq, hkv, page = case['q_heads'], case['kv_heads'], case['page']
    tokens = state['tokens']
    x = state['qkv'][:tokens].float().view(tokens, hq + 2 * hkv, D)
    index = torch.cat([torch.arange(p, p + n, device=DEVICE) for n, p in zip(state['new'], state['past'])])
    seq = torch.cat([torch.full((n,), b, device=DEVICE) for b, n in enumerate(state['new'])])
    cos, sin = state['cos'][index].float().unsqueeze(1), state['sin'][index].float().unsqueeze(1)

    def norm_rope(v, weight):
        v = v * torch.rsqrt((v * v).mean(dim=-1, keepdim=True) + EPS) * weight.float()
        turned = torch.cat((-v[..., D // 2:], v[..., :D // 2]), dim=-1)
        return (v * cos + turned * sin).half()

    state['out'][:tokens] = norm_rope(x[:, :hq], state['q_norm'])
    where = state['page_table'][seq, index // page].long()
    state['key_pages'][where, :, index % page] = norm_rope(x[:, hq:hq + hkv], state['k_norm'])
    state['value_pages'][where, :, index % page] = x[:, hq + hkv:].half()
    return state['out'], state['key_pages'], state['value_pages']


def _plain_attend(state: dict):
    case = state['case']
    hq, hkv, page = case['q_heads'], case['kv_heads'], case['page']
    group = hq // hkv
    out = state['out']
    for b, (n, p) in enumerate(zip(state['new'], state['past'])):
        if n == 0:
            continue
        length, first = n + p, state['starts'][b]
        where = state['page_table'][b, :(length + page - 1) // page].long()
        keys = state['key_pages'][where].transpose(0, 1).reshape(hkv, -1, D)[:, :length].float()
        values = state['value_pages'][where].transpose(0, 1).reshape(hkv, -1, D)[:, :length].float()
        query = state['query'][first:first + n].float().view(n, hkv, group, D).permute(1, 2, 0, 3)
        if 'tree_mask' in state:
            bits = (state['tree_mask'][first:first + n].unsqueeze(1) >> torch.arange(n, device=DEVICE)) & 1
            seen = torch.cat((torch.ones(n, p, dtype=torch.bool, device=DEVICE), bits.bool()), dim=1)
        else:
            seen = (torch.arange(length, device=DEVICE).unsqueeze(0)
                    <= torch.arange(p, length, device=DEVICE).unsqueeze(1))
        scores = torch.matmul(query.reshape(hkv, group * n, D), keys.transpose(1, 2).contiguous())
        scores = (scores * state['scale']).view(hkv, group, n, length).masked_fill(~seen, float('-inf'))
        weights = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
        weights = weights / weights.sum(dim=-1, keepdim=True)
        result = torch.matmul(weights.view(hkv, group * n, length), values).view(hkv, group, n, D)
        out[first:first + n] = result.permute(2, 0, 1, 3).reshape(n, hq, D).half()
    return out


def _plain_sample(state: dict):
    logits = state['logits'].double()
    rows, vocab = logits.shape
    temperature = state['temperature'].double().unsqueeze(1)
    ordered, order = torch.sort(logits, dim=1, descending=True, stable=True)
    top = ordered[:, :1]
    scaled = (ordered - top) / temperature.where(temperature > 0, torch.ones_like(temperature))
    weight = torch.exp(scaled)
    rank = torch.arange(vocab, device=DEVICE).unsqueeze(0)
    top_k = state['top_k'].unsqueeze(1)
    weight = torch.where((top_k > 0) & (rank >= top_k), torch.zeros_like(weight), weight)
    before = torch.cumsum(weight, dim=1) - weight
    top_p = state['top_p'].double().unsqueeze(1)
    drop = (top_p < 1.0) & (before >= top_p * weight.sum(dim=1, keepdim=True))
    min_p = state['min_p'].double().unsqueeze(1)
    drop = (drop | ((min_p > 0) & (scaled < torch.log(min_p)))) & (rank > 0)
    drop = drop | ((temperature == 0) & (rank > 0))
    weight = torch.where(drop, torch.zeros_like(weight), weight)
    weight = torch.zeros_like(weight).scatter_(1, order, weight)      # back in the vocabulary's order
    running = torch.cumsum(weight, dim=1)
    target = state['uniform'].double().unsqueeze(1) * running[:, -1:]
    hit = (running > target) & (weight > 0)
    return torch.argmax(hit.to(torch.int8), dim=1)


def run(state: dict):
    if own:
        return _own(state)
    return {'append': _plain_append, 'attend': _plain_attend, 'tree': _plain_attend,
            'sample': _plain_sample}[state['case']['kind']](state)


# ----------------------------------------------------------------------------- work

def work(case: dict) -> dict:
    """Each input read once and each output written once; the products of attention's visible (query, key) pairs."""
    if case['kind'] == 'sample':
        rows, vocab = case['rows'], case['vocab']
        size = 2 if case['dtype'] == 'fp16' else 4
        return {'bytes': rows * (vocab * size + 28), 'flops': 4 * rows * vocab}
    hq, hkv, page = case['q_heads'], case['kv_heads'], case['page']
    new, past = _lengths(case)
    tokens = sum(new)
    if case['kind'] == 'append':
        return {'bytes': tokens * (2 * 2 * (hq + 2 * hkv) * D + 4 * D), 'flops': 9 * tokens * (hq + hkv) * D}
    cached = sum(n + p for n, p in zip(new, past) if n)
    if case['kind'] == 'attend':
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
    else:
        pairs = sum(n * p for n, p in zip(new, past)) + sum(d + 1 for d in _depths(_tree_masks(new, case['mix'])))
    return {'bytes': 2 * cached * hkv * D * 2 + 2 * tokens * hq * D * 2 + 4 * sum((n + p) // page + 1 for n, p in
                                                                                  zip(new, past)),
            'flops': 4 * pairs * hq * D}


# ----------------------------------------------------------------------------- from the definition, in 64 bits

def _exact_append(case: dict, state: dict):
    hq, hkv, page = case['q_heads'], case['kv_heads'], case['page']
    q_out = state['out'].double()
    keys, values = state['key_pages'].double(), state['value_pages'].double()
    qkv = state['qkv'].double()
    half = D // 2
    for b, (n, p) in enumerate(zip(state['new'], state['past'])):
        if n == 0:
            continue
        t0 = state['starts'][b]
        rows = qkv[t0:t0 + n].reshape(n, hq + 2 * hkv, D)
        c, s = state['cos'][p:p + n].double()[:, None], state['sin'][p:p + n].double()[:, None]
        turned = []
        for part, w in ((rows[:, :hq], state['q_norm']), (rows[:, hq:hq + hkv], state['k_norm'])):
            u = part / torch.sqrt(part.pow(2).sum(-1, keepdim=True) / D + EPS) * w.double()
            lo, hi = u[..., :half], u[..., half:]
            turned.append(torch.cat((lo * c[..., :half] - hi * s[..., :half], hi * c[..., half:] + lo * s[..., half:]),
                                    dim=-1))
        q_out[t0:t0 + n] = turned[0]
        ids = state['page_table'][b].tolist()
        for i in range(n):
            at = p + i
            keys[ids[at // page], :, at % page] = turned[1][i]
            values[ids[at // page], :, at % page] = rows[i, hq + hkv:]
    return q_out, keys, values


def _exact_attend(case: dict, state: dict):
    hq, hkv, page = case['q_heads'], case['kv_heads'], case['page']
    group = hq // hkv
    out = torch.zeros(state['out'].shape, dtype=torch.float64, device=DEVICE)
    for b, (n, p) in enumerate(zip(state['new'], state['past'])):
        if n == 0:
            continue
        length, t0 = n + p, state['starts'][b]
        slot = torch.arange(length, device=DEVICE)
        ids = state['page_table'][b].long()[slot // page]
        if case['kind'] == 'tree':
            rows = [[(m >> j) & 1 for j in range(n)] for m in state['masks'][t0:t0 + n]]
            hide = torch.zeros(n, length, dtype=torch.bool, device=DEVICE)
            hide[:, p:] = torch.tensor(rows, device=DEVICE) == 0
        else:
            hide = slot[None, :] > p + torch.arange(n, device=DEVICE)[:, None]
        for h in range(hkv):
            k = state['key_pages'][ids, h, slot % page].double()
            v = state['value_pages'][ids, h, slot % page].double()
            kt = k.t().contiguous()
            for g in range(group):
                s = state['query'][t0:t0 + n, h * group + g].double() @ kt * state['scale']
                s[hide] = float('-inf')
                out[t0:t0 + n, h * group + g] = torch.softmax(s, dim=1) @ v
    return out


def _exact_sample(case: dict, state: dict):
    tokens = []
    params = _params(case)
    for r in range(case['rows']):
        values = state['logits'][r].double()
        temperature = float(state['temperature'][r])
        order = sorted_by_value = torch.argsort(values, descending=True, stable=True)
        if temperature == 0.0:
            tokens.append(int(order[0]))
            continue
        z = (values[sorted_by_value] - values[order[0]]) / temperature
        kept = z.numel() if params['top_k'][r] <= 0 else min(params['top_k'][r], z.numel())
        z, order = z[:kept], order[:kept]
        w = z.exp()
        top_p = float(state['top_p'][r])
        if top_p < 1.0:
            goal = top_p * w.sum()
            count = int(((torch.cumsum(w, 0) - w) < goal).sum())
            z, w, order = z[:max(count, 1)], w[:max(count, 1)], order[:max(count, 1)]
        min_p = float(state['min_p'][r])
        if min_p > 0.0:
            keep = z >= math.log(min_p)
            keep[0] = True
            w, order = w[keep], order[keep]
        order, back = torch.sort(order)
        running = torch.cumsum(w[back], 0)
        at = int((running <= float(state['uniform'][r]) * running[-1]).sum())
        tokens.append(int(order[min(at, order.numel() - 1)]))
    return torch.tensor(tokens, dtype=torch.int64, device=DEVICE)


def exact(case: dict, seed: int):
    if case['kind'] != 'sample' and work(case)['flops'] > 1e12:
        return None
    state = prepare(case, seed)
    return {'append': _exact_append, 'attend': _exact_attend, 'tree': _exact_attend,
            'sample': _exact_sample}[case['kind']](case, state)
