"""Generation over the quantized Qwen3 model: greedily for one sequence
(``greedy_generate``), sampled for many (``sample_generate``).

Callers' interface as in the reference (``ondeviceinfer/generation.py:15-70``):
``greedy_generate(model, input_ids, *, max_new_tokens, cache, eos_token_id)``
returns ``GenerationResult`` (``token_ids``, ``generated_ids``,
``prefill_seconds``, ``decode_seconds``, ``decode_tokens_per_second`` =
(generated - 1) / decode seconds, the first token being the prefill's).

The loop is built around the decode graph: each step's greedy token stays on
the device (the LM-head kernel picks it, ``CausalLMOutput.next_token``), is
fed straight back as the next input and is written into a preallocated
device row of generated ids, so without an ``eos_token_id`` the host waits
only once, at the end of the decode phase.  With one, every step has to
read the token back to decide whether to stop.
"""
from __future__ import annotations

import time
from dataclasses import dataclass

import torch
from torch import Tensor

from .sampling import sample_tokens


@dataclass
class GenerationResult:
    token_ids: Tensor
    generated_ids: Tensor
    prefill_seconds: float
    decode_seconds: float

    @property
    def decode_tokens_per_second(self) -> float:
        """Tokens of the decode phase per second; the first generated token
        belongs to the prefill."""
        steps = self.generated_ids.shape[1] - 1
        return steps / self.decode_seconds if steps > 0 and self.decode_seconds > 0 else 0.0


def greedy_token(output) -> Tensor:
    """The greedy next token ``[batch, 1]`` of a model output: the decode
    graph's in-kernel pick when present (the first index of the largest fp16
    logit, ``torch.argmax``'s rule), else the argmax of the last position."""
    picked = getattr(output, 'next_token', None)
    if picked is not None:
        return picked
    return torch.argmax(output.logits[:, -1], dim=-1, keepdim=True)


def _wait(device: torch.device) -> None:
    if device.type == 'cuda':
        torch.cuda.synchronize(device)


@torch.inference_mode()
def greedy_generate(model, input_ids: Tensor, *, max_new_tokens: int, cache, eos_token_id: int | None = None
                    ) -> GenerationResult:
    """Prefill ``input_ids [1, S]`` into ``cache``, then decode greedily until
    ``max_new_tokens`` tokens exist (at least the prefill's one) or the last
    one equals ``eos_token_id``."""
    if input_ids.dim() != 2:
        raise ValueError(f'input_ids must be [batch, sequence], got shape {tuple(input_ids.shape)}')
    if input_ids.shape[0] != 1:
        raise NotImplementedError(f'greedy_generate runs batch size 1, got {input_ids.shape[0]}')
    device = input_ids.device
    budget = max(1, max_new_tokens)

    _wait(device)
    t_prefill = time.perf_counter()
    token = greedy_token(model(input_ids, cache=cache, logits_to_keep=1))
    generated = torch.empty((1, budget), dtype=torch.long, device=token.device)
    generated[:, :1].copy_(token)
    _wait(device)
    prefill_seconds = time.perf_counter() - t_prefill

    count = 1
    t_decode = time.perf_counter()
    while count < budget:
        if eos_token_id is not None and bool((token == eos_token_id).all()):
            break
        token = greedy_token(model(token, cache=cache, logits_to_keep=1))
        generated[:, count:count + 1].copy_(token)
        count += 1
    _wait(device)
    decode_seconds = time.perf_counter() - t_decode

    generated = generated[:, :count]
    return GenerationResult(token_ids=torch.cat((input_ids, generated.to(input_ids.dtype)), dim=1),
                            generated_ids=generated, prefill_seconds=prefill_seconds,
                            decode_seconds=decode_seconds)


@torch.inference_mode()
def sample_generate(model, prompts, *, max_new_tokens: int, cache, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                    eos_token_id: int | None = None, generator: torch.Generator | None = None) -> list[list[int]]:
    """The continuations of several prompts (lists or 1-D tensors of token ids),
    sampled together over a paged cache (``model.make_paged_cache``).

    All prompts are prefilled in one step, then every step advances the
    sequences that are not done.  The settings are ``sample_tokens``' (numbers,
    or a device tensor with one entry per prompt); ``generator`` (of the model's
    device) makes a run repeatable.  A sequence ends at ``max_new_tokens`` or
    with ``eos_token_id``, which is kept, or before a token that its row of
    logits does not allow (-1).  Its pages go back to the cache when it ends.
    The tokens are read after every step with an ``eos_token_id`` and once, at
    the end, without; every step's page numbers go to the device in a copy that
    waits for the step before it in either case."""
    prompts = [torch.as_tensor(p, dtype=torch.long).reshape(-1) for p in prompts]
    if not prompts or any(p.numel() == 0 for p in prompts):
        raise ValueError('every prompt needs at least one token')
    device = model.device
    budget = max(1, max_new_tokens)
    settings = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    sequences = [cache.add() for _ in prompts]
    live = list(range(len(prompts)))
    steps: list[tuple[list[int], Tensor]] = []   # per step the prompts it advanced and their tokens, on the device
    done = [False] * len(prompts)

    def pick(logits: Tensor, rows: list[int]) -> Tensor:
        mine = settings
        if len(rows) != len(prompts):
            index = torch.tensor(rows, device=device)
            mine = {k: v[index] if isinstance(v, Tensor) else v for k, v in settings.items()}
        uniform = torch.rand(len(prompts), device=device, generator=generator)   # one per prompt: a sequence's numbers
        if len(rows) != len(prompts):                                            # do not depend on which others live
            uniform = uniform[index]
        return sample_tokens(logits, uniform, **mine)

    try:
        output = model.forward_paged(torch.cat([p.to(device) for p in prompts]), cache, sequences,
                                     [p.numel() for p in prompts])
        tokens = pick(output.logits, live)
        steps.append((live, tokens))
        for _ in range(budget - 1):
            if eos_token_id is not None:
                ended = [t == eos_token_id or t < 0 for t in tokens.tolist()]
                if any(ended):
                    for i, e in zip(live, ended):
                        if e:
                            done[i] = True
                            cache.free(sequences[i])
                    stay = torch.tensor([j for j, e in enumerate(ended) if not e], device=device, dtype=torch.long)
                    tokens, live = tokens[stay], [i for i, e in zip(live, ended) if not e]
                if not live:
                    break
            output = model.forward_paged(tokens, cache, [sequences[i] for i in live], [1] * len(live))
            tokens = pick(output.logits, live)
            steps.append((live, tokens))
    finally:
        for i, seq in enumerate(sequences):
            if not done[i]:
                cache.free(seq)
    result: list[list[int]] = [[] for _ in prompts]
    over = [False] * len(prompts)
    for rows, picked in steps:
        for i, token in zip(rows, picked.tolist()):
            over[i] = over[i] or token < 0
            if not over[i]:
                result[i].append(token)
    return result
