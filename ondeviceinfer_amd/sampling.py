"""Choosing the next token of every sequence of a batch.

The reference generates greedily only (``ondeviceinfer/generation.py:47, :58``:
argmax of the last position); ``sample_tokens`` draws from the logits after
temperature, top-k, top-p and min-p, with random numbers the caller gives, so
that a run can be repeated.
"""
from __future__ import annotations

from torch import Tensor

from . import _native


def sample_tokens(logits: Tensor, uniform: Tensor, *, temperature: Tensor | float = 1.0, top_k: Tensor | int = 0,
                  top_p: Tensor | float = 1.0, min_p: Tensor | float = 0.0, out: Tensor | None = None,
                  workspace: Tensor | None = None) -> Tensor:
    """One token per row of ``logits`` (fp16 or fp32 ``[rows, vocab]``, rows may
    lie apart), int64 ``[rows]``, from ``uniform`` (fp32 ``[rows]`` in [0, 1)).

    Tokens are ordered by logit, equal ones by index, and weigh
    ``exp((logit - largest) / temperature)``.  ``top_k`` > 0 keeps the first
    ``top_k``; ``top_p`` < 1 keeps of those each token in front of which less
    than ``top_p`` of their whole weight lies; ``min_p`` > 0 keeps of those the
    ones that weigh at least ``min_p`` (the largest weighs 1); the first always
    stays.  The result is the first remaining token, in the order of the
    vocabulary, at which their running weight exceeds ``uniform`` times their
    whole weight.  ``temperature`` 0 takes the first token of the order (the
    argmax).  Each setting is a number for all rows or a tensor ``[rows]`` on
    the device (fp32, ``top_k`` int32).

    A row gives -1 if it holds NaN or nothing above -inf, or if a setting of it
    has no meaning (a temperature that is negative or not finite, NaN)."""
    return _native.sample(logits, uniform, temperature, top_k, top_p, min_p, out, workspace)
