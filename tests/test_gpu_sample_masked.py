"""Token sampling of masked rows that are longer than the list of candidates.

Against the oracle, compared as all sampled rows are: tokens equal, probabilities
to the bounds derived there. A masked logit is -inf, or a NaN, which counts as
that; with fewer tokens left than top_k asks for, all of them are kept.
"""
from __future__ import annotations

import math

import pytest
import torch
from test_gpu_sample_tokens import _check, _logits

pytestmark = pytest.mark.gpu

LEFT = (1, 2, 40, 300, 2000)
TOP_K = (2, 50, 256, 257, 500, 5000)
FILTERS = [{}, dict(top_p=0.9), dict(min_p=0.05), dict(top_p=0.9, min_p=0.01)]


def _masked(V, dtype, counts, seed):
    """One row for each of `counts`: so many logits are left, side by side or all over the row, the others -inf or NaN."""
    logits, random = _logits(len(counts), V, dtype, seed)
    gen = torch.Generator().manual_seed(seed + 1)
    for row, n in enumerate(counts):
        if row % 2:
            left = torch.randperm(V, generator=gen)[:n]
        else:
            left = int(torch.randint(0, V - n + 1, (1,), generator=gen)) + torch.arange(n)
        masked = torch.ones(V, dtype=torch.bool)
        masked[left] = False
        logits[row, masked] = math.nan if row // 2 % 2 else -math.inf
    return logits, random


def _check_allowed(logits, random, **kw):
    tokens, probs = _check(logits, random, **kw)
    drawn = logits.gather(1, tokens.unsqueeze(1))  # (out of range raises)
    assert (drawn > -math.inf).all()
    assert not probs[~(logits > -math.inf)].any()


@pytest.mark.parametrize("V", [1025, 32000, 128257])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("kw", FILTERS, ids=str)
def test_top_k(V, dtype, kw):
    """Fewer tokens than top_k, as many, and more."""
    pairs = [(n, k) for n in LEFT if n < V for k in TOP_K]
    logits, random = _masked(V, dtype, [n for n, _ in pairs], seed=V)
    _check_allowed(logits, random, top_k=torch.tensor([k for _, k in pairs]), **kw)


@pytest.mark.parametrize("k", [50, 300, 2000, 2001])
def test_top_k_of_all_rows(k):
    counts = [n for n in (k - 1, k, k + 1, 3000) for _ in range(4)]
    logits, random = _masked(5000, "fp32", counts, seed=k)
    _check_allowed(logits, random, top_k=k, temperature=0.7)


@pytest.mark.parametrize("kw", [{}, dict(top_p=0.5), dict(top_p=0.999), dict(min_p=0.05), dict(temperature=0.0),
                                dict(top_p=0.95, min_p=1e-3, temperature=2.0)], ids=str)
def test_other_filters(kw):
    logits, random = _masked(50021, "bf16", [n for n in LEFT for _ in range(4)], seed=3)
    _check_allowed(logits, random, **kw)


def test_equal_and_far_logits_beside_masked_ones():
    """All that is left in one bin, or at the ends of the range."""
    logits, random = _masked(5000, "fp32", [2000] * 8, seed=5)
    left = logits > -math.inf
    logits[:2] = torch.where(left[:2], 0.25, logits[:2])
    logits[2:4] = torch.where(left[2:4], torch.finfo(torch.float32).min, logits[2:4])
    for row in range(4, 8):
        first = int(left[row].nonzero()[0])
        logits[row, first] = (-1e30, 1e30, math.inf, torch.finfo(torch.float32).min)[row - 4]
    for k in (1500, 2000, 3000):
        _check_allowed(logits, random, top_k=k)
        _check_allowed(logits, random, top_k=k, top_p=0.9)
