"""Random numbers that meet a running sum to the bit: the next token is drawn.

Equal logits have equal weights, so of 2^n kept ones every running sum is a
dyadic share of all, and so is its product with a random number k / 2^m.
"""
from __future__ import annotations

import pytest
import torch
from test_gpu_sample_tokens import _check

pytestmark = pytest.mark.gpu

EIGHTHS = torch.arange(8) / 8.0


def _equal(V, left):
    """Rows of V logits of which the `left` are equal, the others far below the least weight that counts."""
    logits = torch.full((8, V), -1e4)
    logits[:, left] = 0.25
    return logits


@pytest.mark.parametrize("V", [8, 300, 50021])
@pytest.mark.parametrize("kw", [{}, dict(top_k=8), dict(min_p=0.5), dict(top_p=0.999)], ids=str)
def test_eight(V, kw):
    """In a list, and by stretches of a long row."""
    left = torch.linspace(0, V - 1, 8).long()
    tokens, _ = _check(_equal(V, left), EIGHTHS, **kw)
    assert tokens.tolist() == left.tolist()


@pytest.mark.parametrize("kw", [{}, dict(top_k=4096), dict(min_p=0.5), dict(top_p=0.5)], ids=str)
def test_more_than_a_list(kw):
    left = torch.arange(4096) * 12 + 7
    tokens, _ = _check(_equal(50021, left), EIGHTHS, **kw)
    kept = 2048 if "top_p" in kw else 4096
    assert tokens.tolist() == left[torch.arange(8) * (kept // 8)].tolist()
