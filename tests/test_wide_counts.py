"""Lengths and bounds in 64 bits whose values pass 32: held to what there is, as smaller ones are."""
from __future__ import annotations

import pytest
import torch

WIDE = [2 ** 31, 2 ** 32 + 1, 2 ** 63 - 1]
BELOW = [-1, -2 ** 31 - 1, -2 ** 63]


def test_counts_as_the_kernels_read_them():
    from ramnet_ops.impl._delta import _whole
    read = _whole(torch.tensor(WIDE + BELOW + [0, 5, 2 ** 31 - 1]))
    assert read.dtype == torch.int32 and read.tolist() == [2 ** 31 - 1] * 3 + [0] * 3 + [0, 5, 2 ** 31 - 1]
    small = torch.tensor([3, -4], dtype=torch.int32)
    assert _whole(small) is small and _whole(None) is None


def _calls(T):
    """An operator of (lengths or bounds) each, over T tokens of a batch of one."""
    from ramnet_ops import causal_conv, gated_delta_rule, selective_scan
    gen = torch.Generator("cuda").manual_seed(T)

    def randn(*shape):
        return torch.randn(1, T, *shape, device="cuda", generator=gen)

    x, dt, B, C = randn(6), randn(6), randn(2, 5), randn(2, 5)
    q, k, v, g = randn(2, 16), torch.nn.functional.normalize(randn(2, 16), dim=-1), randn(2, 16), -randn(2).abs()
    weight, A = torch.ones(6, 3, device="cuda"), -torch.ones(6, 5, device="cuda")
    return (lambda **kw: causal_conv(x, weight, **kw), lambda **kw: selective_scan(x, dt, A, B, C, softplus=True, **kw),
            lambda **kw: gated_delta_rule(q, k, v, g, torch.sigmoid(g), **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 5, 200])
def test_lengths(T):
    for call in _calls(T):
        for counts, same in ((WIDE, T), (BELOW, 0)):
            want = call(lengths=torch.tensor([same], device="cuda", dtype=torch.int32))
            for n in counts:
                got = call(lengths=torch.tensor([n], device="cuda"))
                assert all(torch.equal(a, b) for a, b in zip(got, want)), n


@pytest.mark.gpu
def test_bounds():
    for call in _calls(200):
        want = call(cu_seqlens=torch.tensor([0, 70, 200], device="cuda", dtype=torch.int32))
        for last in WIDE:
            got = call(cu_seqlens=torch.tensor([-2 ** 40, 70, last], device="cuda"))
            assert all(torch.equal(a, b) for a, b in zip(got, want)), last


@pytest.mark.gpu
def test_draft_lengths():
    from ramnet_ops import verify_drafts
    gen = torch.Generator("cuda").manual_seed(0)
    target = torch.rand(2, 4, 50, device="cuda", generator=gen).softmax(-1)
    draft = torch.rand(2, 3, 50, device="cuda", generator=gen).softmax(-1)
    args = (draft.argmax(-1), target, draft, torch.rand(2, 3, device="cuda", generator=gen),
            torch.rand(2, device="cuda", generator=gen))
    want = verify_drafts(*args, draft_lens=torch.tensor([3, 0], device="cuda", dtype=torch.int32))
    got = verify_drafts(*args, draft_lens=torch.tensor([2 ** 40 + 1, -2 ** 40 + 3], device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
