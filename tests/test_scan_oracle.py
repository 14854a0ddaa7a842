"""The fp64 forms of the convolution, the scan and sampling against closed forms and against themselves (CPU)."""
from __future__ import annotations

import torch

from oracle import scan_oracle as oracle


def test_convolution_is_torchs():
    gen = torch.Generator().manual_seed(0)
    x, w, b = torch.randn(2, 9, 5, generator=gen), torch.randn(5, 4, generator=gen), torch.randn(5, generator=gen)
    y, state = oracle.causal_conv(x, w, b)
    want = torch.nn.functional.conv1d(torch.nn.functional.pad(x.double().mT, (3, 0)), w.double().unsqueeze(1), b.double(),
                                      groups=5).mT
    assert torch.allclose(y, want, rtol=1e-14, atol=1e-14) and torch.equal(state, x[:, -3:].double())
    y, _ = oracle.causal_conv(x, w, b, silu=True)
    assert torch.allclose(y, torch.nn.functional.silu(want), rtol=1e-14, atol=1e-14)


def test_convolution_in_two_calls():
    x, w = torch.randn(1, 9, 5), torch.randn(5, 4)
    y, state = oracle.causal_conv(x, w)
    for cut in (0, 1, 2, 8, 9):
        a, middle = oracle.causal_conv(x[:, :cut], w)
        b, end = oracle.causal_conv(x[:, cut:], w, init_state=middle)
        assert torch.allclose(torch.cat([a.reshape(1, cut, 5), b.reshape(1, 9 - cut, 5)], 1), y) and torch.equal(end, state)


def test_scan_closed_form():
    """Constant inputs: a geometric series."""
    T, D, S = 7, 3, 2
    one = torch.ones(1, T, D)
    A = -torch.rand(D, S)
    y, state = oracle.selective_scan(one, 0.5 * one, A, torch.ones(1, T, 1, S), torch.ones(1, T, 1, S))
    a = (0.5 * A.double()).exp()
    want = 0.5 * (1 - a ** T) / (1 - a)
    assert torch.allclose(state[0], want) and torch.allclose(y[0, -1], want.sum(-1))


def test_scan_parts():
    gen = torch.Generator().manual_seed(1)
    x, dt, z = (torch.randn(1, 6, 4, generator=gen).double() for _ in range(3))
    B, C = (torch.randn(1, 6, 2, 3, generator=gen).double() for _ in range(2))
    A, skip, bias = -torch.rand(4, 3), torch.randn(4, generator=gen), torch.randn(4, generator=gen)
    y, state = oracle.selective_scan(x, dt, A, B, C, skip, z, bias, True)
    step = torch.nn.functional.softplus(dt + bias)
    plain, same = oracle.selective_scan(x, step, A, B, C)
    assert torch.allclose(y, (plain + skip * x) * torch.nn.functional.silu(z)) and torch.allclose(state, same)
    a, middle = oracle.selective_scan(x[:, :2], dt[:, :2], A, B[:, :2], C[:, :2], skip, z[:, :2], bias, True)
    b, end = oracle.selective_scan(x[:, 2:], dt[:, 2:], A, B[:, 2:], C[:, 2:], skip, z[:, 2:], bias, True, init_state=middle)
    assert torch.allclose(torch.cat([a, b], 1), y) and torch.allclose(end, state)


def test_sampling_by_hand():
    logits = torch.log(torch.tensor([0.1, 0.4, 0.1, 0.3, 0.1]))
    assert oracle.sample_row(logits, 0.05)[0] == 0 and oracle.sample_row(logits, 0.15)[0] == 1
    assert oracle.sample_row(logits, 0.99)[0] == 4 and oracle.sample_row(logits, 0.5, temperature=0.0)[0] == 1
    assert torch.allclose(oracle.sample_row(logits, 0.0, top_k=3)[1], torch.tensor([1, 4, 0, 3, 0]).double() / 8)
    # 0.4 + 0.3 = 0.7 of the whole: 0.65 needs both, 0.75 the first of the equal ones too
    assert torch.allclose(oracle.sample_row(logits, 0.0, top_p=0.65)[1], torch.tensor([0, 4, 0, 3, 0]).double() / 7)
    assert torch.allclose(oracle.sample_row(logits, 0.0, top_p=0.75)[1], torch.tensor([1, 4, 0, 3, 0]).double() / 8)
    assert torch.allclose(oracle.sample_row(logits, 0.0, min_p=0.5)[1], torch.tensor([0, 4, 0, 3, 0]).double() / 7)
    nothing = torch.full((4,), -torch.inf)
    assert oracle.sample_row(nothing, 0.5)[0] == 0 and oracle.sample_row(nothing, 0.5)[1].sum() == 0
