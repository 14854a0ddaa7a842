"""The gated delta rule on heads whose matrices pass the 32-bit byte offsets of
the chunked kernels: refused for gradients, walked token by token otherwise."""
from __future__ import annotations

import math

import pytest
import torch

F32, F16, BF16 = 0, 1, 2


@pytest.mark.parametrize("Dk,padded", [(256, 256), (200, 256), (160, 160), (128, 128)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_sizes(Dk, padded, dtype):
    """A matrix of `padded` rows, each padded to a multiple of 8 values, may end at 2^30 bytes."""
    from ramnet_ops import _native
    lib = _native.lib()
    last = (1 << 28) // padded // 8 * 8

    def sizes(Dv, T=64):
        at = (1, T, 1, 1, 1, Dk, Dv, dtype, 0)
        return [lib.ramnet_delta_rule_workspace_bytes(*at, kind) for kind in range(3)] + [
            lib.ramnet_delta_rule_kept_bytes(*at)]
    assert min(sizes(last)) > 0
    assert sizes(last + 1) == [0, -1, -1, -1]
    assert sizes(last, T=8)[0] == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_key_heads(dtype):
    """Rows of dq and dk of all heads: less than 2^22 values."""
    from ramnet_ops import _native
    lib = _native.lib()

    def sizes(Hk):
        at = (1, 64, 1, Hk, Hk, 128, 8, dtype, 0)
        return [lib.ramnet_delta_rule_workspace_bytes(*at, kind) for kind in range(3)] + [
            lib.ramnet_delta_rule_kept_bytes(*at)]
    assert min(sizes((1 << 15) - 1)) > 0
    forward, *others = sizes(1 << 15)
    assert forward > 0 and others == [-1, -1, -1]


@pytest.mark.gpu
@pytest.mark.parametrize("Dv", [(1 << 20) - 5, 1 << 20, (1 << 20) + 3])
def test_values(Dv):
    """Nine tokens at once (in chunks up to 2^20 columns of 256 rows) and as eight and one (token by token)."""
    from ramnet_ops import gated_delta_rule
    gen = torch.Generator(device="cuda").manual_seed(0)
    T, Dk = 9, 256
    q, k = (torch.nn.functional.normalize(torch.randn(1, T, 1, Dk, generator=gen, device="cuda"), dim=-1).bfloat16()
            for _ in range(2))
    v = torch.randn(1, T, 1, Dv, generator=gen, device="cuda").bfloat16()
    g = -torch.rand(1, T, 1, generator=gen, device="cuda")
    beta = torch.rand(1, T, 1, generator=gen, device="cuda").bfloat16()
    o, state = gated_delta_rule(q, k, v, g, beta)
    first, walked = gated_delta_rule(*(t[:, :8] for t in (q, k, v, g, beta)))
    second, _ = gated_delta_rule(*(t[:, 8:] for t in (q, k, v, g, beta)), init_state=walked, inplace=True)
    want = torch.cat([first, second], 1)
    if Dv > 1 << 20:
        assert torch.equal(o, want) and torch.equal(state, walked)
    # both within 8 sqrt(256) 2^-24 of the value; the outputs rounded once each
    arith = 8 * math.sqrt(Dk) * 2.0 ** -24
    assert (state - walked).norm() <= 2 * arith * walked.norm()
    off = float((o.float() - want.float()).norm() / want.float().norm())
    assert off <= math.sqrt(2 * arith * torch.finfo(o.dtype).eps) + 2 * arith
    # the last columns, which share their kernel's tile with columns that are not there
    assert (state[..., -20:] - walked[..., -20:]).norm() <= 2 * arith * walked[..., -20:].norm()
