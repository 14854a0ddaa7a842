"""Packed buffers of which few tokens belong to a sequence, as a server of fixed
sizes has them, on the GPU: zeros elsewhere, in about the time of a full buffer at most."""
from __future__ import annotations

import pytest
import torch

from test_gpu_delta_rule import DEV, _case, _rel

pytestmark = pytest.mark.gpu


def _grads(case, cu, d):
    from ramnet_ops import gated_delta_rule
    x = [t.detach().requires_grad_() for t in case]
    o, state = gated_delta_rule(*x[:5], init_state=x[5], cu_seqlens=cu)
    return [o.detach(), state.detach(), *torch.autograd.grad([o, state], x, [d, torch.ones_like(state)])]


@pytest.mark.parametrize("T,bounds", [
    (3000, [0, 20, 40]), (3000, [2960, 2980, 3000]), (3000, [0, 0, 0]), (3000, [3000, 3000, 3000]),
    (3001, [1500, 1501, 1777]), (3001, [1, 2999, 3000]), (64, [63, 64, 64]), (65, [0, 1, 1]), (130, [65, 65, 65])])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_values(T, bounds, dtype):
    case = [t.to(DEV) for t in _case(T=T, Hk=2, Hv=4, Dk=20, Dv=36, dtype=dtype, g_dtype=dtype, N=2, seed=T)]
    d = torch.randn(1, T, 4, 36, device=DEV).to(case[2].dtype)
    a, b = bounds[0], bounds[-1]
    # memory that is reused holds no zeros
    junk = [torch.full((1, T, 4, 36), 7.0, device=DEV, dtype=case[2].dtype) for _ in range(8)]
    del junk
    got = _grads(case, torch.tensor(bounds, device=DEV, dtype=torch.int32), d)
    for t in (got[0], *got[2:7]):
        assert (t[:, :a] == 0).all() and (t[:, b:] == 0).all()
    if b > a:
        part = [t[:, a:b] for t in case[:5]] + [case[5]]
        want = _grads(part, torch.tensor([n - a for n in bounds], device=DEV, dtype=torch.int32), d[:, a:b])
        for i, (x, y) in enumerate(zip(got, want)):
            x = x if i in (1, 7) else x[:, a:b]
            assert _rel(x, y.cpu()) <= 2 * (torch.finfo(x.dtype).eps if x.dtype != torch.float32 else 2.0 ** -19), i


def _time(f):
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    times = []
    for _ in range(7):
        start.record()
        f()
        end.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(end))
    return min(times)


@pytest.mark.parametrize("train", [False, True])
def test_time(train):
    """100 tokens of 32768 against all of them (half the time; one block that clears the others takes
    seventeen times as long. Twice: a training call's host time is the same for both)."""
    from ramnet_ops import gated_delta_rule
    case = [t.to(DEV) for t in _case(T=32768, Hk=4, Hv=4, Dk=64, Dv=64, dtype="bf16", N=1)]
    few, all_of_them = (torch.tensor([0, n], device=DEV, dtype=torch.int32) for n in (100, 32768))

    def run(cu):
        if train:
            return _grads(case, cu, case[2])
        return gated_delta_rule(*case[:5], init_state=case[5], cu_seqlens=cu)
    assert _time(lambda: run(few)) < 2 * _time(lambda: run(all_of_them))
