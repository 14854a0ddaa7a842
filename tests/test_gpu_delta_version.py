"""A state updated in place counts as changed: autograd refuses what it saved of it before."""
from __future__ import annotations

import pytest
import torch

from test_gpu_delta_rule import DEV, _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 100])
def test_in_place_raises_the_version(T):
    from ramnet_ops import gated_delta_rule
    case = [t.to(DEV) for t in _case(T=T, Dk=16, Dv=16)]
    state = case[5]
    base = state._version
    gated_delta_rule(*case[:5], init_state=state, inplace=True)
    assert state._version > base
    before = state._version
    gated_delta_rule(*case[:5], init_state=state)
    assert state._version == before


@pytest.mark.parametrize("T", [1, 100])
def test_saved_state_is_refused(T):
    from ramnet_ops import gated_delta_rule
    case = [t.to(DEV) for t in _case(T=T, Dk=16, Dv=16)]
    w = torch.ones_like(case[5], requires_grad=True)
    loss = (w * case[5]).sum()  # the gradient of w is the state as it is now
    gated_delta_rule(*case[:5], init_state=case[5], inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_in_inference_mode():
    from ramnet_ops import gated_delta_rule
    with torch.inference_mode():
        case = [t.to(DEV) for t in _case(T=1, Dk=16, Dv=16)]
        state = case[5].clone()
        want = gated_delta_rule(*case[:5], init_state=case[5])[1]
        gated_delta_rule(*case[:5], init_state=state, inplace=True)
        assert torch.equal(state, want)
