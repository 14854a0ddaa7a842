"""Types that the gated delta rule and draft verification do not compute with are refused (CPU)."""
from __future__ import annotations

import pytest
import torch

from test_delta_refusals import _delta, _verify

WRONG = [torch.float64, torch.int32, torch.int64, torch.bool, torch.complex64]


@pytest.mark.parametrize("dtype", WRONG)
def test_init_state(dtype):
    from ramnet_ops import gated_delta_rule
    with pytest.raises(RuntimeError, match="init_state must be one of"):
        gated_delta_rule(**_delta(init_state=torch.zeros(1, 4, 8, 6).to(dtype)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_types_that_are_taken(dtype):
    """They get as far as the device's check."""
    from ramnet_ops import gated_delta_rule, verify_drafts
    with pytest.raises(RuntimeError, match="must be on a GPU"):
        gated_delta_rule(**_delta(init_state=torch.zeros(1, 4, 8, 6).to(dtype)))
    with pytest.raises(RuntimeError, match="must be on a GPU"):
        verify_drafts(**_verify(accept=torch.zeros(2, 3).to(dtype), sample=torch.zeros(2).to(dtype)))


@pytest.mark.parametrize("name", ["accept", "sample"])
@pytest.mark.parametrize("dtype", WRONG[1:])
def test_uniform_numbers(name, dtype):
    from ramnet_ops import verify_drafts
    x = _verify()
    with pytest.raises(RuntimeError, match=f"{name} must be floating-point"):
        verify_drafts(**_verify(**{name: x[name].to(dtype)}))


@pytest.mark.gpu
def test_a_type_once_taken_does_not_let_another_in():
    """Calls of the same sizes share their checks, of the same types alone."""
    from ramnet_ops import gated_delta_rule
    case = [t.cuda() for t in _delta().values()]
    state = torch.zeros(1, 4, 8, 6, device="cuda")
    gated_delta_rule(*case, init_state=state)
    with pytest.raises(RuntimeError, match="init_state must be one of"):
        gated_delta_rule(*case, init_state=state.double())
