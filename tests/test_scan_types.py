"""Types of the selective scan's parameters, as its documentation has them (CPU)."""
from __future__ import annotations

import pytest
import torch

from test_scan_refusals import _scan

SHAPES = dict(A=(6, 5), skip=(6,), dt_bias=(6,), init_state=(2, 6, 5))


@pytest.mark.parametrize("name", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float64, torch.int32, torch.bool, torch.complex64])
def test_others_are_refused(name, dtype):
    from ramnet_ops import selective_scan
    with pytest.raises(RuntimeError, match=f"{name} must be one of"):
        selective_scan(**_scan(**{name: torch.zeros(SHAPES[name]).to(dtype)}))


@pytest.mark.parametrize("name", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_types_that_are_taken(name, dtype):
    """They get as far as the device's check."""
    from ramnet_ops import selective_scan
    with pytest.raises(RuntimeError, match="must be on a GPU"):
        selective_scan(**_scan(**{name: torch.zeros(SHAPES[name]).to(dtype)}))
