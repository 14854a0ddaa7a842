"""Tracing the convolution, the scan and sampling (CPU): shapes, symbolic sizes, what a training call keeps."""
from __future__ import annotations

import itertools

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv, StatelessSymbolicContext


def _fake(mode, shape, dynamic, dtype=torch.float32):
    sizes = [DimDynamic.DYNAMIC if d else DimDynamic.STATIC for d in dynamic]
    return mode.from_tensor(torch.empty(shape, dtype=dtype),
                            symbolic_context=StatelessSymbolicContext(dynamic_sizes=sizes))


@pytest.mark.parametrize("packed", [False, True])
def test_symbolic_sizes(packed):
    import ramnet_ops  # noqa: F401
    ops = torch.ops.ramnet_ops
    env = ShapeEnv()
    mode = FakeTensorMode(shape_env=env)
    dims = (not packed, True, False)
    batch = 1 if packed else 3
    x, dt = (_fake(mode, (batch, 1234, 24), dims) for _ in range(2))
    B, C = (_fake(mode, (batch, 1234, 2, 10), (*dims, False)) for _ in range(2))
    A, weight = _fake(mode, (24, 10), (False, False)), _fake(mode, (24, 4), (False, False))
    cu = _fake(mode, (8,), (True,), torch.int32) if packed else None
    with mode:
        y, state = ops.causal_conv(x, weight, None, None, cu, None, True)
        y2, state2, kept = ops.selective_scan_kept(x, dt, A, B, C, None, None, None, None, cu, None, True)
        for t in (y, y2):
            assert t.shape[1].node.expr.free_symbols
        for t in (state, state2, kept):
            assert t.shape[0].node.expr.free_symbols
        tokens, probs = ops.sample_tokens_with_probabilities(y, y[..., 0], None, None, None, None, 1.0, 0, 1.0, 0.0)
        assert tokens.shape[1].node.expr.free_symbols and probs.dtype == torch.float32
    assert not [s for s, value in env.replacements.items() if not value.free_symbols]


def test_kept_is_what_the_forward_asks_for():
    from ramnet_ops import _native
    from ramnet_ops.impl import _scan
    lib = _native.lib()
    for B, T, D, S, packed in itertools.product((1, 2, 9), (0, 1, 15, 16, 17, 500, 4096), (1, 40), (1, 4, 5, 16, 17, 33, 64),
                                                (0, 1)):
        sizes = (1 if packed else B, T, B, D, S, 1)
        assert lib.ramnet_selective_scan_kept_bytes(*sizes, packed) == _scan._kept_bytes(sizes, bool(packed))
