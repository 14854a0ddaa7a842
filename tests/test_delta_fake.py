"""Tracing a training call of the gated delta rule (CPU): sizes stay symbolic."""
from __future__ import annotations

import itertools

import pytest
import torch
import torch._dynamo.testing
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv, StatelessSymbolicContext

HK, HV, DK, DV = 2, 4, 24, 40


def _fake(mode, shape, dynamic, dtype=torch.float32):
    sizes = [DimDynamic.DYNAMIC if d else DimDynamic.STATIC for d in dynamic]
    return mode.from_tensor(torch.empty(shape, dtype=dtype),
                            symbolic_context=StatelessSymbolicContext(dynamic_sizes=sizes))


def _inputs(mode, B, T, dyn_b, dyn_t, Dk=DK):
    dims = (dyn_b, dyn_t, False, False)
    q, k = (_fake(mode, (B, T, HK, Dk), dims) for _ in range(2))
    v = _fake(mode, (B, T, HV, DV), dims)
    g, beta = (_fake(mode, (B, T, HV), dims[:3]) for _ in range(2))
    return q, k, v, g, beta


@pytest.mark.parametrize("B,dyn_b", [(1, False), (3, True), (40, True)])
@pytest.mark.parametrize("op", ["gated_delta_rule", "gated_delta_rule_kept"])
def test_symbolic_sizes(op, B, dyn_b):
    import ramnet_ops  # noqa: F401
    env = ShapeEnv()
    mode = FakeTensorMode(shape_env=env)
    x = _inputs(mode, B, 1234, dyn_b, True)
    with mode:
        o, state, *kept = getattr(torch.ops.ramnet_ops, op)(*x, None, None, None, 0.3)
        for t in (*x, o):
            assert t.shape[1].node.expr.free_symbols
        for t in kept:
            assert t.shape[0].node.expr.free_symbols
    # nothing but the sizes of different tensors being the same ones is assumed
    assert not [s for s, value in env.replacements.items() if not value.free_symbols]


def test_packed_symbolic_sizes():
    import ramnet_ops  # noqa: F401
    env = ShapeEnv()
    mode = FakeTensorMode(shape_env=env)
    x = _inputs(mode, 1, 1234, False, True)
    cu = _fake(mode, (8,), (True,), torch.int32)
    with mode:
        o, state, kept = torch.ops.ramnet_ops.gated_delta_rule_kept(*x, None, cu, None, 0.3)
        assert state.shape[0].node.expr.free_symbols and kept.shape[0].node.expr.free_symbols
    assert not [s for s, value in env.replacements.items() if not value.free_symbols]


def test_refused_sizes():
    """As the call itself refuses them."""
    import ramnet_ops  # noqa: F401
    with FakeTensorMode():
        x = [torch.empty(shape) for shape in ((1, 70, 1, 200), (1, 70, 1, 200), (1, 70, 1, 8), (1, 70, 1), (1, 70, 1))]
        with pytest.raises(RuntimeError, match="up to 160 for gradients of float32"):
            torch.ops.ramnet_ops.gated_delta_rule_kept(*x, None, None, None, 0.3)


def test_kept_is_large_enough():
    """What is allotted under tracing against what the native forward asks for: that, and no more
    than the maps of the most segments there can be on top."""
    from ramnet_ops import _native
    from ramnet_ops.impl import _delta
    lib = _native.lib()
    for B, T, Hv, Dk, Dv, code, packed in itertools.product(
            (1, 2, 9, 64, 200), (1, 63, 64, 65, 500, 512, 513, 4096, 32768), (1, 8, 16), (1, 33, 128, 160, 256),
            (1, 64, 130), (0, 2), (0, 1)):
        N, rows = (B, 1) if packed else (B, B)
        sizes = rows, T, N, 1, Hv, Dk, Dv
        dtype = torch.float32 if code == 0 else torch.bfloat16
        need = lib.ramnet_delta_rule_kept_bytes(*sizes, code, packed)
        if need < 0:
            with pytest.raises(RuntimeError, match="not supported"):
                _delta._kept_bytes("test", sizes, dtype, bool(packed))
            continue
        have = _delta._kept_bytes("test", sizes, dtype, bool(packed))
        wide = next(w for w in (32, 64, 96, 128, 160, 256) if Dk <= w)
        assert need <= have <= need + N * Hv * min(-(-T // 64) // 4, 64) * wide * wide * 4 + 256


@pytest.mark.gpu
def test_compiled_for_any_length():
    from ramnet_ops import gated_delta_rule
    from test_gpu_delta_rule import DEV, _case
    counter = torch._dynamo.testing.CompileCounterWithBackend("aot_eager")

    def loss(q, k, v, g, beta, init):
        o, state = gated_delta_rule(q, k, v, g, beta, init_state=init)
        return (o * o).sum() + state.sum()
    compiled = torch.compile(loss, backend=counter, fullgraph=True, dynamic=True)
    for T in (70, 100, 129, 1100):
        x = [t.to(DEV).requires_grad_() for t in _case(T=T, Hk=1, Hv=2, Dk=32, Dv=32)]
        got = torch.autograd.grad(compiled(*x), x)
        want = torch.autograd.grad(loss(*x), x)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert counter.frame_count == 1
