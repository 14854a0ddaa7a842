"""The selective scan on the GPU against the fp64 oracle.

Tolerances are relative, in the 2-norm of an output:

* fp32 arithmetic: a state is a sum over at most T tokens of products of decays; each token adds three roundings
  (the decay's argument, its exponential, the sum), 2^-23 at most, at random: 8 sqrt(max(T, 64)) 2^-24.
* outputs in 16 bits: half a step of the type (eps / 2) on top.
* gradients are sums over twice as many tokens (there and back) of terms that cancel: 8 times the arithmetic's.
"""
from __future__ import annotations

import math

import pytest
import torch

from oracle import scan_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
NAMES = ("x", "dt", "A", "B", "C", "skip", "gate", "bias", "init")


def _tol(dtype, T, more=1):
    arith = more * 8 * math.sqrt(max(T, 64)) * 2.0 ** -24
    return arith if dtype == torch.float32 else torch.finfo(dtype).eps / 2 + arith


def _rel(got, want):
    want = want.double()
    norm = want.norm()
    off = (got.cpu().double() - want).norm()
    return float(off / norm) if norm > 0 else float(off)


def _case(B=1, T=37, D=40, S=16, G=1, dtype="fp32", N=None, gate=True, bias=True, skip=True, state=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]

    def rn(*s):
        return torch.randn(*s, generator=gen)
    A = -torch.arange(1, S + 1) * torch.exp(0.3 * rn(D, S))
    # steps from 0.001 to 0.5
    return [rn(B, T, D).to(dt), rn(B, T, D).to(dt), A, rn(B, T, G, S).to(dt), rn(B, T, G, S).to(dt),
            rn(D) if skip else None, rn(B, T, D).to(dt) if gate else None,
            -6 + 5 * torch.rand(D, generator=gen) if bias else None,
            0.5 * rn(N if N is not None else B, D, S) if state else None]


def _run(case, softplus=True, **kw):
    from ramnet_ops import selective_scan
    x, dt, A, B, C, skip, gate, bias, init = case
    return selective_scan(x, dt, A, B, C, skip=skip, gate=gate, dt_bias=bias, softplus=softplus, init_state=init, **kw)


def _call(case, **kw):
    return _run([t.to(DEV) if t is not None else None for t in case], **kw)


def _want(case, lens=None, packed=False, softplus=True):
    x, dt, A, B, C, skip, gate, bias, init = case
    return oracle.selective_scan(x, dt, A, B, C, skip, gate, bias, softplus, init, lens, packed)


def _check(case, got, **kw):
    y, state = _want(case, **kw)
    T, dtype = case[0].shape[1], case[0].dtype
    assert got[0].dtype == dtype and got[0].shape == case[0].shape
    assert got[1].dtype == torch.float32 and got[1].shape == state.shape
    assert _rel(got[0], y) <= _tol(dtype, T), ("y", _rel(got[0], y))
    assert _rel(got[1], state) <= _tol(torch.float32, T), ("state", _rel(got[1], state))


@pytest.mark.parametrize("T", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 130, 200])
def test_lengths(T):
    case = _case(B=2, T=T, seed=T)
    _check(case, _call(case))
    case[8] = None
    _check(case, _call(case))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("T", [3, 90])
def test_types_and_parts(dtype, T):
    for gate in (False, True):
        for bias in (False, True):
            case = _case(T=T, dtype=dtype, gate=gate, bias=bias, skip=not bias, seed=T)
            if not bias:
                case[1] = case[1] - 3
            _check(case, _call(case))
    case[1] = case[1].abs() / 16  # steps as they are
    case[7] = None
    _check(case, _call(case, softplus=False), softplus=False)


@pytest.mark.parametrize("S", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 24, 32, 33, 63, 64])
@pytest.mark.parametrize("T", [5, 70])
def test_states(S, T):
    case = _case(T=T, D=20, S=S, seed=S)
    _check(case, _call(case))


@pytest.mark.parametrize("D,G", [(1, 1), (3, 1), (6, 3), (15, 1), (16, 16), (17, 1), (63, 3), (64, 1), (65, 5), (200, 2)])
@pytest.mark.parametrize("T", [5, 70])
def test_channels_and_groups(D, G, T):
    case = _case(T=T, D=D, G=G, S=6, seed=D)
    _check(case, _call(case))


@pytest.mark.parametrize("lens", [[70], [0, 1, 64, 65], [5, 0, 0, 200, 63, 1], [0, 0], [1] * 40, [130, 128, 64, 0]])
def test_packed(lens):
    case = _case(T=sum(lens), D=20, N=len(lens), seed=len(lens))
    cu = torch.tensor([0] + lens).cumsum(0)
    for dt in (torch.int32, torch.int64):
        _check(case, _call(case, cu_seqlens=cu.to(DEV, dt)), lens=lens, packed=True)
    case[8] = None
    _check(case, _call(case, cu_seqlens=cu.to(DEV)), lens=lens, packed=True)


def test_many_packed_sequences():
    lens = [n % 5 for n in range(2500)]
    case = _case(T=sum(lens), D=4, S=3, N=len(lens), seed=3)
    cu = torch.tensor([0] + lens).cumsum(0).to(DEV, torch.int32)
    _check(case, _call(case, cu_seqlens=cu), lens=lens, packed=True)


def test_tokens_of_no_packed_sequence_are_zero():
    case = _case(T=400, D=16, N=2, seed=5)
    y, state = _call(case, cu_seqlens=torch.tensor([140, 150, 231], device=DEV))
    part = [t[:, 140:231] if t.dim() > 2 and t.shape[1] == 400 else t for t in case]
    _check(part, (y[:, 140:231], state), lens=[10, 81], packed=True)
    assert not y[:, :140].any() and not y[:, 231:].any()


def test_bounds_are_held_to_the_tokens():
    case = _case(T=160, D=16, N=5, seed=6)
    got = _call(case, cu_seqlens=torch.tensor([-7, 20, 10, 130, 25, 900], device=DEV))
    _check(case, got, lens=[20, 0, 110, 0, 30], packed=True)


@pytest.mark.parametrize("T", [1, 6, 150])
def test_counted_lengths(T):
    lens = [T, 0, 1, T - 1, T // 2]
    case = _case(B=5, T=T, seed=T)
    for t in (case[0], case[1], case[3], case[4], case[6]):
        for b, n in enumerate(lens):
            t[b, n:] = math.nan  # (not read into anything)
    y, state = _call(case, lengths=torch.tensor(lens, device=DEV))
    _check(case, (y, state), lens=lens)
    over = _call(case, lengths=torch.tensor([T + 5, -3, 1, T - 1, T // 2], device=DEV))
    assert torch.equal(over[0], y) and torch.equal(over[1], state)


@pytest.mark.parametrize("B,T,D", [(1, 1500, 16), (2, 2100, 40), (1, 700, 300), (9, 600, 20)])
def test_rows_in_pieces(B, T, D):
    """Few channels: rows are cut, and what a piece begins with comes from those before it."""
    case = _case(B=B, T=T, D=D, S=4, seed=T)
    case[7] = case[7] - 2  # (slow decays, so that states reach from piece to piece)
    _check(case, _call(case))
    want = _call(case)
    got = _call(case, inplace=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    case[8] = None
    _check(case, _call(case))
    lens = [T // (b + 1) for b in range(B)]
    _check(case, _call(case, lengths=torch.tensor(lens, device=DEV)), lens=lens)


@pytest.mark.parametrize("lens", [[1600], [30, 1500, 0, 70], [1] * 6 + [900], [64, 128, 500, 65]])
def test_packed_in_pieces(lens):
    case = _case(T=sum(lens), D=24, S=5, N=len(lens), seed=len(lens))
    case[7] = case[7] - 2
    cu = torch.tensor([0] + lens).cumsum(0).to(DEV, torch.int32)
    want = _call(case, cu_seqlens=cu)
    _check(case, want, lens=lens, packed=True)
    got = _call(case, cu_seqlens=cu, inplace=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("T", [2, 12, 140])
def test_steps_continue_a_state(T):
    case = _case(B=2, T=T, D=36, G=2, seed=9)
    d = [t.to(DEV) for t in case]
    cut = T // 2 + 1

    def part(lo, hi, state):
        return [t[:, lo:hi] if i in (0, 1, 3, 4, 6) else t for i, t in enumerate(d[:8])] + [state]
    a, state = _run(part(0, cut, d[8]))
    b, same = _run(part(cut, T, state), inplace=True)
    assert same is state
    _check(case, (torch.cat([a, b], 1), state))
    state = d[8].clone()
    rows = [_run(part(t, t + 1, state), inplace=True)[0] for t in range(T)]
    _check(case, (torch.cat(rows, 1), state))


@pytest.mark.parametrize("T", [3, 90])
def test_layouts(T):
    B, D, G, S = 2, 24, 2, 10
    case = [t.to(DEV) for t in _case(B=B, T=T, D=D, G=G, S=S, dtype="bf16")]
    want = _run(case)
    x, dt, A, Bm, Cm, skip, gate, bias, init = case
    fused = torch.cat([x[..., :1], x, dt, gate, Bm.flatten(2), Cm.flatten(2)], -1)  # one projection, at an odd start
    at = [1, 1 + D, 1 + 2 * D, 1 + 3 * D, 1 + 3 * D + G * S, 1 + 3 * D + 2 * G * S]
    x2, dt2, g2, b2, c2 = (fused[..., a:b] for a, b in zip(at, at[1:]))
    other = [x2, dt2, A.mT.contiguous().mT, b2.unflatten(-1, (G, S)), c2.unflatten(-1, (G, S)), skip, g2, bias,
             init.mT.contiguous().mT]
    back = [t.mT.contiguous().mT if t.dim() > 1 else t for t in case]
    half = [*case[:2], A, *case[3:8], init]
    for alike in (other, back, half):
        got = _run(alike)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # parameters and states in 16 bits are read as what they are
    low = [t.bfloat16() if i in (2, 5, 7, 8) else t for i, t in enumerate(case)]
    same = [t.float() if i in (2, 5, 7, 8) else t for i, t in enumerate(low)]
    assert torch.equal(_run(low)[0], _run(same)[0])


def test_past_32_bits():
    """Rows more than 2^31 elements apart."""
    case = _case(B=2, T=20, D=16, dtype="bf16")
    d = [t.to(DEV) for t in case]
    far = torch.empty(2 ** 31 + 1000, dtype=torch.bfloat16, device=DEV)
    d[0] = far.as_strided((2, 20, 16), (2 ** 31 + 8, 16, 1)).copy_(d[0])
    _check(case, _run(d))


@pytest.mark.parametrize("T", [6, 100])
def test_extreme_steps(T):
    """Steps from 0 to 1e4, decays from none to all of it; very negative and very large arguments of the softplus."""
    case = _case(T=T, D=12, S=5, seed=2)
    case[1][..., 0] = -80.0
    case[1][..., 1] = 80.0
    case[1][..., 2] = torch.where(torch.arange(T) % 2 == 0, 1e4, -1e4)
    case[1][..., 3] = -1e30
    case[2][:, 0] = 0.0
    case[2][:, 1] = -1e-6
    case[2][:, 2] = -1e30
    case[7] = None
    got, (y, state) = _call(case), _want(case)
    for c in range(12):  # each channel by itself: their sizes are far apart
        assert _rel(got[0][..., c], y[..., c]) <= _tol(torch.float32, T)
        assert _rel(got[1][:, c], state[:, c]) <= _tol(torch.float32, T)


@pytest.mark.parametrize("T", [6, 100])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_bad_value_stays_in_its_channel(T, bad):
    case = _case(T=T, D=20)
    good = _call(case)
    case[0][:, T // 2, 7] = bad
    y, state = _call(case)
    rest = [c for c in range(20) if c != 7]
    assert torch.equal(y[..., rest], good[0][..., rest]) and torch.equal(state[:, rest], good[1][:, rest])
    assert torch.equal(y[:, :T // 2, 7], good[0][:, :T // 2, 7]) and not y[:, T // 2, 7].isfinite().any()


@pytest.mark.parametrize("B,T,N", [(0, 5, 0), (2, 0, 2), (1, 0, 3), (1, 7, 0), (1, 70, 0)])
def test_empty(B, T, N):
    packed = B == 1
    case = _case(B=B, T=T, D=6, S=3, N=N)
    kw = dict(cu_seqlens=torch.zeros(N + 1, dtype=torch.int32, device=DEV)) if packed else {}
    y, state = _call(case, **kw)
    assert y.shape == (B, T, 6) and not y.any() and torch.equal(state.cpu(), case[8])
    leaves = [t.to(DEV).requires_grad_() for t in case]
    y, state = _run(leaves, **kw)
    grads = torch.autograd.grad([y, state], leaves, [torch.ones_like(y), torch.ones_like(state)])
    assert not any(g.any() for g in grads[:8]) and (grads[8] == 1).all()


# ---- the same bits whatever the way

@pytest.mark.parametrize("T", [8, 140])
def test_streams_compiled_and_registered(T):
    case = [t.to(DEV) for t in _case(B=2, T=T, dtype="bf16")]

    def f(*case):
        return _run(case)

    def g(*case):
        return _run([*case[:8], case[8].clone()], inplace=True)
    want = f(*case)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = f(*case)
    torch.cuda.current_stream().wait_stream(side)
    for other in (got, f(*case), g(*case), *(torch.compile(h, backend="aot_eager", fullgraph=True)(*case) for h in (f, g)),
                  torch.jit.trace(f, tuple(case), check_trace=False)(*case)):
        assert torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])
    ops = torch.ops.ramnet_ops
    for op in (ops.selective_scan, ops.selective_scan_):
        torch.library.opcheck(op, (*case, None, None, True), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(ops.selective_scan_kept, (*(t.float().requires_grad_() for t in case), None, None, True),
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))


@pytest.mark.parametrize("T", [1, 140, 1500])
def test_graph_replays(T):
    case = [t.to(DEV) for t in _case(B=2, T=T, dtype="bf16", seed=1)]
    state = case[8].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run([*case[:8], state], inplace=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = _run([*case[:8], state], inplace=True)
    state.copy_(case[8])
    want_state = case[8].clone()
    for step in range(3):
        for t, s in zip(case[:8], _case(B=2, T=T, dtype="bf16", seed=2 + step)):
            t.copy_(s)
        want, _ = _run([*case[:8], want_state], inplace=True)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(state, want_state)


@pytest.mark.parametrize("T", [1, 100])
def test_in_place_counts_as_changed(T):
    case = [t.to(DEV) for t in _case(T=T)]
    w = torch.ones_like(case[8], requires_grad=True)
    loss = (w * case[8]).sum()
    _run(case, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


# ---- gradients

def _grads(case, kw=None, lens=None, packed=False, use=(0, 1), softplus=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    got_in = [t.to(DEV).requires_grad_() if t is not None else None for t in case]
    want_in = [t.double().requires_grad_() if t is not None else None for t in case]
    got, want = _run(got_in, softplus=softplus, **(kw or {})), _want(want_in, lens=lens, packed=packed, softplus=softplus)
    d = [torch.randn(t.shape, generator=gen).to(t.dtype) for t in got]
    at = [i for i, t in enumerate(case) if t is not None]
    got = torch.autograd.grad([got[i] for i in use], [got_in[i] for i in at], [d[i].to(DEV) for i in use])
    want = torch.autograd.grad([want[i] for i in use], [want_in[i] for i in at], [d[i].double() for i in use],
                               materialize_grads=True)
    return [(NAMES[i], a, b, case[i]) for i, a, b in zip(at, got, want)]


def _check_grads(case, **kw):
    T = case[0].shape[0] * case[0].shape[1]
    for name, a, b, leaf in _grads(case, **kw):
        assert a.dtype == leaf.dtype and a.shape == leaf.shape, name
        assert _rel(a, b) <= _tol(a.dtype, T, 8), (name, _rel(a, b), _tol(a.dtype, T, 8))


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 100])
def test_gradients(T):
    _check_grads(_case(B=2, T=T, D=20, seed=T))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_gradients_types_and_parts(dtype):
    for gate in (False, True):
        for rest in (False, True):
            case = _case(T=50, D=24, dtype=dtype, gate=gate, bias=rest, skip=rest, state=rest)
            if not rest:
                case[1] = case[1] - 3
            _check_grads(case)
    case[1], case[7] = case[1].abs() / 16, None
    _check_grads(case, softplus=False)


@pytest.mark.parametrize("S", [1, 2, 3, 4, 5, 8, 9, 16, 17, 32, 33, 64])
def test_gradients_states(S):
    _check_grads(_case(T=40, D=20, S=S, seed=S))


@pytest.mark.parametrize("D,G", [(1, 1), (6, 3), (17, 1), (16, 16), (64, 1), (65, 5), (130, 2)])
def test_gradients_channels_and_groups(D, G):
    _check_grads(_case(T=40, D=D, G=G, S=6, seed=D))


@pytest.mark.parametrize("lens", [[70], [0, 1, 64, 65], [5, 0, 0, 200, 63, 1], [1] * 40, [1500, 30, 700]])
def test_gradients_packed(lens):
    case = _case(T=sum(lens), D=12, S=4, N=len(lens), seed=len(lens))
    case[7] = case[7] - 2
    cu = torch.tensor([0] + lens).cumsum(0).to(DEV)
    _check_grads(case, kw=dict(cu_seqlens=cu), lens=lens, packed=True)


@pytest.mark.parametrize("B,T,D", [(1, 1500, 16), (2, 700, 40)])
def test_gradients_rows_in_pieces(B, T, D):
    case = _case(B=B, T=T, D=D, S=4, seed=T)
    case[7] = case[7] - 2
    _check_grads(case)
    lens = [T // (b + 2) for b in range(B)]
    _check_grads(case, kw=dict(lengths=torch.tensor(lens, device=DEV)), lens=lens)


@pytest.mark.parametrize("T", [40, 700])
def test_gradients_of_tokens_that_do_not_count(T):
    lens = [T, 0, 1, T - 1, T // 2]
    case = _case(B=5, T=T, D=12, S=4)
    clean = [t.clone() for t in case]
    for i in (0, 1, 3, 4, 6):
        for b, n in enumerate(lens):
            case[i][b, n:] = math.nan
            clean[i][b, n:] = 0
    kw = dict(kw=dict(lengths=torch.tensor(lens, device=DEV)), lens=lens)
    for (name, a, _, _), (_, _, want, _) in zip(_grads(case, **kw), _grads(clean, **kw)):
        assert not a.isnan().any() and _rel(a, want) <= _tol(a.dtype, 5 * T, 8), name
        if name in ("x", "dt", "B", "C", "gate"):
            assert not any(a[b, n:].any() for b, n in enumerate(lens)), name
    case = _case(T=T, D=12, S=4, N=1)
    for name, a, _, _ in _grads(case, kw=dict(cu_seqlens=torch.tensor([10, 20], device=DEV)), lens=[10], packed=True):
        if name in ("x", "dt", "B", "C", "gate"):
            assert not a[:, :10].any() and not a[:, 20:].any() and a[:, 10:20].any(), name


@pytest.mark.parametrize("use", [(0,), (1,)])
def test_gradients_of_one_output(use):
    for name, a, b, _ in _grads(_case(T=70, D=12), use=use):
        assert _rel(a, b) <= _tol(a.dtype, 70, 8) if b.norm() > 0 else not a.any(), name


def test_gradients_extreme_steps():
    case = _case(T=60, D=12, S=5, seed=2)
    case[1][..., 0] = -80.0
    case[1][..., 1] = 80.0
    case[2][:, 0] = 0.0
    case[2][:, 1] = -1e-6
    case[2][:, 2] = -1e30
    case[7] = None
    for name, a, b, _ in _grads(case):
        assert a.isfinite().all(), name
        if name in ("x", "gate", "dt"):
            for c in range(12):
                assert _rel(a[..., c], b[..., c]) <= _tol(a.dtype, 60, 8), (name, c)


def test_gradients_against_differences():
    """Along one direction, central differences of the operator itself: with a step h the
    formula's error is O(h^2) and rounding adds about arith / h; h = 2^-7 leaves
    2^-14 + 2^7 8 sqrt(70) 2^-24 < 1e-3."""
    case = [t.to(DEV) for t in _case(T=70, D=24, S=6, seed=1)]
    x = [t.clone().requires_grad_() for t in case]
    y, state = _run(x)
    gen = torch.Generator().manual_seed(4)
    d = [torch.randn(t.shape, generator=gen).to(DEV) for t in (y, state)]
    grads = torch.autograd.grad([y, state], x, d)
    h = 2.0 ** -7
    for i, name in enumerate(NAMES):
        step = grads[i] / grads[i].norm()

        def along(sign):
            p = [t + (sign * h * step if j == i else 0) for j, t in enumerate(case)]
            a, b = _run(p)
            return float((a.double() * d[0]).sum() + (b.double() * d[1]).sum())
        want = (along(1) - along(-1)) / (2 * h)
        got = float((grads[i].double() * step).sum())
        assert abs(got - want) <= 1e-3 * abs(want), (name, got, want)


def test_gradients_compiled_strided_and_selected():
    case = [t.to(DEV) for t in _case(B=2, T=100, D=24, G=2)]

    def loss(*case):
        y, state = _run(case)
        return (y * y).sum() + state.sum()
    x = [t.clone().requires_grad_() for t in case]
    want = torch.autograd.grad(loss(*x), x)
    for other in (torch.autograd.grad(loss(*x), x), torch.autograd.grad(torch.compile(
            loss, backend="aot_eager", fullgraph=True)(*x), x)):
        assert all(torch.equal(a, b) for a, b in zip(other, want))
    x = [t.mT.contiguous().mT.requires_grad_() if t.dim() > 1 else t.clone().requires_grad_() for t in case]
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss(*x), x), want))
    x = [t.clone().requires_grad_(i == 2) for i, t in enumerate(case)]
    loss(*x).backward()
    assert torch.equal(x[2].grad, want[2]) and all(t.grad is None for i, t in enumerate(x) if i != 2)
    # B and C of one group for all: the sum of the groups' gradients
    one = [t[:, :, :1].clone().requires_grad_() for t in case[3:5]]
    wide = [t.detach().repeat(1, 1, 2, 1).requires_grad_() for t in one]
    shared = torch.autograd.grad(loss(*case[:3], *(t.expand(-1, -1, 2, -1) for t in one), *case[5:]), one)
    each = torch.autograd.grad(loss(*case[:3], *wide, *case[5:]), wide)
    assert all(torch.equal(a, b.sum(2, keepdim=True)) for a, b in zip(shared, each))


@pytest.mark.parametrize("T", [70, 1100])
def test_gradients_graph_replays(T):
    """A forward and its backward captured together, on leaves that no eager graph holds then."""
    def leaves(seed):
        return [t.to(DEV).requires_grad_() for t in _case(T=T, dtype="bf16", seed=seed)]

    def grads(x):
        y, state = _run(x)
        return torch.autograd.grad([y, state], x, [y.detach(), state.detach()])
    x = leaves(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads(x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = grads(x)
    for n in range(3):
        new = leaves(2 + n)
        with torch.no_grad():
            for t, s in zip(x, new):
                t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, grads(new)))


def test_gradients_beside_an_infinite_gate():
    """B and C are shared: an infinite gradient of one channel stays infinite over a block that has lanes to spare."""
    case = [t.to(DEV) for t in _case(T=1, D=20)]
    case[6][..., -1] = math.inf
    B, C = case[3].requires_grad_(), case[4].requires_grad_()
    y, _ = _run(case)
    dB, dC = torch.autograd.grad(y, (B, C), torch.ones_like(y))
    assert dB.isinf().all() and dC.isinf().all()


@pytest.mark.parametrize("G,S,T", [(64, 64, 5), (300, 3, 70)])
def test_gradients_many_groups(G, S, T):
    _check_grads(_case(B=2, T=T, D=G, G=G, S=S))


@pytest.mark.parametrize("T", [1, 3, 4, 5, 8])
@pytest.mark.parametrize("D,S,G", [(40, 16, 1), (36, 10, 3), (20, 64, 2), (7, 3, 1), (130, 48, 1), (24, 24, 2)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_steps_of_all_sizes(T, D, S, G, dtype):
    case = _case(B=3, T=T, D=D, S=S, G=G, dtype=dtype, seed=T)
    _check(case, _call(case))
    lens = [0, T, (T + 1) // 2]
    case[1][2, lens[2]:], case[4][2, lens[2]:], case[0][0] = math.nan, math.inf, math.nan  # none of them counts
    _check(case, _call(case, lengths=torch.tensor(lens, device=DEV)), lens=lens)


@pytest.mark.parametrize("B,T", [(4500, 1), (4200, 2)])
def test_steps_of_more_rows_than_blocks(B, T):
    """Blocks take several rows: each as one alone, also in place."""
    case = [t.to(DEV) for t in _case(B=B, T=T, D=8, S=16, seed=1)]
    lens = torch.arange(B, device=DEV) % (T + 1)
    y, state = _run(case, lengths=lens)
    for lo, hi in ((0, 3000), (3000, B)):
        part = [t[lo:hi] if i in (0, 1, 3, 4, 6, 8) else t for i, t in enumerate(case)]
        y_part, state_part = _run(part, lengths=lens[lo:hi])
        assert torch.equal(y[lo:hi], y_part) and torch.equal(state[lo:hi], state_part)
    own = case[8].clone()
    y_own, _ = _run(case[:8] + [own], lengths=lens, inplace=True)
    assert torch.equal(y_own, y) and torch.equal(own, state)
