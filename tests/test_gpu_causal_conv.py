"""The short causal convolution on the GPU against the fp64 oracle.

Tolerances are relative, in the 2-norm of an output:

* fp32 arithmetic: W + 1 sums, the sigmoid's argument, exponential, reciprocal and product; each off by
  2^-24 or (hardware functions) 2^-23 of a value no greater than the terms': 16 2^-24 for W <= 8.
* sums over T tokens: sqrt(T) 2^-24 each on top, rounded at random, times 4.
* outputs in 16 bits: half a step of the type (eps / 2) on top.
"""
from __future__ import annotations

import math

import pytest
import torch

from oracle import scan_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
NAMES = ("x", "weight", "bias", "init")


def _tol(dtype, terms=0):
    arith = (16 + 4 * math.sqrt(terms)) * 2.0 ** -24
    return arith if dtype == torch.float32 else torch.finfo(dtype).eps / 2 + arith


def _rel(got, want):
    want = want.double()
    norm = want.norm()
    off = (got.cpu().double() - want).norm()
    return float(off / norm) if norm > 0 else float(off)


def _case(B=1, T=37, D=40, W=4, dtype="fp32", N=None, bias=True, state=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]

    def rn(*s):
        return torch.randn(*s, generator=gen).to(dt)
    return [rn(B, T, D), rn(D, W), rn(D) if bias else None, rn(N if N is not None else B, W - 1, D) if state else None]


def _call(case, **kw):
    from ramnet_ops import causal_conv
    x, w, b, init = (t.to(DEV) if t is not None else None for t in case)
    return causal_conv(x, w, b, init_state=init, **kw)


def _check(case, got, lens=None, packed=False, silu=False):
    y, state = oracle.causal_conv(*case[:3], silu=silu, init_state=case[3], lens=lens, packed=packed)
    dtype = case[0].dtype
    assert got[0].dtype == got[1].dtype == dtype and got[0].shape == case[0].shape and got[1].shape == state.shape
    assert _rel(got[0], y) <= _tol(dtype), _rel(got[0], y)
    assert torch.equal(got[1].cpu().double(), state)


@pytest.mark.parametrize("W", range(1, 9))
@pytest.mark.parametrize("T", [1, 2, 7, 15, 16, 17, 50])
def test_widths_and_lengths(W, T):
    case = _case(B=2, T=T, W=W, seed=T)
    _check(case, _call(case))
    case[3] = None
    _check(case, _call(case, activation="silu"), silu=True)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("D", [1, 3, 4, 7, 8, 9, 31, 64, 517])
def test_channels_and_types(dtype, D):
    for bias in (False, True):
        case = _case(B=2, T=21, D=D, dtype=dtype, bias=bias, seed=D)
        _check(case, _call(case, activation="silu"), silu=True)


@pytest.mark.parametrize("lens", [[70], [0, 1, 2, 3, 4, 65], [5, 0, 0, 200, 63, 1], [0, 0], [1] * 40, [16, 32, 15, 17]])
@pytest.mark.parametrize("D", [8, 13])
def test_packed(lens, D):
    case = _case(T=sum(lens), D=D, N=len(lens), seed=len(lens))
    cu = torch.tensor([0] + lens).cumsum(0)
    for dt in (torch.int32, torch.int64):
        _check(case, _call(case, cu_seqlens=cu.to(DEV, dt)), lens, packed=True)


def test_many_packed_sequences():
    lens = [n % 5 for n in range(2500)]
    case = _case(T=sum(lens), D=9, N=len(lens), seed=3)
    cu = torch.tensor([0] + lens).cumsum(0).to(DEV, torch.int32)
    _check(case, _call(case, cu_seqlens=cu), lens, packed=True)


def test_tokens_of_no_packed_sequence_are_zero():
    case = _case(T=200, D=16, N=2, seed=5)
    y, state = _call(case, cu_seqlens=torch.tensor([40, 50, 131], device=DEV))
    part = [case[0][:, 40:131], *case[1:]]
    _check(part, (y[:, 40:131], state), [10, 81], packed=True)
    assert not y[:, :40].any() and not y[:, 131:].any()


def test_bounds_are_held_to_the_tokens():
    """Bounds out of order or out of range, as they are held: to the one before, and to [0, T]."""
    case = _case(T=60, D=16, N=5, seed=6)
    y, state = _call(case, cu_seqlens=torch.tensor([-7, 20, 10, 30, 25, 900], device=DEV))
    _check(case, (y, state), [20, 0, 10, 0, 30], packed=True)


@pytest.mark.parametrize("T", [1, 5, 40])
def test_counted_lengths(T):
    lens = [T, 0, 1, T - 1, T // 2]
    case = _case(B=5, T=T, seed=T)
    for b, n in enumerate(lens):
        case[0][b, n:] = math.nan  # (not read into anything)
    y, state = _call(case, lengths=torch.tensor(lens, device=DEV), activation="silu")
    _check(case, (y, state), lens, silu=True)
    over = _call(case[:1] + case[1:], lengths=torch.tensor([T + 5, -3, 1, T - 1, T // 2], device=DEV), activation="silu")
    assert torch.equal(over[0], y) and torch.equal(over[1], state)


@pytest.mark.parametrize("D", [3, 16, 21])
@pytest.mark.parametrize("cut", [0, 1, 2, 3, 39, 40])
def test_two_calls_in_place(cut, D):
    from ramnet_ops import causal_conv
    case = _case(B=3, T=40, D=D, seed=cut)
    x, w, b, init = (t.to(DEV) for t in case)
    state = init.clone()
    a, same = causal_conv(x[:, :cut], w, b, init_state=state, inplace=True)
    assert same is state
    c, _ = causal_conv(x[:, cut:], w, b, init_state=state, inplace=True)
    _check(case, (torch.cat([a, c], 1), state))
    whole = causal_conv(x, w, b, init_state=init)
    assert torch.equal(whole[0], torch.cat([a, c], 1)) and torch.equal(whole[1], state)


@pytest.mark.parametrize("lens", [[0, 1, 2, 3, 70], [200, 5]])
def test_packed_in_place(lens):
    case = _case(T=sum(lens), D=13, N=len(lens))
    cu = torch.tensor([0] + lens).cumsum(0).to(DEV)
    want, got = _call(case, cu_seqlens=cu), _call(case, cu_seqlens=cu, inplace=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_state_types():
    """A state of another type is rounded to x's."""
    case = _case(B=2, dtype="bf16")
    want = _call(case)
    case[3] = case[3].float()
    got = _call(case)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_layouts():
    case = [t.to(DEV) for t in _case(B=2, T=33, D=24, dtype="bf16")]
    from ramnet_ops import causal_conv
    want = causal_conv(*case[:3], init_state=case[3], activation="silu")
    x = case[0]
    wide = torch.randn(2, 33, 61, device=DEV).bfloat16()
    wide[..., 5:29] = x  # a slice of a projection, at an odd start
    others = [wide[..., 5:29], x.transpose(0, 1).contiguous().transpose(0, 1), x.mT.contiguous().mT,
              torch.repeat_interleave(x, 2, -1)[..., ::2]]
    for other in others:
        got = causal_conv(other, case[1].mT.contiguous().mT, case[2], activation="silu",
                          init_state=case[3].transpose(0, 1).contiguous().transpose(0, 1))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    rows = x[:1].expand(3, -1, -1)
    got = causal_conv(rows, *case[1:3], activation="silu")
    one = causal_conv(x[:1], *case[1:3], activation="silu")
    assert torch.equal(got[0], one[0].expand(3, -1, -1))


def test_past_32_bits():
    """Rows more than 2^31 elements apart."""
    case = _case(B=2, T=20, D=16, dtype="bf16")
    far = torch.empty(2 ** 31 + 1000, dtype=torch.bfloat16, device=DEV)
    x = far.as_strided((2, 20, 16), (2 ** 31 + 8, 16, 1))
    x.copy_(case[0])
    from ramnet_ops import causal_conv
    _check(case, causal_conv(x, *(t.to(DEV) for t in case[1:3]), init_state=case[3].to(DEV)))


def test_extremes():
    case = _case(B=1, T=64, D=16)
    case[0][:, ::3] *= 1e30
    case[0][:, 1::3] *= 1e-30
    _check(case, _call(case))
    big = [torch.tensor([-3e38, -200.0, -100.0, 0.0, 100.0, 3e38]).view(1, 6, 1), torch.ones(1, 1), None, None]
    y = _call(big, activation="silu")[0].cpu().flatten()
    assert torch.equal(y[3:], big[0].flatten()[3:]) and (y[:3].abs() <= 1e-40).all()


@pytest.mark.parametrize("B,T,N", [(0, 5, 0), (2, 0, 2), (1, 0, 3), (1, 7, 0)])
def test_empty(B, T, N):
    packed = B == 1
    case = _case(B=B, T=T, D=6, N=N)
    kw = dict(cu_seqlens=torch.zeros(N + 1, dtype=torch.int32, device=DEV)) if packed else {}
    y, state = _call(case, **kw)
    assert y.shape == (B, T, 6) and not y.any() and torch.equal(state.cpu(), case[3])
    from ramnet_ops import causal_conv
    leaves = [t.to(DEV).requires_grad_() for t in case]
    y, state = causal_conv(*leaves[:3], init_state=leaves[3], **kw)
    grads = torch.autograd.grad([y, state], leaves, [torch.ones_like(y), torch.ones_like(state)])
    assert not any(g.any() for g in grads[:3]) and (grads[3] == 1).all()


# ---- the same bits whatever the way

def test_streams_compiled_and_registered():
    from ramnet_ops import causal_conv
    case = [t.to(DEV) for t in _case(B=2, T=70, dtype="bf16")]

    def f(x, w, b, init):
        return causal_conv(x, w, b, activation="silu", init_state=init)

    def g(x, w, b, init):
        init = init.clone()
        return causal_conv(x, w, b, activation="silu", init_state=init, inplace=True)
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
    torch.library.opcheck(ops.causal_conv_, (*case, None, None, True), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(ops.causal_conv, (*(t.float().requires_grad_() for t in case), None, None, True),
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))


@pytest.mark.parametrize("T", [1, 40])
def test_graph_replays(T):
    from ramnet_ops import causal_conv
    case = [t.to(DEV) for t in _case(B=2, T=T, D=21, dtype="bf16", seed=1)]
    state = case[3].clone()

    def step(x, state):
        return causal_conv(x, *case[1:3], init_state=state, inplace=True)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(case[0], state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(case[0], state)
    state.copy_(case[3])
    want_state = case[3].clone()
    for n in range(3):
        case[0].copy_(_case(B=2, T=T, D=21, dtype="bf16", seed=2 + n)[0])
        want = step(case[0], want_state)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(state, want_state)


def test_in_place_counts_as_changed():
    from ramnet_ops import causal_conv
    case = [t.to(DEV) for t in _case()]
    w = torch.ones_like(case[3], requires_grad=True)
    loss = (w * case[3]).sum()
    causal_conv(*case[:3], init_state=case[3], inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


# ---- gradients

def _grads(case, kw=None, lens=None, packed=False, silu=False, use=(0, 1), seed=0):
    from ramnet_ops import causal_conv
    gen = torch.Generator().manual_seed(seed)
    got_in = [t.to(DEV).requires_grad_() if t is not None else None for t in case]
    want_in = [t.double().requires_grad_() if t is not None else None for t in case]
    got = causal_conv(*got_in[:3], init_state=got_in[3], activation="silu" if silu else None, **(kw or {}))
    want = oracle.causal_conv(*want_in[:3], silu=silu, init_state=want_in[3], lens=lens, packed=packed)
    d = [torch.randn(t.shape, generator=gen).to(t.dtype) for t in got]
    at = [i for i, t in enumerate(case) if t is not None]
    got = torch.autograd.grad([got[i] for i in use], [got_in[i] for i in at], [d[i].to(DEV) for i in use])
    want = torch.autograd.grad([want[i] for i in use], [want_in[i] for i in at], [d[i].double() for i in use],
                               materialize_grads=True)
    return [(NAMES[i], a, b, case[i]) for i, a, b in zip(at, got, want)]


def _check_grads(case, **kw):
    tokens = case[0].shape[0] * case[0].shape[1]
    for name, a, b, leaf in _grads(case, **kw):
        assert a.dtype == leaf.dtype and a.shape == leaf.shape, name
        tol = _tol(a.dtype, tokens if name in ("weight", "bias") else 0)
        assert _rel(a, b) <= tol, (name, _rel(a, b), tol)


@pytest.mark.parametrize("W", range(1, 9))
@pytest.mark.parametrize("T", [1, 3, 16, 17, 50])
def test_gradients(W, T):
    case = _case(B=2, T=T, W=W, D=12, seed=T)
    _check_grads(case, silu=W % 2 == 0)
    case[2] = case[3] = None
    _check_grads(case, silu=True)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("D", [1, 4, 7, 8, 9, 31, 130])
def test_gradients_channels_and_types(dtype, D):
    _check_grads(_case(B=2, T=70, D=D, dtype=dtype, seed=D), silu=True)


@pytest.mark.parametrize("lens", [[70], [0, 1, 2, 3, 4, 65], [5, 0, 0, 200, 63, 1], [1] * 40, [16, 32, 15, 17]])
def test_gradients_packed(lens):
    case = _case(T=sum(lens), D=13, N=len(lens), seed=len(lens))
    cu = torch.tensor([0] + lens).cumsum(0).to(DEV)
    _check_grads(case, kw=dict(cu_seqlens=cu), lens=lens, packed=True, silu=True)


def test_gradients_of_tokens_that_do_not_count():
    lens = [40, 0, 1, 39, 20]
    case = _case(B=5, T=40, D=12)
    for b, n in enumerate(lens):
        case[0][b, n:] = math.nan
    rows = _grads(case, kw=dict(lengths=torch.tensor(lens, device=DEV)), lens=lens, silu=True)
    for name, a, b, _ in rows:
        assert not a.isnan().any() and _rel(a, b.nan_to_num(0.0)) <= _tol(a.dtype, 200), name
    case = _case(T=60, D=12, N=1)
    (_, dx, _, _), *_ = _grads([case[0][:, :30], *case[1:]], kw=dict(cu_seqlens=torch.tensor([10, 20], device=DEV)), lens=[10],
                               packed=True)
    assert not dx[:, :10].any() and not dx[:, 20:].any() and dx[:, 10:20].all()


@pytest.mark.parametrize("use", [(0,), (1,)])
def test_gradients_of_one_output(use):
    for name, a, b, _ in _grads(_case(T=20, D=12), use=use, silu=True):
        assert _rel(a, b) <= _tol(a.dtype, 20), name


def test_gradients_large():
    """Pieces of every length that the backward takes; sums over all of them."""
    for B, T, D in ((2, 5000, 64), (1, 70000, 264), (4, 40001, 512)):
        gen = torch.Generator(device=DEV).manual_seed(T)
        x = torch.randn(B, T, D, generator=gen, device=DEV).bfloat16().requires_grad_()
        w = torch.randn(D, 4, generator=gen, device=DEV).bfloat16().requires_grad_()
        b = torch.randn(D, generator=gen, device=DEV).bfloat16().requires_grad_()
        d = torch.randn(B, T, D, generator=gen, device=DEV).bfloat16()
        from ramnet_ops import causal_conv
        got = torch.autograd.grad(causal_conv(x, w, b)[0], (x, w, b), d)
        line = torch.nn.functional.pad(x.detach().double(), (0, 0, 3, 0))
        want = [sum(torch.nn.functional.pad(d.double(), (0, 0, 0, 3))[:, 3 - j:T + 3 - j] * w.detach().double()[:, j]
                    for j in range(4)),
                torch.stack([(line[:, j:j + T] * d.double()).sum((0, 1)) for j in range(4)], -1), d.double().sum((0, 1))]
        for a, c in zip(got, want):
            assert _rel(a, c.cpu()) <= _tol(torch.bfloat16, B * T)
        again = torch.autograd.grad(causal_conv(x, w, b)[0], (x, w, b), d)
        assert all(torch.equal(a, c) for a, c in zip(got, again))


def test_gradients_against_differences():
    """The operator is linear in x, weight, bias and the state (no activation): a difference over a step has no
    error of the formula's, and rounding adds about 2^-20 over a step of 1; with silu a step of 2^-7 leaves the
    formula 2^-14 and rounding 2^-13."""
    from ramnet_ops import causal_conv
    for act, h, tol in ((None, 1.0, 1e-4), ("silu", 2.0 ** -7, 1e-3)):
        case = [t.to(DEV) for t in _case(T=40, D=16)]
        x = [t.clone().requires_grad_() for t in case]
        y, state = causal_conv(*x[:3], init_state=x[3], activation=act)
        d = [torch.randn(t.shape, generator=torch.Generator().manual_seed(4)).to(DEV) for t in (y, state)]
        grads = torch.autograd.grad([y, state], x, d)
        for i in range(4):
            step = grads[i] / grads[i].norm()

            def along(sign):
                p = [t + (sign * h * step if j == i else 0) for j, t in enumerate(case)]
                a, b = causal_conv(*p[:3], init_state=p[3], activation=act)
                return float((a.double() * d[0]).sum() + (b.double() * d[1]).sum())
            want = (along(1) - along(-1)) / (2 * h)
            got = float((grads[i].double() * step).sum())
            assert abs(got - want) <= tol * abs(want), (act, NAMES[i], got, want)


def test_gradients_compiled_strided_and_selected():
    from ramnet_ops import causal_conv
    case = [t.to(DEV) for t in _case(B=2, T=50, D=24)]

    def loss(x, w, b, init):
        y, state = causal_conv(x, w, b, activation="silu", init_state=init)
        return (y * y).sum() + state.sum()
    x = [t.clone().requires_grad_() for t in case]
    want = torch.autograd.grad(loss(*x), x)
    got = torch.autograd.grad(torch.compile(loss, backend="aot_eager", fullgraph=True)(*x), x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = [t.mT.contiguous().mT.requires_grad_() if t.dim() > 1 else t.clone().requires_grad_() for t in case]
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss(*x), x), want))
    x = [t.clone().requires_grad_(i == 1) for i, t in enumerate(case)]
    loss(*x).backward()
    assert torch.equal(x[1].grad, want[1]) and all(x[i].grad is None for i in (0, 2, 3))
    # one row for all: its gradient is the sum
    row = case[0][:1].clone().requires_grad_()
    shared = torch.autograd.grad(loss(row.expand(2, -1, -1), *case[1:]), row)[0]
    each = case[0][:1].repeat(2, 1, 1).requires_grad_()
    assert torch.equal(shared, torch.autograd.grad(loss(each, *case[1:]), each)[0].sum(0, keepdim=True))


def test_gradients_graph_replays():
    from ramnet_ops import causal_conv

    def leaves(seed):
        return [t.to(DEV).requires_grad_() for t in _case(B=2, T=50, D=21, dtype="bf16", seed=seed)]

    def grads(x):
        y, state = causal_conv(*x[:3], init_state=x[3], activation="silu")
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
