"""The gated delta rule on the GPU against the fp64 oracle: values, states,
gradients, shapes where a chunk, a tile or a slice ends, masks and extremes.

Tolerances are relative, in the 2-norm of an output:

* fp32 arithmetic: dot products over at most max(Dk, 64) terms, rounded at
  random, sqrt(terms) 2^-24 each; a value passes through fewer than 8 of them
  before the contraction by unit keys takes over:
  8 sqrt(max(Dk, 64)) 2^-24.
* outputs in 16 bits: half a step of the type (eps / 2) on top, and two
  operands rounded to fp16 (2^-11 each) on the way.
* a decay's gradient sums terms that cancel: 8 times the arithmetic's.
"""
from __future__ import annotations

import math

import pytest
import torch

from oracle import delta_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _arith(Dk):
    return 8 * math.sqrt(max(Dk, 64)) * 2.0 ** -24


def _tol(t, Dk):
    if t.dtype == torch.float32:
        return _arith(Dk)
    return torch.finfo(t.dtype).eps / 2 + 2 * 2.0 ** -11 + _arith(Dk)


def _case(B=1, T=65, Hk=1, Hv=1, Dk=64, Dv=64, dtype="fp32", g_dtype=None, N=None, seed=0, state=True, g_scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]

    def rn(*s):
        return torch.randn(*s, generator=gen)
    q = torch.nn.functional.normalize(rn(B, T, Hk, Dk), dim=-1).to(dt)
    k = torch.nn.functional.normalize(rn(B, T, Hk, Dk), dim=-1).to(dt)
    v = rn(B, T, Hv, Dv).to(dt)
    g = (-g_scale * rn(B, T, Hv).abs() * torch.rand(Hv, generator=gen)).to(DTYPES[g_dtype] if g_dtype else torch.float32)
    beta = torch.sigmoid(rn(B, T, Hv)).to(dt)
    init = 0.5 * rn(N if N is not None else B, Hv, Dk, Dv) if state else None
    return [q, k, v, g, beta, init]


def _rel(got, want):
    want = want.double()
    norm = want.norm()
    off = (got.cpu().double() - want).norm()
    return float(off / norm) if norm > 0 else float(off)


def _call(case, **kw):
    from ramnet_ops import gated_delta_rule
    q, k, v, g, beta, init = (t.to(DEV) if t is not None else None for t in case)
    return gated_delta_rule(q, k, v, g, beta, init_state=init, **kw)


def _check(case, got, lens=None, packed=False, scale=None):
    Dk = case[0].shape[-1]
    o, state = oracle.delta_rule(*case[:5], scale=scale, init_state=case[5], lens=lens, packed=packed)
    assert got[0].dtype == case[2].dtype and got[0].shape == case[2].shape
    assert got[1].dtype == torch.float32 and got[1].shape == state.shape
    assert _rel(got[0], o) <= _tol(got[0], Dk), ("o", _rel(got[0], o), _tol(got[0], Dk))
    assert _rel(got[1], state) <= _arith(Dk), ("state", _rel(got[1], state), _arith(Dk))
    return o, state


# ---- values

@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 63, 64, 65, 128, 130, 257])
def test_lengths(T):
    case = _case(B=2, T=T, Hk=2, Hv=2, seed=T)
    _check(case, _call(case))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("T", [3, 150])
def test_types(dtype, T):
    for g_dtype in (None, dtype):
        case = _case(T=T, Hk=1, Hv=2, Dk=128, Dv=128, dtype=dtype, g_dtype=g_dtype, seed=T)
        _check(case, _call(case))


@pytest.mark.parametrize("Dk,Dv", [(1, 1), (5, 3), (20, 33), (37, 64), (64, 37), (72, 96), (96, 16), (128, 200),
                                   (160, 256), (161, 17), (200, 40), (256, 64)])
@pytest.mark.parametrize("T", [5, 100])
def test_head_sizes(Dk, Dv, T):
    case = _case(T=T, Hk=1, Hv=2, Dk=Dk, Dv=Dv, seed=Dk + Dv)
    _check(case, _call(case))


@pytest.mark.parametrize("Hk,Hv", [(1, 3), (3, 6), (4, 4)])
@pytest.mark.parametrize("T", [4, 70])
def test_shared_key_heads(Hk, Hv, T):
    case = _case(T=T, Hk=Hk, Hv=Hv, Dk=32, Dv=48, dtype="bf16", seed=Hv)
    _check(case, _call(case))


@pytest.mark.parametrize("lens", [[70], [0, 1, 64, 65], [5, 0, 0, 200, 63, 1], [0, 0], [1] * 40, [130, 128, 64, 0]])
def test_packed(lens):
    T = sum(lens)
    case = _case(T=T, Hk=1, Hv=2, Dk=48, Dv=40, N=len(lens), seed=len(lens))
    cu = torch.tensor([0] + lens).cumsum(0)
    for dt in (torch.int32, torch.int64):
        _check(case, _call(case, cu_seqlens=cu.to(DEV, dt)), lens, packed=True)


def test_many_packed_sequences():
    lens = [n % 5 for n in range(1500)]
    case = _case(T=sum(lens), Dk=16, Dv=16, N=len(lens), seed=3)
    cu = torch.tensor([0] + lens).cumsum(0).to(DEV, torch.int32)
    _check(case, _call(case, cu_seqlens=cu), lens, packed=True)


@pytest.mark.parametrize("T", [20, 100])
def test_tokens_of_no_packed_sequence_are_zero(T):
    case = _case(T=T, Dk=16, Dv=16, N=2, seed=T)
    a, b, c = 3, T // 2, T - 7
    cu = torch.tensor([a, b, c], dtype=torch.int32, device=DEV)
    o, state = _call(case, cu_seqlens=cu)
    part = [t[:, a:c] for t in case[:5]] + [case[5]]
    _check(part, (o[:, a:c].contiguous(), state), [b - a, c - b], packed=True)
    assert o[:, :a].abs().max() == 0 and o[:, c:].abs().max() == 0


@pytest.mark.parametrize("T", [6, 150])
def test_counted_lengths(T):
    lens = [T, 0, 1, T - 1, T // 2]
    case = _case(B=5, T=T, Hk=1, Hv=2, Dk=32, Dv=32, seed=T)
    got = _call(case, lengths=torch.tensor(lens, device=DEV))
    _check(case, got, lens)
    for b, n in enumerate(lens):
        assert (got[0][b, n:] == 0).all()
    assert torch.equal(got[1][1].cpu(), case[5][1])  # no tokens: the state as it was


@pytest.mark.parametrize("T,Dk,Dv,dtype", [(1024, 16, 16, "fp32"), (1100, 40, 24, "fp32"), (2049, 128, 100, "bf16"),
                                           (1600, 200, 72, "fp16")])
def test_long_rows(T, Dk, Dv, dtype):
    """Rows long enough to be cut into segments that run side by side."""
    _check(_case(T=T, Hk=1, Hv=2, Dk=Dk, Dv=Dv, dtype=dtype, seed=T), _call(_case(T=T, Hk=1, Hv=2, Dk=Dk, Dv=Dv,
                                                                                 dtype=dtype, seed=T)))


def test_long_rows_counted_lengths():
    T, lens = 1500, [1500, 0, 1, 512, 700]
    case = _case(B=5, T=T, Hk=1, Hv=1, Dk=24, Dv=40, seed=2)
    got = _call(case, lengths=torch.tensor(lens, device=DEV))
    _check(case, got, lens)
    for b, n in enumerate(lens):
        assert (got[0][b, n:] == 0).all()
    case[5] = None
    _check(case, _call(case, lengths=torch.tensor(lens, device=DEV)), lens)


def test_long_rows_gradients():
    _check_grads(_case(T=1100, Hk=1, Hv=2, Dk=24, Dv=40, seed=3))


@pytest.mark.parametrize("T", [4, 129])
def test_steps_continue_a_state(T):
    """A prompt in two calls, the second in place, is the prompt in one."""
    case = _case(B=2, T=T, Hk=2, Hv=2, Dk=32, Dv=36, seed=9)
    from ramnet_ops import gated_delta_rule
    d = [t.to(DEV) for t in case]
    cut = T // 2 + 1
    o1, state = gated_delta_rule(*(t[:, :cut] for t in d[:5]), init_state=d[5])
    given = state
    o2, state = gated_delta_rule(*(t[:, cut:] for t in d[:5]), init_state=state, inplace=True)
    assert state is given
    _check(case, (torch.cat([o1, o2], 1), state))


@pytest.mark.parametrize("T", [3, 90])
def test_strided_inputs_and_scale(T):
    B, Hk, Hv, Dk, Dv = 2, 2, 4, 24, 20
    case = _case(B=B, T=T, Hk=Hk, Hv=Hv, Dk=Dk, Dv=Dv, dtype="bf16", g_dtype="bf16", seed=T)
    q, k, v, g, beta, init = (t.to(DEV) for t in case)
    # one projection's slices, heads first, and a gate laid out by head
    fused = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2), g, beta], -1)
    at = [0]
    for n in (Hk * Dk, Hk * Dk, Hv * Dv, Hv, Hv):
        at.append(at[-1] + n)
    q2, k2, v2, g2, b2 = (fused[..., a:b] for a, b in zip(at, at[1:]))
    from ramnet_ops import gated_delta_rule
    got = gated_delta_rule(q2.unflatten(-1, (Hk, Dk)), k2.unflatten(-1, (Hk, Dk)), v2.unflatten(-1, (Hv, Dv)), g2, b2,
                           scale=0.7, init_state=init)
    _check(case, got, scale=0.7)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, g, beta)]
    again = gated_delta_rule(*heads_first, scale=0.7, init_state=init.transpose(2, 3).contiguous().transpose(2, 3))
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])
    # a last dimension with gaps
    gaps = torch.repeat_interleave(q, 2, -1)[..., ::2]
    again = gated_delta_rule(gaps, k, v, g, beta, scale=0.7, init_state=init)
    assert torch.equal(again[0], got[0])


@pytest.mark.parametrize("T", [8, 140])
def test_extreme_decays(T):
    """Decays that underflow within a step, resets (-inf), none at all, and
    strong ones next to weak ones, whose differences would lose their digits in
    a 32-bit running sum."""
    case = _case(T=T, Hk=1, Hv=4, Dk=32, Dv=32, seed=11)
    g = case[3]
    g[..., 0] = 0
    g[..., 1] = torch.where(torch.arange(T) % 3 == 1, -math.inf, -0.01)
    g[..., 2] = torch.where(torch.arange(T) % 2 == 0, -90.0, -1e-3)
    g[..., 3] = -2000.0
    got = _call(case)
    _check(case, got)
    for h in range(4):
        o, state = oracle.delta_rule(*case[:5], init_state=case[5])
        assert _rel(got[0][:, :, h], o[:, :, h]) <= _tol(got[0], 32)
        assert _rel(got[1][:, h], state[:, h]) <= _arith(32)


@pytest.mark.parametrize("T", [8, 140])
@pytest.mark.parametrize("scale", [1e-18, 1e-6, 1e6, 1e18])
def test_magnitudes(T, scale):
    """Values, states and queries of any size: nothing overflows or is lost on the way."""
    for dtype in ("fp32", "bf16"):
        case = _case(T=T, Hk=1, Hv=2, Dk=40, Dv=48, dtype=dtype, seed=5)
        case[2] = (case[2].float() * scale).to(case[2].dtype)
        case[5] = case[5] * scale
        case[0] = (case[0].float() / scale).to(case[0].dtype)
        _check(case, _call(case))


@pytest.mark.parametrize("T", [8, 140])
def test_small_keys(T):
    """Keys far below norm 1 (and one head of zeros) with values to match."""
    case = _case(T=T, Hk=2, Hv=2, Dk=40, Dv=48, dtype="bf16", seed=6)
    case[1] = (case[1].float() * 1e-6).to(torch.bfloat16)
    case[1][:, :, 1] = 0
    case[2] = (case[2].float() * 1e5).to(torch.bfloat16)
    case[5] = case[5] * 0.1
    _check(case, _call(case))


@pytest.mark.parametrize("T", [8, 140])
def test_columns_do_not_meet(T):
    """A column of huge values and one of zeros beside ordinary ones."""
    case = _case(T=T, Dk=32, Dv=32, seed=7)
    case[2][..., 3] *= 1e12
    case[2][..., 4] = 0
    case[5][..., 4] = 0
    o, state = _call(case)
    _check(case, (o, state))
    want, after = oracle.delta_rule(*case[:5], init_state=case[5])
    for c in (0, 3, 5, 31):
        assert _rel(o[..., c], want[..., c]) <= _tol(o, 32) and _rel(state[..., c], after[..., c]) <= _arith(32)
    assert (o[..., 4] == 0).all() and (state[..., 4] == 0).all()


@pytest.mark.parametrize("T", [8, 140])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_bad_value_stays_in_its_column(T, bad):
    case = _case(T=T, Hk=2, Hv=2, Dk=32, Dv=32, seed=8)
    case[2][0, T // 2, 1, 5] = bad
    o, state = _call(case)
    want, _ = oracle.delta_rule(*case[:5], init_state=case[5])
    clean = torch.ones(2, 32, dtype=torch.bool)
    clean[1, 5] = False
    assert torch.isfinite(o.cpu()[:, :, clean]).all() and torch.isfinite(state.cpu().transpose(2, 3)[:, clean]).all()
    assert _rel(o[:, :, clean], want[:, :, clean]) <= _tol(o, 32)
    assert torch.isfinite(o[:, :T // 2, 1, 5]).all() or T > 32  # (a chunk's tokens share products)
    assert not torch.isfinite(o[:, T // 2, 1, 5]).any() and not torch.isfinite(state[0, 1, :, 5]).all()


def test_empty():
    from ramnet_ops import gated_delta_rule
    for B, T in ((0, 5), (2, 0)):
        case = [t.to(DEV) for t in _case(B=B, T=T, Dk=8, Dv=8)]
        o, state = gated_delta_rule(*case[:5], init_state=case[5])
        assert o.shape == (B, T, 1, 8) and torch.equal(state, case[5])
    case = [t.to(DEV) for t in _case(B=1, T=4, Dk=8, Dv=8, N=0)]
    o, state = gated_delta_rule(*case[:5], init_state=case[5], cu_seqlens=torch.zeros(1, dtype=torch.int32, device=DEV))
    assert (o == 0).all() and state.shape == (0, 1, 8, 8)


# ---- the same bits whatever the way

@pytest.mark.parametrize("T", [8, 140])
def test_same_bits_again_on_another_stream_and_compiled(T):
    from ramnet_ops import gated_delta_rule
    case = [t.to(DEV) for t in _case(B=2, T=T, Hk=1, Hv=2, Dk=40, Dv=32, dtype="bf16")]

    def f(q, k, v, g, beta, init):
        return gated_delta_rule(q, k, v, g, beta, init_state=init)
    want = f(*case)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = f(*case)
    torch.cuda.current_stream().wait_stream(side)
    for other in (got, f(*case), torch.compile(f, backend="aot_eager", fullgraph=True)(*case)):
        assert torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])


@pytest.mark.parametrize("T", [1, 140])
def test_graph_replays(T):
    from ramnet_ops import gated_delta_rule
    case = [t.to(DEV) for t in _case(B=2, T=T, Hk=1, Hv=2, Dk=40, Dv=32, dtype="bf16", seed=1)]
    state = case[5].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gated_delta_rule(*case[:5], init_state=state, inplace=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, _ = gated_delta_rule(*case[:5], init_state=state, inplace=True)
    state.copy_(case[5])
    want_state = case[5].clone()
    for step in range(3):
        for t, s in zip(case[:5], _case(B=2, T=T, Hk=1, Hv=2, Dk=40, Dv=32, dtype="bf16", seed=2 + step)):
            t.copy_(s)
        want, _ = gated_delta_rule(*case[:5], init_state=want_state, inplace=True)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(state, want_state)


def test_registrations():
    ops = torch.ops.ramnet_ops
    import ramnet_ops  # noqa: F401
    checks = ("test_schema", "test_autograd_registration", "test_faketensor")
    case = [t.to(DEV) for t in _case(B=2, T=70, Hk=1, Hv=2, Dk=16, Dv=24)]
    for t in (70, 5):
        part = [x[:, :t].contiguous() for x in case[:5]]
        for op in (ops.gated_delta_rule, ops.gated_delta_rule_):
            torch.library.opcheck(op, (*part, case[5], None, None, 0.3), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(ops.gated_delta_rule_kept, (*(x.requires_grad_() for x in case[:5]), case[5].requires_grad_(),
                                                      None, None, 0.3), test_utils=checks)


# ---- gradients

NAMES = ("q", "k", "v", "g", "beta", "init")


def _grads(case, seed=0, kw=None, lens=None, packed=False, use=(True, True)):
    """(got, want): gradients of random combinations of o and the state."""
    from ramnet_ops import gated_delta_rule
    gen = torch.Generator().manual_seed(seed)
    have = [n for n, t in zip(NAMES, case) if t is not None]
    got_in = [t.to(DEV).requires_grad_() for t in case if t is not None]
    got = gated_delta_rule(*got_in[:5], init_state=got_in[5] if len(got_in) > 5 else None, **(kw or {}))
    want_in = [t.double().requires_grad_() for t in case if t is not None]
    want = oracle.delta_rule(*want_in[:5], init_state=want_in[5] if len(want_in) > 5 else None, lens=lens, packed=packed)
    d = [torch.randn(t.shape, generator=gen).to(t.dtype) for t in got]
    pick = [i for i in (0, 1) if use[i]]
    ga = torch.autograd.grad([got[i] for i in pick], got_in, [d[i].to(DEV) for i in pick])
    wa = torch.autograd.grad([want[i] for i in pick], want_in, [d[i].double() for i in pick], materialize_grads=True)
    return have, ga, wa, got_in


def _check_grads(case, **kw):
    Dk = case[0].shape[-1]
    have, got, want, leaves = _grads(case, **kw)
    for n, a, b, x in zip(have, got, want, leaves):
        assert a.dtype == x.dtype and a.shape == x.shape, n
        tol = _tol(a, Dk) + (7 * _arith(Dk) if n == "g" else 0)
        assert _rel(a, b) <= tol, (n, _rel(a, b), tol)


@pytest.mark.parametrize("T", [1, 2, 40, 64, 65, 200])
def test_gradients(T):
    _check_grads(_case(B=2, T=T, Hk=2, Hv=2, Dk=64, Dv=48, seed=T))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_gradients_types(dtype):
    for g_dtype in (None, dtype):
        _check_grads(_case(T=130, Hk=1, Hv=2, Dk=128, Dv=128, dtype=dtype, g_dtype=g_dtype))


@pytest.mark.parametrize("Dk,Dv", [(1, 1), (5, 3), (37, 64), (64, 37), (72, 96), (128, 200), (160, 40)])
def test_gradients_head_sizes(Dk, Dv):
    _check_grads(_case(T=70, Hk=1, Hv=2, Dk=Dk, Dv=Dv, seed=Dk))


@pytest.mark.parametrize("Dk,Dv", [(200, 40), (256, 130)])
def test_gradients_widest_heads(Dk, Dv):
    _check_grads(_case(T=70, Hk=1, Hv=2, Dk=Dk, Dv=Dv, dtype="fp16", seed=Dk))
    from ramnet_ops import gated_delta_rule
    case = [t.to(DEV).requires_grad_() for t in _case(T=70, Dk=Dk, Dv=Dv)]
    with pytest.raises(RuntimeError, match="up to 160 for gradients of float32"):
        gated_delta_rule(*case[:5], init_state=case[5])


@pytest.mark.parametrize("Hk,Hv", [(1, 3), (2, 4)])
def test_gradients_shared_key_heads(Hk, Hv):
    _check_grads(_case(T=70, Hk=Hk, Hv=Hv, Dk=32, Dv=48, state=False, seed=Hv))


@pytest.mark.parametrize("lens", [[70], [0, 1, 64, 65], [5, 0, 0, 100, 63, 1]])
def test_gradients_packed(lens):
    case = _case(T=sum(lens), Hk=1, Hv=2, Dk=48, Dv=40, N=len(lens), seed=len(lens))
    cu = torch.tensor([0] + lens).cumsum(0).to(DEV, torch.int32)
    _check_grads(case, kw=dict(cu_seqlens=cu), lens=lens, packed=True)


def test_gradients_counted_lengths():
    lens = [100, 0, 1, 64, 70]
    case = _case(B=5, T=100, Hk=1, Hv=2, Dk=32, Dv=32)
    kw = dict(kw=dict(lengths=torch.tensor(lens, device=DEV)), lens=lens)
    _check_grads(case, **kw)
    _, got, _, _ = _grads(case, **kw)
    for g in got[:5]:
        for b, n in enumerate(lens):
            assert (g[b, n:] == 0).all()


@pytest.mark.parametrize("use", [(True, False), (False, True)])
def test_gradients_of_one_output(use):
    case = _case(T=70, Hk=1, Hv=2, Dk=32, Dv=32)
    have, got, want, _ = _grads(case, use=use)
    for n, a, b in zip(have, got, want):
        if b.norm() == 0:
            assert a.abs().max() == 0, n
        else:
            assert _rel(a, b) <= _tol(a, 32) + (7 * _arith(32) if n == "g" else 0), n


def test_gradients_extreme_decays():
    T = 140
    case = _case(T=T, Hk=1, Hv=3, Dk=32, Dv=32, seed=11)
    g = case[3]
    g[..., 0] = 0
    g[..., 1] = torch.where(torch.arange(T) % 2 == 0, -30.0, -1e-3)
    g[..., 2] = -2000.0
    _check_grads(case)


def test_gradients_with_zero_strength():
    case = _case(T=70, Hk=1, Hv=2, Dk=32, Dv=32)
    case[4][:, ::3] = 0
    _check_grads(case)


def test_gradients_against_differences():
    """Along one direction, central differences of the operator itself: with a step h the
    formula's error is O(h^2) and rounding adds about arith / h; h = 2^-7 leaves
    2^-14 + 2^7 arith < 1e-3."""
    from ramnet_ops import gated_delta_rule
    case = _case(T=70, Hk=1, Hv=2, Dk=32, Dv=32)
    gen = torch.Generator().manual_seed(4)
    x = [t.to(DEV).requires_grad_() for t in case]
    o, state = gated_delta_rule(*x[:5], init_state=x[5])
    d = [torch.randn(t.shape, generator=gen).to(DEV) for t in (o, state)]
    grads = torch.autograd.grad([o, state], x, d)
    h = 2.0 ** -7

    def along(i, step, sign):
        y = [t.detach() + (sign * h * step if j == i else 0) for j, t in enumerate(x)]
        a, b = gated_delta_rule(*y[:5], init_state=y[5])
        return (a.double() * d[0]).sum() + (b.double() * d[1]).sum()
    for i, n in enumerate(NAMES):
        step = torch.randn(case[i].shape, generator=gen).to(DEV)
        step = step / step.norm()
        step = step + grads[i] / grads[i].norm()
        got = float((grads[i].double() * step).sum())
        want = float(along(i, step, 1) - along(i, step, -1)) / (2 * h)
        assert abs(got - want) <= 1e-3 * abs(want), (n, got, want)


def test_gradients_again_and_strided():
    from ramnet_ops import gated_delta_rule
    case = [t.to(DEV) for t in _case(B=2, T=100, Hk=1, Hv=3, Dk=32, Dv=32, dtype="bf16")]
    d = torch.randn(2, 3, 100, 32, device=DEV).bfloat16().transpose(1, 2)
    out = []
    for strided in (False, False, True):
        x = [t.transpose(1, 2).contiguous().transpose(1, 2) if strided and i < 5 else t
             for i, t in enumerate(case)]
        x = [t.detach().requires_grad_() for t in x]
        o, state = gated_delta_rule(*x[:5], init_state=x[5])
        out.append(torch.autograd.grad([o], x, [d if strided else d.contiguous()]))
    for other in out[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out[0], other))


def test_gradients_compiled_and_selected():
    from ramnet_ops import gated_delta_rule
    case = [t.to(DEV) for t in _case(T=70, Hk=1, Hv=2, Dk=32, Dv=32)]

    def loss(q, k, v, g, beta, init):
        o, state = gated_delta_rule(q, k, v, g, beta, init_state=init)
        return (o * o).sum() + state.sum()
    x = [t.detach().requires_grad_() for t in case]
    want = torch.autograd.grad(loss(*x), x)
    got = torch.autograd.grad(torch.compile(loss, backend="aot_eager", fullgraph=True)(*x), x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = [t.detach().requires_grad_(i == 2) for i, t in enumerate(case)]
    loss(*x).backward()
    assert torch.equal(x[2].grad, want[2]) and all(t.grad is None for i, t in enumerate(x) if i != 2)


# ---- rows cut into segments: packed ones, ones whose tokens do not all count, in place

@pytest.mark.parametrize("lens", [[1600], [30, 1500, 0, 70], [700, 700, 600], [1] * 6 + [1994], [1024] + [0] * 5])
def test_long_packed(lens):
    case = _case(T=sum(lens), Hk=1, Hv=2, Dk=40, Dv=24, N=len(lens), seed=len(lens))
    cu = torch.tensor([0] + lens).cumsum(0).to(DEV, torch.int32)
    _check(case, _call(case, cu_seqlens=cu), lens, packed=True)
    case[5] = None
    _check(case, _call(case, cu_seqlens=cu), lens, packed=True)


def test_long_packed_tokens_of_no_sequence_are_zero():
    case = _case(T=2000, Dk=16, Dv=16, N=3, seed=5)
    cu = torch.tensor([100, 110, 1800, 1801], dtype=torch.int32, device=DEV)
    o, state = _call(case, cu_seqlens=cu)
    part = [t[:, 100:1801] for t in case[:5]] + [case[5]]
    _check(part, (o[:, 100:1801].contiguous(), state), [10, 1690, 1], packed=True)
    assert o[:, :100].abs().max() == 0 and o[:, 1801:].abs().max() == 0


@pytest.mark.parametrize("lens", [[1100], [20, 1500, 0, 70], [1] * 3 + [1200]])
def test_long_packed_gradients(lens):
    case = _case(T=sum(lens), Hk=1, Hv=2, Dk=24, Dv=40, N=len(lens), seed=len(lens))
    cu = torch.tensor([0] + lens).cumsum(0).to(DEV, torch.int32)
    _check_grads(case, kw=dict(cu_seqlens=cu), lens=lens, packed=True)


def test_long_rows_counted_lengths_gradients():
    lens = [1100, 0, 1, 600, 320]
    case = _case(B=5, T=1100, Hk=1, Hv=1, Dk=24, Dv=40, seed=8)
    _check_grads(case, kw=dict(lengths=torch.tensor(lens, device=DEV)), lens=lens)


@pytest.mark.parametrize("T,packed", [(1024, False), (4000, False), (4000, True)])
def test_long_rows_in_place(T, packed):
    """The first segment's state is what the last one writes over."""
    case = _case(T=T, Hk=2, Hv=2, Dk=64, Dv=64, dtype="bf16", seed=T)
    kw = dict(cu_seqlens=torch.tensor([0, T], dtype=torch.int32, device=DEV)) if packed else {}
    want = _call(case, **kw)
    got = _call(case, inplace=True, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("T", [70, 1100])
def test_gradients_graph_replays(T):
    """A forward and its backward captured together, on leaves that no eager graph holds then."""
    from ramnet_ops import gated_delta_rule

    def leaves(seed):
        return [t.to(DEV) for t in _case(T=T, Hk=1, Hv=2, Dk=40, Dv=32, dtype="bf16", seed=seed)]

    def grads(x, w):
        o, state = gated_delta_rule(*x[:5], init_state=x[5])
        return torch.autograd.grad([o, state], x, [w, torch.ones_like(state)])
    x = [t.requires_grad_() for t in leaves(1)]
    w = torch.randn(1, T, 2, 32, device=DEV).to(torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads(x, w)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = grads(x, w)
    for step in range(3):
        new = leaves(2 + step)
        with torch.no_grad():
            for t, s in zip(x, new):
                t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, grads([t.requires_grad_() for t in new], w)):
            assert torch.equal(a, b)
