"""Token sampling on the GPU against the oracle, row by row in 64 bits.

Tokens have to be equal. Probabilities are a weight (fp64 on both sides) over a
sum of weights in parts of 2^-45 or finer, rounded once to fp32: 2^-24 of their value, and
2^-23 leaves room for the sum. A weight that rounds to no part of the sum is compared with it too.
"""
from __future__ import annotations

import math

import pytest
import torch

from oracle import scan_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _logits(R, V, dtype="fp32", seed=0, spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    return (spread * torch.randn(R, V, generator=gen)).to(DTYPES[dtype]), torch.rand(R, generator=gen)


def _at(value, row):
    return value[row].item() if torch.is_tensor(value) else value


def _check(logits, random, temperature=1.0, top_k=None, top_p=None, min_p=None):
    from ramnet_ops import sample_tokens, token_probabilities
    kw = {n: v.to(DEV) if torch.is_tensor(v) else v for n, v in
          dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p).items()}
    tokens, probs = sample_tokens(logits.to(DEV), random.to(DEV), probabilities=True, **kw)
    assert tokens.dtype == torch.int64 and probs.dtype == torch.float32 and probs.shape == logits.shape
    assert torch.equal(sample_tokens(logits.to(DEV), random.to(DEV), **kw), tokens)
    assert torch.equal(token_probabilities(logits.to(DEV), **kw), probs)
    tokens, probs = tokens.cpu(), probs.cpu()
    for r in range(logits.shape[0]):
        token, want = oracle.sample_row(logits[r].tolist(), random[r].item(), _at(temperature, r),
                                        *(off if v is None else _at(v, r) for v, off in
                                          ((top_k, 0), (top_p, 1.0), (min_p, 0.0))))
        assert int(tokens[r]) == token, (r, int(tokens[r]), token)
        assert torch.equal(probs[r] > 0, want.float() > 0), r
        assert ((probs[r].double() - want).abs() <= 2.0 ** -23 * want + 2.0 ** -149).all(), r
    return tokens, probs


FILTERS = [{}, dict(top_k=1), dict(top_k=7), dict(top_p=0.3), dict(top_p=0.9), dict(min_p=0.1), dict(top_p=0.0),
           dict(top_k=20, top_p=0.8), dict(top_k=5, top_p=0.95, min_p=0.05), dict(min_p=1.0), dict(top_k=10 ** 12),
           dict(top_p=1.0, min_p=0.0, top_k=0)]


@pytest.mark.parametrize("V", [1, 2, 3, 7, 8, 63, 64, 65, 1023, 1025, 4097])
@pytest.mark.parametrize("kw", FILTERS, ids=str)
def test_vocabularies(V, kw):
    _check(*_logits(3, V, seed=V), **kw)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("kw", FILTERS[2:9], ids=str)
def test_types(dtype, kw):
    """(Rounded to 16 bits, many logits are equal: the lowest indices go first.)"""
    for temperature in (0.0, 0.3, 1.0, 5.0):
        _check(*_logits(3, 3001, dtype, seed=5), temperature=temperature, **kw)


@pytest.mark.parametrize("kw", [dict(top_k=3000), dict(top_k=20000), dict(top_p=0.5), dict(top_p=0.999),
                                dict(top_k=40000, top_p=0.7), dict(top_k=3, top_p=0.7, min_p=0.2), {}], ids=str)
@pytest.mark.parametrize("spread", [0.0, 1e-4, 2.0])
def test_large(kw, spread):
    """More tokens in a bin than are compared with each other: equal logits, and far more kept than dropped."""
    _check(*_logits(2, 50021, seed=1, spread=spread), **kw)


def test_outliers():
    """All but a few tokens in one bin; ties across its whole width."""
    x, u = _logits(6, 30000, seed=3)
    x[0, 17] = 1e30
    x[1, 17] = -1e30
    x[2] = x[2].bfloat16().float()
    x[2, 5] = -3e38
    x[3, ::2] = 0.25
    x[3, 7] = -1e5
    x[4] = x[4].abs() * 1e-30
    x[4, 9] = -1e9
    x[5] = torch.arange(30000) // 7000 * 1e-3
    x[5, 29999] = -1e4
    for kw in (dict(top_k=2500), dict(top_p=0.6), dict(top_k=9000, top_p=0.9), dict(top_k=1), dict(min_p=0.5)):
        _check(x, u, **kw)


def test_settings_of_each_row():
    R = 24
    x, u = _logits(R, 2000, "bf16", seed=2)
    gen = torch.Generator().manual_seed(9)
    temperature = torch.rand(R, generator=gen) * 2
    temperature[::5] = 0
    top_k = torch.randint(0, 2100, (R,), generator=gen)
    top_k[1::6] = -4
    top_p = torch.rand(R, generator=gen) * 1.2
    min_p = torch.rand(R, generator=gen) * 0.2
    min_p[::4] = 0
    _check(x, u, temperature, top_k, top_p, min_p)
    _check(x, u, temperature, top_k.int())
    _check(x, u, 0.7, None, top_p.double().float(), None)
    _check(x, u, torch.tensor(0.5).expand(R), 30)


def test_masked_and_strange_rows():
    x, u = _logits(12, 300, seed=4)
    inf, nan = math.inf, math.nan
    x[0] = -inf                     # nothing left
    x[1, 1:] = -inf                 # one left
    x[2, ::2] = -inf
    x[3, 5] = nan
    x[4] = nan
    x[5, [7, 40]] = inf             # far above the rest
    x[6] = torch.finfo(torch.float32).min
    x[7, :200] = torch.finfo(torch.float32).min
    x[8, 250:] = -inf
    x[9] = torch.tensor([0.0, -0.0]).repeat(150)
    x[10] = inf
    x[11, 0] = -inf
    for kw in ({}, dict(top_k=3), dict(top_p=0.5), dict(top_k=2, top_p=0.9, min_p=0.01), dict(top_k=299), dict(top_p=0.999999),
               dict(temperature=0.0), dict(temperature=inf), dict(temperature=1e-38), dict(temperature=1e30, top_k=4)):
        tokens, probs = _check(x, u, **kw)
        assert tokens[0] == 0 and not probs[0].any() and not probs[4].any()


def test_random_numbers_at_the_borders():
    """Weights of powers of 2, so that running sums are met to the bit."""
    x = torch.log(torch.tensor([1, 2, 4, 1, 8], dtype=torch.float64)).float().repeat(7, 1)
    x[:, :] = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.0])
    u = torch.tensor([0.0, 0.2, 0.4, 0.5999, 0.7999, 0.99999994, 1.0])
    tokens, _ = _check(x, u)
    assert tokens.tolist() == [0, 1, 2, 2, 3, 4, 4]
    tokens, _ = _check(x, u, top_k=4)
    assert tokens.tolist() == [0, 0, 1, 2, 3, 3, 3]
    _check(x, torch.full((7,), math.nan))


@pytest.mark.parametrize("p", [0.25, 0.5, 0.75])
def test_top_p_at_a_border(p):
    """A prefix whose sum is the share asked for to the bit: the next token does not stay."""
    x = torch.zeros(1, 8)
    _, probs = _check(x, torch.tensor([0.5]), top_p=p)
    assert int((probs > 0).sum()) == int(8 * p)


def test_layouts_and_shapes():
    from ramnet_ops import sample_tokens, token_probabilities
    x, u = (t.to(DEV) for t in _logits(6, 1001, "bf16", seed=7))
    want, probs = sample_tokens(x, u, top_p=0.9, probabilities=True)
    wide = torch.zeros(6, 1500, device=DEV, dtype=torch.bfloat16)
    wide[:, 3:1004] = x
    for other in (wide[:, 3:1004], x.mT.contiguous().mT):
        assert torch.equal(sample_tokens(other, u, top_p=0.9), want)
    for shape in ((2, 3), (1, 6, 1), (3, 1, 2)):
        got, p = sample_tokens(x.view(*shape, 1001), u.view(shape), top_p=0.9, probabilities=True)
        assert torch.equal(got, want.view(shape)) and torch.equal(p, probs.view(*shape, 1001))
        assert torch.equal(token_probabilities(x.view(*shape, 1001), top_p=0.9), p)
    assert torch.equal(sample_tokens(x[0], u[0], top_p=0.9), want[0])
    steps = x.view(2, 3, 1001)[:, -1]  # the last position of each row
    assert torch.equal(sample_tokens(steps, u.view(2, 3)[:, -1], top_p=0.9), want.view(2, 3)[:, -1])
    # a setting of each batch row for all its positions
    t = torch.tensor([[0.5], [2.0]], device=DEV)
    got = token_probabilities(x.view(2, 3, 1001), temperature=t)
    assert torch.equal(got[1], token_probabilities(x[3:], temperature=2.0)) and torch.equal(
        got[0], token_probabilities(x[:3], temperature=0.5))
    for dt in (torch.float64, torch.bfloat16):
        assert torch.equal(sample_tokens(x, u.to(dt)), sample_tokens(x, u.to(dt).float()))
    neg = torch.complex(torch.zeros(6, 1001, device=DEV), -x.float()).conj().imag
    assert neg.is_neg() and torch.equal(sample_tokens(neg, u, top_p=0.9), want)


def test_empty():
    from ramnet_ops import sample_tokens
    tokens, probs = sample_tokens(torch.zeros(0, 5, device=DEV), torch.zeros(0, device=DEV), probabilities=True)
    assert tokens.shape == (0,) and probs.shape == (0, 5)
    assert sample_tokens(torch.zeros(2, 0, 5, device=DEV), torch.zeros(2, 0, device=DEV)).shape == (2, 0)


def test_past_32_bits():
    """Rows more than 2^31 elements apart."""
    x, u = _logits(2, 500, "bf16")
    far = torch.empty(2 ** 31 + 1000, dtype=torch.bfloat16, device=DEV)
    rows = far.as_strided((2, 500), (2 ** 31 + 8, 1)).copy_(x)
    from ramnet_ops import sample_tokens
    assert torch.equal(sample_tokens(rows, u.to(DEV), top_k=9), sample_tokens(x.to(DEV), u.to(DEV), top_k=9))


def test_streams_compiled_and_registered():
    from ramnet_ops import sample_tokens, token_probabilities
    x, u = (t.to(DEV) for t in _logits(5, 3000, seed=8))
    t = torch.rand(5, device=DEV) + 0.5

    def f(x, u, t):
        a, b = sample_tokens(x, u, temperature=t, top_k=100, top_p=0.9, probabilities=True)
        return a, b, sample_tokens(x, u, temperature=t), token_probabilities(x, min_p=0.1)
    want = f(x, u, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = f(x, u, t)
    torch.cuda.current_stream().wait_stream(side)
    for other in (got, torch.compile(f, backend="aot_eager", fullgraph=True)(x, u, t),
                  torch.jit.trace(f, (x, u, t), check_trace=False)(x, u, t)):
        assert all(torch.equal(a, b) for a, b in zip(other, want))
    ops, numbers = torch.ops.ramnet_ops, (1.0, 5, 0.9, 0.0)
    for op, args in ((ops.sample_tokens, (x, u)), (ops.sample_tokens_with_probabilities, (x, u)),
                     (ops.token_probabilities, (x,))):
        torch.library.opcheck(op, (*args, t, None, None, None, *numbers), test_utils=("test_schema", "test_faketensor"))


def test_graph_replays():
    from ramnet_ops import sample_tokens
    x, u = (t.to(DEV) for t in _logits(5, 3000, seed=8))

    def f():
        return sample_tokens(x, u, top_k=100, top_p=0.9, probabilities=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, probs = f()
    for n in range(3):
        for t, s in zip((x, u), _logits(5, 3000, seed=20 + n)):
            t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        want = f()
        assert torch.equal(tokens, want[0]) and torch.equal(probs, want[1])


@pytest.mark.parametrize("kw", [dict(min_p=0.02, top_p=0.9, temperature=1.5), dict(min_p=1e-4, top_p=0.97, temperature=1.5),
                                dict(min_p=1e-3, top_p=0.999), dict(top_k=30000, min_p=1e-3, top_p=0.99),
                                dict(min_p=0.5, top_p=0.01), dict(min_p=1e-9, top_p=0.5, temperature=3.0)], ids=str)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("spread", [0.5, 2.0])
def test_min_p_beside_top_p(kw, dtype, spread):
    """Either one ends first, in a list or far past one."""
    _check(*_logits(3, 50021, dtype, seed=9, spread=spread), **kw)


@pytest.mark.parametrize("V", [8192 * 16, 8192 * 16 + 1, 8192 * 40 + 13])
def test_drawn_tokens_of_long_rows(V):
    logits, _ = _logits(5, V, "bf16", seed=3)
    _check(logits, torch.tensor([0.0, 0.13, 0.5, 0.77, 1 - 2.0 ** -24]))


@pytest.mark.parametrize("V,kw", [(37, {}), (5000, dict(top_k=40)), (5000, dict(top_p=0.9)), (5000, dict(min_p=0.05)), (70001, {})])
def test_random_numbers_out_of_range_draw_a_kept_token(V, kw):
    from ramnet_ops import sample_tokens
    logits = _logits(1, V, seed=7)[0].to(DEV).expand(6, V)
    random = torch.tensor([0.0, -0.5, -math.inf, math.nan, 1.0, math.inf], device=DEV)
    token, probs = sample_tokens(logits, random, probabilities=True, **kw)
    kept = (probs[0] > 0).nonzero().flatten()
    assert token.tolist() == [kept[0]] * 3 + [kept[-1]] * 3
