"""Verification of drafted tokens on the GPU against the fp64 oracle: whole
numbers, so equal (sums are in 64 bits on both sides)."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import delta_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _case(B, S, V, dtype="fp32", drafts=True, seed=0, near=0.5):
    gen = torch.Generator().manual_seed(seed)
    logits = 2 * torch.randn(B, S + 1, V, generator=gen)
    target = torch.softmax(logits, -1).to(DTYPES[dtype])
    draft = torch.softmax(logits[:, :S] + near * torch.randn(B, S, V, generator=gen), -1)
    tokens = torch.multinomial(draft.reshape(B * S, V), 1, generator=gen).view(B, S) if S else torch.zeros(B, 0).long()
    return [tokens, target, draft.to(DTYPES[dtype]) if drafts else None, torch.rand(B, S, generator=gen),
            torch.rand(B, generator=gen)]


def _check(case, lens=None):
    from ramnet_ops import verify_drafts
    want = oracle.verify_drafts(*case, lens)
    d = [t.to(DEV) if t is not None else None for t in case]
    got = verify_drafts(*d, draft_lens=None if lens is None else torch.tensor(lens, device=DEV))
    assert got[0].dtype == torch.int64 and got[1].dtype == torch.int32
    assert torch.equal(got[1].cpu(), want[1]), (got[1], want[1])
    assert torch.equal(got[0].cpu(), want[0])
    return got


@pytest.mark.parametrize("V", [1, 2, 3, 7, 64, 1000, 4097, 32000, 50257])
@pytest.mark.parametrize("drafts", [True, False])
def test_vocabularies(V, drafts):
    for S in (1, 3):
        _check(_case(5, S, V, drafts=drafts, seed=V + S))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("V", [1001, 4096])
def test_types(dtype, drafts, V):
    for seed in range(3):
        _check(_case(16, 4, V, dtype, drafts, seed))


@pytest.mark.parametrize("drafts", [True, False])
def test_lengths(drafts):
    case = _case(6, 4, 500, drafts=drafts, near=0.0)
    case[3][:] = 0  # every draft that counts stays
    got = _check(case, [0, 1, 2, 3, 4, 4])
    assert got[1].tolist() == [0, 1, 2, 3, 4, 4]
    _check(_case(6, 4, 500, drafts=drafts, seed=5), [0, 1, 2, 3, 4, 4])
    _check(_case(4, 0, 300))
    _check(_case(2, 1500, 8, near=0.1))


def test_refusals_at_each_place():
    for place in range(4):
        case = _case(3, 4, 300, near=0.0, seed=place)
        case[3][:] = 0
        case[1][:, place].scatter_(-1, case[0][:, place:place + 1], 0.0)  # the target rules the token out
        got = _check(case)
        assert (got[1] == place).all()
        assert (got[0][:, place].cpu() != case[0][:, place]).all()


def test_nothing_left_goes_to_the_target():
    """A refused draft whose distribution covers the target's: max(p - q, 0) is 0 everywhere."""
    case = _case(4, 2, 100, near=0.0)
    case[2] = case[1][:, :2].clone()
    case[3][:] = 1.0  # 1 * q < p is false where q = p
    got = _check(case)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("drafts", [True, False])
def test_borders_of_the_running_sum(drafts):
    """Samples on the borders of exactly representable sums: the first index that passes."""
    V = 8
    p = torch.tensor([0.0, 0.25, 0.0, 0.25, 0.125, 0.125, 0.25, 0.0])
    sample = torch.tensor([0.0, 0.25, 0.5, 0.625, 0.75, 0.875, 1 - 2.0 ** -24])
    B = len(sample)
    case = [torch.zeros(B, 1).long(), p.expand(B, 2, V).contiguous(), None, torch.zeros(B, 1), sample]
    if drafts:
        case[2] = torch.zeros(B, 1, V)
        case[2][..., 0] = 1
    got = _check(case)
    assert got[0][:, 0].tolist() == [1, 3, 4, 5, 6, 6, 6]


def test_tokens_out_of_range_and_strange_rows():
    case = _case(4, 2, 50)
    case[0][0, 0], case[0][1, 1], case[0][2, 0] = -1, 50, 2 ** 40
    _check(case)
    case[2] = None
    _check(case)
    from ramnet_ops import verify_drafts
    case = [t.to(DEV) if t is not None else None for t in _case(3, 2, 50)]
    case[1][0] = math.nan
    case[1][1] = 0
    out, taken = verify_drafts(*case)
    assert ((out >= -1) & (out < 50)).all() and ((taken >= 0) & (taken <= 2)).all()
    case[4][:] = 1.0  # past the range: still a token with a weight
    out, taken = verify_drafts(*case)
    assert case[1][2, taken[2], out[2, taken[2]]] > 0


def test_strides_types_and_ways():
    from ramnet_ops import verify_drafts
    case = [t.to(DEV) for t in _case(6, 3, 701, "bf16")]
    want = verify_drafts(*case)
    # rows of a padded logits buffer, places first
    target = torch.zeros(4, 6, 710, device=DEV, dtype=torch.bfloat16)
    target[..., :701] = case[1].transpose(0, 1)
    draft = torch.repeat_interleave(case[2], 2, -1)[..., ::2]
    lens = torch.full((6,), 3, device=DEV)
    for tokens in (case[0].int(), case[0].t().contiguous().t()):
        got = verify_drafts(tokens, target.transpose(0, 1)[..., :701], draft, case[3].double(), case[4], lens)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = torch.compile(verify_drafts, backend="aot_eager", fullgraph=True)(*case)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    import ramnet_ops  # noqa: F401
    torch.library.opcheck(torch.ops.ramnet_ops.verify_drafts, (*case, None),
                          test_utils=("test_schema", "test_faketensor"))


def test_graph_replays():
    from ramnet_ops import verify_drafts
    case = [t.to(DEV) for t in _case(6, 3, 701)]
    verify_drafts(*case)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = verify_drafts(*case)
    for seed in range(3):
        for t, s in zip(case, _case(6, 3, 701, seed=seed + 1)):
            t.copy_(s)
        want = verify_drafts(*case)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_empty_batch():
    from ramnet_ops import verify_drafts
    out, taken = verify_drafts(*(t.to(DEV) for t in _case(1, 2, 5)))
    assert out.shape == (1, 3)
    e = lambda *s: torch.zeros(*s, device=DEV)  # noqa: E731
    out, taken = verify_drafts(e(0, 2).long(), e(0, 3, 5), None, e(0, 2), e(0))
    assert out.shape == (0, 3) and taken.shape == (0,)
