"""Refusals of ``gated_delta_rule`` and ``verify_drafts``, before any launch (CPU)."""
from __future__ import annotations

import pytest
import torch


def _delta(**kw):
    x = dict(q=torch.zeros(1, 4, 2, 8), k=torch.zeros(1, 4, 2, 8), v=torch.zeros(1, 4, 4, 6), g=torch.zeros(1, 4, 4),
             beta=torch.zeros(1, 4, 4))
    x.update(kw)
    return x


@pytest.mark.parametrize("kw,error,match", [
    (dict(q=None), TypeError, "q to be a Tensor"),
    (dict(init_state=1.0), TypeError, "init_state"),
    (dict(scale="x"), TypeError, "scale"),
    (dict(inplace=True), ValueError, "init_state"),
    (dict(q=torch.zeros(4, 2, 8)), RuntimeError, "q must have 4"),
    (dict(k=torch.zeros(1, 4, 2, 9)), RuntimeError, "k shape mismatch"),
    (dict(v=torch.zeros(1, 5, 4, 6)), RuntimeError, "v shape mismatch"),
    (dict(g=torch.zeros(1, 4, 2)), RuntimeError, "g shape mismatch"),
    (dict(beta=torch.zeros(1, 4)), RuntimeError, "beta shape mismatch"),
    (dict(v=torch.zeros(1, 4, 3, 6), g=torch.zeros(1, 4, 3), beta=torch.zeros(1, 4, 3)), RuntimeError, "multiple"),
    (dict(q=torch.zeros(1, 4, 2, 0), k=torch.zeros(1, 4, 2, 0)), RuntimeError, "no size 0"),
    (dict(init_state=torch.zeros(1, 4, 6, 8)), RuntimeError, "init_state shape mismatch"),
    (dict(lengths=torch.zeros(2, dtype=torch.int32)), RuntimeError, "lengths shape mismatch"),
    (dict(cu_seqlens=torch.zeros(2, 2, dtype=torch.int32)), RuntimeError, "cu_seqlens must have 1"),
    (dict(k=torch.zeros(1, 4, 2, 8).half()), RuntimeError, "share one of"),
    (dict(g=torch.zeros(1, 4, 4).double()), RuntimeError, "share one of"),
    (dict(), RuntimeError, "must be on a GPU"),
])
def test_delta_rule(kw, error, match):
    from ramnet_ops import gated_delta_rule
    with pytest.raises(error, match=match):
        gated_delta_rule(**_delta(**kw))


def _verify(**kw):
    x = dict(tokens=torch.zeros(2, 3).long(), target=torch.zeros(2, 4, 9), draft=torch.zeros(2, 3, 9),
             accept=torch.zeros(2, 3), sample=torch.zeros(2))
    x.update(kw)
    return x


@pytest.mark.parametrize("kw,error,match", [
    (dict(tokens=3), TypeError, "tokens to be a Tensor"),
    (dict(tokens=torch.zeros(2).long()), RuntimeError, "tokens must have 2"),
    (dict(target=torch.zeros(2, 3, 9)), RuntimeError, "target shape mismatch"),
    (dict(draft=torch.zeros(2, 3, 8)), RuntimeError, "draft shape mismatch"),
    (dict(accept=torch.zeros(2, 4)), RuntimeError, "accept shape mismatch"),
    (dict(sample=torch.zeros(2, 1)), RuntimeError, "sample shape mismatch"),
    (dict(draft_lens=torch.zeros(3)), RuntimeError, "draft_lens shape mismatch"),
    (dict(target=torch.zeros(2, 4, 0), draft=torch.zeros(2, 3, 0)), RuntimeError, "empty vocabulary"),
    (dict(draft=torch.zeros(2, 3, 9).half()), RuntimeError, "share one of"),
    (dict(), RuntimeError, "must be on a GPU"),
])
def test_verify_drafts(kw, error, match):
    from ramnet_ops import verify_drafts
    with pytest.raises(error, match=match):
        verify_drafts(**_verify(**kw))


FAKE = 0x1000  # never dereferenced: every call below fails validation first


def _native():
    from ramnet_ops import _native
    return _native


def _einval(name, args, match):
    nat = _native()
    assert getattr(nat.lib(), name)(*args) == nat.RAMNET_EINVAL
    with pytest.raises(RuntimeError, match=match):
        nat.call(name, *args)


def test_native_delta_rule():
    nat = _native()
    ok = dict(q=FAKE, k=FAKE, v=FAKE, dtype=2, g=FAKE, g_dtype=0, beta=FAKE, beta_dtype=2, init=None, state=FAKE, o=FAKE,
              cu=None, lengths=None, B=2, T=100, N=2, Hk=2, Hv=4, Dk=64, Dv=64, scale=1.0, strides=nat.strides(*[64] * 18),
              kept=None, kept_bytes=0, ws=FAKE, ws_bytes=1 << 30, stream=None)

    def call(match, **kw):
        _einval("ramnet_delta_rule_forward", {**ok, **kw}.values(), match)
    call("shape must have", B=-1)
    call("shape must have", Dk=0)
    call("multiple of Hk", Hv=3)
    call("Dk must be at most", Dk=257)
    call("batch of one", cu=FAKE)
    call("batch of one", N=3)
    call("index overflow", T=1 << 30)
    call("dtype", dtype=3)
    call("dtype", g_dtype=-1)
    call("no lengths", B=1, cu=FAKE, lengths=FAKE)
    call("null tensor", q=None)
    call("null tensor", state=None)
    call("one row to", strides=nat.strides(*[63] * 18))
    call("one row to", strides=nat.strides(*[1 << 22] * 18))
    call("workspace too small", ws_bytes=16)
    call("workspace too small", ws=None)
    call("kept region too small", kept=FAKE, kept_bytes=16)
    back = dict(q=FAKE, k=FAKE, v=FAKE, dtype=2, g=FAKE, g_dtype=0, beta=FAKE, beta_dtype=2, cu=None, lengths=None,
                d_o=FAKE, d_state=None, dq=FAKE, dk=FAKE, dv=FAKE, dg=FAKE, dbeta=FAKE, dinit=None, B=2, T=100, N=2,
                Hk=2, Hv=4, Dk=64, Dv=64, scale=1.0, strides=nat.strides(*[64] * 18), kept=FAKE, kept_bytes=1 << 30,
                ws=FAKE, ws_bytes=1 << 30, stream=None)

    def call_back(match, **kw):
        _einval("ramnet_delta_rule_backward", {**back, **kw}.values(), match)
    call_back("needs tokens", T=0)
    call_back("null tensor", dg=None)
    call_back("kept region too small", kept_bytes=16)
    call_back("Dk up to 160", dtype=0, Dk=200, strides=nat.strides(*[256] * 18))
    call_back("workspace too small", ws_bytes=16)
    lib = nat.lib()
    assert lib.ramnet_delta_rule_workspace_bytes(2, 100, 2, 2, 4, 300, 64, 2, 0, 0) == -1
    assert lib.ramnet_delta_rule_workspace_bytes(2, 1, 2, 2, 4, 64, 64, 2, 0, 0) == 0  # a step needs none
    assert lib.ramnet_delta_rule_kept_bytes(2, 100, 3, 2, 4, 64, 64, 2, 0) == -1
    assert lib.ramnet_delta_rule_kept_bytes(2, 100, 2, 2, 4, 161, 64, 0, 0) == -1
    assert lib.ramnet_delta_rule_kept_bytes(2, 100, 2, 2, 4, 161, 64, 2, 0) > 0


def test_native_verify_drafts():
    nat = _native()
    ok = dict(tokens=FAKE, target=FAKE, draft=None, dtype=0, accept=FAKE, sample=FAKE, lens=None, B=2, S=3, V=100,
              strides=nat.strides(0, 0, 0, 0), out=FAKE, taken=FAKE, stream=None)

    def call(match, **kw):
        _einval("ramnet_verify_drafts", {**ok, **kw}.values(), match)
    call("shape must have", V=0)
    call("shape must have", S=-1)
    call("index overflow", V=1 << 31)
    call("dtype", dtype=5)
    call("null tensor", tokens=None)
    call("null tensor", sample=None)
