"""Refusals of ``gated_delta_rule`` and ``verify_drafts``, before any launch (CPU)."""
from __future__ import annotations

import struct

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


FIELDS = ("q k v g beta init_state state o cu_seqlens lengths kept workspace kept_bytes workspace_bytes "
          "B T N Hk Hv Dk Dv").split()


def _packed(strides=64, **kw):
    """A ramnet_delta_rule_call as bytes."""
    x = dict(dict.fromkeys(FIELDS, 0), q=FAKE, k=FAKE, v=FAKE, g=FAKE, beta=FAKE, state=FAKE, o=FAKE, workspace=FAKE,
             workspace_bytes=1 << 30, B=2, T=100, N=2, Hk=2, Hv=4, Dk=64, Dv=64, dtype=2, g_dtype=0, beta_dtype=2)
    x.update(kw)
    return struct.pack("=12Q2q22q3qd", *(x[n] for n in FIELDS), *[strides] * 15, x["dtype"], x["g_dtype"],
                       x["beta_dtype"], 1.0)


def test_native_delta_rule():
    nat = _native()

    def call(match, **kw):
        _einval("ramnet_delta_rule_forward", (_packed(**kw), None), match)
    _einval("ramnet_delta_rule_forward", (None, None), "null call")
    call("shape must have", B=-1)
    call("shape must have", Dk=0)
    call("multiple of Hk", Hv=3)
    call("Dk must be at most", Dk=257)
    call("batch of one", cu_seqlens=FAKE)
    call("batch of one", N=3)
    call("index overflow", T=1 << 30)
    call("index overflow", Dv=1 << 21)
    call("dtype", dtype=3)
    call("dtype", g_dtype=-1)
    call("no lengths", B=1, cu_seqlens=FAKE, lengths=FAKE)
    call("null tensor", q=0)
    call("null tensor", state=0)
    call("one row to", strides=63)
    call("one row to", strides=1 << 22)
    call("workspace too small", workspace_bytes=16)
    call("workspace too small", workspace=0)
    call("kept region too small", kept=FAKE, kept_bytes=16)
    call("Dk up to 160", kept=FAKE, kept_bytes=1 << 40, dtype=0, Dk=200, strides=256)

    def call_back(match, strides=64, grads=(FAKE,) * 6, **kw):
        kw = dict(dict(kept=FAKE, kept_bytes=1 << 30), **kw)
        _einval("ramnet_delta_rule_backward",
                (_packed(strides=kw.pop("rows", 64), **kw), FAKE, nat.strides(64, strides, 64), None, *grads, None), match)
    call_back("needs tokens", T=0)
    call_back("null tensor", grads=(FAKE, FAKE, FAKE, 0, FAKE, FAKE))
    call_back("null tensor", kept=0)
    call_back("kept region too small", kept_bytes=16)
    call_back("Dk up to 160", dtype=0, Dk=200, rows=256)
    call_back("workspace too small", workspace_bytes=16)
    call_back("tokens of d_o", strides=63)
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


def test_native_delta_rule_backward_in_place():
    nat = _native()
    _einval("ramnet_delta_rule_backward",
            (_packed(kept=FAKE, kept_bytes=1 << 30), FAKE, nat.strides(64, 64, 64), FAKE, *(FAKE,) * 6, None), "dinit")
