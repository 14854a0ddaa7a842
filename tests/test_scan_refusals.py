"""Refusals of ``causal_conv``, ``selective_scan`` and sampling, before any launch (CPU)."""
from __future__ import annotations

import struct

import pytest
import torch


def _conv(**kw):
    return {**dict(x=torch.zeros(2, 4, 6), weight=torch.zeros(6, 3)), **kw}


@pytest.mark.parametrize("kw,error,match", [
    (dict(x=None), TypeError, "x to be a Tensor"),
    (dict(weight=3), TypeError, "weight to be a Tensor"),
    (dict(bias=1.0), TypeError, "bias"),
    (dict(activation="relu"), ValueError, "activation"),
    (dict(activation=True), ValueError, "activation"),
    (dict(inplace=True), ValueError, "init_state"),
    (dict(x=torch.zeros(4, 6)), RuntimeError, "x must have 3"),
    (dict(weight=torch.zeros(6)), RuntimeError, "weight must have 2"),
    (dict(weight=torch.zeros(5, 3)), RuntimeError, "weight shape mismatch"),
    (dict(weight=torch.zeros(6, 9)), RuntimeError, "1 to 8 taps"),
    (dict(weight=torch.zeros(6, 0)), RuntimeError, "1 to 8 taps"),
    (dict(x=torch.zeros(2, 4, 0), weight=torch.zeros(0, 3)), RuntimeError, "needs channels"),
    (dict(bias=torch.zeros(5)), RuntimeError, "bias shape mismatch"),
    (dict(init_state=torch.zeros(2, 3, 6)), RuntimeError, "init_state shape mismatch"),
    (dict(init_state=torch.zeros(2, 2, 6).double()), RuntimeError, "init_state must be one of"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), RuntimeError, "lengths shape mismatch"),
    (dict(lengths=torch.zeros(2)), RuntimeError, "lengths must be int32"),
    (dict(cu_seqlens=torch.zeros(2, dtype=torch.int32)), RuntimeError, "batch of one"),
    (dict(x=torch.zeros(1, 4, 6), cu_seqlens=torch.zeros(0, dtype=torch.int32)), RuntimeError, "N \\+ 1 bounds"),
    (dict(x=torch.zeros(1, 4, 6), cu_seqlens=torch.zeros(2, 2, dtype=torch.int32)), RuntimeError, "cu_seqlens must have 1"),
    (dict(x=torch.zeros(1, 4, 6), cu_seqlens=torch.zeros(2)), RuntimeError, "cu_seqlens must be int32"),
    (dict(weight=torch.zeros(6, 3).half()), RuntimeError, "share one of"),
    (dict(bias=torch.zeros(6).half()), RuntimeError, "share one of"),
    (dict(x=torch.zeros(2, 4, 6).double(), weight=torch.zeros(6, 3).double()), RuntimeError, "share one of"),
    (dict(), RuntimeError, "must be on a GPU"),
])
def test_causal_conv(kw, error, match):
    from ramnet_ops import causal_conv
    with pytest.raises(error, match=match):
        causal_conv(**_conv(**kw))


def _scan(**kw):
    return {**dict(x=torch.zeros(2, 4, 6), dt=torch.zeros(2, 4, 6), A=torch.zeros(6, 5), B=torch.zeros(2, 4, 2, 5),
                   C=torch.zeros(2, 4, 2, 5)), **kw}


@pytest.mark.parametrize("kw,error,match", [
    (dict(x=None), TypeError, "x to be a Tensor"),
    (dict(C=1.0), TypeError, "C to be a Tensor"),
    (dict(gate=1.0), TypeError, "gate"),
    (dict(inplace=True), ValueError, "init_state"),
    (dict(x=torch.zeros(4, 6)), RuntimeError, "x must have 3"),
    (dict(B=torch.zeros(2, 4, 5)), RuntimeError, "B must have 4"),
    (dict(dt=torch.zeros(2, 4, 5)), RuntimeError, "dt shape mismatch"),
    (dict(A=torch.zeros(6, 4)), RuntimeError, "A shape mismatch"),
    (dict(C=torch.zeros(2, 4, 1, 5)), RuntimeError, "C shape mismatch"),
    (dict(B=torch.zeros(2, 3, 2, 5)), RuntimeError, "B shape mismatch"),
    (dict(skip=torch.zeros(5)), RuntimeError, "skip shape mismatch"),
    (dict(gate=torch.zeros(2, 4)), RuntimeError, "gate shape mismatch"),
    (dict(dt_bias=torch.zeros(1)), RuntimeError, "dt_bias shape mismatch"),
    (dict(init_state=torch.zeros(2, 5, 6)), RuntimeError, "init_state shape mismatch"),
    (dict(B=torch.zeros(2, 4, 4, 5), C=torch.zeros(2, 4, 4, 5)), RuntimeError, "multiple of the groups"),
    (dict(B=torch.zeros(2, 4, 0, 5), C=torch.zeros(2, 4, 0, 5)), RuntimeError, "multiple of the groups"),
    (dict(A=torch.zeros(6, 65), B=torch.zeros(2, 4, 2, 65), C=torch.zeros(2, 4, 2, 65)), RuntimeError, "1 to 64 states"),
    (dict(A=torch.zeros(6, 0), B=torch.zeros(2, 4, 2, 0), C=torch.zeros(2, 4, 2, 0)), RuntimeError, "1 to 64 states"),
    (dict(dt=torch.zeros(2, 4, 6).half()), RuntimeError, "share one of"),
    (dict(gate=torch.zeros(2, 4, 6).half()), RuntimeError, "share one of"),
    (dict(A=torch.zeros(6, 5).double()), RuntimeError, "A must be one of"),
    (dict(skip=torch.zeros(6).int()), RuntimeError, "skip must be one of"),
    (dict(init_state=torch.zeros(2, 6, 5).double()), RuntimeError, "init_state must be one of"),
    (dict(lengths=torch.zeros(2).bool()), RuntimeError, "lengths must be int32"),
    (dict(cu_seqlens=torch.zeros(2, dtype=torch.int32)), RuntimeError, "batch of one"),
    (dict(), RuntimeError, "must be on a GPU"),
])
def test_selective_scan(kw, error, match):
    from ramnet_ops import selective_scan
    with pytest.raises(error, match=match):
        selective_scan(**_scan(**kw))


@pytest.mark.parametrize("kw,error,match", [
    (dict(logits=None), TypeError, "logits to be a Tensor"),
    (dict(random=0.5), TypeError, "random to be a Tensor"),
    (dict(temperature="1"), TypeError, "temperature to be a number"),
    (dict(temperature=-1.0), ValueError, "temperature"),
    (dict(temperature=float("nan")), ValueError, "temperature"),
    (dict(top_k=1.5), TypeError, "top_k to be an integer"),
    (dict(top_k=True), TypeError, "top_k to be an integer"),
    (dict(top_k=-1), ValueError, "top_k"),
    (dict(top_p=1.5), ValueError, "top_p"),
    (dict(min_p=-0.5), ValueError, "min_p"),
    (dict(logits=torch.zeros(())), RuntimeError, "vocabulary"),
    (dict(logits=torch.zeros(3, 0)), RuntimeError, "vocabulary"),
    (dict(logits=torch.zeros(3, 7).double()), RuntimeError, "logits must be one of"),
    (dict(random=torch.zeros(3, 1)), RuntimeError, "random shape mismatch"),
    (dict(random=torch.zeros(3).int()), RuntimeError, "random must be floating-point"),
    (dict(top_k=torch.zeros(3)), RuntimeError, "top_k must be int32"),
    (dict(top_p=torch.zeros(3).int()), RuntimeError, "top_p must be floating-point"),
    (dict(), RuntimeError, "must be on a GPU"),
])
def test_sampling(kw, error, match):
    from ramnet_ops import sample_tokens, token_probabilities
    x = {**dict(logits=torch.zeros(3, 7), random=torch.zeros(3)), **kw}
    with pytest.raises(error, match=match):
        sample_tokens(**x)
    if "random" not in kw:
        del x["random"]
        with pytest.raises(error, match=match):
            token_probabilities(**x)


@pytest.mark.gpu
def test_settings_that_do_not_broadcast():
    from ramnet_ops import sample_tokens
    x = torch.zeros(3, 7, device="cuda")
    with pytest.raises(RuntimeError, match="top_p must broadcast"):
        sample_tokens(x, x[:, 0], top_p=torch.zeros(2, device="cuda"))
    with pytest.raises(RuntimeError, match="share a device"):
        sample_tokens(x, x[:, 0], min_p=torch.zeros(3))


@pytest.mark.gpu
def test_in_place_refusals():
    from ramnet_ops import causal_conv, selective_scan
    c = {k: v.cuda() for k, v in _conv().items()}
    with pytest.raises(RuntimeError, match="in place must be contiguous"):
        causal_conv(**c, init_state=torch.zeros(2, 2, 6, device="cuda").half(), inplace=True)
    with pytest.raises(ValueError, match="no gradients"):
        causal_conv(**{**c, "x": c["x"].requires_grad_()}, init_state=torch.zeros(2, 2, 6, device="cuda"), inplace=True)
    s = {k: v.cuda() for k, v in _scan().items()}
    with pytest.raises(RuntimeError, match="in place must be contiguous"):
        selective_scan(**s, init_state=torch.zeros(2, 5, 6, device="cuda").mT, inplace=True)
    with pytest.raises(ValueError, match="no gradients"):
        selective_scan(**{**s, "A": s["A"].requires_grad_()}, init_state=torch.zeros(2, 6, 5, device="cuda"), inplace=True)


# ---- the C ABI

FAKE = 0x1000  # never dereferenced: every call below fails validation first


def _native():
    from ramnet_ops import _native
    return _native


def _einval(name, args, match):
    nat = _native()
    assert getattr(nat.lib(), name)(*args) == nat.RAMNET_EINVAL
    with pytest.raises(RuntimeError, match=match):
        nat.call(name, *args)


def _conv_call(x=FAKE, weight=FAKE, state=FAKE, y=FAKE, cu=0, lengths=0, ws=0, n=0, B=1, T=8, N=1, D=16, W=4, dtype=0):
    return struct.pack("=9Qq9q", x, weight, 0, 0, state, y, cu, lengths, ws, n, B, T, N, D, W, T * D, D, dtype, 0)


@pytest.mark.parametrize("kw,match", [
    (dict(x=0), "null tensor"), (dict(weight=0), "null tensor"), (dict(state=0), "null tensor"), (dict(y=0), "null tensor"),
    (dict(B=-1), "shape"), (dict(N=2), "one to a row"), (dict(cu=FAKE, B=2), "batch of one"), (dict(D=0), "D must be above"),
    (dict(W=9), "W from 1 to 8"), (dict(W=0), "W from 1 to 8"), (dict(dtype=5), "dtype"), (dict(T=2 ** 31), "index overflow"),
    (dict(B=2 ** 20, N=2 ** 20, T=2 ** 12), "index overflow"), (dict(D=2 ** 24), "index overflow"),
    (dict(cu=FAKE, lengths=FAKE), "no lengths"), (dict(cu=FAKE), "workspace too small"),
])
def test_conv_call(kw, match):
    _einval("ramnet_causal_conv_forward", (_conv_call(**kw), None), match)


def test_conv_backward_call():
    strides = _native().strides(0, 0)
    name, grads = "ramnet_causal_conv_backward", [FAKE] * 4
    _einval(name, (_conv_call(), FAKE, strides, None, *grads, None), "workspace too small")
    ok = _conv_call(ws=FAKE, n=1 << 30)
    _einval(name, (ok, None, strides, None, *grads, None), "null tensor")
    _einval(name, (ok, FAKE, strides, None, FAKE, None, None, None, None), "null tensor")
    _einval(name, (ok, FAKE, strides, FAKE, FAKE, FAKE, FAKE, FAKE, None), "dinit must not be dstate")
    _einval(name, (_conv_call(ws=FAKE, n=1 << 30, B=0, N=0), FAKE, strides, None, *grads, None), "needs rows")


def _scan_call(x=FAKE, A=FAKE, state=FAKE, y=FAKE, cu=0, lengths=0, kept=0, ws=FAKE, kept_n=0, n=1 << 30, B=1, T=80, N=1,
               D=16, S=4, G=1, dtype=0, gate=0):
    return struct.pack("=15Q2q20q", x, FAKE, gate, FAKE, FAKE, A, 0, 0, 0, state, y, cu, lengths, kept, ws, kept_n, n,
                       B, T, N, D, S, G, *[0] * 12, dtype, 0)


@pytest.mark.parametrize("kw,match", [
    (dict(x=0), "null tensor"), (dict(A=0), "null tensor"), (dict(state=0), "null tensor"), (dict(y=0), "null tensor"),
    (dict(T=-1), "shape"), (dict(N=0), "one to a row"), (dict(cu=FAKE, B=2), "batch of one"),
    (dict(G=3), "multiple of G"), (dict(G=0), "multiple of G"), (dict(S=65), "S must be from 1 to 64"),
    (dict(S=0), "S must be from 1 to 64"), (dict(dtype=3), "dtype"), (dict(T=2 ** 31), "index overflow"),
    (dict(D=2 ** 24), "index overflow"), (dict(B=2 ** 24, N=2 ** 24, D=2 ** 15), "index overflow"),
    (dict(cu=FAKE, lengths=FAKE), "no lengths"), (dict(n=8, T=4096), "workspace too small"),
    (dict(kept=FAKE, kept_n=8), "kept region too small"),
])
def test_scan_call(kw, match):
    _einval("ramnet_selective_scan_forward", (_scan_call(**kw), None), match)


def test_scan_backward_call():
    strides = _native().strides(0, 0)
    name = "ramnet_selective_scan_backward"
    kept = dict(kept=FAKE, kept_n=1 << 30)

    def args(call, dy=FAKE, dstate=None, **kw):
        out = dict(dx=FAKE, ddt=FAKE, dgate=None, dB=FAKE, dC=FAKE, dA=FAKE, dskip=None, dbias=None, dinit=None)
        return call, dy, strides, dstate, *{**out, **kw}.values(), None
    _einval(name, args(_scan_call(**kept), dy=None), "null tensor")
    _einval(name, args(_scan_call()), "null tensor")
    _einval(name, args(_scan_call(**kept), dA=None), "null tensor")
    _einval(name, args(_scan_call(**kept, gate=FAKE)), "null tensor")
    _einval(name, args(_scan_call(**kept), dstate=FAKE, dinit=FAKE), "dinit must not be dstate")
    _einval(name, args(_scan_call(**kept, n=8)), "workspace too small")
    _einval(name, args(_scan_call(**kept, T=0)), "needs tokens")


def _sample_call(logits=FAKE, random=FAKE, tokens=FAKE, probs=0, R=2, V=9, dtype=0):
    return struct.pack("=8Q3d5q", logits, random, 0, 0, 0, 0, tokens, probs, 1.0, 1.0, 0.0, 0, R, V, V, dtype)


@pytest.mark.parametrize("kw,match", [
    (dict(logits=0), "null tensor"), (dict(random=0), "null tensor"), (dict(tokens=0), "null tensor"), (dict(R=-1), "shape"),
    (dict(V=0), "shape"), (dict(V=2 ** 30), "index overflow"), (dict(R=2 ** 31), "index overflow"), (dict(dtype=4), "dtype"),
])
def test_sample_call(kw, match):
    _einval("ramnet_sample_tokens", (_sample_call(**kw), None), match)


def test_null_calls():
    strides = _native().strides(0, 0)
    for name in ("ramnet_causal_conv_forward", "ramnet_selective_scan_forward", "ramnet_sample_tokens"):
        _einval(name, (None, None), "null call")
    _einval("ramnet_causal_conv_backward", (None, FAKE, strides, *[None] * 6), "null call")
    _einval("ramnet_selective_scan_backward", (None, FAKE, strides, *[None] * 11), "null call")


def test_workspace_queries():
    lib = _native().lib()
    assert lib.ramnet_causal_conv_workspace_bytes(2, 8, 2, 16, 4, 0, 0, 0) == 0
    assert lib.ramnet_causal_conv_workspace_bytes(2, 8, 2, 16, 9, 0, 0, 0) == -1
    assert lib.ramnet_causal_conv_workspace_bytes(2, 8, 2, 16, 4, 7, 0, 0) == -1
    assert lib.ramnet_selective_scan_workspace_bytes(2, 8, 2, 16, 4, 1, 0, 0) == 0
    assert lib.ramnet_selective_scan_workspace_bytes(2, 8, 2, 16, 4, 3, 0, 0) == -1
    assert lib.ramnet_selective_scan_workspace_bytes(2, 8, 2, 16, 4, 1, 0, 3) == -1
    assert lib.ramnet_selective_scan_kept_bytes(2, 8, 3, 16, 4, 1, 0) == -1
    for kind in range(3):
        assert lib.ramnet_selective_scan_workspace_bytes(0, 500, 0, 16, 4, 1, 0, kind) >= 0


def test_sizes_past_a_launch():
    """A launch has less than 2^32 threads: rows, sequences or channels past it are refused before any launch."""
    lib, mega = _native().lib(), 2 ** 20
    conv, scan = lib.ramnet_causal_conv_workspace_bytes, lib.ramnet_selective_scan_workspace_bytes
    # a thread takes 4 channels of a row, or one of up to 7
    assert conv(3 * mega, 1, 3 * mega, 4096, 4, 2, 0, 0) == 0
    assert conv(4 * mega, 1, 4 * mega, 4096, 4, 2, 0, 0) == -1
    assert conv(1024 * mega - 1, 1, 1024 * mega - 1, 3, 4, 2, 0, 0) == 0
    assert conv(1024 * mega - 1, 1, 1024 * mega - 1, 4, 4, 2, 0, 0) == -1
    assert conv(1, 16, 4 * mega, 4096, 4, 2, 1, 0) == -1
    # 256 threads take 64 channels
    assert scan(200000, 1, 200000, 4096, 16, 1, 0, 0) == 0
    assert scan(270000, 1, 270000, 4096, 16, 1, 0, 0) == -1
    assert scan(5000, 1, 5000, 4096, 16, 4096, 0, 0) == -1
    assert scan(1, 1, 270000, 4096, 16, 1, 1, 0) == -1
    # 1024 threads add up 64 sums over pieces
    assert scan(1, 1, 1, 4 * mega - 1, 32, 1, 0, 2) > 0
    assert scan(1, 1, 1, 4 * mega - 1, 64, 1, 0, 2) == -1
    _einval("ramnet_sample_tokens", (_sample_call(R=4 * mega), None), "index overflow")


def test_scan_tokens_far_apart():
    strides = [80 * 16, 16, 0, 0, 0, 0] + [0] * 6
    for i in (1, 3, 5, 7, 10):
        far = list(strides)
        far[i] = 2 ** 22
        call = struct.pack("=15Q2q20q", FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 0, 0, 0, FAKE, FAKE, 0, 0, 0, FAKE, 0, 1 << 30,
                           1, 80, 1, 16, 4, 1, *far, 0, 0)
        _einval("ramnet_selective_scan_forward", (call, None), "2\\*\\*22 elements apart")
