"""Native calls with packed tokens and no sequences: every token is one of no
sequence, so the output and all gradients are 0."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [5, 100])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_zeros(T, dtype):
    from ramnet_ops import _native as nat
    from ramnet_ops.impl import _delta
    Hk, Hv, Dk, Dv = 2, 4, 24, 20
    q, k = (torch.randn(1, T, Hk, Dk, device="cuda").to(dtype) for _ in range(2))
    v = torch.randn(1, T, Hv, Dv, device="cuda").to(dtype)
    g, beta = torch.zeros(1, T, Hv, device="cuda"), torch.ones(1, T, Hv, device="cuda", dtype=dtype)
    cu = torch.zeros(1, dtype=torch.int32, device="cuda")
    plan, *_ = _delta._plan("test", q, k, v, g, beta, None, cu, None)
    room = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")

    def call(o, kept):
        return _delta._HEAD.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), 0,
                                 room.data_ptr(), o, cu.data_ptr(), 0, kept, room.data_ptr(), room.numel(),
                                 room.numel()) + plan.tail + _delta._SCALE.pack(1.0)
    o = torch.ones_like(v)
    nat.call("ramnet_delta_rule_forward", call(o.data_ptr(), 0), nat.stream_of(q))
    assert (o == 0).all()
    grads = [torch.ones_like(t) for t in (q, k, v, g, beta)]
    nat.call("ramnet_delta_rule_backward", call(0, room.data_ptr()), v.data_ptr(), nat.strides(*v.stride()[:3]), None,
             *(t.data_ptr() for t in grads), None, nat.stream_of(q))
    for t in grads:
        assert (t == 0).all()
