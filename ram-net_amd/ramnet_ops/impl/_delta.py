"""``torch.library`` operators of the gated delta rule and of draft verification.

``_forward``, ``_verify`` and their like make the native call; the operators
registered around them carry the schemas, fakes and gradients that tracing,
autograd and ``torch.func`` need. The public functions call the former where
nothing of the latter is wanted: a call through the dispatcher costs the host
several times what a decode step costs the GPU.
"""
from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd import forward_ad

from .. import _native as nat
from ._ops import _check_shapes, _code, _dims, _NS, _require_gpu

_FLOATS = tuple(nat.DTYPE_CODES)


def is_eager(*tensors: Tensor | None) -> bool:
    """Whether a call on these tensors loses nothing beside the dispatcher: no
    tracing, mode, transform, forward-mode level or tensor subclass."""
    return (not torch.compiler.is_compiling() and torch._C._functorch.peek_interpreter_stack() is None
            and torch._C._len_torch_dispatch_stack() == 0 and forward_ad._current_level < 0
            and all(t is None or type(t) in (Tensor, torch.nn.Parameter) for t in tensors))


def wants_grad(*tensors: Tensor | None) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# --------------------------------------------------------------------------
# gated delta rule

def _check(op: str, q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, init_state: Tensor | None,
           cu_seqlens: Tensor | None, lengths: Tensor | None) -> tuple[int, ...]:
    """Sizes (B, T, N, Hk, Hv, Dk, Dv) of a call, its tensors checked against them."""
    B, T, Hk, Dk = _dims(op, "q", q, 4)
    Hv, Dv = _dims(op, "v", v, 4)[2:]
    N = B if cu_seqlens is None else _dims(op, "cu_seqlens", cu_seqlens, 1)[0] - 1
    if k.shape != q.shape or v.shape[:2] != q.shape[:2] or g.shape != v.shape[:3] or beta.shape != g.shape \
            or init_state is not None and init_state.shape != (N, Hv, Dk, Dv) \
            or lengths is not None and lengths.shape != (B,):
        _check_shapes(op, k=(k, (B, T, Hk, Dk)), v=(v, (B, T, Hv, Dv)), g=(g, (B, T, Hv)), beta=(beta, (B, T, Hv)),
                      init_state=(init_state, (N, Hv, Dk, Dv)), lengths=(lengths, (B,)))
    if Hk == 0 or Hv == 0 or Hv % Hk or Dk == 0 or Dv == 0:
        raise RuntimeError(f"{op}: the heads of v must be a multiple of those of q and k and no size 0, got "
                           f"q {tuple(q.shape)} and v {tuple(v.shape)}")
    if q.dtype not in _FLOATS or k.dtype != q.dtype or v.dtype != q.dtype or g.dtype not in _FLOATS \
            or beta.dtype not in _FLOATS:
        raise RuntimeError(f"{op}: q, k and v must share one of {_FLOATS}, g and beta have one of them, got "
                           f"{q.dtype}, {k.dtype}, {v.dtype}, {g.dtype} and {beta.dtype}")
    device = q.device
    for t in (q, k, v, g, beta, init_state, cu_seqlens, lengths):
        if t is not None and t.device != device:
            raise RuntimeError(f"{op}: tensors must share a device, got {t.device} beside {device}")
    if not q.is_cuda:
        _require_gpu(op, q)
    if cu_seqlens is not None:
        if B != 1 or lengths is not None:
            raise RuntimeError(f"{op}: sequences packed by cu_seqlens lie in a batch of one, without lengths")
        if N < 0:
            raise RuntimeError(f"{op}: cu_seqlens needs N + 1 bounds of N sequences")
    for name, t in (("cu_seqlens", cu_seqlens), ("lengths", lengths)):
        if t is not None and t.dtype not in (torch.int32, torch.int64):
            raise RuntimeError(f"{op}: {name} must be int32 or int64, got {t.dtype}")
    return B, T, N, Hk, Hv, Dk, Dv


def _dense(t: Tensor) -> Tensor:
    """t with adjacent elements along its last dimension."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _rows(t: Tensor) -> Tensor:
    """t (B, T, H, D) whose heads are dense and whose tokens lie apart, within the kernels' reach."""
    D, (_, step, _, last) = t.shape[3], t.stride()
    return t if (last == 1 or D == 1) and (D <= step < 2 ** 22 or t.shape[1] == 1) else t.contiguous()


def _whole(t: Tensor | None) -> Tensor | None:
    if t is None or (t.dtype == torch.int32 and t.is_contiguous()):
        return t
    return t.to(torch.int32).contiguous()


def _args(q, k, v, g, beta, cu_seqlens, lengths):
    """The inputs as the native calls read them."""
    return _rows(q), _rows(k), _rows(v), g, beta, _whole(cu_seqlens), _whole(lengths)


def _at(q, k, v, g, beta, *more):
    s = q.stride()[:3] + k.stride()[:3] + v.stride()[:3] + g.stride() + beta.stride()
    for t in more:
        s += t.stride()[:3]
    return nat.strides(*s)


def _bytes(op: str, count: int, sizes) -> int:
    if count < 0:
        raise RuntimeError(f"{op}: sizes (B, T, N, Hk, Hv, Dk, Dv) = {tuple(sizes)} are not supported "
                           "(Dk up to 256, up to 160 for gradients of float32; tokens within int32)")
    return count


def _forward(op: str, q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, init_state: Tensor | None,
             cu_seqlens: Tensor | None, lengths: Tensor | None, scale: float, state: Tensor | None = None,
             keep: bool = False) -> tuple[Tensor, Tensor, Tensor | None]:
    """(o, state, kept). ``state``: where the state goes (init_state itself in place)."""
    sizes = _check(op, q, k, v, g, beta, init_state, cu_seqlens, lengths)
    B, T, N, Hk, Hv, Dk, Dv = sizes
    packed = cu_seqlens is not None
    q, k, v, g, beta, cu_seqlens, lengths = _args(q, k, v, g, beta, cu_seqlens, lengths)
    if init_state is not None and init_state is not state:
        init_state = init_state.to(torch.float32).contiguous()
    if state is None:
        state = torch.empty((N, Hv, Dk, Dv), dtype=torch.float32, device=q.device)
    o = torch.empty((B, T, Hv, Dv), dtype=q.dtype, device=q.device)
    lib = nat.lib()
    kept = None
    kept_bytes = 0
    if keep:
        kept_bytes = _bytes(op, lib.ramnet_delta_rule_kept_bytes(*sizes, _code(q), packed), sizes)
        kept = torch.empty(kept_bytes, dtype=torch.uint8, device=q.device)
    n = _bytes(op, lib.ramnet_delta_rule_workspace_bytes(*sizes, _code(q), packed, int(keep)), sizes)
    ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    if N == 0:
        return o.zero_(), state, kept
    with nat.on_device(q):
        nat.call("ramnet_delta_rule_forward", q.data_ptr(), k.data_ptr(), v.data_ptr(), _code(q), g.data_ptr(), _code(g),
                 beta.data_ptr(), _code(beta), nat.ptr(init_state), state.data_ptr(), o.data_ptr(),
                 nat.ptr(cu_seqlens), nat.ptr(lengths), *sizes, scale, _at(q, k, v, g, beta), nat.ptr(kept), kept_bytes,
                 nat.ptr(ws), n, nat.stream_of(q))
    return o, state, kept


def _out_shapes(q, k, v, cu_seqlens):
    N = q.shape[0] if cu_seqlens is None else cu_seqlens.shape[0] - 1
    return v.new_empty(v.shape), v.new_empty((N, v.shape[2], q.shape[3], v.shape[3]), dtype=torch.float32)


@torch.library.custom_op(f"{_NS}::gated_delta_rule", mutates_args=(), device_types="cuda")
def gated_delta_rule(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, init_state: Tensor | None,
                     cu_seqlens: Tensor | None, lengths: Tensor | None, scale: float) -> tuple[Tensor, Tensor]:
    """(o, state); no gradients (``gated_delta_rule_kept`` has them)."""
    return _forward("gated_delta_rule", q, k, v, g, beta, init_state, cu_seqlens, lengths, scale)[:2]


@gated_delta_rule.register_fake
def _(q, k, v, g, beta, init_state, cu_seqlens, lengths, scale):
    return _out_shapes(q, k, v, cu_seqlens)


def _require_state(op: str, state: Tensor) -> None:
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise RuntimeError(f"{op}: a state updated in place must be contiguous float32, got {state.dtype}")


@torch.library.custom_op(f"{_NS}::gated_delta_rule_", mutates_args=("state",), device_types="cuda")
def gated_delta_rule_(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, state: Tensor,
                      cu_seqlens: Tensor | None, lengths: Tensor | None, scale: float) -> Tensor:
    """o; updates ``state`` in place."""
    _require_state("gated_delta_rule_", state)
    return _forward("gated_delta_rule_", q, k, v, g, beta, state, cu_seqlens, lengths, scale, state)[0]


@gated_delta_rule_.register_fake
def _(q, k, v, g, beta, state, cu_seqlens, lengths, scale):
    return v.new_empty(v.shape)


@torch.library.custom_op(f"{_NS}::gated_delta_rule_kept", mutates_args=(), device_types="cuda")
def gated_delta_rule_kept(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, init_state: Tensor | None,
                          cu_seqlens: Tensor | None, lengths: Tensor | None,
                          scale: float) -> tuple[Tensor, Tensor, Tensor]:
    """(o, state, kept): ``gated_delta_rule`` that leaves its backward the state
    before each chunk of 64 tokens and each token's v - S^T k."""
    return _forward("gated_delta_rule_kept", q, k, v, g, beta, init_state, cu_seqlens, lengths, scale, keep=True)


@gated_delta_rule_kept.register_fake
def _(q, k, v, g, beta, init_state, cu_seqlens, lengths, scale):
    B, T, Hk, Dk = q.shape
    N = B if cu_seqlens is None else cu_seqlens.shape[0] - 1
    n = nat.lib().ramnet_delta_rule_kept_bytes(B, T, N, Hk, v.shape[2], Dk, v.shape[3], _code(q), cu_seqlens is not None)
    return *_out_shapes(q, k, v, cu_seqlens), q.new_empty((n,), dtype=torch.uint8)


@torch.library.custom_op(f"{_NS}::gated_delta_rule_backward", mutates_args=(), device_types="cuda")
def gated_delta_rule_backward(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, cu_seqlens: Tensor | None,
                              lengths: Tensor | None, scale: float, kept: Tensor, d_o: Tensor,
                              d_state: Tensor | None) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """Gradients (dq, dk, dv, dg, dbeta, dinit) of ``gated_delta_rule_kept``."""
    op = "gated_delta_rule_backward"
    sizes = _check(op, q, k, v, g, beta, None, cu_seqlens, lengths)
    B, T, N, Hk, Hv, Dk, Dv = sizes
    packed = cu_seqlens is not None
    _check_shapes(op, d_o=(d_o, (B, T, Hv, Dv)), d_state=(d_state, (N, Hv, Dk, Dv)))
    q, k, v, g, beta, cu_seqlens, lengths = _args(q, k, v, g, beta, cu_seqlens, lengths)
    d_o = _rows(d_o.to(q.dtype))
    if d_state is not None:
        d_state = d_state.to(torch.float32).contiguous()
    grads = [torch.empty(t.shape, dtype=t.dtype, device=q.device) for t in (q, k, v, g, beta)]
    dinit = torch.empty((N, Hv, Dk, Dv), dtype=torch.float32, device=q.device)
    n = _bytes(op, nat.lib().ramnet_delta_rule_workspace_bytes(*sizes, _code(q), packed, 2), sizes)
    if N == 0 or T == 0 or B == 0:
        for t in grads:
            t.zero_()
        dinit.zero_() if d_state is None else dinit.copy_(d_state)
        return *grads, dinit
    ws = torch.empty(n, dtype=torch.uint8, device=q.device)
    with nat.on_device(q):
        nat.call("ramnet_delta_rule_backward", q.data_ptr(), k.data_ptr(), v.data_ptr(), _code(q), g.data_ptr(), _code(g),
                 beta.data_ptr(), _code(beta), nat.ptr(cu_seqlens), nat.ptr(lengths), d_o.data_ptr(),
                 nat.ptr(d_state), *(t.data_ptr() for t in grads), dinit.data_ptr(), *sizes, scale,
                 _at(q, k, v, g, beta, d_o), kept.data_ptr(), kept.numel(), ws.data_ptr(), n, nat.stream_of(q))
    return *grads, dinit


@gated_delta_rule_backward.register_fake
def _(q, k, v, g, beta, cu_seqlens, lengths, scale, kept, d_o, d_state):
    return (*(t.new_empty(t.shape) for t in (q, k, v, g, beta)), _out_shapes(q, k, v, cu_seqlens)[1])


def _setup(ctx, inputs, output):
    q, k, v, g, beta, init_state, cu_seqlens, lengths, scale = inputs
    kept = output[2]
    ctx.scale = scale
    ctx.init_dtype = None if init_state is None else init_state.dtype
    ctx.save_for_backward(q, k, v, g, beta, cu_seqlens, lengths, kept)
    ctx.mark_non_differentiable(kept)
    ctx.set_materialize_grads(False)


def _backward(ctx, d_o, d_state, d_kept):
    q, k, v, g, beta, cu_seqlens, lengths, kept = ctx.saved_tensors
    if d_o is None and d_state is None:
        return (None,) * 9
    if d_o is None:
        d_o = torch.zeros_like(v)
    *grads, dinit = gated_delta_rule_backward(q, k, v, g, beta, cu_seqlens, lengths, ctx.scale, kept, d_o, d_state)
    need = ctx.needs_input_grad
    return (*(t if n else None for t, n in zip(grads, need)),
            dinit.to(ctx.init_dtype) if need[5] else None, None, None, None)


gated_delta_rule_kept.register_autograd(_backward, setup_context=_setup)


# --------------------------------------------------------------------------
# verification of drafted tokens

def _verify(tokens: Tensor, target: Tensor, draft: Tensor | None, accept: Tensor, sample: Tensor,
            draft_lens: Tensor | None) -> tuple[Tensor, Tensor]:
    op = "verify_drafts"
    B, S = _dims(op, "tokens", tokens, 2)
    V = _dims(op, "target", target, 3)[2]
    if target.shape != (B, S + 1, V) or draft is not None and draft.shape != (B, S, V) or accept.shape != (B, S) \
            or sample.shape != (B,) or draft_lens is not None and draft_lens.shape != (B,):
        _check_shapes(op, target=(target, (B, S + 1, V)), draft=(draft, (B, S, V)), accept=(accept, (B, S)),
                      sample=(sample, (B,)), draft_lens=(draft_lens, (B,)))
    if V == 0:
        raise RuntimeError(f"{op}: an empty vocabulary")
    device = target.device
    for t in (tokens, draft, accept, sample, draft_lens):
        if t is not None and t.device != device:
            raise RuntimeError(f"{op}: tensors must share a device, got {t.device} beside {device}")
    if target.dtype not in _FLOATS or draft is not None and draft.dtype != target.dtype:
        raise RuntimeError(f"{op}: target and draft must share one of {_FLOATS}, got {target.dtype} and "
                           f"{None if draft is None else draft.dtype}")
    if not target.is_cuda:
        _require_gpu(op, target)
    for name, t in (("tokens", tokens), ("draft_lens", draft_lens)):
        if t is not None and t.dtype not in (torch.int32, torch.int64):
            raise RuntimeError(f"{op}: {name} must be int32 or int64, got {t.dtype}")
    tokens = tokens.to(torch.int64).contiguous()
    accept, sample = accept.to(torch.float32).contiguous(), sample.to(torch.float32).contiguous()
    target, draft, draft_lens = _dense(target), None if draft is None else _dense(draft), _whole(draft_lens)
    out = torch.empty((B, S + 1), dtype=torch.int64, device=device)
    taken = torch.empty((B,), dtype=torch.int32, device=device)
    at = target.stride()[:2] + (draft.stride()[:2] if draft is not None else (0, 0))
    with nat.on_device(target):
        nat.call("ramnet_verify_drafts", tokens.data_ptr(), target.data_ptr(), nat.ptr(draft), _code(target),
                 accept.data_ptr(), sample.data_ptr(), nat.ptr(draft_lens), B, S, V, nat.strides(*at), out.data_ptr(),
                 taken.data_ptr(), nat.stream_of(target))
    return out, taken


@torch.library.custom_op(f"{_NS}::verify_drafts", mutates_args=(), device_types="cuda")
def verify_drafts(tokens: Tensor, target: Tensor, draft: Tensor | None, accept: Tensor, sample: Tensor,
                  draft_lens: Tensor | None) -> tuple[Tensor, Tensor]:
    return _verify(tokens, target, draft, accept, sample, draft_lens)


@verify_drafts.register_fake
def _(tokens, target, draft, accept, sample, draft_lens):
    B, S = tokens.shape
    return tokens.new_empty((B, S + 1), dtype=torch.int64), tokens.new_empty((B,), dtype=torch.int32)
