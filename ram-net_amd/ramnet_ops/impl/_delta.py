"""``torch.library`` operators of the gated delta rule and of draft verification.

``_forward``, ``_verify`` and their like make the native call; the operators
registered around them carry the schemas, fakes and gradients that tracing,
autograd and ``torch.func`` need. The public functions call the former where
nothing of the latter is wanted: a call through the dispatcher costs the host
several times what a decode step costs the GPU.
"""
from __future__ import annotations

import struct
from typing import NamedTuple

import torch
from torch import Tensor
from torch.autograd import forward_ad

from .. import _native as nat
from ._ops import _check_shapes, _code, _dims, _NS, _require_gpu

_FLOATS = tuple(nat.DTYPE_CODES)


_peek, _modes = torch._C._functorch.peek_interpreter_stack, torch._C._len_torch_dispatch_stack
_jit_trace = torch._C._get_tracing_state
_PLAIN = {Tensor, torch.nn.Parameter}


def is_eager(*tensors: Tensor | None) -> bool:
    """Whether a call on these tensors loses nothing beside the dispatcher: no
    tracing (by torch.compile or torch.jit.trace), mode, transform, forward-mode
    level, tensor subclass or view whose memory holds the negated values (the
    imaginary part of a conjugated tensor)."""
    if (torch.compiler.is_compiling() or _jit_trace() is not None or _peek() is not None or _modes()
            or forward_ad._current_level >= 0):
        return False
    for t in tensors:
        if t is not None and (type(t) not in _PLAIN or t.is_neg()):
            return False
    return True


def wants_grad(*tensors: Tensor | None) -> bool:
    if not torch.is_grad_enabled():
        return False
    return any(t is not None and t.requires_grad for t in tensors)


class _Plans(dict):
    """What calls of the same sizes, strides, types and devices share, by these."""

    def keep(self, key, plan):
        if len(self) >= 1024:
            self.clear()
        self[key] = plan
        return plan


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
    if init_state is not None and init_state.dtype not in _FLOATS:
        raise RuntimeError(f"{op}: init_state must be one of {_FLOATS}, got {init_state.dtype}")
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


def _kept_bytes(op: str, sizes, dtype: torch.dtype, packed: bool):
    """Bytes of what a training forward keeps, in arithmetic that tracing leaves
    symbolic: ramnet_delta_rule_kept_bytes, but room for the maps of the most
    segments that rows of these sizes can be cut into."""
    B, T, N, Hk, Hv, Dk, Dv = sizes
    wide = next((w for w in (32, 64, 96, 128, 160, 256) if Dk <= w), 0)
    row = (Dv + 7) // 8 * 8
    if wide == 0 or dtype == torch.float32 and wide > 160 or wide * row > 2 ** 28 or Hk * Dk >= 2 ** 22:
        _bytes(op, -1, sizes)
    per_row = (T + 63) // 64
    records = (per_row + N if packed else N * per_row) * Hv

    def region(floats):
        return (floats * 4 + 255) // 256 * 256
    count = region(records * 64 * row) + region(records * Dk * row)
    if N * Hv * ((Dv + 63) // 64) <= 128:
        count += region(N * Hv * torch.sym_min(per_row // 4, 64) * wide * wide)
    return count


def _bytes(op: str, count: int, sizes) -> int:
    if count < 0:
        raise RuntimeError(f"{op}: sizes (B, T, N, Hk, Hv, Dk, Dv) = {tuple(sizes)} are not supported "
                           "(Dk up to 256, up to 160 for gradients of float32; Hk Dk below 2**22 and Dk Dv up to "
                           "2**28 for gradients; tokens within int32)")
    return count


# ramnet_delta_rule_call: pointers and region sizes; sizes, strides and types; scale
_HEAD, _TAIL, _SCALE = struct.Struct("=12Q2q"), struct.Struct("=22q3q"), struct.Struct("=d")


class _Plan(NamedTuple):
    sizes: tuple[int, ...]
    tail: bytes
    state_shape: tuple[int, ...]
    workspace: tuple[int, int, int]  # bytes of kinds 0 to 2; -1: sizes not taken
    kept: int


_plans = _Plans()


def _plan(op: str, q, k, v, g, beta, init_state, cu_seqlens, lengths):
    """The call's plan, with q, k and v as the native calls read them."""
    key = (q.shape, k.shape, v.shape, g.shape, beta.shape, q.stride(), k.stride(), v.stride(), g.stride(),
           beta.stride(), q.dtype, k.dtype, v.dtype, g.dtype, beta.dtype, q.device, k.device, v.device, g.device,
           beta.device, None if init_state is None else (init_state.shape, init_state.dtype, init_state.device),
           None if cu_seqlens is None else (cu_seqlens.shape, cu_seqlens.dtype, cu_seqlens.device),
           None if lengths is None else (lengths.shape, lengths.dtype, lengths.device))
    plan = _plans.get(key)
    if plan is not None:
        return plan, q, k, v
    sizes = _check(op, q, k, v, g, beta, init_state, cu_seqlens, lengths)
    as_read = _rows(q), _rows(k), _rows(v)
    if any(a is not b for a, b in zip(as_read, (q, k, v))):
        return _plan(op, *as_read, g, beta, init_state, cu_seqlens, lengths)
    B, T, N, Hk, Hv, Dk, Dv = sizes
    packed = cu_seqlens is not None
    lib, code = nat.lib(), _code(q)
    tail = _TAIL.pack(*sizes, *(s for t in (q, k, v, g, beta) for s in t.stride()[:3]), code, _code(g), _code(beta))
    return _plans.keep(key, _Plan(
        sizes, tail, (N, Hv, Dk, Dv),
        tuple(lib.ramnet_delta_rule_workspace_bytes(*sizes, code, packed, kind) for kind in range(3)),
        lib.ramnet_delta_rule_kept_bytes(*sizes, code, packed))), q, k, v


def _forward(op: str, q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, init_state: Tensor | None,
             cu_seqlens: Tensor | None, lengths: Tensor | None, scale: float, state: Tensor | None = None,
             keep: bool = False, kept: Tensor | None = None) -> tuple[Tensor, Tensor, Tensor | None]:
    """(o, state, kept). ``state``: where the state goes (init_state itself in place);
    ``kept``: where what is kept goes."""
    plan, q, k, v = _plan(op, q, k, v, g, beta, init_state, cu_seqlens, lengths)
    if init_state is not None and init_state is not state and not (init_state.dtype == torch.float32
                                                                   and init_state.is_contiguous()):
        init_state = init_state.to(torch.float32).contiguous()
    if state is None:
        state = q.new_empty(plan.state_shape, dtype=torch.float32)
    o = q.new_empty(v.shape)
    n = _bytes(op, plan.workspace[keep], plan.sizes)
    kept_bytes = 0
    if keep:
        if kept is None:
            kept = q.new_empty((_bytes(op, plan.kept, plan.sizes),), dtype=torch.uint8)
        kept_bytes = kept.numel()
    ws = q.new_empty((n,), dtype=torch.uint8) if n else None
    if plan.sizes[2] == 0:
        return o.zero_(), state, kept
    cu_seqlens, lengths = _whole(cu_seqlens), _whole(lengths)
    with nat.on_device(q):
        nat.call("ramnet_delta_rule_forward", _HEAD.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), _ptr(init_state), state.data_ptr(),
            o.data_ptr(), _ptr(cu_seqlens), _ptr(lengths), _ptr(kept), _ptr(ws), kept_bytes, n) + plan.tail
            + _SCALE.pack(scale), nat.stream_of(q))
    return o, state, kept


def _ptr(t: Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


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
    op = "gated_delta_rule_kept"
    sizes = _check(op, q, k, v, g, beta, init_state, cu_seqlens, lengths)
    kept = q.new_empty((_kept_bytes(op, sizes, q.dtype, cu_seqlens is not None),), dtype=torch.uint8)
    return _forward(op, q, k, v, g, beta, init_state, cu_seqlens, lengths, scale, keep=True, kept=kept)


@gated_delta_rule_kept.register_fake
def _(q, k, v, g, beta, init_state, cu_seqlens, lengths, scale):
    B, T, Hk, Dk = q.shape
    N = B if cu_seqlens is None else cu_seqlens.shape[0] - 1
    n = _kept_bytes("gated_delta_rule_kept", (B, T, N, Hk, v.shape[2], Dk, v.shape[3]), q.dtype,
                    cu_seqlens is not None)
    return *_out_shapes(q, k, v, cu_seqlens), q.new_empty((n,), dtype=torch.uint8)


@torch.library.custom_op(f"{_NS}::gated_delta_rule_backward", mutates_args=(), device_types="cuda")
def gated_delta_rule_backward(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, cu_seqlens: Tensor | None,
                              lengths: Tensor | None, scale: float, kept: Tensor, d_o: Tensor,
                              d_state: Tensor | None) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """Gradients (dq, dk, dv, dg, dbeta, dinit) of ``gated_delta_rule_kept``."""
    return _gradients(q, k, v, g, beta, cu_seqlens, lengths, scale, kept, d_o, d_state)


def _gradients(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, cu_seqlens: Tensor | None,
               lengths: Tensor | None, scale: float, kept: Tensor, d_o: Tensor, d_state: Tensor | None) -> tuple:
    op = "gated_delta_rule_backward"
    plan, q, k, v = _plan(op, q, k, v, g, beta, None, cu_seqlens, lengths)
    B, T, N, Hk, Hv, Dk, Dv = plan.sizes
    _check_shapes(op, d_o=(d_o, (B, T, Hv, Dv)), d_state=(d_state, plan.state_shape))
    d_o = _rows(d_o.resolve_neg().to(q.dtype))
    if d_state is not None:
        d_state = d_state.resolve_neg().to(torch.float32).contiguous()
    grads = [torch.empty(t.shape, dtype=t.dtype, device=q.device) for t in (q, k, v, g, beta)]
    dinit = q.new_empty(plan.state_shape, dtype=torch.float32)
    n = _bytes(op, plan.workspace[2], plan.sizes)
    if N == 0 or T == 0 or B == 0:
        for t in grads:
            t.zero_()
        dinit.zero_() if d_state is None else dinit.copy_(d_state)
        return *grads, dinit
    ws = q.new_empty((n,), dtype=torch.uint8)
    cu_seqlens, lengths = _whole(cu_seqlens), _whole(lengths)
    with nat.on_device(q):
        nat.call("ramnet_delta_rule_backward", _HEAD.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), 0, 0, 0, _ptr(cu_seqlens),
            _ptr(lengths), kept.data_ptr(), ws.data_ptr(), kept.numel(), n) + plan.tail + _SCALE.pack(scale),
            d_o.data_ptr(), nat.strides(*d_o.stride()[:3]), nat.ptr(d_state), *(t.data_ptr() for t in grads),
            dinit.data_ptr(), nat.stream_of(q))
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


def _backward(ctx, d_o, d_state, d_kept, run=gated_delta_rule_backward):
    q, k, v, g, beta, cu_seqlens, lengths, kept = ctx.saved_tensors
    if d_o is None and d_state is None:
        return (None,) * 9
    if d_o is None:
        d_o = torch.zeros_like(v)
    *grads, dinit = run(q, k, v, g, beta, cu_seqlens, lengths, ctx.scale, kept, d_o, d_state)
    need = ctx.needs_input_grad
    return (*(t if n else None for t, n in zip(grads, need)),
            dinit.to(ctx.init_dtype) if need[5] else None, None, None, None)


gated_delta_rule_kept.register_autograd(_backward, setup_context=_setup)


class Trained(torch.autograd.Function):
    """``gated_delta_rule_kept`` for eager calls, beside the dispatcher (a
    training step of few tokens: 260 us with it, 208 so)."""

    @staticmethod
    def forward(ctx, *inputs):
        output = _forward("gated_delta_rule_kept", *inputs, keep=True)
        _setup(ctx, inputs, output)
        return output

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, d_state, d_kept):
        return _backward(ctx, d_o, d_state, d_kept, _gradients)


# --------------------------------------------------------------------------
# verification of drafted tokens

_verify_plans = _Plans()


def _verify_plan(key, tokens, target, draft, accept, sample, draft_lens):
    """(B, S, V, dtype code, strides) of a call, its tensors checked."""
    op = "verify_drafts"
    B, S = _dims(op, "tokens", tokens, 2)
    V = _dims(op, "target", target, 3)[2]
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
    for name, t in (("accept", accept), ("sample", sample)):
        if not t.dtype.is_floating_point:
            raise RuntimeError(f"{op}: {name} must be floating-point, got {t.dtype}")
    _require_gpu(op, target)
    for name, t in (("tokens", tokens), ("draft_lens", draft_lens)):
        if t is not None and t.dtype not in (torch.int32, torch.int64):
            raise RuntimeError(f"{op}: {name} must be int32 or int64, got {t.dtype}")
    at = target.stride()[:2] + (draft.stride()[:2] if draft is not None else (0, 0))
    return _verify_plans.keep(key, (B, S, V, _code(target), nat.strides(*at)))


def _as(t: Tensor, dtype: torch.dtype) -> Tensor:
    return t if t.dtype == dtype and t.is_contiguous() else t.to(dtype).contiguous()


def _verify(tokens: Tensor, target: Tensor, draft: Tensor | None, accept: Tensor, sample: Tensor,
            draft_lens: Tensor | None) -> tuple[Tensor, Tensor]:
    if target.dim() == 3:
        target = _dense(target)
    if draft is not None and draft.dim() == 3:
        draft = _dense(draft)
    key = (tokens.shape, target.shape, accept.shape, sample.shape, target.stride(), target.dtype, tokens.dtype,
           tokens.device, target.device, accept.device, sample.device, accept.dtype, sample.dtype,
           None if draft is None else (draft.shape, draft.stride(), draft.dtype, draft.device),
           None if draft_lens is None else (draft_lens.shape, draft_lens.dtype, draft_lens.device))
    plan = _verify_plans.get(key) or _verify_plan(key, tokens, target, draft, accept, sample, draft_lens)
    B, S, V, code, at = plan
    tokens, draft_lens = _as(tokens, torch.int64), _whole(draft_lens)
    accept, sample = _as(accept, torch.float32), _as(sample, torch.float32)
    out = tokens.new_empty((B, S + 1))
    taken = tokens.new_empty((B,), dtype=torch.int32)
    with nat.on_device(target):
        nat.call("ramnet_verify_drafts", tokens.data_ptr(), target.data_ptr(), nat.ptr(draft), code,
                 accept.data_ptr(), sample.data_ptr(), nat.ptr(draft_lens), B, S, V, at, out.data_ptr(),
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
