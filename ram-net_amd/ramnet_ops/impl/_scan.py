"""``torch.library`` operators of the short causal convolution and of the selective scan.

As with the gated delta rule, ``_conv``, ``_scan`` and their like make the native
calls, the operators registered around them serve tracing, autograd and
``torch.func``, and eager calls go beside the dispatcher.
"""
from __future__ import annotations

import struct
from typing import NamedTuple

import torch
from torch import Tensor

from .. import _native as nat
from ._delta import _as, _dense, _FLOATS, _Plans, _ptr, _whole
from ._ops import _check_shapes, _code, _dims, _NS, _require_gpu

_MAX_WIDTH, _MAX_STATES, _KEPT = 8, 64, 16


def _check_sequences(op: str, B: int, cu_seqlens: Tensor | None, lengths: Tensor | None) -> int:
    """How many sequences there are."""
    if lengths is not None and tuple(lengths.shape) != (B,):
        _check_shapes(op, lengths=(lengths, (B,)))
    for name, t in (("cu_seqlens", cu_seqlens), ("lengths", lengths)):
        if t is not None and t.dtype not in (torch.int32, torch.int64):
            raise RuntimeError(f"{op}: {name} must be int32 or int64, got {t.dtype}")
    if cu_seqlens is None:
        return B
    N = _dims(op, "cu_seqlens", cu_seqlens, 1)[0] - 1
    if B != 1 or lengths is not None:
        raise RuntimeError(f"{op}: sequences packed by cu_seqlens lie in a batch of one, without lengths")
    if N < 0:
        raise RuntimeError(f"{op}: cu_seqlens needs N + 1 bounds of N sequences")
    return N


def _check_devices(op: str, first: Tensor, *others: Tensor | None) -> None:
    for t in others:
        if t is not None and t.device != first.device:
            raise RuntimeError(f"{op}: tensors must share a device, got {t.device} beside {first.device}")
    _require_gpu(op, first)


def _key(*tensors: Tensor | None) -> tuple:
    return tuple([None if t is None else (t.shape, t.stride(), t.dtype, t.device) for t in tensors])


def _as_read(t: Tensor | None, dtype: torch.dtype) -> bool:
    """Whether a tensor that is read whole, as `dtype`, needs no copy."""
    return t is None or t.dtype == dtype and t.is_contiguous()


def _gradient(t: Tensor, dtype: torch.dtype) -> Tensor:
    """An output's gradient in the type and with the sign that memory has."""
    return t if t.dtype == dtype and not t.is_neg() else t.resolve_neg().to(dtype)


def _rows_of(t: Tensor) -> Tensor:
    """A tensor that the kernels read along its last dimension."""
    return _dense(t) if t.dim() else t


def _near_rows_of(t: Tensor) -> Tensor:
    """Likewise, its tokens (dimension 1) within the scan's reach of each other."""
    t = _rows_of(t)
    return t.contiguous() if t.dim() > 2 and t.stride(1) >= 2 ** 22 and t.shape[1] > 1 else t


# --------------------------------------------------------------------------
# short causal convolution

_CONV_HEAD, _CONV_TAIL = struct.Struct("=9Qq"), struct.Struct("=9q")


class _ConvPlan(NamedTuple):
    sizes: tuple[int, ...]       # B, T, N, D, W
    tails: tuple[bytes, bytes]   # without and with silu
    workspace: tuple[int, int]   # bytes of forward and backward
    plain: bool                  # whether all but x are read as they are


_conv_plans = _Plans()


def _conv_sizes(op: str, x, weight, bias, init_state, cu_seqlens, lengths) -> tuple[int, ...]:
    B, T, D = _dims(op, "x", x, 3)
    W = _dims(op, "weight", weight, 2)[1]
    _check_shapes(op, weight=(weight, (D, W)), bias=(bias, (D,)))
    if D == 0 or not 1 <= W <= _MAX_WIDTH:
        raise RuntimeError(f"{op}: needs channels and a weight of 1 to {_MAX_WIDTH} taps, got {tuple(weight.shape)}")
    N = _check_sequences(op, B, cu_seqlens, lengths)
    _check_shapes(op, init_state=(init_state, (N, W - 1, D)))
    if x.dtype not in _FLOATS or weight.dtype != x.dtype or bias is not None and bias.dtype != x.dtype:
        raise RuntimeError(f"{op}: x, weight and bias must share one of {_FLOATS}, got {x.dtype}, {weight.dtype} and "
                           f"{None if bias is None else bias.dtype}")
    if init_state is not None and init_state.dtype not in _FLOATS:
        raise RuntimeError(f"{op}: init_state must be one of {_FLOATS}, got {init_state.dtype}")
    _check_devices(op, x, weight, bias, init_state, cu_seqlens, lengths)
    return B, T, N, D, W


def _conv_plan(op: str, x, weight, bias, init_state, cu_seqlens, lengths) -> tuple[_ConvPlan, Tensor]:
    """The call's plan, with x as the native calls read it."""
    key = _key(x, weight, bias, init_state, cu_seqlens, lengths)
    plan = _conv_plans.get(key)
    if plan is not None:
        return plan, x
    sizes = _conv_sizes(op, x, weight, bias, init_state, cu_seqlens, lengths)
    rows = _rows_of(x)
    if rows is not x:
        return _conv_plan(op, rows, weight, bias, init_state, cu_seqlens, lengths)
    code, lib, packed = _code(x), nat.lib(), cu_seqlens is not None
    return _conv_plans.keep(key, _ConvPlan(
        sizes, tuple(_CONV_TAIL.pack(*sizes, *x.stride()[:2], code, silu) for silu in (0, 1)),
        tuple(_bytes_of(op, lib.ramnet_causal_conv_workspace_bytes(*sizes, code, packed, back), sizes)
              for back in (0, 1)),
        all(_as_read(t, x.dtype) for t in (weight, bias, init_state))
        and all(_as_read(t, torch.int32) for t in (cu_seqlens, lengths)))), x


def _conv_inputs(weight, bias, init_state, cu_seqlens, lengths, state=None) -> tuple:
    """Those that are read whole, as the native calls read them (a state updated in place as it is)."""
    return (weight.contiguous(), None if bias is None else bias.contiguous(),
            init_state if init_state is None or init_state is state else _as(init_state, weight.dtype),
            _whole(cu_seqlens), _whole(lengths))


def _bytes_of(op: str, count: int, sizes) -> int:
    if count < 0:
        raise RuntimeError(f"{op}: sizes {tuple(sizes)} are not supported (tokens within int32, channels below 2**22)")
    return count


def _conv(op: str, x: Tensor, weight: Tensor, bias: Tensor | None, init_state: Tensor | None,
          cu_seqlens: Tensor | None, lengths: Tensor | None, silu: bool,
          state: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """(y, state). ``state``: where the state goes (init_state itself in place)."""
    plan, x = _conv_plan(op, x, weight, bias, init_state, cu_seqlens, lengths)
    B, T, N, D, W = plan.sizes
    if not plan.plain:
        weight, bias, init_state, cu_seqlens, lengths = _conv_inputs(weight, bias, init_state, cu_seqlens, lengths, state)
    if state is None:
        state = x.new_empty((N, W - 1, D))
    y = x.new_empty((B, T, D))
    n = plan.workspace[0]
    ws = x.new_empty((n,), dtype=torch.uint8) if n else None
    with nat.on_device(x):
        nat.call("ramnet_causal_conv_forward", _CONV_HEAD.pack(
            x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(init_state), state.data_ptr(), y.data_ptr(),
            _ptr(cu_seqlens), _ptr(lengths), _ptr(ws), n) + plan.tails[silu], nat.stream_of(x))
    return y, state


def _conv_shapes(x, weight, cu_seqlens):
    N = x.shape[0] if cu_seqlens is None else cu_seqlens.shape[0] - 1
    return x.new_empty(x.shape), x.new_empty((N, weight.shape[1] - 1, x.shape[2]))


@torch.library.custom_op(f"{_NS}::causal_conv", mutates_args=(), device_types="cuda")
def causal_conv(x: Tensor, weight: Tensor, bias: Tensor | None, init_state: Tensor | None, cu_seqlens: Tensor | None,
                lengths: Tensor | None, silu: bool) -> tuple[Tensor, Tensor]:
    """(y, state)."""
    return _conv("causal_conv", x, weight, bias, init_state, cu_seqlens, lengths, silu)


@causal_conv.register_fake
def _(x, weight, bias, init_state, cu_seqlens, lengths, silu):
    return _conv_shapes(x, weight, cu_seqlens)


def _require_conv_state(op: str, x: Tensor, state: Tensor) -> None:
    if state.dtype != x.dtype or not state.is_contiguous():
        raise RuntimeError(f"{op}: a state updated in place must be contiguous and of x's type {x.dtype}, got "
                           f"{state.dtype}")


@torch.library.custom_op(f"{_NS}::causal_conv_", mutates_args=("state",), device_types="cuda")
def causal_conv_(x: Tensor, weight: Tensor, bias: Tensor | None, state: Tensor, cu_seqlens: Tensor | None,
                 lengths: Tensor | None, silu: bool) -> Tensor:
    """y; updates ``state`` in place."""
    _require_conv_state("causal_conv_", x, state)
    return _conv("causal_conv_", x, weight, bias, state, cu_seqlens, lengths, silu, state)[0]


@causal_conv_.register_fake
def _(x, weight, bias, state, cu_seqlens, lengths, silu):
    return x.new_empty(x.shape)


@torch.library.custom_op(f"{_NS}::causal_conv_backward", mutates_args=(), device_types="cuda")
def causal_conv_backward(x: Tensor, weight: Tensor, bias: Tensor | None, init_state: Tensor | None,
                         cu_seqlens: Tensor | None, lengths: Tensor | None, silu: bool, d_y: Tensor,
                         d_state: Tensor | None) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """Gradients (dx, dweight, dbias, dinit) of ``causal_conv``."""
    return _conv_gradients(x, weight, bias, init_state, cu_seqlens, lengths, silu, d_y, d_state)


def _conv_gradients(x, weight, bias, init_state, cu_seqlens, lengths, silu, d_y, d_state) -> tuple:
    op = "causal_conv_backward"
    plan, x = _conv_plan(op, x, weight, bias, init_state, cu_seqlens, lengths)
    B, T, N, D, W = plan.sizes
    _check_shapes(op, d_y=(d_y, (B, T, D)), d_state=(d_state, (N, W - 1, D)))
    d_y = _rows_of(_gradient(d_y, x.dtype))
    if d_state is not None:
        d_state = _gradient(d_state, x.dtype).contiguous()
    dx, dweight, dbias, dinit = x.new_empty((B, T, D)), x.new_empty((D, W)), x.new_empty((D,)), x.new_empty((N, W - 1, D))
    if B == 0:
        return dx, dweight.zero_(), dbias.zero_(), dinit
    if not plan.plain:
        weight, bias, init_state, cu_seqlens, lengths = _conv_inputs(weight, bias, init_state, cu_seqlens, lengths)
    n = plan.workspace[1]
    ws = x.new_empty((n,), dtype=torch.uint8)
    with nat.on_device(x):
        nat.call("ramnet_causal_conv_backward", _CONV_HEAD.pack(
            x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(init_state), 0, 0, _ptr(cu_seqlens), _ptr(lengths),
            ws.data_ptr(), n) + plan.tails[silu], d_y.data_ptr(), nat.strides(*d_y.stride()[:2]), nat.ptr(d_state),
            dx.data_ptr(), dweight.data_ptr(), dbias.data_ptr(), dinit.data_ptr(), nat.stream_of(x))
    return dx, dweight, dbias, dinit


@causal_conv_backward.register_fake
def _(x, weight, bias, init_state, cu_seqlens, lengths, silu, d_y, d_state):
    return (x.new_empty(x.shape), weight.new_empty(weight.shape), x.new_empty((x.shape[2],)),
            _conv_shapes(x, weight, cu_seqlens)[1])


def _conv_setup(ctx, inputs, output):
    x, weight, bias, init_state, cu_seqlens, lengths, silu = inputs
    ctx.silu = silu
    ctx.save_for_backward(x, weight, bias, init_state, cu_seqlens, lengths)
    ctx.set_materialize_grads(False)


def _conv_backward(ctx, d_y, d_state, run=causal_conv_backward):
    x, weight, bias, init_state, cu_seqlens, lengths = ctx.saved_tensors
    if d_y is None and d_state is None:
        return (None,) * 7
    if d_y is None:
        d_y = torch.zeros_like(x)
    dx, dweight, dbias, dinit = run(x, weight, bias, init_state, cu_seqlens, lengths, ctx.silu, d_y, d_state)
    need = ctx.needs_input_grad
    return (dx if need[0] else None, dweight if need[1] else None, dbias if need[2] else None,
            dinit.to(init_state.dtype) if need[3] else None, None, None, None)


causal_conv.register_autograd(_conv_backward, setup_context=_conv_setup)


class TrainedConv(torch.autograd.Function):
    """``causal_conv`` for eager calls that want gradients, beside the dispatcher."""

    @staticmethod
    def forward(ctx, *inputs):
        output = _conv("causal_conv", *inputs)
        _conv_setup(ctx, inputs, output)
        return output

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y, d_state):
        return _conv_backward(ctx, d_y, d_state, _conv_gradients)


# --------------------------------------------------------------------------
# selective scan

_SCAN_HEAD, _SCAN_TAIL = struct.Struct("=15Q2q"), struct.Struct("=20q")


class _ScanPlan(NamedTuple):
    sizes: tuple[int, ...]             # B, T, N, D, S, G
    tails: tuple[bytes, bytes]         # without and with softplus
    workspace: tuple[int, int, int]    # bytes of kinds 0 to 2
    kept: int
    plain: bool                        # whether all but x, dt, B, C and gate are read as they are


_scan_plans = _Plans()


def _scan_sizes(op: str, x, dt, A, B, C, skip, gate, dt_bias, init_state, cu_seqlens, lengths) -> tuple[int, ...]:
    batch, T, D = _dims(op, "x", x, 3)
    G, S = _dims(op, "B", B, 4)[2:]
    _check_shapes(op, dt=(dt, (batch, T, D)), A=(A, (D, S)), B=(B, (batch, T, G, S)), C=(C, (batch, T, G, S)),
                  skip=(skip, (D,)), gate=(gate, (batch, T, D)), dt_bias=(dt_bias, (D,)))
    if D == 0 or G == 0 or D % G or not 1 <= S <= _MAX_STATES:
        raise RuntimeError(f"{op}: the channels of x must be a multiple of the groups of B and C, none 0, with 1 to "
                           f"{_MAX_STATES} states, got x {tuple(x.shape)} and B {tuple(B.shape)}")
    N = _check_sequences(op, batch, cu_seqlens, lengths)
    _check_shapes(op, init_state=(init_state, (N, D, S)))
    if x.dtype not in _FLOATS or any(t is not None and t.dtype != x.dtype for t in (dt, B, C, gate)):
        raise RuntimeError(f"{op}: x, dt, B, C and gate must share one of {_FLOATS}, got {x.dtype}, {dt.dtype}, "
                           f"{B.dtype}, {C.dtype} and {None if gate is None else gate.dtype}")
    for name, t in (("A", A), ("skip", skip), ("dt_bias", dt_bias), ("init_state", init_state)):
        if t is not None and t.dtype not in _FLOATS:
            raise RuntimeError(f"{op}: {name} must be one of {_FLOATS}, got {t.dtype}")
    _check_devices(op, x, dt, A, B, C, skip, gate, dt_bias, init_state, cu_seqlens, lengths)
    return batch, T, N, D, S, G


def _scan_plan(op: str, x, dt, A, B, C, skip, gate, dt_bias, init_state, cu_seqlens, lengths) -> tuple[_ScanPlan, tuple]:
    """The call's plan, with x, dt, B, C and gate as the native calls read them."""
    key = _key(x, dt, A, B, C, skip, gate, dt_bias, init_state, cu_seqlens, lengths)
    plan = _scan_plans.get(key)
    if plan is not None:
        return plan, (x, dt, B, C, gate)
    sizes = _scan_sizes(op, x, dt, A, B, C, skip, gate, dt_bias, init_state, cu_seqlens, lengths)
    rows = tuple(None if t is None else _near_rows_of(t) for t in (x, dt, B, C, gate))
    if any(a is not b for a, b in zip(rows, (x, dt, B, C, gate))):
        x, dt, B, C, gate = rows
        return _scan_plan(op, x, dt, A, B, C, skip, gate, dt_bias, init_state, cu_seqlens, lengths)
    lib, packed = nat.lib(), cu_seqlens is not None
    strides = (*x.stride()[:2], *dt.stride()[:2], *(gate.stride()[:2] if gate is not None else (0, 0)),
               *B.stride()[:3], *C.stride()[:3])
    return _scan_plans.keep(key, _ScanPlan(
        sizes, tuple(_SCAN_TAIL.pack(*sizes, *strides, _code(x), softplus) for softplus in (0, 1)),
        tuple(_bytes_of(op, lib.ramnet_selective_scan_workspace_bytes(*sizes, packed, kind), sizes)
              for kind in range(3)),
        _bytes_of(op, lib.ramnet_selective_scan_kept_bytes(*sizes, packed), sizes),
        all(_as_read(t, torch.float32) for t in (A, skip, dt_bias, init_state))
        and all(_as_read(t, torch.int32) for t in (cu_seqlens, lengths)))), rows


def _kept_bytes(sizes, packed: bool):
    """ramnet_selective_scan_kept_bytes in arithmetic that tracing leaves symbolic."""
    batch, T, N, D, S, _ = sizes
    slots = T // _KEPT + N + 1 if packed else batch * ((T + _KEPT - 1) // _KEPT)
    return slots * D * 16 * next(w for w in (1, 2, 3, 4, 6, 8, 12, 16) if S <= 4 * w)


def _head(x, dt, gate, B, C, A, skip, dt_bias, init_state, state, y, cu_seqlens, lengths, kept, ws) -> bytes:
    return _SCAN_HEAD.pack(
        x.data_ptr(), dt.data_ptr(), _ptr(gate), B.data_ptr(), C.data_ptr(), A.data_ptr(), _ptr(skip), _ptr(dt_bias),
        _ptr(init_state), _ptr(state), _ptr(y), _ptr(cu_seqlens), _ptr(lengths), _ptr(kept), _ptr(ws),
        0 if kept is None else kept.numel(), 0 if ws is None else ws.numel())


def _parameter(t: Tensor | None) -> Tensor | None:
    return None if t is None else _as(t, torch.float32)


def _scan(op: str, x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, skip: Tensor | None, gate: Tensor | None,
          dt_bias: Tensor | None, init_state: Tensor | None, cu_seqlens: Tensor | None, lengths: Tensor | None,
          softplus: bool, state: Tensor | None = None, keep: bool = False) -> tuple[Tensor, Tensor, Tensor | None]:
    """(y, state, kept). ``state``: where the state goes (init_state itself in place)."""
    plan, (x, dt, B, C, gate) = _scan_plan(op, x, dt, A, B, C, skip, gate, dt_bias, init_state, cu_seqlens, lengths)
    batch, T, N, D, S, G = plan.sizes
    if not plan.plain:
        A, skip, dt_bias = _parameter(A), _parameter(skip), _parameter(dt_bias)
        init_state = init_state if init_state is state else _parameter(init_state)
        cu_seqlens, lengths = _whole(cu_seqlens), _whole(lengths)
    if state is None:
        state = x.new_empty((N, D, S), dtype=torch.float32)
    y = x.new_empty((batch, T, D))
    kept = x.new_empty((plan.kept,), dtype=torch.uint8) if keep else None
    n = plan.workspace[keep]
    ws = x.new_empty((n,), dtype=torch.uint8) if n else None
    with nat.on_device(x):
        nat.call("ramnet_selective_scan_forward", _head(
            x, dt, gate, B, C, A, skip, dt_bias, init_state, state, y, cu_seqlens, lengths, kept, ws)
            + plan.tails[softplus], nat.stream_of(x))
    return y, state, kept


def _scan_shapes(x, B, cu_seqlens):
    N = x.shape[0] if cu_seqlens is None else cu_seqlens.shape[0] - 1
    return x.new_empty(x.shape), x.new_empty((N, x.shape[2], B.shape[3]), dtype=torch.float32)


@torch.library.custom_op(f"{_NS}::selective_scan", mutates_args=(), device_types="cuda")
def selective_scan(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, skip: Tensor | None, gate: Tensor | None,
                   dt_bias: Tensor | None, init_state: Tensor | None, cu_seqlens: Tensor | None,
                   lengths: Tensor | None, softplus: bool) -> tuple[Tensor, Tensor]:
    """(y, state); no gradients (``selective_scan_kept`` has them)."""
    return _scan("selective_scan", x, dt, A, B, C, skip, gate, dt_bias, init_state, cu_seqlens, lengths, softplus)[:2]


@selective_scan.register_fake
def _(x, dt, A, B, C, skip, gate, dt_bias, init_state, cu_seqlens, lengths, softplus):
    return _scan_shapes(x, B, cu_seqlens)


def _require_scan_state(op: str, state: Tensor) -> None:
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise RuntimeError(f"{op}: a state updated in place must be contiguous float32, got {state.dtype}")


@torch.library.custom_op(f"{_NS}::selective_scan_", mutates_args=("state",), device_types="cuda")
def selective_scan_(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, skip: Tensor | None, gate: Tensor | None,
                    dt_bias: Tensor | None, state: Tensor, cu_seqlens: Tensor | None, lengths: Tensor | None,
                    softplus: bool) -> Tensor:
    """y; updates ``state`` in place."""
    _require_scan_state("selective_scan_", state)
    return _scan("selective_scan_", x, dt, A, B, C, skip, gate, dt_bias, state, cu_seqlens, lengths, softplus, state)[0]


@selective_scan_.register_fake
def _(x, dt, A, B, C, skip, gate, dt_bias, state, cu_seqlens, lengths, softplus):
    return x.new_empty(x.shape)


@torch.library.custom_op(f"{_NS}::selective_scan_kept", mutates_args=(), device_types="cuda")
def selective_scan_kept(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, skip: Tensor | None,
                        gate: Tensor | None, dt_bias: Tensor | None, init_state: Tensor | None,
                        cu_seqlens: Tensor | None, lengths: Tensor | None,
                        softplus: bool) -> tuple[Tensor, Tensor, Tensor]:
    """(y, state, kept): ``selective_scan`` that leaves its backward the state before every 16 tokens."""
    return _scan("selective_scan_kept", x, dt, A, B, C, skip, gate, dt_bias, init_state, cu_seqlens, lengths, softplus,
                 keep=True)


@selective_scan_kept.register_fake
def _(x, dt, A, B, C, skip, gate, dt_bias, init_state, cu_seqlens, lengths, softplus):
    y, state = _scan_shapes(x, B, cu_seqlens)
    sizes = (*x.shape[:2], state.shape[0], x.shape[2], B.shape[3], B.shape[2])
    return y, state, x.new_empty((_kept_bytes(sizes, cu_seqlens is not None),), dtype=torch.uint8)


@torch.library.custom_op(f"{_NS}::selective_scan_backward", mutates_args=(), device_types="cuda")
def selective_scan_backward(
        x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, skip: Tensor | None, gate: Tensor | None,
        dt_bias: Tensor | None, cu_seqlens: Tensor | None, lengths: Tensor | None, softplus: bool, sequences: int,
        kept: Tensor, d_y: Tensor, d_state: Tensor | None,
) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """Gradients (dx, ddt, dA, dB, dC, dskip, dgate, dbias, dinit) of ``selective_scan_kept``."""
    return _scan_gradients(x, dt, A, B, C, skip, gate, dt_bias, cu_seqlens, lengths, softplus, sequences, kept, d_y,
                           d_state)


def _scan_gradients(x, dt, A, B, C, skip, gate, dt_bias, cu_seqlens, lengths, softplus, sequences, kept, d_y,
                    d_state) -> tuple:
    op = "selective_scan_backward"
    plan, (x, dt, B, C, gate) = _scan_plan(op, x, dt, A, B, C, skip, gate, dt_bias, None, cu_seqlens, lengths)
    batch, T, N, D, S, G = plan.sizes
    _check_shapes(op, d_y=(d_y, (batch, T, D)), d_state=(d_state, (N, D, S)))
    d_y = _near_rows_of(_gradient(d_y, x.dtype))
    if d_state is not None:
        d_state = _gradient(d_state, torch.float32).contiguous()
    dx, ddt, dgate = x.new_empty((batch, T, D)), x.new_empty((batch, T, D)), x.new_empty((batch, T, D))
    dB, dC = x.new_empty((batch, T, G, S)), x.new_empty((batch, T, G, S))
    if not plan.plain:
        A, skip, dt_bias = _parameter(A), _parameter(skip), _parameter(dt_bias)
        cu_seqlens, lengths = _whole(cu_seqlens), _whole(lengths)
    dA, dskip, dbias = A.new_empty((D, S)), A.new_empty((D,)), A.new_empty((D,))
    dinit = A.new_empty((N, D, S))
    if batch * T == 0 or N == 0:
        for t in (dx, ddt, dgate, dB, dC, dA, dskip, dbias):
            t.zero_()
        dinit.zero_() if d_state is None else dinit.copy_(d_state)
        return dx, ddt, dA, dB, dC, dskip, dgate, dbias, dinit
    if gate is None:
        dgate.zero_()
    n = plan.workspace[2]
    ws = x.new_empty((n,), dtype=torch.uint8)
    with nat.on_device(x):
        nat.call("ramnet_selective_scan_backward", _head(
            x, dt, gate, B, C, A, skip, dt_bias, None, None, None, cu_seqlens, lengths, kept, ws)
            + plan.tails[softplus], d_y.data_ptr(), nat.strides(*d_y.stride()[:2]), nat.ptr(d_state),
            *(t.data_ptr() for t in (dx, ddt, dgate, dB, dC, dA, dskip, dbias, dinit)), nat.stream_of(x))
    return dx, ddt, dA, dB, dC, dskip, dgate, dbias, dinit


@selective_scan_backward.register_fake
def _(x, dt, A, B, C, skip, gate, dt_bias, cu_seqlens, lengths, softplus, sequences, kept, d_y, d_state):
    D, S = A.shape

    def wide(*shape):
        return A.new_empty(shape, dtype=torch.float32)
    return (x.new_empty(x.shape), x.new_empty(x.shape), wide(D, S), B.new_empty(B.shape), C.new_empty(C.shape), wide(D),
            x.new_empty(x.shape), wide(D), wide(sequences, D, S))


def _scan_setup(ctx, inputs, output):
    x, dt, A, B, C, skip, gate, dt_bias, init_state, cu_seqlens, lengths, softplus = inputs
    ctx.softplus, ctx.sequences = softplus, output[1].shape[0]
    ctx.init_dtype = None if init_state is None else init_state.dtype
    ctx.save_for_backward(x, dt, A, B, C, skip, gate, dt_bias, cu_seqlens, lengths, output[2])
    ctx.mark_non_differentiable(output[2])
    ctx.set_materialize_grads(False)


def _scan_backward(ctx, d_y, d_state, d_kept, run=selective_scan_backward):
    x, dt, A, B, C, skip, gate, dt_bias, cu_seqlens, lengths, kept = ctx.saved_tensors
    if d_y is None and d_state is None:
        return (None,) * 12
    if d_y is None:
        d_y = torch.zeros_like(x)
    dx, ddt, dA, dB, dC, dskip, dgate, dbias, dinit = run(
        x, dt, A, B, C, skip, gate, dt_bias, cu_seqlens, lengths, ctx.softplus, ctx.sequences, kept, d_y, d_state)
    need = ctx.needs_input_grad

    def of(i, grad, dtype):
        return grad.to(dtype) if need[i] else None
    return (of(0, dx, x.dtype), of(1, ddt, x.dtype), of(2, dA, A.dtype), of(3, dB, x.dtype), of(4, dC, x.dtype),
            of(5, dskip, skip.dtype) if skip is not None else None, of(6, dgate, x.dtype),
            of(7, dbias, dt_bias.dtype) if dt_bias is not None else None, of(8, dinit, ctx.init_dtype),
            None, None, None)


selective_scan_kept.register_autograd(_scan_backward, setup_context=_scan_setup)


class TrainedScan(torch.autograd.Function):
    """``selective_scan_kept`` for eager calls, beside the dispatcher."""

    @staticmethod
    def forward(ctx, *inputs):
        output = _scan("selective_scan_kept", *inputs, keep=True)
        _scan_setup(ctx, inputs, output)
        return output

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y, d_state, d_kept):
        return _scan_backward(ctx, d_y, d_state, d_kept, _scan_gradients)
