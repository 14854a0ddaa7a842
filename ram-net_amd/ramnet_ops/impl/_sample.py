"""``torch.library`` operator of token sampling, and its native call."""
from __future__ import annotations

import struct

import torch
from torch import Tensor

from .. import _native as nat
from ._delta import _as, _dense, _FLOATS, _ptr
from ._ops import _check_shapes, _code, _NS, _require_gpu

# ramnet_sample_tokens_call
_CALL = struct.Struct("=8Q3d5q")


def _rows(op: str, name: str, t: Tensor | None, shape, dtype: torch.dtype) -> Tensor | None:
    """A setting of each row, one number a row."""
    if t is None:
        return None
    try:
        t = t.expand(shape)
    except RuntimeError:
        raise RuntimeError(f"{op}: {name} must broadcast to the rows {tuple(shape)}, got {tuple(t.shape)}") from None
    return _as(t, dtype)


def _sample(op: str, logits: Tensor, random: Tensor | None, temperature: Tensor | None, top_k: Tensor | None,
            top_p: Tensor | None, min_p: Tensor | None, temperature_of_all: float, top_k_of_all: int,
            top_p_of_all: float, min_p_of_all: float, probabilities: bool) -> tuple[Tensor | None, Tensor | None]:
    """(tokens or None, probabilities or None)."""
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise RuntimeError(f"{op}: logits need a vocabulary in their last dimension, got shape {tuple(logits.shape)}")
    *rows, V = logits.shape
    if logits.dtype not in _FLOATS:
        raise RuntimeError(f"{op}: logits must be one of {_FLOATS}, got {logits.dtype}")
    if random is not None:
        _check_shapes(op, random=(random, tuple(rows)))
    for name, t in (("random", random), ("temperature", temperature), ("top_p", top_p), ("min_p", min_p)):
        if t is not None and not t.dtype.is_floating_point:
            raise RuntimeError(f"{op}: {name} must be floating-point, got {t.dtype}")
    if top_k is not None and top_k.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"{op}: top_k must be int32 or int64, got {top_k.dtype}")
    for t in (random, temperature, top_k, top_p, min_p):
        if t is not None and t.device != logits.device:
            raise RuntimeError(f"{op}: tensors must share a device, got {t.device} beside {logits.device}")
    _require_gpu(op, logits)
    flat = _dense(logits.reshape(-1, V)) if len(rows) != 1 else _dense(logits)
    R = flat.shape[0]
    if random is not None:
        random = _as(random, torch.float32)
    temperature, top_p = _rows(op, "temperature", temperature, rows, torch.float32), _rows(op, "top_p", top_p, rows, torch.float32)
    min_p = _rows(op, "min_p", min_p, rows, torch.float32)
    if top_k is not None:  # (more than the vocabulary is all of it)
        top_k = _rows(op, "top_k", top_k.clamp(0, V) if top_k.dtype == torch.int64 else top_k, rows, torch.int32)
    tokens = logits.new_empty(rows, dtype=torch.int64) if random is not None else None
    probs = logits.new_empty((*rows, V), dtype=torch.float32) if probabilities else None
    with nat.on_device(logits):
        nat.call("ramnet_sample_tokens", _CALL.pack(
            flat.data_ptr(), _ptr(random), _ptr(temperature), _ptr(top_p), _ptr(min_p), _ptr(top_k), _ptr(tokens),
            _ptr(probs), temperature_of_all, top_p_of_all, min_p_of_all, top_k_of_all, R, V,
            flat.stride(0) if R > 1 else V, _code(flat)), nat.stream_of(logits))
    return tokens, probs


@torch.library.custom_op(f"{_NS}::sample_tokens", mutates_args=(), device_types="cuda")
def sample_tokens(logits: Tensor, random: Tensor, temperature: Tensor | None, top_k: Tensor | None,
                  top_p: Tensor | None, min_p: Tensor | None, temperature_of_all: float, top_k_of_all: int,
                  top_p_of_all: float, min_p_of_all: float) -> Tensor:
    """Tokens. A setting is a tensor, of the rows, or the number of all beside it."""
    return _sample("sample_tokens", logits, random, temperature, top_k, top_p, min_p, temperature_of_all, top_k_of_all,
                   top_p_of_all, min_p_of_all, False)[0]


@sample_tokens.register_fake
def _(logits, random, *settings):
    return logits.new_empty(logits.shape[:-1], dtype=torch.int64)


@torch.library.custom_op(f"{_NS}::sample_tokens_with_probabilities", mutates_args=(), device_types="cuda")
def sample_tokens_with_probabilities(
        logits: Tensor, random: Tensor, temperature: Tensor | None, top_k: Tensor | None, top_p: Tensor | None,
        min_p: Tensor | None, temperature_of_all: float, top_k_of_all: int, top_p_of_all: float,
        min_p_of_all: float) -> tuple[Tensor, Tensor]:
    """(tokens, probabilities)."""
    return _sample("sample_tokens", logits, random, temperature, top_k, top_p, min_p, temperature_of_all, top_k_of_all,
                   top_p_of_all, min_p_of_all, True)


@sample_tokens_with_probabilities.register_fake
def _(logits, random, *settings):
    return logits.new_empty(logits.shape[:-1], dtype=torch.int64), logits.new_empty(logits.shape, dtype=torch.float32)


@torch.library.custom_op(f"{_NS}::token_probabilities", mutates_args=(), device_types="cuda")
def token_probabilities(logits: Tensor, temperature: Tensor | None, top_k: Tensor | None, top_p: Tensor | None,
                        min_p: Tensor | None, temperature_of_all: float, top_k_of_all: int, top_p_of_all: float,
                        min_p_of_all: float) -> Tensor:
    """Probabilities."""
    return _sample("token_probabilities", logits, None, temperature, top_k, top_p, min_p, temperature_of_all,
                   top_k_of_all, top_p_of_all, min_p_of_all, True)[1]


@token_probabilities.register_fake
def _(logits, *settings):
    return logits.new_empty(logits.shape, dtype=torch.float32)
