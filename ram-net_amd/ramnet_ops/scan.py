"""Public API of the short causal convolution and of the selective scan.

The reference has neither; both follow this package's rules, as the gated delta
rule does (``delta_rule.py``).
"""
from __future__ import annotations

import torch

from .delta_rule import _delta, _require_tensors
from .ram_attn import _unavailable

try:
    from .impl import _scan
except ImportError:  # library not built: fail at call time
    _scan = None


def causal_conv(
        x: torch.Tensor,
        weight: torch.Tensor,
        bias: torch.Tensor | None = None,
        activation: str | None = None,
        init_state: torch.Tensor | None = None,
        cu_seqlens: torch.Tensor | None = None,
        lengths: torch.Tensor | None = None,
        inplace: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Causal convolution of each channel over its last W tokens, for prompts and for single tokens.

    ``s[t, d] = bias[d] + sum_j weight[d, j] x[t - (W - 1) + j, d]`` and y is s, or silu(s). Inputs before a
    sequence's first token are those of its state. Differentiable in x, weight, bias and init_state.

    :param x: Inputs (B, T, D); last dimension dense, any other strides.
    :param weight: Taps (D, W), the last one of the token itself; W up to 8; x's type.
    :param bias: (D) in x's type.
    :param activation: ``"silu"`` or None.
    :param init_state: The W - 1 inputs before the first token (N, W - 1, D), a float type of 32 bits or fewer;
        default zeros.
    :param cu_seqlens: (N + 1) bounds of N sequences packed one after the other in a batch of one.
    :param lengths: (B) tokens of each row that count; the others leave the state and have y = 0.
    :param inplace: Update init_state in place (contiguous, of x's type, no gradients).
    :return: ``(y, state)``: (B, T, D) and (N, W - 1, D) in x's type. N is B without cu_seqlens.
    """
    if _scan is None:
        raise _unavailable("causal_conv")
    eager = _delta.is_eager(x, weight, bias, init_state, cu_seqlens, lengths)
    if not eager or x is None or weight is None:
        _require_tensors("x weight bias init_state cu_seqlens lengths", 2, x, weight, bias, init_state, cu_seqlens,
                         lengths)
    if activation is not None and activation != "silu":
        raise ValueError(f"`activation` must be 'silu' or None, got {activation!r}.")
    silu = activation is not None
    if inplace and init_state is None:
        raise ValueError("`inplace` needs an init_state to update.")
    grad = _delta.wants_grad(x, weight, bias, init_state)
    if inplace:
        if grad:
            raise ValueError("`inplace` has no gradients.")
        if eager:
            _scan._require_conv_state("causal_conv", x, init_state)
            out = _scan._conv("causal_conv", x, weight, bias, init_state, cu_seqlens, lengths, silu, init_state)
            torch.autograd.graph.increment_version(init_state)  # (as the dispatcher does)
            return out
        return _scan.causal_conv_(x, weight, bias, init_state, cu_seqlens, lengths, silu), init_state
    if eager:
        run = _scan.TrainedConv.apply if grad else lambda *inputs: _scan._conv("causal_conv", *inputs)
    else:
        run = _scan.causal_conv
    return run(x, weight, bias, init_state, cu_seqlens, lengths, silu)


def selective_scan(
        x: torch.Tensor,
        dt: torch.Tensor,
        A: torch.Tensor,
        B: torch.Tensor,
        C: torch.Tensor,
        skip: torch.Tensor | None = None,
        gate: torch.Tensor | None = None,
        dt_bias: torch.Tensor | None = None,
        softplus: bool = False,
        init_state: torch.Tensor | None = None,
        cu_seqlens: torch.Tensor | None = None,
        lengths: torch.Tensor | None = None,
        inplace: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Selective scan: S numbers of state per sequence and channel, each with a decay of its own.

    Per token and channel d of group g: ``dt = softplus(dt + dt_bias)``,
    ``h = exp(dt A[d]) h + dt x B[g]``, ``y = C[g] . h + skip x``, times silu(gate). Differentiable in x, dt, A, B,
    C, skip, gate, dt_bias and init_state. States and sums are in 32 bits.

    :param x: Inputs (batch, T, D); last dimension dense, any other strides, as for dt, B, C and gate.
    :param dt: Step of each token and channel (batch, T, D), before dt_bias and the softplus.
    :param A: Rates (D, S), below 0 for decays; S up to 64; a float type of 32 bits or fewer, used in
        32, as for skip and dt_bias.
    :param B: What the state takes up (batch, T, G, S); channel d reads group ``d // (D // G)``.
    :param C: What is read of it (batch, T, G, S).
    :param skip: Share of x in y (D).
    :param gate: (batch, T, D).
    :param dt_bias: (D).
    :param softplus: Whether dt goes through a softplus.
    :param init_state: State before the first token (N, D, S), a float type of 32 bits or fewer; default zeros.
    :param cu_seqlens: (N + 1) bounds of N sequences packed one after the other in a batch of one.
    :param lengths: (batch) tokens of each row that count; the others leave the state and have y = 0.
    :param inplace: Update init_state in place (contiguous float32, no gradients).
    :return: ``(y, state)``: (batch, T, D) in x's type and (N, D, S) float32. N is the batch without cu_seqlens.
    """
    if _scan is None:
        raise _unavailable("selective_scan")
    eager = _delta.is_eager(x, dt, A, B, C, skip, gate, dt_bias, init_state, cu_seqlens, lengths)
    if not eager or x is None or dt is None or A is None or B is None or C is None:
        _require_tensors("x dt A B C skip gate dt_bias init_state cu_seqlens lengths", 5, x, dt, A, B, C, skip, gate,
                         dt_bias, init_state, cu_seqlens, lengths)
    softplus = bool(softplus)
    if inplace and init_state is None:
        raise ValueError("`inplace` needs an init_state to update.")
    grad = _delta.wants_grad(x, dt, A, B, C, skip, gate, dt_bias, init_state)
    if inplace:
        if grad:
            raise ValueError("`inplace` has no gradients.")
        if eager:
            _scan._require_scan_state("selective_scan", init_state)
            out = _scan._scan("selective_scan", x, dt, A, B, C, skip, gate, dt_bias, init_state, cu_seqlens, lengths,
                              softplus, init_state)[:2]
            torch.autograd.graph.increment_version(init_state)  # (as the dispatcher does)
            return out
        return _scan.selective_scan_(x, dt, A, B, C, skip, gate, dt_bias, init_state, cu_seqlens, lengths,
                                     softplus), init_state
    inputs = (x, dt, A, B, C, skip, gate, dt_bias, init_state, cu_seqlens, lengths, softplus)
    if grad:
        run = _scan.TrainedScan.apply if eager else _scan.selective_scan_kept
        return run(*inputs)[:2]
    return _scan._scan("selective_scan", *inputs)[:2] if eager else _scan.selective_scan(*inputs)
