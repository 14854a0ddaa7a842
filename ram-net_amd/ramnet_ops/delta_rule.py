"""Public API of the gated delta rule and of draft verification.

The reference has neither; both follow this package's rules: argument errors
before any launch (``TypeError`` for wrong kinds, ``ValueError`` for wrong
choices, ``RuntimeError`` for tensors the kernels do not take), work on the
current stream of the inputs' device, no fallback.
"""
from __future__ import annotations

import torch

from .ram_attn import _unavailable

try:
    from .impl import _delta
    _delta_error: Exception | None = None
except ImportError as exc:  # library not built: fail at call time
    _delta = None
    _delta_error = exc


def _require_tensors(names: str, needed: int, *tensors) -> None:
    """TypeError unless the first `needed` are tensors and the others are or are None."""
    for i, (name, t) in enumerate(zip(names.split(), tensors)):
        if not isinstance(t, torch.Tensor) and (t is not None or i < needed):
            raise TypeError(f"Expected {name} to be a Tensor{' or None' if i >= needed else ''}, "
                            f"got {type(t).__name__}.")


def gated_delta_rule(
        q: torch.Tensor,
        k: torch.Tensor,
        v: torch.Tensor,
        g: torch.Tensor,
        beta: torch.Tensor,
        scale: float | None = None,
        init_state: torch.Tensor | None = None,
        cu_seqlens: torch.Tensor | None = None,
        lengths: torch.Tensor | None = None,
        inplace: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Gated delta rule: one (Dk, Dv) state per sequence and value head.

    Per token: ``S = exp(g) S``, ``S = S + k (beta (v - S^T k))^T``, ``o = scale S^T q``.
    Differentiable in q, k, v, g, beta and init_state. Whole prompts run in
    chunks of 64 tokens, decode steps and short prompts (up to 8 tokens) token by
    token. In chunks, values far below the largest of their column of v within a
    chunk (2^-15 and less) have fewer than 24 bits, and a NaN or infinity reaches
    the tokens of its chunk before it as well as those after (one in v: its column).

    :param q: Queries (B, T, Hk, Dk), Dk up to 256; their last dimension dense, any other strides.
    :param k: Keys (B, T, Hk, Dk), as a rule of norm 1.
    :param v: Values (B, T, Hv, Dv); value head h reads key head ``h // (Hv // Hk)``.
    :param g: Logarithm of the decay (B, T, Hv), any float type; -inf clears the state.
    :param beta: Write strength (B, T, Hv).
    :param scale: Factor of o; default ``Dk ** -0.5``.
    :param init_state: State before the first token (N, Hv, Dk, Dv), a float type of 32 bits or fewer; default zeros.
    :param cu_seqlens: (N + 1) bounds of N sequences packed one after the other in a batch of one.
    :param lengths: (B) tokens of each row that count; the others leave the state and have o = 0.
    :param inplace: Update init_state in place (contiguous float32, no gradients).
    :return: ``(o, state)``: (B, T, Hv, Dv) in v's type and (N, Hv, Dk, Dv) float32. N is B without cu_seqlens.
    """
    if _delta is None:
        raise _unavailable("gated_delta_rule")
    eager = _delta.is_eager(q, k, v, g, beta, init_state, cu_seqlens, lengths)
    if not eager or q is None or k is None or v is None or g is None or beta is None:
        _require_tensors("q k v g beta init_state cu_seqlens lengths", 5, q, k, v, g, beta, init_state, cu_seqlens,
                         lengths)
    if scale is None:
        scale = q.shape[-1] ** -0.5 if q.dim() and q.shape[-1] else 1.0
    elif not isinstance(scale, (int, float)):
        raise TypeError(f"Expected scale to be a number or None, got {type(scale).__name__}.")
    else:
        scale = float(scale)
    if inplace and init_state is None:
        raise ValueError("`inplace` needs an init_state to update.")
    grad = _delta.wants_grad(q, k, v, g, beta, init_state)
    if inplace:
        if grad:
            raise ValueError("`inplace` has no gradients.")
        if eager:
            _delta._require_state("gated_delta_rule", init_state)
            out = _delta._forward("gated_delta_rule", q, k, v, g, beta, init_state, cu_seqlens, lengths, scale,
                                  init_state)[:2]
            torch.autograd.graph.increment_version(init_state)  # (as the dispatcher does)
            return out
        return _delta.gated_delta_rule_(q, k, v, g, beta, init_state, cu_seqlens, lengths, scale), init_state
    if grad:
        run = _delta.Trained.apply if eager else _delta.gated_delta_rule_kept
        return run(q, k, v, g, beta, init_state, cu_seqlens, lengths, scale)[:2]
    if eager:
        return _delta._forward("gated_delta_rule", q, k, v, g, beta, init_state, cu_seqlens, lengths, scale)[:2]
    return _delta.gated_delta_rule(q, k, v, g, beta, init_state, cu_seqlens, lengths, scale)


def verify_drafts(
        tokens: torch.Tensor,
        target: torch.Tensor,
        draft: torch.Tensor | None,
        accept: torch.Tensor,
        sample: torch.Tensor,
        draft_lens: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Which drafted tokens stay, and the token after them, from given random numbers.

    Draft s stays if all before it did and ``accept[s] * draft[s, x] < target[s, x]`` for its token x. Then one
    token is drawn with ``sample``: at the first refused place from ``max(target - draft, 0)`` (from target where
    that is 0 everywhere), after the last draft from target. Tokens so taken are distributed as the target's own.

    :param tokens: Drafted tokens (B, S).
    :param target: The target's probabilities after each of 0 .. S drafts (B, S + 1, V).
    :param draft: Probabilities the drafts were drawn from (B, S, V), in target's type; None for drafts without
        (looked up, or greedy): 1 at the drafted token.
    :param accept: Uniform numbers in [0, 1) (B, S), any float type; used in 32 bits.
    :param sample: Uniform numbers in [0, 1) (B), likewise.
    :param draft_lens: Drafts of each row (B); default S.
    :return: ``(tokens, taken)``: (B, S + 1) int64 -- the drafts that stay, the drawn token, then -1 -- and (B) int32.
    """
    if _delta is None:
        raise _unavailable("verify_drafts")
    if (_delta.is_eager(tokens, target, draft, accept, sample, draft_lens) and tokens is not None and target is not None
            and accept is not None and sample is not None):
        return _delta._verify(tokens, target, draft, accept, sample, draft_lens)
    _require_tensors("tokens target accept sample draft draft_lens", 4, tokens, target, accept, sample, draft, draft_lens)
    return _delta.verify_drafts(tokens, target, draft, accept, sample, draft_lens)
