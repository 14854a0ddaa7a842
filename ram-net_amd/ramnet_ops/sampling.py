"""Public API of token sampling (the reference has none of it)."""
from __future__ import annotations

import torch

from .delta_rule import _delta, _require_tensors
from .ram_attn import _unavailable

try:
    from .impl import _sample
except ImportError:  # library not built: fail at call time
    _sample = None


def _settings(temperature, top_k, top_p, min_p) -> tuple[tuple, tuple]:
    """Each setting as a tensor or None, and as the number of all rows; checked where it is a number."""
    tensors, numbers = [], []
    for name, value, off, whole in (("temperature", temperature, 1.0, False), ("top_k", top_k, 0, True),
                                    ("top_p", top_p, 1.0, False), ("min_p", min_p, 0.0, False)):
        if isinstance(value, torch.Tensor):
            tensors.append(value)
            numbers.append(off)
            continue
        if value is None:
            value = off
        elif isinstance(value, bool) or not isinstance(value, int if whole else (int, float)):
            raise TypeError(f"Expected {name} to be {'an integer' if whole else 'a number'}, a Tensor or None, got "
                            f"{type(value).__name__}.")
        if name in ("temperature", "top_k") and not value >= 0 or name in ("top_p", "min_p") and not 0 <= value <= 1:
            raise ValueError(f"`{name}` must be {'at least 0' if name in ('temperature', 'top_k') else 'in [0, 1]'}, "
                             f"got {value}.")
        tensors.append(None)
        numbers.append(min(value, 2 ** 31 - 1) if whole else float(value))
    return tuple(tensors), tuple(numbers)


def sample_tokens(
        logits: torch.Tensor,
        random: torch.Tensor,
        temperature: float | torch.Tensor = 1.0,
        top_k: int | torch.Tensor | None = None,
        top_p: float | torch.Tensor | None = None,
        min_p: float | torch.Tensor | None = None,
        probabilities: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """One token a row from given random numbers, with temperature, top-k, top-p and min-p.

    A token's weight is ``exp((logit - max) / temperature)``. Tokens are ordered by descending logit, equal ones by
    index, and each filter keeps a prefix of that order: the first `top_k`; of these, tokens with less than `top_p`
    of their weights before them; tokens of at least `min_p` times the greatest weight. The first is always kept.
    The token is the lowest index whose running sum of kept weights passes ``random`` times their sum. Sums are in
    64 bits. A NaN logit counts as -inf; a row of nothing else gives token 0 and probabilities of 0.

    Settings are numbers, used in 64 bits, or tensors that broadcast to the rows (any float type, used in 32 bits; top_k
    int32 or int64); a tensor's values are not checked. No gradients.

    :param logits: (..., V), a float type of 32 bits or fewer.
    :param random: Uniform numbers in [0, 1) (...), any float type; used in 32 bits. Below 0 counts as 0, from 1 on
        draws the last kept token.
    :param temperature: 0 takes the greatest logit (of equal ones the first).
    :param top_k: 0 or None keeps all.
    :param top_p: 1 or None keeps all.
    :param min_p: 0 or None keeps all.
    :param probabilities: Whether the kept weights over their sum come too, as ``verify_drafts`` takes them.
    :return: tokens (...) int64, or ``(tokens, probabilities)``, the latter (..., V) float32.
    """
    if _sample is None:
        raise _unavailable("sample_tokens")
    tensors, numbers = _settings(temperature, top_k, top_p, min_p)
    eager = _delta.is_eager(logits, random, *tensors)
    if not eager or logits is None or random is None:
        _require_tensors("logits random", 2, logits, random)
    if eager:
        out = _sample._sample("sample_tokens", logits, random, *tensors, *numbers, bool(probabilities))
        return out if probabilities else out[0]
    run = _sample.sample_tokens_with_probabilities if probabilities else _sample.sample_tokens
    return run(logits, random, *tensors, *numbers)


def token_probabilities(
        logits: torch.Tensor,
        temperature: float | torch.Tensor = 1.0,
        top_k: int | torch.Tensor | None = None,
        top_p: float | torch.Tensor | None = None,
        min_p: float | torch.Tensor | None = None,
) -> torch.Tensor:
    """The probabilities that ``sample_tokens`` draws with: (..., V) float32."""
    if _sample is None:
        raise _unavailable("token_probabilities")
    tensors, numbers = _settings(temperature, top_k, top_p, min_p)
    eager = _delta.is_eager(logits, *tensors)
    if not eager or logits is None:
        _require_tensors("logits", 1, logits)
    if eager:
        return _sample._sample("token_probabilities", logits, None, *tensors, *numbers, True)[1]
    return _sample.token_probabilities(logits, *tensors, *numbers)
