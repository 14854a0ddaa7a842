"""Config-5 caller harness: a RAM-Net language model above the operator.

Not part of the operator library. It exercises ``ramnet_ops`` the way the
reference's model does (``packages/ramnet``: ``ram_attn_block.py:281-350``,
``modeling_ramnet.py:71-107``): a prefill over a prompt with a fresh state,
then greedy single-token steps that update each layer's state in place.

``delta_lm`` does the same for the gated delta rule and draft verification: a
language model on the one, decoded speculatively with the other.
"""
from .delta_lm import DeltaConfig, DeltaLayer, DeltaLM, speculative_generate
from .lm import HarnessConfig, RamLM, RamLayer, greedy_generate

__all__ = ["DeltaConfig", "DeltaLM", "DeltaLayer", "HarnessConfig", "RamLM", "RamLayer", "greedy_generate",
           "speculative_generate"]
