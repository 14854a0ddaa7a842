"""RAM-Net operators on AMD MI355X (gfx950).

Drop-in for the reference ``ramnet_ops`` package
(packages/ramnet-ops/src/ramnet_ops/__init__.py:1-6): the same two public
functions, computed by hand-written HIP kernels through a C ABI. Beside them
the gated delta rule and the selective scan (states of fixed size, for hybrid
models), the short causal convolution before them, the sampling of tokens and
the verification of drafted ones, which the reference does not have.
"""
from .delta_rule import gated_delta_rule, verify_drafts
from .ram_attn import random_access_memory_attention, topk_addr
from .sampling import sample_tokens, token_probabilities
from .scan import causal_conv, selective_scan

__all__ = [
    'causal_conv',
    'gated_delta_rule',
    'random_access_memory_attention',
    'sample_tokens',
    'selective_scan',
    'token_probabilities',
    'topk_addr',
    'verify_drafts',
]
