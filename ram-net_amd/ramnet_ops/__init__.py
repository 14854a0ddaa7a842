"""RAM-Net operators on AMD MI355X (gfx950).

Drop-in for the reference ``ramnet_ops`` package
(packages/ramnet-ops/src/ramnet_ops/__init__.py:1-6): the same two public
functions, computed by hand-written HIP kernels through a C ABI. Beside them
the gated delta rule (a dense fixed-size state, for hybrid models) and the
verification of drafted tokens, which the reference does not have.
"""
from .delta_rule import gated_delta_rule, verify_drafts
from .ram_attn import random_access_memory_attention, topk_addr

__all__ = [
    'gated_delta_rule',
    'random_access_memory_attention',
    'topk_addr',
    'verify_drafts',
]
