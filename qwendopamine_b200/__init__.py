"""B200-native GatedDeltaNet2 (GDN-2) token mixer.

Drop-in for ``qwendopamine.models.gdn2``: :class:`GatedDeltaNet2` keeps the
reference module's API; :func:`chunk_gdn2` and :func:`fused_recurrent_gdn2`
keep the reference kernel entry points.  Next to them stand a gated linear
recurrence (:func:`gated_scan`, :func:`gated_scan_step`), log probabilities of
given tokens (:func:`token_logprobs`) and the optimizer (:class:`AdamW`,
:func:`adamw_step`).  All compute runs in
``libgdn2_b200.so`` (hand-written CUDA for sm_100a) through a C ABI.
"""

from .gdn2 import GDN2_BACKENDS, GatedDeltaNet2, RMSNormGated, ShortConvolution, resolve_gdn2_backend
from .gdn2_ops import (AdamW, ChunkGDN2Function, adamw_step, chunk_gdn2, fused_recurrent_gdn2,
                       fused_recurrent_gdn2_fwd, gated_scan, gated_scan_step, TokenLogprobs,
                       token_logprobs)
from .registry import BLOCKS, build_block

__all__ = [
    "AdamW",
    "BLOCKS",
    "ChunkGDN2Function",
    "GDN2_BACKENDS",
    "GatedDeltaNet2",
    "RMSNormGated",
    "ShortConvolution",
    "TokenLogprobs",
    "adamw_step",
    "build_block",
    "chunk_gdn2",
    "fused_recurrent_gdn2",
    "fused_recurrent_gdn2_fwd",
    "gated_scan",
    "gated_scan_step",
    "resolve_gdn2_backend",
    "token_logprobs",
]
