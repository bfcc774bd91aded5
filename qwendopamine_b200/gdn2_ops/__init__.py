"""B200 kernels behind the GDN-2 token mixer (chunkwise and recurrent), and the
operators that a decoder runs next to it."""

from .adamw import AdamW, adamw_step
from .chunk_gdn2 import ChunkGDN2Function, chunk_gdn2
from .block_ops import gated_rms_norm, short_conv
from .cp import CPChunkGDN2Function, chunk_gdn2_cp, gather_span_maps, short_conv_cp
from .fused_recurrent_gdn2 import fused_recurrent_gdn2, fused_recurrent_gdn2_fwd
from .gated_scan import GatedScanFunction, gated_scan, gated_scan_step
from .token_logprobs import TokenLogprobs, TokenLogprobsFunction, token_logprobs

__all__ = ["AdamW", "CPChunkGDN2Function", "ChunkGDN2Function", "GatedScanFunction",
           "TokenLogprobs", "TokenLogprobsFunction", "adamw_step", "chunk_gdn2", "chunk_gdn2_cp",
           "fused_recurrent_gdn2", "fused_recurrent_gdn2_fwd", "gated_rms_norm", "gated_scan",
           "gated_scan_step", "gather_span_maps", "short_conv", "short_conv_cp", "token_logprobs"]
