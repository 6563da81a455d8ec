"""gdn_b200 -- B200-native chunked Gated DeltaNet forward (sm_100a).

Drop-in for the forward entry point of 123123213weqw/v100-attention-lab
(``gdn_triton.gdn_chunk_fwd``); see ``ops.gdn_chunk_fwd``.  Beside it: the
elementwise gated recurrence (``recurrence``), windowed attention (``windowed``)
and the single-token forms of all three.
"""

from .fla_compat import chunk_delta_rule, chunk_gated_delta_rule
from .ops import (GdnError, check_status, gdn_chunk_fwd, gdn_chunk_fwd_fixed, gdn_chunk_fwd_v2, gdn_step,
                  gdn_wy_prep)
from .recurrence import gated_scan, gated_scan_step
from .windowed import window_attention, window_attention_step

__all__ = ["gdn_chunk_fwd", "gdn_chunk_fwd_v2", "gdn_chunk_fwd_fixed", "gdn_wy_prep", "chunk_gated_delta_rule",
           "chunk_delta_rule", "gdn_step", "gated_scan", "gated_scan_step", "window_attention",
           "window_attention_step", "GdnError", "check_status"]
