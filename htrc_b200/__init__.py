"""htrc_b200: the flat (tree-free) HTRC attention operator for NVIDIA B200 (sm_100a).

Drop-in for the production path of ASarych/HTRC's flat operator (h3/htrc_flat.py,
h3/htrc_flat_runner.py): PyTorch host code over the C-ABI library libhtrc_flat.so of hand-written
sm_100a kernels.  See include/htrc_flat.h for the C ABI.
"""
from .cross import cross_attention, cross_attention_backward, cross_status  # noqa: F401
from .flat import (PROD, dequant_rows, fake_quant, flat_attention, flat_attention_heads,  # noqa: F401
                   flat_attention_prod, forward_into, run_stages, workspace_bytes)
from .linear8 import Int8Rows, int8_linear, int8_linear_status, int8_rows, quantize_rows  # noqa: F401
from .norm import layer_norm, layer_norm_backward, layer_norm_int8  # noqa: F401
from .rotary import (grid_positions, rotary_axes, rotary_axes_backward, rotary_qk,  # noqa: F401
                     rotary_qk_backward)
from .runner import CHUNKS, MODES, FlatRunner, plan_chunk, predicted_peak_mib  # noqa: F401

__all__ = ["PROD", "MODES", "CHUNKS", "flat_attention", "flat_attention_heads", "flat_attention_prod", "FlatRunner",
           "plan_chunk",
           "predicted_peak_mib", "run_stages", "workspace_bytes", "forward_into", "fake_quant", "dequant_rows",
           "cross_attention", "cross_attention_backward", "cross_status",
           "grid_positions", "rotary_axes", "rotary_axes_backward", "rotary_qk", "rotary_qk_backward",
           "layer_norm", "layer_norm_backward", "layer_norm_int8",
           "Int8Rows", "int8_rows", "quantize_rows", "int8_linear", "int8_linear_status"]
