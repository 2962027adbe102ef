"""gfx950 operators of the NF4 + multi-LoRA serving path (mirror of ``loraforge.ops``)."""

from .experts import ExpertRouting, combine_experts, expert_linear, expert_mlp, route_experts
from .fp8 import FP8Tensor, dequantize_fp8, fp8_linear, quantize_fp8
from .fused import LoraBatch, lora_apply, nf4_lora_linear, segments_to_slots, workspace_bytes
from .lora_rows import row_expand, row_shrink
from .mxfp4 import MXFP4Tensor, dequantize_mxfp4, mxfp4_linear, quantize_mxfp4
from .nf4 import NF4State, NestedState, dequantize_nf4, dequantize_nf4_nested, prepare_scales, quantize_nf4
from . import rowexpand
from .quant_state import load_nf4_weight, quant_state_entries, quant_state_from_entries, save_nf4_weights

__all__ = [
    "ExpertRouting",
    "FP8Tensor",
    "LoraBatch",
    "MXFP4Tensor",
    "NF4State",
    "NestedState",
    "combine_experts",
    "dequantize_fp8",
    "dequantize_mxfp4",
    "dequantize_nf4",
    "dequantize_nf4_nested",
    "expert_linear",
    "expert_mlp",
    "fp8_linear",
    "load_nf4_weight",
    "lora_apply",
    "mxfp4_linear",
    "nf4_lora_linear",
    "prepare_scales",
    "quant_state_entries",
    "quant_state_from_entries",
    "quantize_fp8",
    "quantize_mxfp4",
    "quantize_nf4",
    "route_experts",
    "row_expand",
    "row_shrink",
    "rowexpand",
    "save_nf4_weights",
    "segments_to_slots",
    "workspace_bytes",
]
