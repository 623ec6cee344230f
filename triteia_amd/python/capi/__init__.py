from .marlin import mul_2_4, bmm_2_4, sbmm_2_4, sbmm_2_4_multilaunch
from .marlin import sbmm_2_4_routed, sbmm_2_4_planned, route_plan, routed_workspace, pack_2_4
from .punica import add_lora_sgmv_cutlass, add_lora_bgmv, sgmv_routed, lora_scratch, lora_shrink, lora_expand
from .attention import AttentionPlan, PagedCache, attention_plan, cache_read, paged_attention, rotary_cache
from .fp8 import dequantize_fp8, matmul_fp8, quantize_fp8

__all__ = ["mul_2_4", "bmm_2_4", "sbmm_2_4", "sbmm_2_4_multilaunch", "add_lora_sgmv_cutlass", "add_lora_bgmv",
           "sbmm_2_4_routed", "sbmm_2_4_planned", "route_plan", "routed_workspace", "sgmv_routed", "pack_2_4", "lora_scratch", "lora_shrink",
           "lora_expand", "AttentionPlan", "PagedCache", "attention_plan", "cache_read", "paged_attention", "rotary_cache",
           "quantize_fp8", "dequantize_fp8", "matmul_fp8"]
