"""vates_amd: MI355X-native speculative-decode MoE hot path (HIP kernels behind a C ABI).

Public surface:
  fused_moe_slots   -- mirror of the reference native_moe_ext.fused_moe_slots
  fused_moe_staged  -- mirror of native_moe_ext.fused_moe_staged (pre-sliced weights)
  MoELayer          -- routed MoE layer (router, top-k, experts, shared expert)
  QuantizedProj     -- one affine-quantised projection stack
  expert_plan, sort_by_expert, combine_experts
                    -- routes sorted by expert and combined again, with gradients
  head_loss         -- the loss of tokens under a head, with its gradients
"""
from ._lib import VmiError, LIB_PATH
from .head import head_loss, head_loss_grad
from .moe import (ExpertPlan, MoELayer, QuantizedProj, combine_experts, expert_plan, fused_moe_slots, fused_moe_staged,
                  sort_by_expert, workspace_status)

__all__ = ["VmiError", "LIB_PATH", "MoELayer", "QuantizedProj", "fused_moe_slots", "fused_moe_staged",
           "workspace_status", "ExpertPlan", "expert_plan", "sort_by_expert", "combine_experts", "head_loss",
           "head_loss_grad"]
