"""W4A4 MXFP4 fused-MoE scheme: weights and activations in blocks of 32 four-bit floats that share a power of two, activations
quantised on the fly.  The contract of the other schemes (``apply(layer, x, topk_weights, topk_ids, shared_experts,
shared_experts_input)``, ``vllm_ascend/quantization/methods/base.py:206-287``) for ``QuantType.W4A4MXFP``
(``vllm_ascend/quantization/quant_type.py:26-37``).

Checkpoint form: codes two a byte along K (the first in the low half), ``w13_weight`` ``[E, 2I, H / 2]`` and ``w2_weight``
``[E, H, I / 2]``; one E8M0 byte a block, ``w13_weight_scale`` ``[E, 2I, H / 32]`` and ``w2_weight_scale`` ``[E, H, I / 32]``.  H
and I are multiples of 64."""
from __future__ import annotations

from typing import Any

import torch

from .. import kernels, npu_ops
from ..fused_moe.contracts import FusedExpertsResult
from ..quant_type import QuantType
from .base import AscendMoEScheme, register_scheme


@register_scheme("W4A4_MXFP4", "moe")
class AscendW4A4MXFP4DynamicFusedMoEMethod(AscendMoEScheme):
    supports_eplb = False
    quant_type: QuantType = QuantType.W4A4MXFP

    def __init__(self, in_dtype: torch.dtype = torch.bfloat16):
        if in_dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"in_dtype must be bfloat16 or float16, got {in_dtype}")
        self.in_dtype = in_dtype
        self.dynamic_eplb = False
        self.use_expert_weight_list = False

    def get_weight(self, num_experts: int, intermediate_size_per_partition: int, hidden_sizes: int,
                   params_dtype: torch.dtype) -> dict[str, Any]:
        if hidden_sizes % 64 or intermediate_size_per_partition % 64:
            raise ValueError("MXFP4 experts: hidden and intermediate size must be multiples of 64, got "
                             f"{hidden_sizes} and {intermediate_size_per_partition}")
        return {
            "w13_weight": torch.empty(num_experts, 2 * intermediate_size_per_partition, hidden_sizes // 2,
                                      dtype=torch.uint8),
            "w2_weight": torch.empty(num_experts, hidden_sizes, intermediate_size_per_partition // 2, dtype=torch.uint8),
        }

    def get_dynamic_quant_param(self, num_experts: int, intermediate_size_per_partition: int, hidden_sizes: int,
                                params_dtype: torch.dtype) -> dict[str, Any]:
        block = kernels.MX_BLOCK
        return {
            "w13_weight_scale": torch.empty(num_experts, 2 * intermediate_size_per_partition, hidden_sizes // block,
                                            dtype=torch.uint8),
            "w2_weight_scale": torch.empty(num_experts, hidden_sizes, intermediate_size_per_partition // block,
                                           dtype=torch.uint8),
        }

    def process_weights_after_loading(self, layer) -> None:
        """Checkpoint order -> the storage that the products stream."""
        for name in ("w13", "w2"):
            codes, scale = getattr(layer, f"{name}_weight"), getattr(layer, f"{name}_weight_scale")
            codes.data, scale.data = npu_ops.npu_format_cast_mx(codes.data, scale.data)

    def apply(self, layer, x: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor,
              shared_experts: Any | None = None, shared_experts_input: torch.Tensor | None = None):
        """Hidden states [T, H] in 16 bits, quantised here once a token, or MXFP4 codes [T, H / 2] of the caller's (their
        scales in ``layer.ascend_pertoken_scale``).  The rows stay in token order: the gate_up product reads them through
        the row -> token map of the routing."""
        self._refuse(layer)
        scale = layer.ascend_pertoken_scale
        if scale is None:
            if x.dtype != self.in_dtype:
                raise TypeError(f"hidden states are {x.dtype}, the scheme was built for {self.in_dtype}")
            H = x.shape[-1]
        else:
            x = kernels._bytes(x, "hidden states quantised by the caller")
            H = x.shape[-1] * 2
            if x.dim() != 2:
                scale = scale.reshape(-1, scale.shape[-1])
        lead = x.shape[:-1]
        if x.dim() != 2:
            x = x.reshape(-1, x.shape[-1])
        if topk_weights.dtype != self.in_dtype:
            topk_weights = topk_weights.to(self.in_dtype)
        if topk_ids.dim() != 2 or topk_ids.shape[0] != x.shape[0] or topk_weights.shape != topk_ids.shape:
            raise ValueError(f"{x.shape[0]} tokens, but topk_ids {tuple(topk_ids.shape)} and topk_weights "
                             f"{tuple(topk_weights.shape)}")
        limit = layer.moe_config.swiglu_limit or 0.0
        if shared_experts is None:
            # one native call; no events are recorded, which are for what runs beside the routed experts
            out, expert_tokens = kernels.mx_experts(x, scale, topk_ids, topk_weights, layer.w13_weight, layer.w13_weight_scale,
                                                    layer.w2_weight, layer.w2_weight_scale, limit)
            return FusedExpertsResult(routed_out=out if len(lead) == 1 else out.reshape(*lead, H), group_list_type=1,
                                      expert_tokens=expert_tokens)
        stream = torch.cuda.current_stream()
        before_dispatch_evt = stream.record_event()
        if shared_experts_input is None:
            shared_experts_input = x if scale is None else npu_ops.npu_mx_dequant(x, scale, dst_type=self.in_dtype)
        shared_out = shared_experts(shared_experts_input)
        if scale is None:
            x, scale = npu_ops.npu_dynamic_mx_quant(x)
        expanded_row_idx, row_token, expert_tokens = kernels.route_map(topk_ids, layer.w13_weight.shape[0], 1)
        hidden, hidden_scale = npu_ops.npu_grouped_matmul_swiglu_quant_v2(
            x, layer.w13_weight, layer.w13_weight_scale, scale, expert_tokens, group_list_type=1, swiglu_limit=limit,
            row_map=row_token)
        before_gmm2_evt = stream.record_event()
        out = npu_ops.npu_grouped_matmul([hidden], [layer.w2_weight], scale=[layer.w2_weight_scale],
                                         per_token_scale=[hidden_scale], group_list=expert_tokens, split_item=2,
                                         group_type=0, group_list_type=1, output_dtype=self.in_dtype)[0]
        before_combine_evt = stream.record_event()
        shared_experts.wait()
        routed_out = kernels.token_unpermute(out, expanded_row_idx, topk_weights, shared_out.reshape(-1, H))
        return FusedExpertsResult(routed_out=routed_out.reshape(*lead, H), before_dispatch_evt=before_dispatch_evt,
                                  before_gmm2_evt=before_gmm2_evt, before_combine_evt=before_combine_evt,
                                  group_list_type=1, expert_tokens=expert_tokens, shared_out=shared_out)

    @staticmethod
    def _refuse(layer) -> None:
        act = getattr(layer, "activation", "silu")
        if (getattr(act, "value", act) or "silu") != "silu":
            raise NotImplementedError(f"activation {act!r}: MXFP4 experts have SwiGLU (silu) only")
        for name in ("apply_router_weight_on_input", "global_redundant_expert_num"):
            if getattr(layer, name, False):
                raise NotImplementedError(f"MXFP4 experts: {name} is not supported")
        for name in ("ascend_expert_map", "ascend_mc2_mask"):
            if getattr(layer, name, None) is not None:
                raise NotImplementedError(f"MXFP4 experts: {name} is not supported")
