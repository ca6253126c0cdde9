"""Per-expert MXFP4 tensors of a checkpoint directory -> one layer: the bytes, whichever name their type has there."""
import json

import numpy as np
import pytest
import torch

import _mxfp4 as ref
from test_checkpoint_loader import PREFIX, _CpuLayer
from vllm_ascend_amd.quantization.checkpoint import load_routed_experts, routed_experts_from_checkpoint
from vllm_ascend_amd.quantization.modelslim_config import MODELSLIM_CONFIG_FILENAME, AscendModelSlimConfig

E, I, H = 3, 64, 320  # a last, shorter window of K


def write(path, scale_type):
    from safetensors.torch import save_file

    rng = np.random.default_rng(5)
    held, tensors = {}, {}
    for name, rows, cols in (("w13", 2 * I, H), ("w2", H, I)):
        code, scale = ref.random_mx(rng, (E, rows, cols))
        held[name + "_weight"], held[name + "_weight_scale"] = torch.from_numpy(ref.pack(code)), torch.from_numpy(scale - 5)
    for e in range(E):
        for module, name, rows in (("gate_proj", "w13", slice(0, I)), ("up_proj", "w13", slice(I, 2 * I)), ("down_proj", "w2", slice(None))):
            tensors[f"{PREFIX}.{e}.{module}.weight"] = held[name + "_weight"][e, rows].contiguous()
            tensors[f"{PREFIX}.{e}.{module}.weight_scale"] = held[name + "_weight_scale"][e, rows].contiguous().view(scale_type)
    save_file(tensors, str(path / "model.safetensors"))
    (path / MODELSLIM_CONFIG_FILENAME).write_text(json.dumps({n: "W4A4_MXFP4" for n in tensors}))
    return held


@pytest.mark.parametrize("scale_type", [torch.uint8, torch.float8_e8m0fnu], ids=str)
def test_stacking(tmp_path, scale_type):
    held = write(tmp_path, scale_type)
    conf = AscendModelSlimConfig()
    conf.maybe_update_config(str(tmp_path))
    layer = _CpuLayer(conf.get_moe_scheme(PREFIX, "qwen3_moe"), E, I, H)
    assert len(load_routed_experts(layer, str(tmp_path), PREFIX, post_process=False)) == 6 * E
    assert all(torch.equal(getattr(layer, n).data, t) for n, t in held.items())


@pytest.mark.gpu
def test_layer_from_checkpoint(tmp_path):
    from vllm_ascend_amd.fused_moe.contracts import FusedMoEConfig
    from vllm_ascend_amd.fused_moe.layer import AscendRoutedExperts
    from vllm_ascend_amd.fused_moe.router import AscendFusedTopKRouter
    from vllm_ascend_amd.quantization import get_scheme_class

    print("MXFP4 layer from a checkpoint", flush=True)
    held = write(tmp_path, torch.float8_e8m0fnu)
    config = FusedMoEConfig(num_experts=E, experts_per_token=2, hidden_dim=H, intermediate_size_per_partition=I)
    layer = routed_experts_from_checkpoint(str(tmp_path), PREFIX, config, AscendFusedTopKRouter(2, E), device="cuda:0")
    direct = AscendRoutedExperts(config, get_scheme_class("W4A4_MXFP4", "moe")(), AscendFusedTopKRouter(2, E), device="cuda:0")
    direct.load_weights(held)
    g = torch.Generator().manual_seed(0)
    x, logits = torch.randn(40, H, generator=g).to(torch.bfloat16).to("cuda:0"), torch.randn(40, E, generator=g).to("cuda:0")
    assert torch.equal(layer(x, logits), direct(x, logits))
