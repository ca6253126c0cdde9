"""The MXFP4 operators and the norm on more than 2^31 values, and the layer beside a shared expert in its other forms."""
import numpy as np
import pytest
import torch

import _mxfp4 as ref
from test_gpu_mxfp4 import DEV, HALF, build, check_both, close, both_products, dev, experts_ref, make_product, say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from vllm_ascend_amd import kernels

    return kernels


@pytest.fixture(scope="module")
def ops():
    from vllm_ascend_amd import npu_ops

    return npu_ops


@pytest.mark.parametrize("rows", [2, 40, 700])
def test_rows_far_into_x(K, rows):
    """As many rows of x as the products take: offsets past 2^31 and up to 2^32 less 1 MiB, the last rows, and rows behind them."""
    say("far rows", rows)
    E, N, Kd = 3, 192, 256
    _, counts, _, xc, xs, wc, ws = make_product(E, N, Kd, rows, "zipf")
    x_rows, half = 0xfff00000 // (Kd // 2), (1 << 31) // (Kd // 2)
    x = torch.zeros(x_rows, Kd // 2, dtype=torch.uint8, device=DEV)
    x_scale = torch.full((x_rows, Kd // 32), 127, dtype=torch.uint8, device=DEV)
    where = np.array([x_rows - 1, half, 0, half - 1, x_rows - 2] + [7919 * i % x_rows for i in range(3, rows)])[:rows]
    where = np.concatenate([where, (half + 48611 * np.arange(max(rows - len(where), 0))) % x_rows])
    where[10::9] = [(x_rows, -1, 2**31 - 1)[i % 3] for i in range(len(where[10::9]))]
    there = (where >= 0) & (where < x_rows)
    assert len(set(where[there])) == there.sum()
    on = torch.from_numpy(where[there]).to(DEV)
    x[on], x_scale[on] = dev(ref.pack(xc[there])), dev(xs[there])
    w, s = K.format_cast_mx(dev(ref.pack(wc)), dev(ws))
    held = np.where(there[:, None], ref.values(xc, xs), 0.0)
    got = both_products(K, E, N, Kd, x, x_scale, w, s, dev(counts.astype(np.int64)), row_map=dev(where.astype(np.int32)))
    check_both(got, ref.products(held, ref.values(wc, ws), counts))


def test_quantisation_of_more_than_2_31_values(ops):
    say("far quantisation")
    rows, cols = 66000, 32768
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator().manual_seed(0)
    at = [0, 32767, 65535, 65536, rows - 1]
    some = torch.randn(len(at), cols, generator=g).to(torch.bfloat16)
    x[at] = some.to(DEV)
    codes, scale = ops.npu_dynamic_mx_quant(x)
    c, s = ref.quantise(some.double().numpy())
    assert np.array_equal(codes[at].cpu().numpy(), ref.pack(c)) and np.array_equal(scale[at].cpu().numpy(), s)
    assert torch.count_nonzero(scale).item() == np.count_nonzero(s)
    del x
    back = ops.npu_mx_dequant(codes, scale)
    assert np.array_equal(back[at].double().cpu().numpy(), ref.values(c, s))


@pytest.mark.parametrize("kind", [1, 2])
def test_norm_of_more_than_2_31_values(K, kind):
    say("far norm", kind)
    rows, cols = 132000, 16384
    x1 = torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator().manual_seed(0)
    at = [0, 65536, 131071, 131072, rows - 1]
    x1[at] = torch.randn(len(at), cols, generator=g).to(torch.bfloat16).to(DEV)
    gamma = torch.rand(cols, generator=g).to(torch.bfloat16).to(DEV)
    got = K.add_rms_norm_quant(x1, x1, gamma, None, 1e-6, kind)
    want = K.add_rms_norm_quant(x1[at], x1[at], gamma, None, 1e-6, kind)
    assert all(torch.equal(a[at], b) for a, b in zip(got, want))
    assert torch.count_nonzero(got[2].view(torch.int16).amax(1)).item() == len(at)


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("T", [1, 33])
def test_shared_expert_beside_rows_that_the_caller_quantised(ops, T, dtype):
    from vllm_ascend_amd.fused_moe.shared_experts import AscendSharedExperts

    say("shared expert beside codes", T, dtype)
    E, k, H, I = 8, 2, 256, 128
    g = torch.Generator().manual_seed(2)
    up = torch.randint(-127, 128, (2 * I, H), generator=g, dtype=torch.int8).to(DEV)
    down = torch.randint(-127, 128, (H, I), generator=g, dtype=torch.int8).to(DEV)
    su, sd = (torch.rand(n, generator=g).to(DEV) * 1e-3 for n in (2 * I, H))
    shared = AscendSharedExperts(up, su, down, sd)
    layer, w13, w2 = build(E, k, H, I, dtype, shared=shared)
    x = torch.randn(T, H, generator=g).to(dtype).to(DEV)
    logits = torch.randn(T, E, generator=g).to(DEV)
    weights, ids = layer.router.select_experts(x, logits)
    codes, scale = ops.npu_dynamic_mx_quant(x)
    held = ops.npu_mx_dequant(codes, scale, dst_type=dtype)
    for rows, given, pertoken in ((x, x, None), (held, codes, scale), (held, codes.view(torch.float4_e2m1fn_x2), scale)):
        layer.ascend_pertoken_scale = None
        extra = shared(rows)
        shared.wait()
        assert extra.dtype == dtype
        want = experts_ref(x, ids.cpu().numpy(), weights, w13, w2, dtype, extra.double().cpu().numpy())
        layer.ascend_pertoken_scale = pertoken
        assert close(layer(given, logits), want, dtype, k + 1)
    layer.ascend_pertoken_scale = scale
    three = layer.quant_method.apply(layer, codes.view(1, T, -1), weights, ids, shared).routed_out
    assert torch.equal(three, layer.quant_method.apply(layer, codes, weights, ids, shared).routed_out.view(1, T, H))
