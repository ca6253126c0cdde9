"""What the MXFP4 operators and the norm refuse, and what they say about themselves, without a GPU."""
import numpy as np
import pytest
import torch

import _mxfp4 as ref

FP4 = torch.float4_e2m1fn_x2


@pytest.fixture(scope="module")
def lib():
    from vllm_ascend_amd import _lib

    return _lib.load()


@pytest.fixture(scope="module")
def ops():
    from vllm_ascend_amd import npu_ops

    return npu_ops


def test_the_definition_used_by_the_tests():
    v = np.array([0.0, 0.25, 0.2500001, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.000001, 7.9, -0.25, -5.0, -7.0] + [4.0] * 18)[None]
    code, scale = ref.quantise(v)
    assert scale.tolist() == [[127]]
    held = ref.values(code, scale)[0, :14]
    assert held.tolist() == [0, 0, 0.5, 1, 1, 2, 2, 4, 4, 6, 6, 0, -4, -6]
    assert np.array_equal(ref.unpack(ref.pack(code)), code)
    assert ref.quantise(np.full((1, 32), 2.0 ** -140))[1].tolist() == [[0]]
    assert ref.quantise(np.full((1, 32), np.nan))[1].tolist() == [[255]]


P = 1 << 20  # a device address that nothing may read: every call below is refused first


def test_quantiser_refuses(lib):
    q = lib.moe355_dynamic_mx_quant
    assert q(P, 1, 0, 32, P, P, None) == 0  # nothing to do
    assert q(P, 3, 1, 32, P, P, None) == -1 and q(P, 1, -1, 32, P, P, None) == -1 and q(P, 1, 1, 0, P, P, None) == -1
    assert q(None, 1, 1, 32, P, P, None) == -1 and q(P, 1, 1, 32, None, P, None) == -1 and q(P, 1, 1, 32, P, None, None) == -1
    assert q(P, 1, 1, 48, P, P, None) == -2 and q(P + 8, 1, 1, 32, P, P, None) == -2 and q(P, 1, 1, 32, P + 2, P, None) == -2
    assert q(P, 1, 1 << 39, 32, P, P, None) == -2 and q(P, 1, 1, 1 << 21, P, P, None) == -2
    d = lib.moe355_mx_dequant
    assert d(P, P, 0, 32, P, 1, None) == 0
    assert d(P, P, 1, 32, P, 3, None) == -1 and d(None, P, 1, 32, P, 1, None) == -1 and d(P, P, 1, 40, P, 1, None) == -2
    assert d(P, P, 1, 32, P + 8, 1, None) == -2


def test_norm_refuses(lib):
    n = lib.moe355_add_rms_norm_quant

    def call(x1=P, x2=P, gamma=P, beta=None, dt=1, wdt=1, rows=1, cols=64, eps=1e-6, kind=1, x=P, y=P, q=P, scale=P):
        return n(x1, x2, gamma, beta, dt, wdt, rows, cols, eps, kind, x, y, q, scale, None)

    assert call(rows=0) == 0
    for bad in (dict(x1=None), dict(gamma=None), dict(q=None), dict(scale=None), dict(kind=0, y=None), dict(kind=3), dict(kind=-1),
                dict(dt=0), dict(wdt=2), dict(rows=-1), dict(cols=0), dict(eps=-1.0), dict(eps=float("nan"))):
        assert call(**bad) == -1, bad
    for bad in (dict(cols=36), dict(kind=2, cols=40), dict(x1=P + 2), dict(x2=P + 8), dict(x=P + 8), dict(y=P + 8), dict(q=P + 4),
                dict(cols=(1 << 20) + 8)):
        assert call(**bad) == -2, bad


def test_products_refuse(lib):
    def call(swiglu, x=P, xs=P, rt=None, x_rows=4, w=P, ws=P, gl=P, glt=1, rows=4, k=128, n=64, E=2, out=P, out_scale=P, dt=1):
        space = lib.moe355_gmm_mx_workspace(rows, n, E, int(swiglu))
        if swiglu:
            return lib.moe355_gmm_mx_swiglu_quant(x, xs, rt, x_rows, w, ws, gl, glt, rows, k, n, E, 0.0, out, out_scale, P, space,
                                                  None)
        return lib.moe355_gmm_mx(x, xs, rt, x_rows, w, ws, gl, glt, rows, k, n, E, out, dt, P, space, None)

    for swiglu in (False, True):
        assert call(swiglu, rows=0) == 0
        for bad in (dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(gl=None), dict(out=None), dict(glt=2),
                    dict(rows=-1), dict(x_rows=-1), dict(k=0), dict(n=0), dict(E=0)):
            assert call(swiglu, **bad) == -1, bad
        for bad in (dict(k=96), dict(n=48), dict(x=P + 8), dict(w=P + 8), dict(ws=P + 2), dict(out=P + 8), dict(rows=1 << 31),
                    dict(x_rows=1 << 31), dict(E=1 << 20), dict(k=1 << 21), dict(n=1 << 21), dict(x_rows=1 << 26)):
            assert call(swiglu, **bad) == -2, bad
    assert call(True, n=96) == -2 and call(True, out_scale=None) == -1 and call(False, dt=0) == -1
    f = lib.moe355_format_cast_mx
    assert f(P, P, 1, 32, 64, None, P, None) == -1 and f(P, P, 0, 32, 64, P, P, None) == -1
    assert f(P, P, 1, 33, 64, P, P, None) == -2 and f(P, P, 1, 32, 96, P, P, None) == -2 and f(P + 4, P, 1, 32, 64, P, P, None) == -2


def test_operators_refuse_what_they_have_no_kernel_for(ops):
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    for kw in (dict(axis=0), dict(block_size=16), dict(round_mode="floor"), dict(scale_alg=1), dict(dst_type=torch.float8_e4m3fn)):
        with pytest.raises(NotImplementedError):
            ops.npu_dynamic_mx_quant(x, **kw)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.npu_dynamic_mx_quant(x)
    with pytest.raises(ValueError, match="multiple of 32"):
        ops.npu_dynamic_mx_quant(x[:, :48])
    with pytest.raises(TypeError):
        ops.npu_dynamic_mx_quant(x.to(torch.int32))
    c, s = torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)
    with pytest.raises(ValueError, match="belong together"):
        ops.npu_mx_dequant(c, s[:, :1])
    with pytest.raises(TypeError):
        ops.npu_mx_dequant(c.to(torch.int8), s)
    with pytest.raises(TypeError):
        ops.npu_mx_dequant(c, s, dst_type=torch.float64)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.npu_mx_dequant(c, s)

    g = torch.ones(64, dtype=torch.bfloat16)
    norm = ops.npu_add_rms_norm_dynamic_quant
    with pytest.raises(NotImplementedError):
        norm(x, x, g, dst_type=torch.float8_e4m3fn)
    for bad in ((x, x[:1], g), (x, x.half(), g), (x, x, g[:8]), (x, x, g.half()), (x[:, :4], None, g[:4])):
        with pytest.raises(ValueError):
            norm(*bad)
    with pytest.raises(ValueError, match="beta"):
        norm(x, x, g, beta=g.float())
    with pytest.raises(ValueError, match="multiple of 32"):
        norm(x[:, :40], None, g[:40], dst_type=FP4)
    with pytest.raises(TypeError):
        norm(x.float(), None, g.float())
    with pytest.raises(RuntimeError, match="GPU"):
        norm(x, x, g)


def test_products_refuse_operands_that_do_not_belong_together(ops):
    E, N, K, M = 2, 64, 128, 5
    x, xs = torch.zeros(M, K // 2, dtype=torch.uint8), torch.zeros(M, K // 32, dtype=torch.uint8)
    w, ws = torch.zeros(E, N, K // 2, dtype=torch.uint8), torch.zeros(E, N, 8, dtype=torch.uint8)
    gl = torch.tensor([2, 3])

    def swiglu(x=x, w=w, ws=ws, xs=xs, gl=gl, **kw):
        return ops.npu_grouped_matmul_swiglu_quant_v2(x, [w], [ws], xs, gl, **kw)

    def plain(x=x, w=w, ws=ws, xs=xs, gl=gl, **kw):
        return ops.npu_grouped_matmul([x], [w], scale=[ws], per_token_scale=[xs], group_list=gl,
                                      **{"split_item": 2, "group_type": 0, "group_list_type": 1, **kw})

    for f in (swiglu, plain):
        for bad in (dict(x=x[:, :32]), dict(xs=xs[:3]), dict(w=w[0]), dict(ws=ws[:, :, :4]), dict(gl=gl[:1]), dict(gl=None),
                    dict(gl=gl.float()), dict(w=w[:, :48], ws=ws[:, :48])):
            with pytest.raises(ValueError):
                f(**bad)
        with pytest.raises(TypeError):
            f(w=w.to(torch.int8))
        with pytest.raises(RuntimeError, match="GPU"):
            f()
    for bad in (dict(bias=gl), dict(smooth_scale=gl), dict(quant_mode=0), dict(dequant_mode=0), dict(quant_dtype=torch.int8),
                dict(dequant_dtype=torch.bfloat16)):
        with pytest.raises(NotImplementedError):
            swiglu(**bad)
    with pytest.raises(NotImplementedError):
        ops.npu_grouped_matmul_swiglu_quant_v2(x, [w, w], [ws, ws], xs, gl)
    with pytest.raises(TypeError, match="row_map"):
        swiglu(row_map=gl)
    for bad in (dict(bias=gl), dict(output_dtype=torch.float32), dict(group_type=1)):
        with pytest.raises(NotImplementedError):
            plain(**bad)
    with pytest.raises(ValueError):
        ops.npu_format_cast_mx(w[:, :33], ws[:, :33])
    with pytest.raises(ValueError):
        ops.npu_format_cast_mx(w, ws)  # [E, N, K / 32] belongs to these codes
    with pytest.raises(NotImplementedError):
        ops.npu_quant_matmul(x, w[0], ws[0], output_dtype=torch.bfloat16)  # no row scales
    with pytest.raises(NotImplementedError):
        ops.npu_quant_matmul(x, w[0], ws[0], pertoken_scale=xs, output_dtype=torch.int32)


def test_device_operator_has_the_mx_calls():
    from vllm_ascend_amd.device_op import DeviceOperator

    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        DeviceOperator.npu_dynamic_quant(x, act_quant_type=FP4, use_mxfp_quant=True)
    with pytest.raises(NotImplementedError):
        DeviceOperator.npu_dynamic_quant(x, act_quant_type=torch.float8_e4m3fn, use_mxfp_quant=True)
    codes, scale = torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)
    assert DeviceOperator.npu_dynamic_quant(codes, scale, act_quant_type=FP4, use_mxfp_quant=True) == (codes, scale)
    kw = DeviceOperator.get_quant_gmm2_kwargs(input_dtype=torch.float16, act_quant_type=FP4, use_mxfp_quant=True)
    assert kw == {"output_dtype": torch.float16}


def test_scheme():
    from vllm_ascend_amd.fused_moe.contracts import FusedMoEConfig
    from vllm_ascend_amd.fused_moe.layer import AscendRoutedExperts
    from vllm_ascend_amd.fused_moe.router import AscendFusedTopKRouter
    from vllm_ascend_amd.quant_type import QuantType
    from vllm_ascend_amd.quantization import get_scheme_class

    cls = get_scheme_class("W4A4_MXFP4", "moe")
    scheme = cls()
    assert scheme.quant_type == QuantType.W4A4MXFP
    w, q = scheme.get_weight(8, 1408, 1024, torch.bfloat16), scheme.get_dynamic_quant_param(8, 1408, 1024, torch.bfloat16)
    assert w["w13_weight"].shape == (8, 2816, 512) and w["w2_weight"].shape == (8, 1024, 704)
    assert q["w13_weight_scale"].shape == (8, 2816, 32) and q["w2_weight_scale"].shape == (8, 1024, 44)
    assert all(t.dtype == torch.uint8 for t in (*w.values(), *q.values()))
    with pytest.raises(ValueError):
        scheme.get_weight(8, 96, 1024, torch.bfloat16)
    with pytest.raises(TypeError):
        cls(in_dtype=torch.float32)

    layer = AscendRoutedExperts(FusedMoEConfig(num_experts=8, experts_per_token=2, hidden_dim=64, intermediate_size_per_partition=64),
                                scheme, AscendFusedTopKRouter(2, 8), device="cpu")
    x, tw, ids = torch.zeros(3, 64, dtype=torch.bfloat16), torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int32)
    for name, value in (("activation", "gelu"), ("apply_router_weight_on_input", True), ("global_redundant_expert_num", 2),
                        ("ascend_expert_map", ids), ("ascend_mc2_mask", ids)):
        was = getattr(layer, name)
        setattr(layer, name, value)
        with pytest.raises(NotImplementedError):
            scheme.apply(layer, x, tw, ids)
        setattr(layer, name, was)


def test_checkpoint_tensors_under_the_names_of_their_types():
    """E8M0 scales and E2M1 codes are loaded as the bytes they are, not as the numbers they stand for."""
    from vllm_ascend_amd.fused_moe.contracts import FusedMoEConfig
    from vllm_ascend_amd.fused_moe.layer import AscendRoutedExperts
    from vllm_ascend_amd.fused_moe.router import AscendFusedTopKRouter
    from vllm_ascend_amd.quantization import get_scheme_class

    scheme = get_scheme_class("W4A4_MXFP4", "moe")()
    scheme.process_weights_after_loading = lambda layer: None
    layer = AscendRoutedExperts(FusedMoEConfig(num_experts=2, experts_per_token=1, hidden_dim=64, intermediate_size_per_partition=64),
                                scheme, AscendFusedTopKRouter(1, 2), device="cpu")
    g = torch.Generator().manual_seed(0)
    raw = {n: torch.randint(0, 255, p.shape, generator=g, dtype=torch.uint8) for n, p in layer.named_parameters()}
    layer.load_weights({n: t.view(torch.float8_e8m0fnu if n.endswith("scale") else FP4) for n, t in raw.items()})
    assert all(torch.equal(getattr(layer, n), t) for n, t in raw.items())


def test_checkpoint_loader_keeps_the_bytes():
    from vllm_ascend_amd.quantization.checkpoint import moe_weight_loader

    g = torch.Generator().manual_seed(1)
    codes, scale = torch.randint(0, 256, (64, 32), generator=g, dtype=torch.uint8), torch.randint(0, 255, (64, 2), generator=g, dtype=torch.uint8)
    w, s = (torch.nn.Parameter(torch.zeros(2, 128, n, dtype=torch.uint8), requires_grad=False) for n in (32, 2))
    for c, sc in ((codes, scale), (codes.view(FP4), scale.view(torch.float8_e8m0fnu))):
        w.data.zero_(), s.data.zero_()
        moe_weight_loader(w, c, "w13_weight", "w3", 1)
        moe_weight_loader(s, sc, "w13_weight_scale", "w3", 1)
        assert torch.equal(w[1, 64:], codes) and torch.equal(s[1, 64:], scale) and not w[0].any() and not w[1, :64].any()


def test_experts_refuse(lib):
    def call(x=P, xs=None, dt=1, T=4, H=128, ids=P, tw=P, k=2, w13=P, s13=P, w2=P, s2=P, I=64, E=8, res=None, tokens=P, out=P, ws=P,
             less=0):
        space = lib.moe355_mx_experts_workspace(T, k, H, I, E, int(xs is not None))
        return lib.moe355_mx_experts(x, xs, dt, T, H, ids, tw, k, w13, s13, w2, s2, I, E, 0.0, res, tokens, out, ws, space - less, None)

    assert call(T=0) == 0
    for bad in (dict(x=None), dict(ids=None), dict(tw=None), dict(w13=None), dict(s13=None), dict(w2=None), dict(s2=None),
                dict(tokens=None), dict(out=None), dict(dt=0), dict(T=-1), dict(k=0), dict(H=0), dict(I=0), dict(E=0)):
        assert call(**bad) == -1, bad
    for bad in (dict(H=96), dict(I=96), dict(k=65), dict(E=2049), dict(T=1 << 30), dict(x=P + 8), dict(w13=P + 8), dict(s13=P + 2),
                dict(w2=P + 8), dict(s2=P + 1), dict(out=P + 8), dict(res=P + 8), dict(H=(1 << 20) + 64), dict(I=(1 << 19) + 64)):
        assert call(**bad) == -2, bad
    assert call(ws=None) == -3 and call(ws=P + 16) == -3 and call(less=1) == -3


def test_launches_larger_than_there_are(lib):
    """More threads than a launch has."""
    assert lib.moe355_dynamic_mx_quant(P, 1, 1 << 15, 1 << 20, P, P, None) == -2
    assert lib.moe355_mx_dequant(P, P, 1 << 15, 1 << 20, P, 1, None) == -2
    norm = lambda rows, cols: lib.moe355_add_rms_norm_quant(P, P, P, None, 1, 1, rows, cols, 1e-6, 1, P, P, P, P, None)
    assert norm(1 << 26, 512) == -2 and norm(1 << 22, 16384) == -2
    assert lib.moe355_format_cast_mx(P, P, 32768, 1 << 16, 64, P, P, None) == -2
    gmm = lambda rows, n: lib.moe355_gmm_mx(P, P, P, 4, P, P, P, 1, rows, 64, n, 2, P, 1, None, 0, None)
    assert gmm((1 << 31) - 1, 1 << 20) == -2


def test_tiles_wait_for_the_tokens_of_their_first_window(tmp_path):
    """The compiler orders loads to LDS only by what it sees, and the kernel's own wait counts loads: in front of the first barrier
    the four loads of the first window's tokens must have landed, whatever order the others were put in."""
    import subprocess

    from test_abi_and_host import _code_objects
    from vllm_ascend_amd import _lib

    data, kernels = open(_lib.LIB_PATH, "rb").read(), 0
    for at in _code_objects(data):
        if b"gmm_mx_tiled_kernel" not in data[at:at + (1 << 22)]:
            continue
        part = tmp_path / "code"
        part.write_bytes(data[at:at + (1 << 22)])
        text = subprocess.run(["/opt/rocm/llvm/bin/llvm-objdump", "-d", "--mcpu=gfx950", str(part)], capture_output=True, text=True).stdout
        for body in text.split("\n\n"):
            lines = body.strip().split("\n")
            if "gmm_mx_tiled_kernel" not in lines[0]:
                continue
            kernels += 1
            pending, tokens = [], 0  # loads on their way, oldest first: True is one to LDS
            for line in lines[1:]:
                op = line.split("//")[0].split()
                if not op:
                    continue
                if op[0].startswith(("buffer_load", "global_load", "scratch_", "buffer_store", "global_store")):
                    pending.append(op[-1] == "lds")
                    tokens += op[-1] == "lds"
                elif op[0] == "s_waitcnt" and "vmcnt" in line:
                    left = int(line.split("vmcnt(")[1].split(")")[0])
                    pending = pending[max(len(pending) - left, 0):]
                elif op[0] == "s_barrier" and tokens:
                    assert tokens == 8 and sum(pending) <= 4, lines[0]  # two windows asked for, one of them still on its way
                    break
    assert kernels == 6


@pytest.mark.parametrize("name", [torch.uint8, FP4], ids=str)
def test_layer_asks_the_router_for_weights_of_the_model_type(name):
    """Rows that the caller has quantised, under either of the names of their type."""
    from vllm_ascend_amd.fused_moe.contracts import FusedExpertsResult, FusedMoEConfig
    from vllm_ascend_amd.fused_moe.layer import AscendRoutedExperts
    from vllm_ascend_amd.fused_moe.router import AscendFusedTopKRouter
    from vllm_ascend_amd.quantization import get_scheme_class

    asked = []

    class Router(AscendFusedTopKRouter):
        def select_experts(self, hidden_states, router_logits, **kw):
            asked.append(kw["weights_dtype"])
            return torch.ones(3, 1), torch.zeros(3, 1, dtype=torch.int32)

    for dtype in (torch.bfloat16, torch.float16):
        scheme = get_scheme_class("W4A4_MXFP4", "moe")(in_dtype=dtype)
        scheme.apply = lambda layer, x, *a: FusedExpertsResult(routed_out=x)
        layer = AscendRoutedExperts(FusedMoEConfig(num_experts=2, experts_per_token=1, hidden_dim=64, intermediate_size_per_partition=64),
                                    scheme, Router(1, 2), device="cpu")
        layer.ascend_pertoken_scale = torch.zeros(3, 2, dtype=torch.uint8)
        layer(torch.zeros(3, 32, dtype=torch.uint8).view(name), torch.zeros(3, 2))
        assert asked.pop() is dtype and not asked


@pytest.mark.parametrize("T,H,k,E,fits", [(8190, 1 << 20, 64, 8, False), (8190, 1 << 20, 63, 8, True), (1 << 24, 64, 1, 8, False),
                                          ((1 << 24) - 1, 64, 1, 8, True)])
def test_experts_of_more_threads_than_a_launch_has(lib, T, H, k, E, fits):
    """The down product's tiles, or the combine's tokens: refused before the first launch, and no workspace asked for."""
    assert (lib.moe355_mx_experts_workspace(T, k, H, 64, E, 0) > 0) == fits
    if not fits:
        assert lib.moe355_mx_experts(P, None, 1, T, H, P, P, k, P, P, P, P, 64, E, 0.0, None, P, P, P, 1 << 60, None) == -2


def test_device_operator_takes_mx_calls_for_what_they_say():
    """An MX call of int8 rows or weights is not the int8 product; a type other than four bits is refused wherever it is named."""
    from vllm_ascend_amd.device_op import DeviceOperator as D

    E, N, K, M = 2, 64, 128, 5
    x, xs = torch.zeros(M, K // 2, dtype=torch.uint8), torch.zeros(M, K // 32, dtype=torch.uint8)
    w, ws = torch.zeros(E, N, K // 2, dtype=torch.uint8), torch.zeros(E, N, 8, dtype=torch.uint8)
    gl = torch.tensor([2, 3])
    int8 = dict(x=torch.zeros(M, K, dtype=torch.int8), xs=torch.ones(M), w=torch.zeros(E, K, N, dtype=torch.int8), ws=torch.ones(E, N))

    def down(x=x, xs=xs, w=w, ws=ws, **kw):
        return D.npu_grouped_matmul_gmm2(hidden_states=x, weight=[w], weight_scale=[ws], per_token_scale=xs, group_list=gl,
                                         group_list_type=1, input_dtype=torch.bfloat16, use_mxfp_quant=True, **kw)

    def up(x=x, xs=xs, w=w, ws=ws, **kw):
        return D.npu_grouped_matmul_swiglu_quant(x=x, weight=w, group_list=gl, weight_scale=ws, x_scale=xs, group_list_type=1,
                                                 use_mxfp_quant=True, **kw)

    for call in (up, down):
        for name in (None, FP4, torch.uint8):
            with pytest.raises(RuntimeError, match="GPU"):
                call(act_quant_type=name, weight_quant_type=name, mxfp_quant_dtype=name)
        for name in ("act_quant_type", "weight_quant_type", "mxfp_quant_dtype"):
            with pytest.raises(NotImplementedError):
                call(**{name: torch.float8_e4m3fn})
        with pytest.raises(TypeError):
            call(**int8)
        with pytest.raises(TypeError):
            call(x=int8["x"], xs=int8["xs"])
        with pytest.raises(TypeError):
            call(w=int8["w"], ws=int8["ws"])
