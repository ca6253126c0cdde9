"""Performance cases of the operators around a layer with microscaled 4-bit (MXFP4) experts.

An MXFP4 row is 32 values a block: a power of two that the block shares (one byte, exponent + 127) and a code of four
bits a value (sign, two bits of exponent, one of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6), two codes a byte, the first one in
the low half.  The operators:

- ``norm``: residual addition, RMS norm, the norm's 16-bit output and its quantised form (int8 with a scale a row, or MXFP4);
- ``mx_quant``: quantisation of hidden states to MXFP4, and the values that the codes stand for;
- ``gate_up``: product of MXFP4 rows with their experts' gate and up weights, SwiGLU, quantisation to MXFP4;
- ``down``: product of MXFP4 rows with their experts' weights to 16 bits; ``dense``: the same with one weight for all rows;
- ``experts``: all experts of a layer on a batch of tokens whose routing is known: quantisation, both products, combine."""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

# hidden size, experts, experts per token, expert width
MODELS = {
    "small": dict(H=1024, E=8, k=2, I=1408),
    "qwen3": dict(H=2048, E=128, k=8, I=768),
    "dsv3": dict(H=7168, E=256, k=8, I=2048),
}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
CODES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _rows(name, op, tokens, hidden, dtype="bf16", **more):
    c = dict(op=op, tokens=tokens, hidden=hidden, dtype=dtype, **more)
    return dict(name=name, **c) if name else c


def _moe(name, op, tokens, model, dtype="bf16", zipf=0.0):
    """zipf: exponent of the experts' popularity (0: uniform)."""
    c = dict(op=op, tokens=tokens, dtype=dtype, zipf=zipf, **(MODELS[model] if isinstance(model, str) else model))
    return dict(name=name, **c) if name else c


def listed():
    return [
        # one user's chat turn, large layer: latency between two tokens
        _rows("norm_int8_1", "norm", 1, 7168, to="int8"),
        # a prefill batch of the large layer: bandwidth
        _rows("norm_int8_4096", "norm", 4096, 7168, to="int8"),
        # a step that mixes decoding sequences with a piece of a prompt, fp16, in front of MXFP4 experts
        _rows("norm_mx_777", "norm", 777, 2048, "fp16", to="mxfp4"),
        # the width of an expert, a few rows
        _rows("mx_quant_37", "mx_quant", 37, 1408, "fp16"),
        # a full prefill batch's hidden states
        _rows("mx_quant_8192", "mx_quant", 8192, 7168),
        # a serving engine's decode batch: four rows an expert, the weights stream from HBM
        _moe("gate_up_decode_64", "gate_up", 64, "qwen3"),
        # a full prefill batch: 512 rows an expert, matrix units
        _moe("gate_up_prefill_8192", "gate_up", 8192, "qwen3"),
        # the large layer's decode batch
        _moe("down_decode_64", "down", 64, "dsv3"),
        # a full prefill batch, prompts of one domain: few experts take most of the tokens
        _moe("down_zipf_4096", "down", 4096, "qwen3", "fp16", 1.1),
        # a linear layer on a piece of a prompt
        dict(name="dense_2048", op="dense", tokens=2048, K=7168, N=4096, dtype="bf16"),
        # one token through a layer's experts
        _moe("experts_1", "experts", 1, "qwen3"),
        # the large layer under skewed routing: the weights of all touched experts stream, a few have many rows
        _moe("experts_zipf_512", "experts", 512, "dsv3", zipf=1.1),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "mx_quant", "gate_up", "gate_up", "down", "down", "dense", "experts", "experts"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "norm":
        to = rng.choice(["int8", "mxfp4"])
        return _rows(None, op, _log(rng, 1, 4096), 32 * _log(rng, 2, 224) if to == "mxfp4" else 8 * _log(rng, 8, 896), dtype, to=to)
    if op == "mx_quant":
        return _rows(None, op, _log(rng, 1, 8192), 32 * _log(rng, 1, 224), dtype)
    if op == "dense":
        return dict(op=op, tokens=_log(rng, 1, 2048), K=64 * _log(rng, 1, 112), N=32 * _log(rng, 1, 128), dtype=dtype)
    if rng.random() < 0.5:
        model = rng.choice(["small", "qwen3", "qwen3"] + (["dsv3"] if op != "gate_up" else []))
    else:
        E = rng.choice([1, 4, 16, 60, 100, 160])
        model = dict(H=64 * _log(rng, 4, 64), E=E, k=rng.randint(1, min(E, 8)), I=64 * _log(rng, 2, 24))
    most = 512 if model == "dsv3" else 2048 if op == "experts" else 4096
    return _moe(None, op, _log(rng, 1, most), model, dtype, rng.choice([0.0, 0.0, 1.1]))


# ---------------------------------------------------------------------------------------------------- inputs
def _mx_parts(v):
    """float values [..., K] -> the exponent of every block (as the power of two's) and the values over that power,
    rounded to what four bits hold: nearest, ties to the even code, at most 6."""
    v = v.unflatten(-1, (-1, 32))
    largest = v.abs().amax(-1, keepdim=True)
    e = torch.frexp(largest).exponent - 3  # largest = m 2^(e + 3), m in [0.5, 1): floor(log2) - 2
    e = torch.where(largest > 0, e, -127).clamp(-127, 127)
    v = torch.ldexp(v, -e)
    a = v.abs().clamp(max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
    return e, torch.copysign(torch.round(a / step) * step, v)


def _pack(e, v):
    """The parts as bytes: codes [..., K / 2], scales [..., K / 32]."""
    order = torch.tensor(CODES[1:8], device=v.device, dtype=v.dtype)
    code = torch.bucketize(v.abs(), order, right=True).to(torch.uint8) + 8 * torch.signbit(v).to(torch.uint8)
    code = code.flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], (e.squeeze(-1) + 127).to(torch.uint8)


def _quantised(gen, shape, heavy):
    """Hidden states that an earlier operator has quantised. heavy: with a SwiGLU's tails."""
    x = torch.randn(shape, generator=gen, device="cuda")
    if heavy:
        x = x * torch.randn(shape, generator=gen, device="cuda")
    return _pack(*_mx_parts(x))


def _weights(gen, shape):
    """MXFP4 weights [..., N, K] with entries of about 0.02: codes as often as a bell shape has them, a slice at a time."""
    weight = [0.13, 0.25, 0.22, 0.14, 0.15, 0.07, 0.03, 0.01]
    often = torch.tensor([w / 2 for w in weight * 2], dtype=torch.float64)
    nibble = torch.searchsorted(often.cumsum(0).clamp(max=1 - 1e-9), (torch.arange(256, dtype=torch.float64) + 0.5) / 256)
    nibble = nibble.clamp(max=15).to(torch.uint8).cuda()
    codes = torch.empty((*shape[:-1], shape[-1] // 2), dtype=torch.uint8, device="cuda")
    for part in codes.view(-1).split(1 << 27):
        low, high = (nibble[torch.randint(0, 256, (part.numel(),), generator=gen, device="cuda", dtype=torch.uint8).int()]
                     for _ in range(2))
        part.copy_(low + 16 * high)
    scales = torch.randint(119, 122, (*shape[:-1], shape[-1] // 32), generator=gen, device="cuda", dtype=torch.uint8)
    return codes, scales


def _routing(gen, case):
    """Experts of every token, and the maps of their rows: sorted row -> token, rows of every expert."""
    T, E, k = case["tokens"], case["E"], case["k"]
    logits = torch.randn(T, E, generator=gen, device="cuda")
    if case["zipf"]:
        logits -= case["zipf"] * (torch.randperm(E, generator=gen, device="cuda").float() + 1).log()
    weights, ids = torch.softmax(logits, -1).topk(k, -1)
    row = ids.flatten().sort(stable=True).indices
    return (ids.int(), (weights / weights.sum(-1, keepdim=True)).to(DTYPES[case["dtype"]]), row,
            torch.bincount(ids.flatten(), minlength=E))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, T, dtype = case["op"], case["tokens"], DTYPES[case["dtype"]]
    s = {"case": case, "op": op, "dtype": dtype}
    if op in ("norm", "mx_quant"):
        H = case["hidden"]
        s["x"] = torch.randn(T, H, generator=gen, device="cuda").to(dtype)
        if op == "norm":
            s["residual"] = (3.0 * torch.randn(T, H, generator=gen, device="cuda")).to(dtype)
            s["gamma"] = (1.0 + 0.1 * torch.randn(H, generator=gen, device="cuda")).to(dtype)
        return s
    if op == "dense":
        s["x"], s["x_scale"] = _quantised(gen, (T, case["K"]), False)
        s["w"], s["w_scale"] = _weights(gen, (case["N"], case["K"]))
    else:
        E, H, I = case["E"], case["H"], case["I"]
        s["ids"], s["topk_weights"], row, s["counts"] = _routing(gen, case)
        s["most"] = int(s["counts"].max())
        if op != "down":
            s["row_token"] = (row // case["k"]).int()
            s["w13"], s["w13_scale"] = _weights(gen, (E, 2 * I, H))
        if op != "gate_up":
            s["w2"], s["w2_scale"] = _weights(gen, (E, H, I))
        if op == "experts":
            s["x"] = torch.randn(T, H, generator=gen, device="cuda").to(dtype)
            s["row"] = row
        else:
            s["x"], s["x_scale"] = _quantised(gen, (T, H) if op == "gate_up" else (row.numel(), I), op == "down")
    if own:
        # a program lays its weights out once, when it loads them
        from vllm_ascend_amd import npu_ops

        if op == "experts":
            s["layer"] = _layer(case, s)
        for name in ("w", "w13", "w2") if op != "experts" else ():
            if name in s:
                s[name + "_laid"], s[name + "_scale_laid"] = npu_ops.npu_format_cast_mx(s[name], s[name + "_scale"])
    return s


def _layer(case, s):
    from vllm_ascend_amd.fused_moe.contracts import FusedMoEConfig
    from vllm_ascend_amd.fused_moe.layer import AscendRoutedExperts
    from vllm_ascend_amd.fused_moe.router import AscendFusedTopKRouter
    from vllm_ascend_amd.quantization import get_scheme_class

    E, k, H, I = (case[n] for n in ("E", "k", "H", "I"))
    layer = AscendRoutedExperts(
        FusedMoEConfig(num_experts=E, experts_per_token=k, hidden_dim=H, intermediate_size_per_partition=I),
        get_scheme_class("W4A4_MXFP4", "moe")(in_dtype=s["dtype"]), AscendFusedTopKRouter(k, E))
    layer.load_weights({"w13_weight": s["w13"], "w13_weight_scale": s["w13_scale"], "w2_weight": s["w2"],
                        "w2_weight_scale": s["w2_scale"]})
    return layer


# ---------------------------------------------------------------------------------------------------- one pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from vllm_ascend_amd import npu_ops

    op, dtype = s["op"], s["dtype"]
    if op == "norm":
        int8 = s["case"]["to"] == "int8"
        q, scale, y, x = npu_ops.npu_add_rms_norm_dynamic_quant(
            s["x"], s["residual"], s["gamma"], epsilon=EPS, dst_type=torch.int8 if int8 else torch.float4_e2m1fn_x2)
        values = q * scale[:, None] if int8 else npu_ops.npu_mx_dequant(q, scale, dst_type=dtype)
        return {"x": x, "y": y, "values": values}
    if op == "mx_quant":
        return npu_ops.npu_mx_dequant(*npu_ops.npu_dynamic_mx_quant(s["x"]), dst_type=dtype)
    if op == "dense":
        return npu_ops.npu_quant_matmul(s["x"], s["w_laid"], s["w_scale_laid"], pertoken_scale=s["x_scale"],
                                        output_dtype=dtype)
    if op == "gate_up":
        q, scale = npu_ops.npu_grouped_matmul_swiglu_quant_v2(
            s["x"], s["w13_laid"], s["w13_scale_laid"], s["x_scale"], s["counts"], group_list_type=1,
            row_map=s["row_token"])
        return npu_ops.npu_mx_dequant(q, scale, dst_type=dtype)
    if op == "down":
        return npu_ops.npu_grouped_matmul(
            [s["x"]], [s["w2_laid"]], scale=[s["w2_scale_laid"]], per_token_scale=[s["x_scale"]],
            group_list=s["counts"], split_item=2, group_type=0, group_list_type=1, output_dtype=dtype)[0]
    layer = s["layer"]
    return layer.quant_method.apply(layer, s["x"], s["topk_weights"], s["ids"]).routed_out


def _values(codes, scales):
    """float32 values of packed codes and their blocks' scales."""
    pairs = torch.tensor([[CODES[b & 15], CODES[b >> 4]] for b in range(256)], device=codes.device)
    v = torch.nn.functional.embedding(codes.int(), pairs).flatten(-2)
    v.unflatten(-1, (-1, 32)).mul_(torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127).unsqueeze(-1))
    return v


def _mx(v):
    """Values [..., K] as MXFP4 holds them."""
    e, q = _mx_parts(v)
    return torch.ldexp(q, e).flatten(-2)


def _products(x, w, w_scale, counts, most):
    """Rows x [R, K] (sorted by expert) with their experts' weights [E, N, K]: float32 [R, N]."""
    R, E = x.shape[0], w.shape[0]
    expert = torch.repeat_interleave(torch.arange(E, device=x.device), counts, output_size=R)
    if R <= E:  # few rows: each with a copy of its expert's weights
        return torch.bmm(_values(w[expert], w_scale[expert]), x.unsqueeze(-1)).squeeze(-1)
    at = torch.arange(R, device=x.device) - (counts.cumsum(0) - counts)[expert]
    padded = x.new_zeros(E, most, x.shape[1])
    padded[expert, at] = x
    return torch.bmm(padded, _values(w, w_scale).transpose(1, 2))[expert, at]


def _swiglu_mx(acc):
    """SwiGLU in 64 bits (values next to the border between two codes), rounded to 32 and quantised."""
    gate, up = acc.double().chunk(2, -1)
    return _mx((gate / (1.0 + torch.exp(-gate)) * up).float())


def _run_plain(s):
    op, dtype = s["op"], s["dtype"]
    if op == "norm":
        x = s["x"] + s["residual"]
        # in 64 bits: a value next to the border between two codes goes to the right side of it
        v = x.double()
        v = v * (1.0 / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)) * s["gamma"].double()
        y = v.float().to(dtype)
        if s["case"]["to"] == "mxfp4":
            return {"x": x, "y": y, "values": _mx(y.float()).to(dtype)}
        f = y.float()
        scale = f.abs().amax(-1, keepdim=True) / torch.full((), 127.0, device=f.device)
        return {"x": x, "y": y, "values": torch.where(scale > 0, torch.round(f / scale), 0.0) * scale}
    if op == "mx_quant":
        return _mx(s["x"].float()).to(dtype)
    if op == "dense":
        return torch.mm(_values(s["x"], s["x_scale"]), _values(s["w"], s["w_scale"]).t()).to(dtype)
    if op == "gate_up":
        x = _values(s["x"], s["x_scale"])[s["row_token"]]
        return _swiglu_mx(_products(x, s["w13"], s["w13_scale"], s["counts"], s["most"])).to(dtype)
    if op == "down":
        x = _values(s["x"], s["x_scale"])
        return _products(x, s["w2"], s["w2_scale"], s["counts"], s["most"]).to(dtype)
    x = _mx(s["x"].float())[s["row_token"]]
    h = _swiglu_mx(_products(x, s["w13"], s["w13_scale"], s["counts"], s["most"]))
    out = _products(h, s["w2"], s["w2_scale"], s["counts"], s["most"]).to(dtype)
    pairs = torch.empty_like(out)
    pairs[s["row"]] = out
    pairs = pairs.view(*s["ids"].shape, -1).float() * s["topk_weights"].float().unsqueeze(-1)
    return pairs.sum(1).to(dtype)


# ---------------------------------------------------------------------------------------------------- from the definition
def _exact_values(codes, scales):
    table = torch.tensor(CODES, dtype=torch.float64, device=codes.device)
    v = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], -1).flatten(-2)
    return v * (2.0 ** (scales.double() - 127)).repeat_interleave(32, -1)


def _exact_mx(v):
    """Nearest of the values that four bits hold, by comparing with the middles between neighbours."""
    shape, v = v.shape, v.reshape(-1, 32)
    largest = v.abs().amax(-1, keepdim=True)
    power = 2.0 ** (torch.floor(torch.log2(torch.where(largest > 0, largest, 1.0))) - 2)
    a = v.abs() / power
    held = torch.tensor(CODES[:8], dtype=torch.float64, device=v.device)
    middle = (held[1:] + held[:-1]) / 2
    # at a middle the even one of the two codes: the upper one where its number is even
    up = torch.searchsorted(middle, a.contiguous())
    tie = torch.searchsorted(middle, a.contiguous(), right=True)
    code = torch.where((tie != up) & (tie % 2 == 0), tie, up)
    return (torch.sign(v) * held[code] * power).view(shape)


def _exact_products(x, w, w_scale, counts):
    out, begin = [], 0
    for e, n in enumerate(counts.tolist()):
        if n:
            out.append(x[begin:begin + n] @ _exact_values(w[e], w_scale[e]).t().contiguous())
        begin += n
    return torch.cat(out)


def _exact_swiglu_mx(acc):
    half = acc.shape[1] // 2
    gate, up = acc[:, :half], acc[:, half:]
    return _exact_mx((gate * torch.sigmoid(gate) * up).float().double())


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op, dtype = case["op"], s["dtype"]
    if op == "norm":
        x = s["x"].double() + s["residual"].double()
        v = x.float().to(dtype).double()
        y = v * s["gamma"].double() / torch.sqrt((v * v).sum(-1, keepdim=True) / v.shape[-1] + EPS)
        held = y.float().to(dtype).double()
        if case["to"] == "mxfp4":
            return {"x": x, "y": y, "values": _exact_mx(held)}
        scale = (held.abs().amax(-1, keepdim=True) / 127.0).float().double()
        return {"x": x, "y": y, "values": torch.round((held / scale.clamp(min=1e-300)).float().double()) * scale}
    if op == "mx_quant":
        return _exact_mx(s["x"].double())
    if op == "dense":
        return _exact_values(s["x"], s["x_scale"]) @ _exact_values(s["w"], s["w_scale"]).t().contiguous()
    if op == "down":
        return _exact_products(_exact_values(s["x"], s["x_scale"]), s["w2"], s["w2_scale"], s["counts"])
    if op == "gate_up":
        x = _exact_values(s["x"], s["x_scale"])[s["row_token"].long()]
        return _exact_swiglu_mx(_exact_products(x, s["w13"], s["w13_scale"], s["counts"]))
    x = _exact_mx(s["x"].double())[s["row_token"].long()]
    h = _exact_swiglu_mx(_exact_products(x, s["w13"], s["w13_scale"], s["counts"]))
    o = _exact_products(h, s["w2"], s["w2_scale"], s["counts"]).to(dtype).double()
    weight = s["topk_weights"].double().flatten()[s["row"]].unsqueeze(-1)
    return torch.zeros_like(s["x"], dtype=torch.float64).index_add_(0, s["row"] // case["k"], o * weight)


# ---------------------------------------------------------------------------------------------------- the least work
def _touched(case):
    """How many experts such a batch touches, by drawing one."""
    E, k = case["E"], case["k"]
    rng = np.random.default_rng(1)
    prior = -case["zipf"] * np.log(np.arange(1, E + 1))
    hit = np.zeros(E, dtype=bool)
    for _ in range(min(case["tokens"], 2048)):
        hit[np.argpartition(-(rng.standard_normal(E) + prior), k - 1)[:k]] = True
    return int(hit.sum())


def work(case):
    op, T = case["op"], case["tokens"]
    held = 17 / 32  # bytes of an MXFP4 value with its share of the scale
    if op == "norm":
        n = T * case["hidden"]
        return {"bytes": n * (8 + (1 if case["to"] == "int8" else held)) + 2 * case["hidden"], "flops": 10 * n}
    if op == "mx_quant":  # the codes are what the path writes; the values are their reading
        n = T * case["hidden"]
        return {"bytes": n * (2 + 2 * held + 2), "flops": 4 * n}
    if op == "dense":
        K, N = case["K"], case["N"]
        return {"bytes": held * K * (T + N) + 2 * T * N, "flops": 2 * T * K * N}
    H, I, R, E = case["H"], case["I"], T * case["k"], _touched(case)
    if op == "gate_up":
        return {"bytes": held * (T * H + E * 2 * I * H + 2 * R * I) + 2 * R * I + 4 * R, "flops": 4 * R * H * I}
    if op == "down":
        return {"bytes": held * (R * I + E * I * H) + 2 * R * H, "flops": 2 * R * H * I}
    return {"bytes": held * E * 3 * I * H + 4 * T * H, "flops": 6 * R * H * I}
