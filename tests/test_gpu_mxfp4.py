"""The MXFP4 operators and the norm on the GPU against their definition in 64 bits.  What is compared is equal bit for bit: sums
of products of four-bit values are exact in 32 bits for scales a few powers of two apart (24 bits hold K * 36 / 0.25 * 2^spread
for every K and spread here that matters: a sum's typical size is sqrt(K) * 8 units, 2^10 for K = 7168, times 2^(2 * spread)), and
what is rounded is rounded once from the value of the formula."""
import numpy as np
import pytest
import torch

import _mxfp4 as ref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def K():
    from vllm_ascend_amd import kernels

    return kernels


@pytest.fixture(scope="module")
def ops():
    from vllm_ascend_amd import npu_ops

    return npu_ops


def say(*a):
    print(*a, flush=True)


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
    return t if dtype is None else t.to(dtype)


def same_bits(a, b):
    return torch.equal(a.cpu().view(torch.int16), b.cpu().view(torch.int16))


# ------------------------------------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (37, 1408), (2, 5, 7168), (513, 64), (1, 8224)], ids=str)
def test_mx_quant(ops, dtype, shape):
    say("mx_quant", dtype, shape)
    g = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-9, 9, (*shape[:-1], 1), generator=g).float())
    x = x.to(dtype)
    codes, scale = ops.npu_dynamic_mx_quant(x.to(DEV))
    c, s = ref.quantise(x.double().numpy())
    assert codes.shape == (*shape[:-1], shape[-1] // 2) and scale.shape == (*shape[:-1], shape[-1] // 32)
    assert np.array_equal(codes.cpu().numpy(), ref.pack(c)) and np.array_equal(scale.cpu().numpy(), s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_mx_quant_borders_and_special_values(ops, dtype):
    say("mx_quant borders", dtype)
    info = torch.finfo(dtype)
    rows = []
    borders = [0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0]
    for power in (0, -3, 5):
        for b in borders:  # the border, its neighbours of the type, under a largest value that fixes the scale
            t = torch.tensor([b], dtype=torch.float64).to(dtype)
            up, down = t * (1 + info.eps), t * (1 - info.eps / 2)
            block = torch.cat([t, up, down, -t, -up, -down, torch.tensor([4.0, 0.0, -0.0], dtype=dtype)])
            rows.append(torch.cat([block.double() * 2.0 ** power, torch.zeros(32 - len(block)).double()]))
    rows.append(torch.zeros(32).double())
    rows.append(-torch.zeros(32).double())
    for v in (info.max, info.tiny, info.smallest_normal, float(torch.finfo(dtype).smallest_normal) / 4):
        rows.append(torch.linspace(-1, 1, 32).double() * v)
    for v in (float("inf"), -float("inf"), float("nan")):
        r = torch.linspace(-1, 1, 32).double()
        r[7] = v
        rows.append(r)
    x = torch.stack(rows).to(dtype)
    codes, scale = ops.npu_dynamic_mx_quant(x.to(DEV))
    c, s = ref.quantise(x.double().numpy())
    assert np.array_equal(scale.cpu().numpy(), s)
    assert np.array_equal(codes.cpu().numpy(), ref.pack(c))


def test_mx_quant_of_views(ops):
    """Transposed rows, and rows that start at an address no wide load may start at."""
    say("mx_quant views")
    x = torch.randn(64, 96, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    flat = torch.empty(32 * 5 + 1, dtype=torch.bfloat16, device=DEV)
    flat.copy_(torch.arange(161) / 7)
    for v in (x.t(), x[:, :64], x[::2], flat[1:].view(5, 32)):
        c, s = ref.quantise(v.double().cpu().numpy())
        codes, scale = ops.npu_dynamic_mx_quant(v)
        assert np.array_equal(codes.cpu().numpy(), ref.pack(c)) and np.array_equal(scale.cpu().numpy(), s)
    codes, scale = ops.npu_dynamic_mx_quant(torch.empty(0, 64, dtype=torch.bfloat16, device=DEV))
    assert codes.shape == (0, 32) and scale.shape == (0, 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_mx_dequant_of_every_code_and_scale(ops, dtype):
    say("mx_dequant", dtype)
    code = np.tile(np.arange(32, dtype=np.uint8) % 16, (256, 1))
    scale = np.arange(256, dtype=np.uint8)[:, None]
    got = ops.npu_mx_dequant(dev(ref.pack(code)), dev(scale), dst_type=dtype).cpu()
    with np.errstate(over="ignore"):
        want = torch.from_numpy(ref.values(code, scale).astype(np.float32)).to(dtype)
    assert torch.equal(got.nan_to_num(nan=-7.0), want.nan_to_num(nan=-7.0)) and torch.equal(got.isnan(), want.isnan())
    assert torch.equal(torch.signbit(got[:255]), torch.signbit(want[:255]))


# ------------------------------------------------------------------------------------------------ norm
def norm_ref(x1, x2, gamma, beta, eps):
    x = x1 if x2 is None else (x1.float() + x2.float()).to(x1.dtype)
    v = x.double().numpy()
    y = v * (1.0 / np.sqrt((v * v).mean(-1, keepdims=True) + eps)) * gamma.double().numpy()
    if beta is not None:
        y = y + beta.double().numpy()
    return x, ref.rounded(y, x1.dtype)


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("rows,cols,residual,bias,wide", [
    (1, 32, True, False, False), (3, 96, False, True, False), (5, 1024, True, True, True), (777, 2048, True, False, False),
    (2, 7168, True, False, True), (4, 8192, False, False, False), (3, 8224, True, True, False), (2, 16384, True, False, False),
    (2, 16416, True, True, False), (3, 40960, False, False, True)])
def test_norm_with_every_kind_of_output(K, dtype, rows, cols, residual, bias, wide):
    say("norm", dtype, rows, cols, residual, bias, wide)
    g = torch.Generator().manual_seed(rows + cols)
    x1 = (torch.randn(rows, cols, generator=g) * 3).to(dtype)
    x2 = torch.randn(rows, cols, generator=g).to(dtype) if residual else None
    kind = torch.float32 if wide else dtype
    gamma = (1 + 0.2 * torch.randn(cols, generator=g)).to(kind)
    beta = (0.1 * torch.randn(cols, generator=g)).to(kind) if bias else None
    x, y = norm_ref(x1, x2, gamma, beta, 1e-6)
    on = [None if t is None else t.to(DEV) for t in (x1, x2, gamma, beta)]
    for to in (K.NORM_INT8, K.NORM_MXFP4, K.NORM_PLAIN):
        q, scale, got_y, got_x = K.add_rms_norm_quant(*on, 1e-6, to)
        assert same_bits(got_x, x) and same_bits(got_y, y)
        if to == K.NORM_INT8:  # what the token quantiser of the framework makes of y
            want_q, want_scale = K.dynamic_quant(got_y)
            assert torch.equal(q, want_q) and torch.equal(scale, want_scale)
        elif to == K.NORM_MXFP4:
            want_q, want_scale = ref.quantise(y.double().numpy())
            assert np.array_equal(q.cpu().numpy(), ref.pack(want_q)) and np.array_equal(scale.cpu().numpy(), want_scale)
        else:
            assert q is None and scale is None


@pytest.mark.parametrize("cols", [8, 40, 1000, 8200, 20488])
def test_norm_to_int8_of_odd_widths(ops, K, cols):
    say("norm int8", cols)
    g = torch.Generator().manual_seed(cols)
    x1, x2 = (torch.randn(7, cols, generator=g).to(torch.bfloat16) for _ in range(2))
    gamma = torch.rand(cols, generator=g).to(torch.bfloat16)
    x1[3], x2[3] = 0, 0      # a row of zeros
    x1[4, 0] = float("nan")  # and rows that are not numbers
    x1[5, 1] = float("inf")
    q, scale, y, x = ops.npu_add_rms_norm_dynamic_quant(x1.to(DEV), x2.to(DEV), gamma.to(DEV))
    keep = [0, 1, 2, 3, 6]
    want_x, want_y = norm_ref(x1[keep], x2[keep], gamma, None, 1e-6)
    assert same_bits(x[keep], want_x) and same_bits(y[keep], want_y)
    assert y[4].isnan().all() and y[5, 1].isnan()
    want_q, want_scale = K.dynamic_quant(y)
    assert torch.equal(q, want_q) and torch.equal(scale.nan_to_num(nan=-1.0), want_scale.nan_to_num(nan=-1.0))
    assert not q[3].any() and scale[3] == 0


@pytest.mark.parametrize("cols", [7168, 16384, 20480])
@pytest.mark.parametrize("kind", [1, 2])
def test_norm_in_place(K, cols, kind):
    """The sum may be written over either of its operands."""
    from vllm_ascend_amd import _lib

    say("norm in place", cols, kind)
    g = torch.Generator().manual_seed(cols)
    x1, x2 = (torch.randn(3, cols, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    gamma = torch.rand(cols, generator=g).to(torch.bfloat16).to(DEV)
    q, scale, y, x = K.add_rms_norm_quant(x1, x2, gamma, None, 1e-6, kind)
    for over in (0, 1):
        a, b = x1.clone(), x2.clone()
        q2, scale2, y2 = torch.empty_like(q), torch.empty_like(scale), torch.empty_like(y)
        _lib.check(_lib.load().moe355_add_rms_norm_quant(
            a.data_ptr(), b.data_ptr(), gamma.data_ptr(), None, 1, 1, 3, cols, 1e-6, kind, (a, b)[over].data_ptr(),
            y2.data_ptr(), q2.data_ptr(), scale2.data_ptr(), torch.cuda.current_stream().cuda_stream), "norm")
        assert torch.equal((a, b)[over], x) and torch.equal(y2, y) and torch.equal(q2, q) and torch.equal(scale2, scale)


# ------------------------------------------------------------------------------------------------ products
def counts_of(rng, E, rows, kind):
    if kind == "even":
        return np.bincount(np.arange(rows) % E, minlength=E)
    if kind == "one":  # all rows at the last expert but one, the others empty
        c = np.zeros(E, dtype=np.int64)
        c[max(E - 2, 0)] = rows
        return c
    p = 1.0 / np.arange(1, E + 1) ** 1.1
    return np.bincount(rng.choice(E, rows, p=rng.permutation(p / p.sum())), minlength=E)


PRODUCTS = [
    # E, N, K, rows, how they are spread
    (1, 64, 64, 1, "even"), (1, 64, 128, 33, "even"), (3, 128, 192, 7, "zipf"), (4, 64, 256, 64, "one"),
    (5, 192, 320, 100, "zipf"), (8, 2816, 1024, 64, "zipf"), (8, 1024, 1408, 130, "even"), (128, 1536, 2048, 512, "zipf"),
    (16, 128, 7168, 32, "zipf"), (2, 256, 704, 300, "zipf"), (7, 320, 448, 700, "zipf"), (1, 512, 512, 1000, "even"),
    (3, 1088, 576, 1900, "zipf"), (300, 64, 64, 900, "zipf"), (2, 4096, 512, 5, "one"), (1, 320, 1024, 257, "even"),
    (4, 704, 960, 2100, "zipf"),
]


def make_product(E, N, Kd, rows, kind, seed=0, spread=2, tokens=None, heavy=False):
    rng = np.random.default_rng(seed + E * 1000 + N + Kd + rows)
    counts = counts_of(rng, E, rows, kind)
    row_token = None if tokens is None else rng.integers(0, tokens, rows).astype(np.int32)
    xc, xs = ref.random_mx(rng, (rows if tokens is None else tokens, Kd), spread, heavy)
    wc, ws = ref.random_mx(rng, (E, N, Kd), spread)
    ws = ws - 5  # weights of about 0.03
    return rng, counts, row_token, xc, xs, wc, ws


@pytest.mark.parametrize("case", PRODUCTS, ids=str)
@pytest.mark.parametrize("dtype", HALF, ids=str)
def test_product_to_16_bits(ops, case, dtype):
    say("gmm_mx", case, dtype)
    _, counts, _, xc, xs, wc, ws = make_product(*case, heavy=True)
    w, s = ops.npu_format_cast_mx(dev(ref.pack(wc)), dev(ws))
    want = ref.rounded(ref.products(ref.values(xc, xs), ref.values(wc, ws), counts), dtype)
    for list_type, group_list in ((1, counts), (0, counts.cumsum())):
        out = ops.npu_grouped_matmul([dev(ref.pack(xc))], [w], scale=[s], per_token_scale=[dev(xs)],
                                     group_list=dev(group_list.astype(np.int64)), split_item=2, group_type=0,
                                     group_list_type=list_type, output_dtype=dtype)[0]
        assert out.dtype == dtype and same_bits(out, want)


@pytest.mark.parametrize("case", PRODUCTS, ids=str)
@pytest.mark.parametrize("limit", [0.0, 0.75])
def test_product_with_swiglu(ops, case, limit):
    """Codes and scales are those of the formula in 64 bits, next to the borders between two codes as well."""
    say("gmm_mx_swiglu_quant", case, limit)
    tokens = max(1, case[3] // 3)
    _, counts, row_token, xc, xs, wc, ws = make_product(*case, seed=1, tokens=tokens)
    w, s = ops.npu_format_cast_mx(dev(ref.pack(wc)), dev(ws))
    codes, scale = ops.npu_grouped_matmul_swiglu_quant_v2(
        dev(ref.pack(xc)), [w], [s], dev(xs), dev(counts.astype(np.int64)), group_list_type=1, swiglu_limit=limit,
        row_map=dev(row_token))
    y = ref.swiglu(ref.products(ref.values(xc, xs), ref.values(wc, ws), counts, row_token), limit)
    c, sc = ref.quantise(y)
    assert np.array_equal(scale.cpu().numpy(), sc) and np.array_equal(codes.cpu().numpy(), ref.pack(c))


@pytest.mark.parametrize("rows", [40, 700])
def test_rows_that_no_group_has_stay_as_they_were(K, rows):
    from vllm_ascend_amd import _lib

    say("rows outside the groups", rows)
    E, N, Kd = 5, 192, 320
    _, counts, _, xc, xs, wc, ws = make_product(E, N, Kd, rows, "zipf")
    counts = np.maximum(counts - 3, 0)
    used = int(counts.sum())
    w, s = K.format_cast_mx(dev(ref.pack(wc)), dev(ws))
    x, x_scale, lib = dev(ref.pack(xc)), dev(xs), _lib.load()
    n = max(lib.moe355_gmm_mx_workspace(rows, N, E, swiglu) for swiglu in (0, 1))
    space = torch.empty(max(n, 1), dtype=torch.uint8, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    want = ref.rounded(ref.products(ref.values(xc, xs), ref.values(wc, ws), counts)[:used], torch.bfloat16)
    for list_type, gl in ((1, counts), (0, counts.cumsum())):
        gl = dev(gl.astype(np.int64))
        out = torch.full((rows, N), 7.0, dtype=torch.bfloat16, device=DEV)
        _lib.check(lib.moe355_gmm_mx(x.data_ptr(), x_scale.data_ptr(), None, rows, w.data_ptr(), s.data_ptr(), gl.data_ptr(),
                                     list_type, rows, Kd, N, E, out.data_ptr(), 1, space.data_ptr(), n, stream), "gmm_mx")
        assert same_bits(out[:used], want) and (out[used:] == 7.0).all()
        codes = torch.full((rows, N // 4), 9, dtype=torch.uint8, device=DEV)
        scale = torch.full((rows, N // 64), 9, dtype=torch.uint8, device=DEV)
        _lib.check(lib.moe355_gmm_mx_swiglu_quant(
            x.data_ptr(), x_scale.data_ptr(), None, rows, w.data_ptr(), s.data_ptr(), gl.data_ptr(), list_type, rows, Kd, N, E,
            0.0, codes.data_ptr(), scale.data_ptr(), space.data_ptr(), n, stream), "gmm_mx_swiglu_quant")
        assert (codes[used:] == 9).all() and (scale[used:] == 9).all()
        y = ref.swiglu(ref.products(ref.values(xc, xs), ref.values(wc, ws), counts)[:used])
        c, sc = ref.quantise(y)
        assert np.array_equal(codes[:used].cpu().numpy(), ref.pack(c)) and np.array_equal(scale[:used].cpu().numpy(), sc)


@pytest.mark.parametrize("rows", [40, 700])
def test_group_lists_that_ask_for_more_than_there_is(ops, rows):
    """Counts past the last row, negative ones, sums that go back: rows are cut to those that exist, none is written twice by
    two experts of a list of counts, and nothing outside is read or written."""
    say("group lists out of range", rows)
    E, N, Kd = 4, 64, 128
    _, _, _, xc, xs, wc, ws = make_product(E, N, Kd, rows, "even")
    w, s = ops.npu_format_cast_mx(dev(ref.pack(wc)), dev(ws))
    x, x_scale = dev(ref.pack(xc)), dev(xs)
    half = rows // 2
    for list_type, gl, counts in (
            (1, [half, 10 * rows, 5, 1 << 40], [half, rows - half, 0, 0]),
            (1, [-4, half, -1, rows], [0, half, 0, rows - half]),
            (0, [half, half, 1 << 50, 1 << 50], [half, 0, rows - half, 0])):
        out = ops.npu_grouped_matmul([x], [w], scale=[s], per_token_scale=[x_scale], group_list=torch.tensor(gl, device=DEV),
                                     split_item=2, group_type=0, group_list_type=list_type)[0]
        assert same_bits(out, ref.rounded(ref.products(ref.values(xc, xs), ref.values(wc, ws), counts), torch.bfloat16))


@pytest.mark.parametrize("rows", [9, 600])
def test_row_map_with_rows_that_are_not_there(ops, rows):
    """An index outside the rows counts as a row of zeros; the same index may come any number of times."""
    say("row map out of range", rows)
    E, N, Kd, tokens = 2, 128, 192, 5
    _, counts, row_token, xc, xs, wc, ws = make_product(E, N, Kd, rows, "even", tokens=tokens)
    row_token[::4] = [-1, tokens, 2**31 - 1, -(2**31)][: len(row_token[::4])] if rows < 16 else -1
    row_token[1::4] = 3
    w, s = ops.npu_format_cast_mx(dev(ref.pack(wc)), dev(ws))
    codes, scale = ops.npu_grouped_matmul_swiglu_quant_v2(
        dev(ref.pack(xc)), w, s, dev(xs), dev(counts.astype(np.int64)), group_list_type=1, row_map=dev(row_token))
    c, sc = ref.quantise(ref.swiglu(ref.products(ref.values(xc, xs), ref.values(wc, ws), counts, row_token)))
    assert np.array_equal(codes.cpu().numpy(), ref.pack(c)) and np.array_equal(scale.cpu().numpy(), sc)


@pytest.mark.parametrize("rows", [6, 600])
def test_scales_that_stand_for_nan_and_far_powers(ops, rows):
    """A block without a value makes its row's results NaN and no other row's; powers of two at the ends of fp32 hold."""
    say("special scales", rows)
    E, N, Kd = 2, 64, 128
    rng, counts, _, xc, xs, wc, ws = make_product(E, N, Kd, rows, "even")
    xs[0], xs[1], xs[2] = 255, 0, 250  # NaN; 2^-127, a weight's 2^-8 on top: below fp32; 2^123
    xs[3, 1] = 255
    wc[0, 5, :32] = 0
    ws[0, 5, 0], ws[:, 7] = 255, 0
    w, s = ops.npu_format_cast_mx(dev(ref.pack(wc)), dev(ws))
    out = ops.npu_grouped_matmul([dev(ref.pack(xc))], [w], scale=[s], per_token_scale=[dev(xs)],
                                 group_list=dev(counts.astype(np.int64)), split_item=2, group_type=0, group_list_type=1)[0]
    out = out.cpu().double().numpy()
    x, wv = ref.values(xc, xs), ref.values(wc, ws)
    with np.errstate(invalid="ignore", over="ignore"):
        want = ref.rounded(ref.products(x, wv, counts), torch.bfloat16).double().numpy()
    assert np.array_equal(np.isnan(out), np.isnan(want))
    # results below the smallest normal number may be zero
    keep = ~np.isnan(want) & ((np.abs(want) >= 2.0 ** -126) | (want == 0))
    assert np.array_equal(out[keep], want[keep])
    assert (np.abs(out[~keep & ~np.isnan(want)]) < 2.0 ** -125).all()


@pytest.mark.parametrize("rows", [20, 600])
def test_swiglu_of_gates_far_from_zero(ops, rows):
    """Gates below the range of a 32-bit exponential, results that overflow, results of zero."""
    say("far gates", rows)
    E, N, Kd = 2, 128, 64
    rng, counts, _, xc, xs, wc, ws = make_product(E, N, Kd, rows, "even", spread=0)
    for i, p in enumerate([0, 3, 4, 5, 6, 8, 40, 60, 70]):
        xs[i::9] = 127 + p
    xc[4] = 0
    w, s = ops.npu_format_cast_mx(dev(ref.pack(wc)), dev(ws + 5))
    codes, scale = ops.npu_grouped_matmul_swiglu_quant_v2(
        dev(ref.pack(xc)), w, s, dev(xs), dev(counts.astype(np.int64)), group_list_type=1)
    with np.errstate(over="ignore", invalid="ignore"):
        c, sc = ref.quantise(ref.swiglu(ref.products(ref.values(xc, xs), ref.values(wc, ws + 5), counts)))
    assert np.array_equal(scale.cpu().numpy(), sc)
    c[np.repeat(sc == 0, 32, -1)] = 0  # blocks at the smallest scale: subnormal values
    got = ref.unpack(codes.cpu().numpy())
    got[np.repeat(sc == 0, 32, -1)] = 0
    assert np.array_equal(got, c)


@pytest.mark.parametrize("rows,N,Kd", [(1, 32, 64), (5, 96, 320), (130, 4096, 7168), (1000, 672, 1408)])
def test_dense_product(ops, rows, N, Kd):
    say("dense", rows, N, Kd)
    _, _, _, xc, xs, wc, ws = make_product(1, N, Kd, rows, "even")
    w, s = ops.npu_format_cast_mx(dev(ref.pack(wc[0])), dev(ws[0]))
    out = ops.npu_quant_matmul(dev(ref.pack(xc)), w, s, pertoken_scale=dev(xs), output_dtype=torch.float16)
    assert same_bits(out, ref.rounded(ref.values(xc, xs) @ ref.values(wc, ws)[0].T, torch.float16))
    lead = ops.npu_quant_matmul(dev(ref.pack(xc))[None], w, s, pertoken_scale=dev(xs)[None], output_dtype=torch.float16)
    assert lead.shape == (1, rows, N) and torch.equal(lead[0], out)


# ------------------------------------------------------------------------------------------------ together
def build(E, k, H, I, dtype=torch.bfloat16, seed=0, shared=None, **layer_kw):
    from vllm_ascend_amd.fused_moe.contracts import FusedMoEConfig
    from vllm_ascend_amd.fused_moe.layer import AscendRoutedExperts
    from vllm_ascend_amd.fused_moe.router import AscendFusedTopKRouter
    from vllm_ascend_amd.quantization import get_scheme_class

    rng = np.random.default_rng(seed)
    w13, s13 = ref.random_mx(rng, (E, 2 * I, H), 1)
    w2, s2 = ref.random_mx(rng, (E, H, I), 1)
    s13, s2 = s13 - 5, s2 - 5
    layer = AscendRoutedExperts(
        FusedMoEConfig(num_experts=E, experts_per_token=k, hidden_dim=H, intermediate_size_per_partition=I),
        get_scheme_class("W4A4_MXFP4", "moe")(in_dtype=dtype), AscendFusedTopKRouter(k, E, renormalize=True), device=DEV,
        shared_experts=shared, **layer_kw)
    layer.load_weights({"w13_weight": torch.from_numpy(ref.pack(w13)), "w13_weight_scale": torch.from_numpy(s13),
                        "w2_weight": torch.from_numpy(ref.pack(w2)), "w2_weight_scale": torch.from_numpy(s2)})
    return layer, ref.values(w13, s13), ref.values(w2, s2)


def experts_ref(y, ids, weights, w13, w2, dtype, residual=None):
    """The layer of hidden states y, expert by expert in 64 bits, rounded where the path rounds."""
    T, k = ids.shape
    order = np.argsort(ids.reshape(-1), kind="stable")
    counts = np.bincount(ids.reshape(-1), minlength=len(w13))
    x = ref.values(*ref.quantise(y.double().cpu().numpy()))[order // k]
    h = ref.values(*ref.quantise(ref.swiglu(ref.products(x, w13, counts))))
    o = ref.rounded(ref.products(h, w2, counts), dtype).double().numpy()
    pairs = np.empty_like(o)
    pairs[order] = o
    out = (pairs.reshape(T, k, -1) * weights.double().cpu().numpy()[:, :, None]).sum(1)
    return out if residual is None else out + residual


def close(got, want, dtype, k):
    """One rounding to 16 bits (half a step) and k additions in 32 bits: 2^-8 or 2^-11 of the value plus k 2^-24 of the terms'
    size, for which the row's largest value times sqrt(k) stands.  Below the smallest normal number 2^m the type's steps are all
    2^m eps (fp16: 2^-14 2^-10 = 2^-24), so the rounding there is off by up to 2^m eps / 2 however small the value."""
    got = got.double().cpu().numpy()
    info = torch.finfo(dtype)
    bound = np.maximum(np.abs(want), info.smallest_normal) * info.eps / 2 * 1.001
    bound += k * 2.0 ** -24 * np.abs(want).max(-1, keepdims=True) * 4
    return bool((np.abs(got - want) <= bound).all())


@pytest.mark.parametrize("T,E,k,H,I,dtype", [
    (1, 8, 2, 256, 192, torch.bfloat16), (5, 8, 2, 1024, 1408, torch.float16), (64, 60, 4, 448, 128, torch.bfloat16),
    (300, 16, 8, 512, 320, torch.bfloat16), (700, 4, 2, 576, 704, torch.float16)])
def test_norm_and_layer_together(ops, T, E, k, H, I, dtype):
    """Residual addition and norm, the router on the norm's output, the experts on its MXFP4 form."""
    say("norm and layer", T, E, k, H, I, dtype)
    layer, w13, w2 = build(E, k, H, I, dtype)
    g = torch.Generator().manual_seed(T)
    x1, x2 = (torch.randn(T, H, generator=g).to(dtype).to(DEV) for _ in range(2))
    gamma = (1 + 0.1 * torch.randn(H, generator=g)).to(dtype).to(DEV)
    logits = torch.randn(T, E, generator=g).to(DEV)
    codes, scale, y, x = ops.npu_add_rms_norm_dynamic_quant(x1, x2, gamma, dst_type=torch.float4_e2m1fn_x2)
    weights, ids = layer.router.select_experts(y, logits)
    want = experts_ref(y, ids.cpu().numpy(), weights, w13, w2, dtype)
    out = layer(y, logits)
    assert out.shape == y.shape and out.dtype == dtype and close(out, want, dtype, k)
    layer.ascend_pertoken_scale = scale  # the rows as the norm has quantised them
    assert torch.equal(layer(codes, logits), out)
    res = layer.forward_impl(codes, logits)
    assert torch.equal(res.expert_tokens.cpu(), torch.bincount(ids.flatten().cpu().long(), minlength=E))


def test_layer_with_a_shared_expert(ops):
    from vllm_ascend_amd.fused_moe.shared_experts import AscendSharedExperts

    say("layer with a shared expert")
    T, E, k, H, I = 33, 8, 2, 256, 128
    g = torch.Generator().manual_seed(2)
    up = torch.randint(-127, 128, (2 * I, H), generator=g, dtype=torch.int8).to(DEV)
    down = torch.randint(-127, 128, (H, I), generator=g, dtype=torch.int8).to(DEV)
    su, sd = (torch.rand(n, generator=g).to(DEV) * 1e-3 for n in (2 * I, H))
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV)
    logits = torch.randn(T, E, generator=g).to(DEV)
    for overlap in (False, True):
        shared = AscendSharedExperts(up, su, down, sd, multistream_overlap=overlap)
        layer, w13, w2 = build(E, k, H, I, shared=shared)
        weights, ids = layer.router.select_experts(x, logits)
        extra = shared(x)
        shared.wait()
        want = experts_ref(x, ids.cpu().numpy(), weights, w13, w2, torch.bfloat16, extra.double().cpu().numpy())
        assert close(layer(x, logits), want, torch.bfloat16, k + 1)


def test_int8_layer_on_rows_that_the_norm_quantised(ops):
    """The norm's int8 rows and the 16-bit ones give the W8A8 layer the same bits."""
    from _inputs import CONFIGS, make_layer
    from _layer_utils import build_layer

    say("int8 layer behind the norm")
    cfg = CONFIGS["c2_small"]
    layer = build_layer(cfg, make_layer(cfg, seed=0), DEV)
    g = torch.Generator().manual_seed(3)
    x1, x2 = (torch.randn(cfg.T, cfg.H, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    gamma = (1 + 0.1 * torch.randn(cfg.H, generator=g)).to(torch.bfloat16).to(DEV)
    logits = torch.randn(cfg.T, cfg.E, generator=g).to(DEV)
    q, scale, y, _ = ops.npu_add_rms_norm_dynamic_quant(x1, x2, gamma)
    want = layer(y, logits)
    layer.ascend_pertoken_scale = scale
    assert torch.equal(layer(q, logits), want)


@pytest.mark.parametrize("T", [4, 400])
def test_captured_and_replayed(ops, T):
    """Norm and layer in a graph, replayed on other inputs with eager calls between."""
    say("graph", T)
    E, k, H, I = 8, 2, 512, 256
    layer, _, _ = build(E, k, H, I)
    g = torch.Generator().manual_seed(T)
    x1, x2 = (torch.empty(T, H, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    logits = torch.empty(T, E, device=DEV)
    gamma = torch.ones(H, dtype=torch.bfloat16, device=DEV)

    def fill():
        for t in (x1, x2, logits):
            t.copy_(torch.randn(t.shape, generator=g))

    def step():
        codes, scale, y, x = ops.npu_add_rms_norm_dynamic_quant(x1, x2, gamma, dst_type=torch.float4_e2m1fn_x2)
        weights, ids = layer.router.select_experts(y, logits)
        return x, layer.quant_method.apply(layer, y, weights, ids).routed_out

    fill()
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs over the same layer
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for i in range(4):
        fill()
        for graph, _ in graphs:
            graph.replay()
        want = step()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_on_another_stream(ops):
    say("other stream")
    layer, _, _ = build(8, 2, 512, 256)
    g = torch.Generator().manual_seed(5)
    x, logits = torch.randn(50, 512, generator=g).to(torch.bfloat16).to(DEV), torch.randn(50, 8, generator=g).to(DEV)
    want = layer(x, logits)
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams * 3:
        with torch.cuda.stream(s):
            outs.append(layer(x, logits))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_layer_of_no_tokens(ops):
    say("no tokens")
    layer, _, _ = build(8, 2, 512, 256)
    out = layer.quant_method.apply(layer, torch.empty(0, 512, dtype=torch.bfloat16, device=DEV),
                                   torch.empty(0, 2, device=DEV), torch.empty(0, 2, dtype=torch.int32, device=DEV)).routed_out
    assert out.shape == (0, 512)


# ------------------------------------------------------------------------------------------------ where it can go wrong
def both_products(K, E, N, Kd, x, x_scale, w, s, gl, list_type=1, row_map=None):
    """-> (16-bit rows, codes, scales) of the two forms of output."""
    return (K.gmm_mx(x, x_scale, w, s, gl, list_type, row_map=row_map),
            *K.gmm_mx_swiglu_quant(x, x_scale, w, s, gl, list_type, row_map=row_map))


def check_both(got, acc, used=None):
    out, codes, scale = (t[:used] for t in got)
    acc = acc[:used]
    with np.errstate(invalid="ignore"):
        want = ref.rounded(acc, out.dtype)
        c, sc = ref.quantise(ref.swiglu(acc))
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(out.cpu()), nan)
    assert same_bits(out.cpu().masked_fill(nan, 0), want.masked_fill(nan, 0))
    assert np.array_equal(scale.cpu().numpy(), sc) and np.array_equal(codes.cpu().numpy(), ref.pack(c))


@pytest.mark.parametrize("rows", [9, 600])
def test_rows_that_are_not_there_have_nobodys_scale(K, rows):
    """Row 0 of x has no value (its scales stand for NaN), and a block of weights has none either: a row that is not there is
    zeros times the weights, NaN in that block's channel only."""
    say("absent rows beside NaN", rows)
    E, N, Kd, tokens = 2, 128, 320, 5
    _, counts, row_token, xc, xs, wc, ws = make_product(E, N, Kd, rows, "even", tokens=tokens)
    xs[0] = 255
    ws[1, 3, 2] = 255
    row_token[row_token == 0] = 1
    row_token[::3] = -1
    row_token[1::5] = tokens
    row_token[2::7] = 0
    w, s = K.format_cast_mx(dev(ref.pack(wc)), dev(ws))
    got = both_products(K, E, N, Kd, dev(ref.pack(xc)), dev(xs), w, s, dev(counts.astype(np.int64)), row_map=dev(row_token))
    with np.errstate(invalid="ignore"):
        check_both(got, ref.products(ref.values(xc, xs), ref.values(wc, ws), counts, row_token))


@pytest.mark.parametrize("E,rows,kind", [(600, 4000, "zipf"), (1100, 4500, "even"), (600, 3700, "one")])
@pytest.mark.parametrize("list_type", [0, 1])
def test_tiles_from_a_list(K, E, rows, kind, list_type):
    """Many experts with many rows each could have: the products make a list of the tiles first."""
    from vllm_ascend_amd import _lib

    say("listed tiles", E, rows, kind, list_type)
    N, Kd = 64, 128
    assert _lib.load().moe355_gmm_mx_workspace(rows, N, E, 0) and _lib.load().moe355_gmm_mx_workspace(rows, N, E, 1)
    _, counts, _, xc, xs, wc, ws = make_product(E, N, Kd, rows, kind)
    counts[0] = max(counts[0] - 5, 0)  # rows behind the last group
    used = int(counts.sum())
    w, s = K.format_cast_mx(dev(ref.pack(wc)), dev(ws))
    gl = dev(np.asarray(counts if list_type else counts.cumsum()).astype(np.int64))
    x, x_scale = dev(ref.pack(xc)), dev(xs)
    acc = ref.products(ref.values(xc, xs), ref.values(wc, ws), counts)
    check_both(both_products(K, E, N, Kd, x, x_scale, w, s, gl, list_type), acc, used)
    check_both(both_products(K, E, N, Kd, x, x_scale, w, s, gl.int(), list_type), acc, used)


@pytest.mark.parametrize("list_type", [0, 1])
def test_lists_of_tiles_out_of_range(K, list_type):
    say("listed tiles, lists out of range", list_type)
    E, N, Kd, rows = 600, 64, 64, 4000
    _, _, _, xc, xs, wc, ws = make_product(E, N, Kd, rows, "even")
    counts = np.zeros(E, dtype=np.int64)
    counts[[0, 2, 599]] = [1500, 1, 2499]
    gl = np.zeros(E, dtype=np.int64)
    if list_type:
        gl[0], gl[1], gl[2], gl[599] = 1500, -7, 1, 1 << 45
    else:
        gl[:2], gl[2:599], gl[599] = 1500, 1501, 1 << 45
    w, s = K.format_cast_mx(dev(ref.pack(wc)), dev(ws))
    got = both_products(K, E, N, Kd, dev(ref.pack(xc)), dev(xs), w, s, dev(gl), list_type)
    check_both(got, ref.products(ref.values(xc, xs), ref.values(wc, ws), counts))


@pytest.mark.parametrize("rows", [5, 300])
def test_operands_that_are_views(K, rows):
    """Scales at odd addresses, codes that no wide load may start at, transposed and strided operands, lists of int32."""
    say("views", rows)
    E, N, Kd = 2, 128, 192
    _, counts, _, xc, xs, wc, ws = make_product(E, N, Kd, rows, "even")
    x, x_scale = dev(ref.pack(xc)), dev(xs)
    w, s = K.format_cast_mx(dev(ref.pack(wc)), dev(ws))
    acc = ref.products(ref.values(xc, xs), ref.values(wc, ws), counts)

    def at(t, offset):
        room = torch.zeros(t.numel() + offset, dtype=torch.uint8, device=DEV)
        room[offset:] = t.flatten()
        return room[offset:].view(t.shape)

    gl = dev(counts.astype(np.int32))
    check_both(both_products(K, E, N, Kd, at(x, 8), at(x_scale, 1), at(w, 4), at(s, 3), gl), acc)
    check_both(both_products(K, E, N, Kd, x.t().contiguous().t(), x_scale.t().contiguous().t(), w, s, gl), acc)
    check_both(both_products(K, E, N, Kd, x.repeat_interleave(2, 0)[::2], x_scale.repeat(1, 2)[:, :Kd // 32], w, s, gl), acc)
    w2, s2 = K.format_cast_mx(at(dev(ref.pack(wc)), 8), at(dev(ws), 1))
    assert torch.equal(w2, w) and torch.equal(s2, s)


def test_one_row_with_two_scales(ops):
    """K = 64: less memory at the scales than the kernels read at a time."""
    say("two scales")
    _, _, _, xc, xs, wc, ws = make_product(1, 32, 64, 1, "even")
    w, s = ops.npu_format_cast_mx(dev(ref.pack(wc[0])), dev(ws[0]))
    out = ops.npu_quant_matmul(dev(ref.pack(xc)), w, s, pertoken_scale=dev(xs), output_dtype=torch.bfloat16)
    assert same_bits(out, ref.rounded(ref.values(xc, xs) @ ref.values(wc, ws)[0].T, torch.bfloat16))


def test_output_larger_than_the_last_cache(K):
    """Such an output is stored past it; channels repeat, so that the reference stays small."""
    say("far stores")
    rows, Kd, distinct, times = 3210, 64, 1024, 32
    _, _, _, xc, xs, wc, ws = make_product(1, distinct, Kd, rows, "even")
    w, s = K.format_cast_mx(dev(ref.pack(wc)).repeat(1, times, 1), dev(ws).repeat(1, times, 1))
    out = K.gmm_mx(dev(ref.pack(xc)), dev(xs), w, s, None, 1)
    want = ref.rounded(ref.values(xc, xs) @ ref.values(wc, ws)[0].T, torch.bfloat16).to(DEV)
    for part in out.view(rows, times, distinct).unbind(1):
        assert torch.equal(part, want)


def op_by_op(K, x, x_scale, ids, weights, w13, s13, w2, s2, limit, residual):
    if x_scale is None:
        x, x_scale = K.dynamic_mx_quant(x)
    dst, row_token, tokens = K.route_map(ids, w13.shape[0], 1)
    h, hs = K.gmm_mx_swiglu_quant(x, x_scale, w13, s13, tokens, 1, limit, row_token)
    out = K.gmm_mx(h, hs, w2, s2, tokens, 1, weights.dtype)
    return K.token_unpermute(out, dst, weights, residual), tokens


@pytest.mark.parametrize("T,E,k,H,I,dtype", [
    (1, 8, 2, 64, 64, torch.bfloat16), (40, 16, 4, 320, 192, torch.float16), (900, 8, 2, 256, 448, torch.bfloat16),
    (2100, 600, 2, 64, 64, torch.bfloat16),   # listed tiles, more experts than one launch of the routing has
    (1200, 400, 5, 64, 64, torch.float16),    # listed tiles, their list made by the routing
    (9000, 16, 8, 128, 64, torch.bfloat16)])  # more rows than one launch of the routing has
def test_experts_as_one_call(K, T, E, k, H, I, dtype):
    """The same bits as the operators one after the other; ids outside the experts count for nothing."""
    say("experts", T, E, k, H, I, dtype)
    rng = np.random.default_rng(T)
    w13, s13 = ref.random_mx(rng, (E, 2 * I, H), 1)
    w2, s2 = ref.random_mx(rng, (E, H, I), 1)
    held = (*K.format_cast_mx(dev(ref.pack(w13)), dev(s13 - 5)), *K.format_cast_mx(dev(ref.pack(w2)), dev(s2 - 5)))
    g = torch.Generator().manual_seed(T)
    x, residual = (torch.randn(T, H, generator=g).to(dtype).to(DEV) for _ in range(2))
    weights = torch.rand(T, k, generator=g).to(dtype).to(DEV)
    ids = torch.from_numpy((rng.zipf(1.3, (T, k)) % E).astype(np.int32)).to(DEV)
    outside = ids.clone()
    outside.view(-1)[::3] = -1
    outside.view(-1)[1::7] = E
    for chosen in (ids, outside):
        for limit, res in ((0.0, None), (0.5, residual)):
            want, want_tokens = op_by_op(K, x, None, chosen, weights, *held, limit, res)
            for given in ((x, None), K.dynamic_mx_quant(x)):
                out, tokens = K.mx_experts(*given, chosen, weights, *held, limit, res)
                assert torch.equal(tokens, want_tokens) and torch.equal(out, want)
    nothing, none = K.mx_experts(x, None, torch.full_like(ids, -1), weights, *held)
    assert not nothing.any() and not none.any()
    # the rows whose ids are all inside, against the formula
    y = experts_ref(x[:64], ids[:64].cpu().numpy(), weights[:64], ref.values(w13, s13 - 5), ref.values(w2, s2 - 5), dtype)
    assert close(K.mx_experts(x, None, ids, weights, *held)[0][:64], y, dtype, k)


def test_layer_of_rows_in_three_dimensions(ops):
    say("three dimensions")
    layer, _, _ = build(8, 2, 512, 256)
    g = torch.Generator().manual_seed(6)
    x, logits = torch.randn(30, 512, generator=g).to(torch.bfloat16).to(DEV), torch.randn(30, 8, generator=g).to(DEV)
    weights, ids = layer.router.select_experts(x, logits)
    want = layer.quant_method.apply(layer, x, weights, ids).routed_out
    assert torch.equal(layer.quant_method.apply(layer, x.view(3, 10, 512), weights, ids).routed_out, want.view(3, 10, 512))
    codes, layer.ascend_pertoken_scale = (t.view(3, 10, -1) for t in ops.npu_dynamic_mx_quant(x))
    assert torch.equal(layer.quant_method.apply(layer, codes, weights, ids).routed_out, want.view(3, 10, 512))


def test_products_captured_and_replayed_on_two_streams(K):
    """Two graphs of the same product, one of listed tiles, replayed on two streams at once on changing rows."""
    say("products in graphs")
    E, N, Kd, rows = 600, 64, 128, 4000
    _, counts, _, xc, xs, wc, ws = make_product(E, N, Kd, rows, "zipf")
    w, s = K.format_cast_mx(dev(ref.pack(wc)), dev(ws))
    x, x_scale, gl = dev(ref.pack(xc)), dev(xs), dev(counts.astype(np.int64))
    both_products(K, E, N, Kd, x, x_scale, w, s, gl)
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for _ in streams:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both_products(K, E, N, Kd, x, x_scale, w, s, gl)
        graphs.append((graph, out))
    for i in range(4):
        x.copy_(torch.roll(x, 1, 0))
        gl.copy_(torch.roll(gl, 7, 0))
        want = both_products(K, E, N, Kd, x, x_scale, w, s, gl)
        torch.cuda.synchronize()
        for stream, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("E,rows,kind", [(300, 40, "zipf"), (300, 299, "even"), (1100, 9, "even"), (700, 650, "one"), (2, 1, "even"),
                                         (256, 255, "zipf"), (257, 200, "zipf"), (65, 64, "even")])
@pytest.mark.parametrize("list_type", [0, 1])
def test_fewer_rows_than_experts(K, E, rows, kind, list_type):
    say("few rows", E, rows, kind, list_type)
    N, Kd = 64, 576
    rng, counts, _, xc, xs, wc, ws = make_product(E, N, Kd, rows, kind)
    counts = rng.permutation(counts)
    counts[counts.argmax()] -= 1  # a row behind the last group
    used = int(counts.sum())
    w, s = K.format_cast_mx(dev(ref.pack(wc)), dev(ws))
    gl = dev(np.asarray(counts if list_type else counts.cumsum()).astype(np.int64))
    check_both(both_products(K, E, N, Kd, dev(ref.pack(xc)), dev(xs), w, s, gl, list_type),
               ref.products(ref.values(xc, xs), ref.values(wc, ws), counts), used)


@pytest.mark.parametrize("list_type,gl,counts", [
    (1, {3: -9, 4: 7, 90: 1 << 50, 200: 4, 299: -1}, {4: 7, 90: 33}),
    (1, {0: 40, 7: 40, 299: 40}, {0: 40}),
    (0, [(0, -5), (10, 3), (100, 1 << 50)], {10: 3, 100: 37}),
    (0, [(0, 40), (299, 41)], {0: 40}),
    (1, {}, {}), (0, [], {})])
def test_fewer_rows_than_experts_and_lists_out_of_range(K, list_type, gl, counts):
    say("few rows, lists out of range", list_type, gl)
    E, N, Kd, rows = 300, 64, 64, 40
    _, _, _, xc, xs, wc, ws = make_product(E, N, Kd, rows, "even")
    given, want = np.zeros(E, dtype=np.int64), np.zeros(E, dtype=np.int64)
    for e, n in gl.items() if list_type else gl:
        if list_type:
            given[e] = n
        else:
            given[e:] = n
    for e, n in counts.items():
        want[e] = n
    w, s = K.format_cast_mx(dev(ref.pack(wc)), dev(ws))
    check_both(both_products(K, E, N, Kd, dev(ref.pack(xc)), dev(xs), w, s, dev(given), list_type),
               ref.products(ref.values(xc, xs), ref.values(wc, ws), want), int(want.sum()))


@pytest.mark.parametrize("T,E,k,H,I", [
    (1, 8, 1, 64, 64), (3, 5, 3, 192, 320), (16, 4, 4, 1024, 704), (8, 300, 8, 448, 64), (1, 128, 8, 2048, 768), (2, 8, 2, 7168, 192),
    (1, 2, 2, 64, 2048), (5, 16, 7, 576, 128), (1, 1, 1, 16384, 64), (4, 2048, 6, 320, 256), (7, 6, 5, 8192, 64),
    (17, 8, 2, 64, 64), (13, 8, 5, 64, 64), (32, 16, 4, 512, 256), (16, 128, 8, 192, 64),
    # just past what the form takes: 33 tokens, 9 slots, 130 pairs, more weights or more read again than it is worth
    (33, 8, 2, 64, 64), (2, 16, 9, 64, 64), (26, 8, 5, 64, 64), (8, 64, 6, 2048, 1408), (32, 8, 2, 1024, 1408)])
@pytest.mark.parametrize("dtype", HALF, ids=str)
def test_experts_of_a_few_tokens(K, T, E, k, H, I, dtype):
    """The bits of the operators one after the other: ids that repeat, within a token too, ids outside, infinities and NaN in a row."""
    say("few tokens", T, E, k, H, I, dtype)
    rng = np.random.default_rng(T * 100 + E)
    w13, s13 = ref.random_mx(rng, (E, 2 * I, H), 1)
    w2, s2 = ref.random_mx(rng, (E, H, I), 1)
    held = (*K.format_cast_mx(dev(ref.pack(w13)), dev(s13 - 5)), *K.format_cast_mx(dev(ref.pack(w2)), dev(s2 - 5)))
    g = torch.Generator().manual_seed(T)
    x, residual = (torch.randn(T, H, generator=g).to(dtype).to(DEV) for _ in range(2))
    weights = torch.rand(T, k, generator=g).to(dtype).to(DEV)
    ids = torch.from_numpy(rng.integers(0, E, (T, k)).astype(np.int32)).to(DEV)
    outside, same = ids.clone(), torch.full_like(ids, E - 1)
    outside.view(-1)[::3], outside.view(-1)[1::4] = -1, E
    odd = x.clone()
    odd[0, 0], odd[-1, 33] = float("inf"), float("nan")
    for rows, chosen in ((x, ids), (x, outside), (x, same), (odd, ids)):
        for limit, res in ((0.0, None), (0.5, residual)):
            want, want_tokens = op_by_op(K, rows, None, chosen, weights, *held, limit, res)
            for given in ((rows, None), K.dynamic_mx_quant(rows)):
                out, tokens = K.mx_experts(*given, chosen, weights, *held, limit, res)
                assert torch.equal(tokens, want_tokens)
                assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(nan=9.0), want.nan_to_num(nan=9.0))
    if H * I * T * k < 1 << 24:  # against the formula
        y = experts_ref(x, ids.cpu().numpy(), weights, ref.values(w13, s13 - 5), ref.values(w2, s2 - 5), dtype)
        assert close(K.mx_experts(x, None, ids, weights, *held)[0], y, dtype, k)


@pytest.mark.parametrize("E,N,Kd,rows", [(1, 64, 7168, 1), (1, 4096, 4096, 20), (4, 128, 2048, 9), (2, 512, 4096, 700),
                                        (1, 1024, 8192, 300), (600, 64, 1024, 4000)])
def test_sums_that_32_bits_do_not_hold(K, E, N, Kd, rows):
    """Blocks up to 2^40 apart.  Every addition of at most K, to a sum of 24 bits that may be cut off instead of rounded, is off by
    at most 2^-23 of what the magnitudes add up to, and the result by half a step of bf16 on top: its steps are 2^-7 of the power of
    two below a value, half of one is at most 2^-8 of the value."""
    say("inexact sums", E, N, Kd, rows)
    rng, counts, _, xc, xs, wc, ws = make_product(E, N, Kd, rows, "even")
    xs = rng.integers(107, 147, xs.shape).astype(np.uint8)
    w, s = K.format_cast_mx(dev(ref.pack(wc)), dev(ws))
    got = K.gmm_mx(dev(ref.pack(xc)), dev(xs), w, s, dev(counts.astype(np.int64)), 1).double().cpu().numpy()
    x, wv = ref.values(xc, xs), ref.values(wc, ws)
    want = ref.products(x, wv, counts)
    bound = np.abs(want) * 2.0 ** -8 * 1.001 + Kd * 2.0 ** -23 * ref.products(np.abs(x), np.abs(wv), counts)
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("E,rows", [(3, 2), (3, 9), (3, 900), (600, 4000)])
def test_group_lists_at_the_ends_of_64_bits(K, E, rows):
    say("group lists at the ends", E, rows)
    N, Kd = 1600 if E == 3 else 64, 64
    _, _, _, xc, xs, wc, ws = make_product(E, N, Kd, rows, "even")
    w, s = K.format_cast_mx(dev(ref.pack(wc)), dev(ws))
    most, least = (1 << 63) - 1, -(1 << 63)
    acc = ref.products(ref.values(xc, xs), ref.values(wc, ws), [0, rows] + [0] * (E - 2))
    for list_type, gl in ((1, [least, most, most]), (0, [least, most, most]), (0, [0, most, least]), (1, [least, rows, least])):
        gl = gl + [gl[-1]] * (E - 3)
        check_both(both_products(K, E, N, Kd, dev(ref.pack(xc)), dev(xs), w, s, torch.tensor(gl, device=DEV), list_type), acc)


@pytest.mark.parametrize("T", [3, 100])
def test_experts_from_two_threads_and_streams(K, T):
    """Calls at once on two streams, each thread with tensors of its own, against calls one after the other."""
    import threading

    say("two threads", T)
    E, k, H, I = 8, 2, 512, 256
    rng = np.random.default_rng(T)
    w13, s13 = ref.random_mx(rng, (E, 2 * I, H), 1)
    w2, s2 = ref.random_mx(rng, (E, H, I), 1)
    held = (*K.format_cast_mx(dev(ref.pack(w13)), dev(s13 - 5)), *K.format_cast_mx(dev(ref.pack(w2)), dev(s2 - 5)))
    inputs = []
    for i in range(2):
        g = torch.Generator().manual_seed(i)
        inputs.append((torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV), None,
                       torch.from_numpy(rng.integers(0, E, (T, k)).astype(np.int32)).to(DEV),
                       torch.rand(T, k, generator=g).to(torch.bfloat16).to(DEV)))
    want = [K.mx_experts(*a, *held) for a in inputs]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(K.mx_experts(*inputs[i], *held))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert len(got[i]) == 20
        assert all(torch.equal(o, want[i][0]) and torch.equal(n, want[i][1]) for o, n in got[i])


@pytest.mark.parametrize("case", [(128, 1536, 2048, 512, "zipf"), (3, 1088, 576, 1900, "zipf"), (4, 704, 960, 2100, "zipf"),
                                  (1, 512, 192, 1000, "even"), (600, 64, 320, 4000, "zipf"), (16, 128, 2048, 200, "zipf")], ids=str)
def test_products_on_cold_caches(K, case):
    """Rows and weights come late, out of the memory itself: nothing may be used in front of its arrival."""
    say("cold caches", case)
    E, N, Kd, _, _ = case
    _, counts, _, xc, xs, wc, ws = make_product(*case)
    w, s = K.format_cast_mx(dev(ref.pack(wc)), dev(ws))
    x, x_scale, gl = dev(ref.pack(xc)), dev(xs), dev(counts.astype(np.int64))
    acc = ref.products(ref.values(xc, xs), ref.values(wc, ws), counts)
    other = torch.empty(1 << 28, dtype=torch.float32, device=DEV)
    first = None
    for i in range(12):
        other.fill_(i)
        got = both_products(K, E, N, Kd, x, x_scale, w, s, gl)
        if first is None:
            check_both(got, acc)
            first = got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


@pytest.mark.parametrize("E,rows", [(3, 9), (3, 900), (600, 4000), (300, 40)])
def test_counts_far_past_the_last_row_behind_other_groups(K, E, rows):
    """A count that no sum of 64 bits holds is cut like any other, in every form: the rest of the rows are its expert's."""
    say("far counts", E, rows)
    N, Kd, first = 1600 if E == 3 else 64, 64, 5
    _, _, _, xc, xs, wc, ws = make_product(E, N, Kd, rows, "even")
    w, s = K.format_cast_mx(dev(ref.pack(wc)), dev(ws))
    most = (1 << 63) - 1
    acc = ref.products(ref.values(xc, xs), ref.values(wc, ws), [first, rows - first] + [0] * (E - 2))
    for count, behind in ((most, 0), (most, most), (most - first, 1), (most - first + 1, 0), (most - rows, most)):
        gl = torch.tensor([first, count] + [behind] * (E - 2), device=DEV)
        check_both(both_products(K, E, N, Kd, dev(ref.pack(xc)), dev(xs), w, s, gl), acc)


@pytest.mark.parametrize("dtype", HALF, ids=str)
def test_layer_of_codes_under_the_names_of_their_types(ops, dtype):
    say("layer of named codes", dtype)
    layer, _, _ = build(8, 2, 512, 256, dtype)
    g = torch.Generator().manual_seed(7)
    x, logits = torch.randn(30, 512, generator=g).to(dtype).to(DEV), torch.randn(30, 8, generator=g).to(DEV)
    want = layer(x, logits)
    codes, scale = ops.npu_dynamic_mx_quant(x)
    layer.ascend_pertoken_scale = scale.view(torch.float8_e8m0fnu)
    for given in (codes, codes.view(torch.float4_e2m1fn_x2)):
        assert torch.equal(layer(given, logits), want)
