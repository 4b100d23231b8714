"""The block operators (``native.fp8_quantize`` / ``fp8_gemm`` / ``fp8_linear``, ``native.block_norm``, ``native.rotary``)
against plain 64-bit forms written here.

Tolerances.  ``half_step(t)`` = ``finfo(t).eps / 2`` is the largest relative error of one rounding (bf16 2^-8, fp16 2^-11);
every output is rounded once.  To it comes the error of fp32 arithmetic, counted in units of U = 2^-24 of the magnitudes
that were added: stated where each bound is written."""
import importlib
import itertools
import math

import pytest
import torch

P = "fastwamjoint_quantization_b200."
U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def native(pkg):
    return importlib.import_module(P + "native")


@pytest.fixture(scope="module")
def quant(pkg):
    return importlib.import_module(P + "quant")


@pytest.fixture(scope="module")
def rope(pkg):
    return importlib.import_module(P + "rotary")


@pytest.fixture(autouse=True)
def no_device_timeouts(request, pkg):
    yield
    if "gpu" in request.keywords and torch.cuda.is_available():
        torch.cuda.synchronize()
        assert importlib.import_module(P + "native").device_status() == 0


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def within(got, want, slack, dtype):
    """|got - want| <= one rounding of the result + ``slack`` (fp32 error), NaN exactly where NaN is wanted."""
    got, want = got.double(), want.double()
    assert torch.equal(got.isnan(), want.isnan())
    finite = want.isfinite()
    assert torch.equal(got[~finite & ~want.isnan()], want[~finite & ~want.isnan()])
    slack = torch.as_tensor(slack, dtype=torch.float64, device=want.device).expand_as(want)
    # a subnormal result is rounded to a fixed grid: half of its spacing
    allowed = half_step(dtype) * (want.abs() + slack) + slack + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    bad = ((got - want).abs() > allowed) & finite
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() - allowed)[finite].max()))


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


# ------------------------------------------------------------------------------------------------- e4m3 linear
def fp8_case(quant, m, n, k, dtype, bias=True, seed=0):
    x = randn(m, k, seed=seed) * torch.where(randn(k, seed=seed + 1).abs() > 2.5, 20.0, 1.0)
    codes, scales = quant.quantize_token_runs(x.to(dtype))
    weight, weight_scales = quant.quantize_weight_block(randn(n, k, seed=seed + 2, scale=0.02))
    b = randn(n, seed=seed + 3, dtype=dtype, scale=0.1) if bias else None
    return x.to(dtype), codes.contiguous(), scales, weight, weight_scales, b


def fp8_product(codes, scales, weight, weight_scales, bias):
    """(y, sum of magnitudes) in 64 bits."""
    n, k = weight.shape
    a = codes.double() * scales.double().repeat_interleave(128, dim=1)[:, :k]
    w = weight.double() * weight_scales.double().repeat_interleave(128, dim=0)[:n].repeat_interleave(128, dim=1)[:, :k]
    y, size = a @ w.t(), a.abs() @ w.abs().t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size


def fp8_slack(size, k):
    # a sum of at most 128 products on the tensor core, 2 multiplications by scales, the runs added one by one, the bias:
    # each step off by at most 2 U (the tensor core may cut instead of round) of the magnitudes added
    return 2 * U * (128 + 2 + -(-k // 128) + 1) * size


GEMM_SHAPES = [(1, 8, 16), (1, 4096, 4096), (3, 136, 144), (16, 128, 128), (17, 264, 1024), (32, 4096, 1024), (64, 200, 2000),
               (65, 1480, 272), (127, 128, 4096), (128, 1024, 1040), (129, 1032, 128), (256, 256, 256), (257, 264, 384),
               (294, 1024, 14336), (500, 1488, 2000), (1592, 4096, 1024), (2049, 2056, 528)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", GEMM_SHAPES)
def test_fp8_gemm_against_64_bits(native, quant, m, n, k, dtype):
    _, codes, scales, weight, weight_scales, bias = fp8_case(quant, m, n, k, dtype, bias=(m + n) % 3 != 0)
    got = native.fp8_gemm(codes, scales, weight, weight_scales, bias, out_dtype=dtype)
    want, size = fp8_product(codes, scales, weight, weight_scales, bias)
    assert got.shape == (m, n) and got.dtype == dtype
    within(got, want, fp8_slack(size, k), dtype)
    # the same bits again, and whatever strides the scales have
    assert torch.equal(got, native.fp8_gemm(codes, scales.t().contiguous().t(), weight, weight_scales, bias, out_dtype=dtype))


@gpu
def test_fp8_gemm_of_many_tiles_equals_its_rows(native, quant):
    """Long K and several waves of tiles: every row of the whole product against 64 bits, in slices."""
    m, n, k = 4100, 3080, 4096
    _, codes, scales, weight, weight_scales, bias = fp8_case(quant, m, n, k, torch.bfloat16)
    got = native.fp8_gemm(codes, scales, weight, weight_scales, bias, out_dtype=torch.bfloat16)
    want, size = fp8_product(codes, scales, weight, weight_scales, bias)
    within(got, want, fp8_slack(size, k), torch.bfloat16)


@gpu
def test_fp8_gemm_writes_its_rows_and_nothing_else(native, quant):
    for m, n, k in ((1, 8, 16), (33, 72, 128), (130, 136, 256), (300, 264, 512)):
        _, codes, scales, weight, weight_scales, bias = fp8_case(quant, m, n, k, torch.bfloat16)
        room = torch.full((m + 64, n), 7.0, device="cuda", dtype=torch.bfloat16)
        out = native.fp8_gemm(codes, scales, weight, weight_scales, bias, out_dtype=torch.bfloat16, out=room[:m])
        assert out.data_ptr() == room.data_ptr() and (room[m:] == 7.0).all()


@gpu
@pytest.mark.parametrize("m", [5, 300, 1100])
def test_fp8_bias_off_the_vector_grid_and_strided_codes(native, quant, m):
    n, k = 264, 512
    _, codes, scales, weight, weight_scales, bias = fp8_case(quant, m, n, k, torch.bfloat16)
    want = native.fp8_gemm(codes, scales, weight, weight_scales, bias, out_dtype=torch.bfloat16)
    shifted = torch.zeros(n + 1, device="cuda", dtype=torch.bfloat16)
    shifted[1:] = bias
    wide = torch.zeros(m, 2 * k, device="cuda", dtype=torch.uint8)
    wide[:, :k] = codes.view(torch.uint8)
    got = native.fp8_gemm(wide.view(torch.float8_e4m3fn)[:, :k], scales.contiguous(), weight, weight_scales, shifted[1:],
                          out_dtype=torch.bfloat16)
    assert torch.equal(got, want)
    one = scales[:, :1].expand(m, scales.shape[1])  # one scale per token, broadcast over the runs
    got = native.fp8_gemm(codes, one, weight, weight_scales, out_dtype=torch.bfloat16)
    assert torch.equal(got, native.fp8_gemm(codes, one.contiguous(), weight, weight_scales, out_dtype=torch.bfloat16))


@gpu
def test_fp8_non_finite_values_stay_in_their_rows(native, quant):
    m, n, k = 40, 256, 384
    x, _, _, weight, weight_scales, _ = fp8_case(quant, m, n, k, torch.bfloat16)
    x[3, 130], x[17, 0], x[39, 383] = float("nan"), float("inf"), float("-inf")
    codes, scales = native.fp8_quantize(x)
    y = native.fp8_gemm(codes, scales, weight, weight_scales, out_dtype=torch.bfloat16)
    bad = torch.zeros(m, dtype=torch.bool, device="cuda")
    bad[[3, 17, 39]] = True
    assert torch.equal(y.isnan().all(dim=1), bad) and torch.equal(y.isnan().any(dim=1), bad)
    want, size = fp8_product(codes[~bad], scales[~bad], weight, weight_scales, None)
    within(y[~bad], want, fp8_slack(size, k), torch.bfloat16)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 16), (1, 128), (2, 144), (5, 256), (33, 1040), (7, 14336), (294, 4096), (4097, 272)])
def test_fp8_quantize_is_the_rule_bit_for_bit(native, quant, rows, k, dtype):
    x = randn(rows, k, dtype=dtype, scale=3.0)
    x[0, : min(k, 128)] = 0            # a run of zeros: the smallest scale, zero codes
    x[-1, -1] = torch.finfo(dtype).max  # the largest value of the type
    if rows > 2:
        x[1] = torch.finfo(dtype).smallest_normal
    codes, scales = native.fp8_quantize(x)
    want_codes, want_scales = quant.quantize_token_runs(x.cpu())  # IEEE division on the host
    assert codes.shape == x.shape and scales.shape == (rows, -(-k // 128))
    assert torch.equal(scales.cpu(), want_scales)
    assert torch.equal(codes.cpu().view(torch.uint8), want_codes.contiguous().view(torch.uint8))


@gpu
@pytest.mark.parametrize("m,n,k", [(1, 64, 128), (32, 1024, 1024), (300, 264, 2000), (1592, 512, 4096)])
@pytest.mark.parametrize("gelu", [False, True])
def test_fp8_linear_is_quantizer_and_product(native, quant, m, n, k, gelu):
    x, _, _, weight, weight_scales, bias = fp8_case(quant, m, n, k, torch.bfloat16)
    act = "gelu" if gelu else None
    codes, scales = native.fp8_quantize(x, input_activation=act)
    two = native.fp8_gemm(codes, scales, weight, weight_scales, bias, out_dtype=torch.bfloat16)
    for _ in range(3):  # back to back: the set-up of each product overlaps the quantizer in front of it
        one = native.fp8_linear(x, weight, weight_scales, bias, input_activation=act)
        assert torch.equal(one, two)
    if gelu:  # the activation itself: a code is off by half a step of e4m3 (2^-4, or half of 2^-9 scales) and erf by a few U
        value = x.double() * torch.special.ndtr(x.double())
        s = scales.double().repeat_interleave(128, dim=1)[:, :k]
        err = (codes.double() * s - value).abs()
        assert (err <= value.abs() * 2.0 ** -4 * (1 + 1e-5) + s * 2.0 ** -10 + 16 * U * x.double().abs()).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gelu_of_every_value(native, dtype):
    """Every finite 16-bit value, one per run so that its code is 448 and its scale carries the activation: what the kernel
    computes of x * Phi(x) to fp32.  The bound: fit 1.1e-7; t 2 U (reciprocal and sum), exp 2 U and its argument 2 U of
    x^2 / 2, eight products and sums of P at U each, four products, the scale's two divisions."""
    bits = torch.arange(-32768, 32768, dtype=torch.int32, device="cuda").to(torch.int16).view(dtype)
    x = bits[torch.isfinite(bits)]
    x = x[: x.numel() // 16 * 16].contiguous()
    rows = torch.zeros(x.numel(), 128, device="cuda", dtype=dtype)
    rows[:, 0] = x
    codes, scales = native.fp8_quantize(rows, input_activation="gelu")
    exact = x.double() * torch.special.ndtr(x.double())
    seen = exact.abs() > 448e-8  # below, the scale is the floor's
    got = codes[:, 0].double().sign() * scales[:, 0].double() * 448
    assert (codes[seen, 0].float().abs() == 448).all() and not codes[:, 1:].float().any()
    bound = 1.1e-7 + U * (20 + x.double() ** 2 * (x < 0))
    assert ((got - exact).abs()[seen] <= (bound * exact.abs())[seen]).all()
    odd = torch.zeros(4, 128, device="cuda", dtype=dtype)
    odd[0, 5], odd[1, 5], odd[2, 5] = math.inf, -math.inf, math.nan
    scales = native.fp8_quantize(odd, input_activation="gelu")[1].cpu()[:, 0]
    assert torch.isinf(scales[0]) and torch.isnan(scales[1:3]).all() and scales[3] == 1e-8


@gpu
def test_fp8_linear_views_streams_graphs(native, quant):
    m, n, k = 96, 512, 1024
    x, _, _, weight, weight_scales, bias = fp8_case(quant, m, n, k, torch.bfloat16)
    want = native.fp8_linear(x, weight, weight_scales, bias)
    wide = torch.zeros(m, k + 8, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:k + 3] = x  # rows that are not contiguous and start off the vector grid
    assert torch.equal(native.fp8_linear(wide[:, 3:k + 3], weight, weight_scales, bias), want)
    flat = torch.zeros(m * k + 1, device="cuda", dtype=torch.bfloat16)
    flat[1:] = x.flatten()  # contiguous, off by one element
    assert torch.equal(native.fp8_linear(flat[1:].view(2, m // 2, k), weight, weight_scales, bias), want.view(2, m // 2, n))
    assert native.fp8_linear(x[:0], weight, weight_scales, bias).shape == (0, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = native.fp8_linear(x, weight, weight_scales, bias)
    side.synchronize()
    assert torch.equal(on_side, want)
    # two graphs with workspaces of their own from the graph pools, replayed in either order on new inputs
    graphs = []
    for i in range(2):
        static = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = native.fp8_linear(static, weight, weight_scales, bias)
            y2 = native.fp8_linear(static * 2, weight, weight_scales, bias)
        graphs.append((static, graph, y, y2))
    for i in (1, 0, 1):
        static, graph, y, y2 = graphs[i]
        fresh = randn(m, k, seed=50 + i, dtype=torch.bfloat16)
        static.copy_(fresh)
        graph.replay()
        assert torch.equal(y, native.fp8_linear(fresh, weight, weight_scales, bias))
        assert torch.equal(y2, native.fp8_linear(fresh * 2, weight, weight_scales, bias))


# ------------------------------------------------------------------------------------------------- block norms
def plain_norm(v, kind, weight, bias, eps):
    """(value, magnitude of what fp32 adds to get it): the deviations carry the error of the mean, a few U of the
    largest magnitude in the row."""
    size = v.abs()
    if kind == "layer":
        size = size + v.abs().mean(-1, keepdim=True)
        v = v - v.mean(-1, keepdim=True)
    r = (v.square().mean(-1, keepdim=True) + eps).rsqrt()
    v, size = v * r, size * r
    if weight is not None:
        v, size = v * weight.double(), size * weight.double().abs()
    if bias is not None:
        v, size = v + bias.double(), size + bias.double().abs()
    return v, size


def plain_block_norm(x, branch, kw):
    rows = x.shape[0]
    spread = lambda t: t.double().reshape(-1, x.shape[1]).repeat_interleave(rows // t.reshape(-1, x.shape[1]).shape[0], dim=0)
    h = x.double()
    size = h.abs()
    eps = kw.get("eps", 1e-6)
    if branch is not None:
        b, b_size = branch.double(), branch.double().abs()
        if kw.get("post_norm"):
            b, b_size = plain_norm(b, kw["post_norm"], kw.get("post_weight"), kw.get("post_bias"), eps)
        if kw.get("gate") is not None:
            b, b_size = b * spread(kw["gate"]), b_size * spread(kw["gate"]).abs()
        scale = kw.get("residual_scale", 1.0)
        h, size = scale * h + b, abs(scale) * size + b_size
    if kw.get("norm", "rms") is None:
        return h, size, None, None
    z, _ = plain_norm(h, kw.get("norm", "rms"), kw.get("weight"), kw.get("bias"), eps)
    # errors of h pass through the norm like h itself; the mean's error reaches every element
    mean = size.mean(-1, keepdim=True)
    centred = h - h.mean(-1, keepdim=True) if kw.get("norm", "rms") == "layer" else h
    z_size = (size + mean) * (centred.square().mean(-1, keepdim=True) + eps).rsqrt()
    if kw.get("weight") is not None:
        z_size = z_size * kw["weight"].double().abs()
    z_size = z_size + z.abs()
    if kw.get("bias") is not None:
        z_size = z_size + kw["bias"].double().abs()
    if kw.get("mod_scale") is not None:
        z, z_size = z * (1 + spread(kw["mod_scale"])), z_size * (1 + spread(kw["mod_scale"]).abs())
    if kw.get("mod_shift") is not None:
        z, z_size = z + spread(kw["mod_shift"]), z_size + spread(kw["mod_shift"]).abs()
    return h, size, z, z_size


# fp32 steps of a row's statistics: a thread adds up to 32 values, then 5 shuffles and up to 16 warps, then rsqrt (2), the
# multiplications and additions around it (8): below 64 steps of U; two norms in a row: twice that
NORM_STEPS = 128


def check_block_norm(native, x, branch=None, **kw):
    got_h, got_z = native.block_norm(x, branch, **kw)
    flat = lambda t: t.reshape(-1, x.shape[-1])
    want_h, h_size, want_z, z_size = plain_block_norm(flat(x), None if branch is None else flat(branch), kw)
    if branch is None:
        assert got_h is x
    else:
        within(flat(got_h), want_h, NORM_STEPS * U * h_size, x.dtype)
    if want_z is None:
        assert got_z is None
    elif not kw.get("quantize"):
        assert got_z.dtype == x.dtype and got_z.shape == x.shape
        within(flat(got_z), want_z, NORM_STEPS * U * z_size, x.dtype)
    else:
        codes, scales = got_z
        width = x.shape[-1]
        slack = NORM_STEPS * U * z_size
        run = lambda t: torch.nn.functional.pad(t, (0, -width % 128)).view(t.shape[0], -1, 128)
        amax = run(want_z.abs()).amax(-1)
        assert ((scales.double() - amax / 448).abs() <= run(slack).amax(-1) / 448 + 2 * U * amax / 448 + 1.001e-8).all()
        s = scales.double().repeat_interleave(128, dim=1)[:, :width]
        err = (flat(codes).double() * s - want_z).abs()
        # half a step of e4m3 (2^-4 of the value, half of 2^-9 scales near zero), the product with 1 / scale (3 U)
        assert (err <= 2.0 ** -4 * (want_z.abs() + slack) * (1 + 8 * U) + s * 2.0 ** -10 + slack).all()
    return got_h, got_z


WIDTHS = [8, 16, 64, 136, 256, 264, 512, 520, 1024, 1032, 2048, 2056, 3080, 4096, 4104, 6144, 8192, 8200, 12288, 14336, 16384]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_block_norm_widths(native, width, dtype):
    x = randn(13, width, dtype=dtype, scale=2.0)
    branch = randn(13, width, seed=1, dtype=dtype)
    gate, scale, shift = (randn(1, width, seed=s, dtype=torch.float32, scale=0.3) for s in (2, 3, 4))
    check_block_norm(native, x, norm="rms")
    check_block_norm(native, x, norm="layer", mod_scale=scale, mod_shift=shift)
    check_block_norm(native, x, branch, post_norm="layer", gate=gate, norm="rms", residual_scale=0.7)
    if width % 16 == 0:
        check_block_norm(native, x, branch, gate=gate, norm="layer", mod_scale=scale, mod_shift=shift, quantize=True)


COMBINATIONS = list(itertools.product([None, "rms", "layer"], [None, "rms", "layer"], [False, True]))


@gpu
@pytest.mark.parametrize("post,norm,params", COMBINATIONS)
def test_block_norm_combinations(native, post, norm, params):
    dtype, rows, width = torch.bfloat16, 24, 640
    x, branch = randn(rows, width, dtype=dtype), randn(rows, width, seed=1, dtype=dtype)
    kw = {"post_norm": post, "norm": norm}
    if params:
        table = randn(6, 3, width, seed=2, dtype=dtype, scale=0.3)
        kw.update(gate=table[:, 2], residual_scale=-1.5, eps=1e-3)
        if post:
            kw.update(post_weight=randn(width, seed=3), post_bias=randn(width, seed=4, dtype=dtype))
        if norm:
            kw.update(weight=randn(width, seed=5, dtype=dtype), bias=randn(width, seed=6), mod_scale=table[:, 1],
                      mod_shift=randn(24, width, seed=7))
    check_block_norm(native, x.view(4, 6, width), branch.view(4, 6, width), **kw)
    if norm:
        check_block_norm(native, x, branch, quantize=True, **kw)


@gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 147, 1001])
@pytest.mark.parametrize("groups", ["one", "each", "some"])
def test_block_norm_groups_of_rows(native, rows, groups):
    count = {"one": 1, "each": rows, "some": next(g for g in (7, 11, 2, 3, 5, 1) if rows % g == 0)}[groups]
    x = randn(rows, 520, dtype=torch.float16)
    branch = randn(rows, 520, seed=1, dtype=torch.float16)
    table = randn(count, 6, 520, seed=2, dtype=torch.float16, scale=0.5)
    check_block_norm(native, x, branch, gate=table[:, 5], mod_scale=table[:, 1], mod_shift=table[:, 0], norm="layer")


@gpu
@pytest.mark.parametrize("width", [8208, 12288, 13504, 16384])
@pytest.mark.parametrize("rows", [295, 296])
def test_block_norm_wide_rows(native, rows, width):
    """Rows beyond 8192 elements, with and without a block for each SM's second place."""
    x, branch = randn(rows, width, dtype=torch.bfloat16), randn(rows, width, seed=1, dtype=torch.bfloat16)
    table = randn(rows, width, seed=2, scale=0.3)
    check_block_norm(native, x, branch, post_norm="layer", gate=table[:1], norm="layer", mod_scale=table, mod_shift=table[1:2])
    check_block_norm(native, x, norm="rms", mod_scale=table, quantize=True)


@gpu
def test_block_norm_hard_rows(native):
    """A large mean, constant rows, zeros, the smallest and the largest values, non-finite values in single rows."""
    x = randn(12, 1024, scale=0.01)
    x[0] += 1000.0
    x[1] = 3.0
    x[2] = 0.0
    x[3] *= 1e-30
    x[4] *= 1e30
    x = x.bfloat16()
    check_block_norm(native, x, norm="layer")
    check_block_norm(native, x[:4].contiguous(), norm="rms")
    x[5, 7], x[6, 9] = float("nan"), float("inf")
    _, z = native.block_norm(x, norm="layer")
    bad = torch.tensor([5, 6], device="cuda")
    assert z[bad].isnan().all() and not z[[0, 1, 2, 3, 7, 8, 9, 10, 11]].isnan().any()
    _, (codes, scales) = native.block_norm(x, norm="rms", quantize=True)
    assert scales[5].isnan().all() and codes.float()[5].isnan().all()
    _, z = native.block_norm(x, norm="rms")
    assert z[6, 9].isnan() and (z[6, :9] == 0).all()  # inf / inf, and finite / inf


@gpu
def test_block_norm_in_place_views_graph(native):
    x, branch = randn(40, 1024, dtype=torch.bfloat16), randn(40, 1024, seed=1, dtype=torch.bfloat16)
    gate = randn(1024, seed=2)
    want_h, want_z = native.block_norm(x, branch, gate=gate)
    for target in ("x", "branch"):
        tensors = {"x": x.clone(), "branch": branch.clone()}
        h, z = native.block_norm(tensors["x"], tensors["branch"], gate=gate, out=tensors[target])
        assert h is tensors[target] and torch.equal(h, want_h) and torch.equal(z, want_z)
    odd = torch.zeros(40 * 1024 + 1, device="cuda", dtype=torch.bfloat16)
    odd[1:] = x.flatten()
    h, z = native.block_norm(odd[1:].view(40, 1024), branch, gate=gate)
    assert torch.equal(h, want_h) and torch.equal(z, want_z)
    h, z = native.block_norm(x.t().contiguous().t(), branch, gate=gate)
    assert torch.equal(h, want_h) and torch.equal(z, want_z)
    odd_table = randn(40, 3 * 1024 + 2, seed=3)[:, 1:1025]  # parameter rows off the vector grid
    check_block_norm(native, x, branch, gate=odd_table)
    empty_h, empty_z = native.block_norm(x[:0], branch[:0], gate=gate)
    assert empty_h.shape == empty_z.shape == (0, 1024)
    graph = torch.cuda.CUDAGraph()
    static = x.clone()
    with torch.cuda.graph(graph):
        gh, (codes, scales) = native.block_norm(static, branch, gate=gate, quantize=True)
    fresh = randn(40, 1024, seed=9, dtype=torch.bfloat16)
    static.copy_(fresh)
    graph.replay()
    eh, (ec, es) = native.block_norm(fresh, branch, gate=gate, quantize=True)
    assert torch.equal(gh, eh) and torch.equal(codes.view(torch.uint8), ec.view(torch.uint8)) and torch.equal(scales, es)


# ------------------------------------------------------------------------------------------------------ rotary
def plain_rotary(x, positions, inv_freq, sections, layout, norm, weight, eps=1e-6):
    v = x.double()
    if norm:
        axes = (-1,) if norm == "head" else (-2, -1)
        v = v * (v.square().mean(axes, keepdim=True) + eps).rsqrt()
        if weight is not None:
            v = v * weight.double().reshape(x.shape[2:] if norm == "token" else x.shape[3:])
    phase, first = [], 0
    for a, n in enumerate(sections):
        phase.append(positions[..., a].double()[..., None] * inv_freq[first:first + n])
        first += n
    phase = torch.cat(phase, -1)
    phase = (phase if phase.ndim == 3 else phase[None])[:, :, None]
    c, s = phase.cos(), phase.sin()
    pairs = sum(sections)
    out, size = v.clone(), v.abs()
    first, second = ((slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if layout == "interleaved"
                     else (slice(0, pairs), slice(pairs, 2 * pairs)))
    a, b = v[..., first], v[..., second]
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    size[..., first] = size[..., second] = a.abs() + b.abs()
    return out, size


# one norm (below 64 steps), the angle (a turn's fraction rounded once: pi U), sincospi (4), two products and a sum
ROTARY_STEPS = 80


def check_rotary(native, rope, q, k, positions, sections, *, layout="interleaved", norm=None, weights=(None, None), out=None,
                 per_axis=True):
    inv_freq = rope.rotary_frequencies(sections, per_axis=per_axis, device="cuda")
    want = [None if t is None else plain_rotary(t, positions, inv_freq, sections, layout, norm, w)
            for t, w in zip((q, k), weights)]
    got = native.rotary(q, k, positions, inv_freq, sections=sections, layout=layout, norm=norm, q_weight=weights[0],
                        k_weight=weights[1], out=out)
    for g, w in zip(got, want):
        if w is None:
            assert g is None
        else:
            within(g, w[0], ROTARY_STEPS * U * w[1], q.dtype)
    return got


ROTARY_HEADS = [(1, 1, 8), (1, 1, 16), (3, 1, 40), (2, 2, 64), (10, 5, 72), (5, 1, 80), (12, 4, 96), (7, 7, 112), (24, 24, 128),
                (8, 1, 128), (17, 3, 136), (6, 2, 192), (4, 4, 256), (60, 20, 128), (28, 4, 256)]


@gpu
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("heads,kv_heads,dim", ROTARY_HEADS)
def test_rotary_head_shapes(native, rope, heads, kv_heads, dim, layout):
    for i, (norm, dtype) in enumerate(itertools.product([None, "head", "token"], DTYPES)):
        tokens = (1, 37, 64)[i % 3]
        qkv = randn(2, tokens, heads + 2 * kv_heads, dim, seed=i, dtype=dtype)
        q, k = qkv[:, :, :heads], qkv[:, :, heads:heads + kv_heads]
        positions = torch.randint(0, 900, (2, tokens, 3), device="cuda", dtype=(torch.int32, torch.int64)[i % 2])
        weights = (None, None)
        if norm:
            width = (lambda n: dim) if norm == "head" else (lambda n: n * dim)
            weights = (1 + 0.2 * randn(width(heads), seed=7, dtype=dtype), 1 + 0.2 * randn(width(kv_heads), seed=8))
            weights = (weights[0].to(dtype), weights[1])
        sections = rope.even_sections(dim)
        check_rotary(native, rope, q, k, positions, sections, layout=layout, norm=norm, weights=weights)
        partial = (dim // 8, 0, max(dim // 16, 1) if dim > 8 else 1)  # part of the head rotates, an axis without pairs
        check_rotary(native, rope, q, k, positions[0], partial, layout=layout, norm=norm, weights=weights, per_axis=False)


@gpu
def test_rotary_far_negative_and_fractional_positions(native, rope):
    q, k = randn(1, 50, 4, 128, dtype=torch.float16), randn(1, 50, 2, 128, seed=1, dtype=torch.float16)
    for positions in (torch.arange(50, device="cuda", dtype=torch.int64)[:, None] * 99991 + 2 ** 31,
                      -torch.arange(50, device="cuda", dtype=torch.int32)[:, None] * 1000003,
                      torch.linspace(-3, 1000.5, 50, device="cuda")[:, None]):
        check_rotary(native, rope, q, k, positions, (64,))
    # turning back gives the input: two roundings of the rotated pair
    positions = torch.arange(50, device="cuda", dtype=torch.int32)[:, None] * 17
    inv_freq = rope.rotary_frequencies((64,), device="cuda")
    there, _ = native.rotary(q, None, positions, inv_freq, sections=(64,))
    back, _ = native.rotary(there, None, -positions, inv_freq, sections=(64,))
    pair = q.double().unflatten(-1, (64, 2)).norm(dim=-1).repeat_interleave(2, dim=-1)
    assert ((back.double() - q.double()).abs() <= 2 * half_step(torch.float16) * 2 * pair + 1e-6).all()


@gpu
def test_rotary_grid_of_a_clip(native, rope):
    positions = rope.grid_positions(3, 4, 5, start=(2, 0, 0), device="cuda")
    assert positions.shape == (60, 3) and positions[0].tolist() == [2, 0, 0] and positions[-1].tolist() == [4, 3, 4]
    q, k = randn(2, 60, 3, 128, dtype=torch.bfloat16), randn(2, 60, 3, 128, seed=1, dtype=torch.bfloat16)
    got = check_rotary(native, rope, q, k, positions, (22, 21, 21), norm="head")
    inv_freq = rope.rotary_frequencies((22, 21, 21), device="cuda")
    plain = rope.rotary_reference(q, positions, inv_freq, sections=(22, 21, 21), norm="head")
    within(got[0], plain, half_step(torch.bfloat16) * plain.double().abs() + 1e-5, torch.bfloat16)


@gpu
def test_rotary_outputs_in_place_and_strided(native, rope):
    for layout, norm, dim in (("interleaved", "token", 128), ("half", None, 72), ("half", "head", 128)):
        qkv = randn(2, 21, 12, dim, dtype=torch.bfloat16)
        q, k = qkv[:, :, :8], qkv[:, :, 8:10]
        v = qkv[:, :, 10:].clone()
        positions = rope.grid_positions(21, device="cuda") + 5
        sections = (dim // 2,)
        want = check_rotary(native, rope, q, k, positions, sections, layout=layout, norm=norm)
        inv_freq = rope.rotary_frequencies(sections, device="cuda")
        # [batch, heads, tokens, dim] storage, and k into the middle of a longer cache whose other rows stay
        q_to = torch.empty(2, 8, 21, dim, device="cuda", dtype=torch.bfloat16).transpose(1, 2)
        cache = torch.full((2, 64, 2, dim), 3.0, device="cuda", dtype=torch.bfloat16)
        got = native.rotary(q, k, positions, inv_freq, sections=sections, layout=layout, norm=norm, out=(q_to, cache[:, 30:51]))
        assert got[0] is q_to and torch.equal(q_to, want[0]) and torch.equal(cache[:, 30:51], want[1])
        assert (cache[:, :30] == 3).all() and (cache[:, 51:] == 3).all()
        native.rotary(q, k, positions, inv_freq, sections=sections, layout=layout, norm=norm, out=(q, k))
        assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, :, 10:], v)


@gpu
def test_rotary_inputs_off_the_vector_grid_empty_and_broadcast(native, rope):
    positions = rope.grid_positions(9, device="cuda")
    base = randn(1, 9, 4, 67, dtype=torch.bfloat16)
    check_rotary(native, rope, base[..., 1:65], None, positions, (32,))
    shared = randn(1, 1, 4, 64, dtype=torch.bfloat16).expand(3, 9, 4, 64)
    check_rotary(native, rope, shared, shared, positions, (32,), layout="half")
    inv_freq = rope.rotary_frequencies((32,), device="cuda")
    q, k = native.rotary(base[:, :0, :, :64].contiguous(), None, positions[:0], inv_freq, sections=(32,))
    assert q.shape == (1, 0, 4, 64) and k is None
    wide = torch.zeros(9, 5, device="cuda", dtype=torch.int64)
    wide[:, 1:2] = positions.long()
    q = randn(1, 9, 4, 64, dtype=torch.bfloat16)
    check_rotary(native, rope, q, None, wide[:, 1:2], (32,))


# ------------------------------------------------------------------------------------------------ together
@gpu
def test_block_operators_in_a_row(native, quant, rope):
    """Norm with codes -> qkv product -> q/k norm and rotation -> attention -> output product -> gate, residual and next
    norm, captured as one graph, against the same chain in plain torch on the kernels' own intermediate roundings."""
    tokens, heads, dim = 60, 8, 64
    width = heads * dim
    x = randn(1, tokens, width, dtype=torch.bfloat16)
    qkv_w, qkv_s = quant.quantize_weight_block(randn(3 * width, width, seed=1, scale=0.05))
    o_w, o_s = quant.quantize_weight_block(randn(width, width, seed=2, scale=0.05))
    table = randn(1, 6, width, seed=3, dtype=torch.bfloat16, scale=0.2)
    positions = rope.grid_positions(3, 4, 5, device="cuda")
    sections = rope.even_sections(dim)
    inv_freq = rope.rotary_frequencies(sections, device="cuda")

    def chain(t):
        _, (codes, scales) = native.block_norm(t, norm="rms", mod_scale=table[:, 1], mod_shift=table[:, 0], quantize=True)
        qkv = native.fp8_gemm(codes, scales, qkv_w, qkv_s, out_dtype=torch.bfloat16).view(1, tokens, 3 * heads, dim)
        q, k = native.rotary(qkv[:, :, :heads], qkv[:, :, heads:2 * heads], positions, inv_freq, sections=sections, norm="head")
        v = qkv[:, :, 2 * heads:]
        a = torch.nn.functional.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2))
        y = native.fp8_linear(a.transpose(1, 2).reshape(1, tokens, width), o_w, o_s)
        return native.block_norm(t, y, gate=table[:, 2], norm="rms", mod_scale=table[:, 4], mod_shift=table[:, 3])

    with torch.no_grad():
        h, z = chain(x)
        static = torch.zeros_like(x)
        chain(static)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            gh, gz = chain(static)
        static.copy_(x)
        graph.replay()
        assert torch.equal(gh, h) and torch.equal(gz, z)
        # the plain chain
        f = x.float().view(tokens, width)
        n = f * (f.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * (1 + table[:, 1].float()) + table[:, 0].float()
        qkv = (quant.fake_quant_token_runs(n) @ quant.dequantize_weight_block(qkv_w, qkv_s).t()).bfloat16()
        qkv = qkv.view(1, tokens, 3 * heads, dim)
        q, k = (rope.rotary_reference(t, positions, inv_freq, sections=sections, norm="head")
                for t in (qkv[:, :, :heads], qkv[:, :, heads:2 * heads]))
        att = torch.softmax(q.float().transpose(1, 2) @ k.float().transpose(1, 2).transpose(2, 3) * dim ** -0.5, -1)
        a = (att @ qkv[:, :, 2 * heads:].float().transpose(1, 2)).transpose(1, 2).reshape(tokens, width).bfloat16()
        y = (quant.fake_quant_token_runs(a) @ quant.dequantize_weight_block(o_w, o_s).t()).bfloat16().float()
        want_h = f + table[:, 2].float() * y
        want_z = want_h * (want_h.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * (1 + table[:, 4].float()) + table[:, 3].float()
    # codes flip where a bf16 rounding moved a value across a step of e4m3 (2^-4 of it): seldom, and averaged over the K of
    # a product; what is left is a few roundings of bf16
    rel = lambda g, w: float((g.float().view(tokens, width) - w).norm() / w.norm())
    assert rel(h, want_h) < 4 * half_step(torch.bfloat16) and rel(z, want_z) < 4 * half_step(torch.bfloat16)


@pytest.fixture(scope="module")
def dit(pkg):
    return importlib.import_module(P + "dit")


def small_dit(dit, **kw):
    return dit.DiTConfig(**{**dict(blocks=2, hidden=512, heads=4, ffn=1024, latent_tokens=168, action_tokens=32, grid=(3, 7, 8),
                                   linear="fp8", modulated=True, rotary=True), **kw})


@gpu
@pytest.mark.parametrize("kw", [{}, {"linear": "int4"}, {"modulated": False}, {"rotary": False}, {"heads": 8, "latent_tokens": 7, "grid": (1, 1, 7)}])
def test_extended_dit_blocks_against_plain_torch(native, dit, kw):
    """The stack's blocks with e4m3 linears, modulation and positions, on both backends, and as one graph."""
    cfg = small_dit(dit, **kw)
    model = dit.SyntheticDiT(cfg, device="cuda", backend="native")
    x = randn(1, cfg.tokens, cfg.hidden, dtype=torch.bfloat16)
    with torch.no_grad():
        parity = dit.extended_parity(model, x)
        # On the reference's own input of a block both backends round the same four or five bf16 tensors and the same codes; a
        # value that lands on the other side of a rounding moves by one step, and what codes flip by it is averaged over K.
        # The bar of a linear on its own is 1e-2 (test_gpu_modules); a branch chains four of them.
        assert parity["block_stream_max"] < 1e-2 and parity["block_branch_max"] < 4e-2, parity
        eager = model(x)
        graph = torch.cuda.CUDAGraph()
        static = torch.zeros_like(x)
        model(static)
        with torch.cuda.graph(graph):
            out = model(static)
        static.copy_(x)
        graph.replay()
        assert torch.equal(out, eager)


CAPTURE_FIRST = '''
import importlib, sys
import torch
sys.path.insert(0, {root!r})
import __graft_entry__ as entry
entry.load_package()
native = importlib.import_module("fastwamjoint_quantization_b200.native")
x = torch.randn(64, 512, device="cuda").bfloat16()
w = torch.randn(256, 512, device="cuda").to(torch.float8_e4m3fn)
ws = torch.ones(2, 4, device="cuda")
q = torch.randn(1, 64, 4, 128, device="cuda").bfloat16()
pos = torch.arange(64, device="cuda", dtype=torch.int32)[:, None]
f = torch.ones(64, device="cuda", dtype=torch.float64)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = native.fp8_linear(x, w, ws)
    big = native.fp8_linear(x.repeat(32, 1), w, ws)
    h, z = native.block_norm(x, x)
    r, _ = native.rotary(q, None, pos, f, sections=(64,))
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, native.fp8_linear(x, w, ws)) and torch.equal(big[:64], big[64:128])
assert torch.equal(z, native.block_norm(x, x)[1]) and torch.equal(r, native.rotary(q, None, pos, f, sections=(64,))[0])
assert native.device_status() == 0
print("captured first")
'''


@gpu
def test_first_call_of_a_process_under_capture():
    """Nothing a first call does (attributes, occupancy, symbol and driver lookups) is refused while a stream is captured."""
    import subprocess
    import sys
    from pathlib import Path
    root = str(Path(__file__).resolve().parents[1])
    done = subprocess.run([sys.executable, "-c", CAPTURE_FIRST.format(root=root)], capture_output=True, text=True, timeout=180)
    assert done.returncode == 0 and "captured first" in done.stdout, done.stderr[-2000:]


@gpu
def test_out_may_be_an_input_but_not_part_of_one(native):
    buffer = randn(9, 64, seed=3, dtype=torch.bfloat16)
    x, branch = buffer[:8], randn(8, 64, seed=4, dtype=torch.bfloat16)
    want, _ = native.block_norm(x, branch)
    for bad in (dict(out=buffer[1:]), dict(out=branch, gate=branch), dict(out=x, mod_scale=x[:1]), dict(out=x, weight=x[7])):
        with pytest.raises(ValueError, match="share no memory"):
            native.block_norm(x, branch, **bad)
    kept = buffer.clone()
    h, _ = native.block_norm(x, branch, out=branch)
    assert h is branch and torch.equal(h, want) and torch.equal(buffer, kept)


@gpu
@pytest.mark.parametrize("offset", [1, 4, 8])
def test_parameters_of_any_alignment(native, offset):
    """Parameters whose address is off the kernels' vectors of 16 or 32 bytes give what aligned ones do."""
    x, branch = (randn(6, 136, seed=i, dtype=torch.bfloat16) for i in (1, 2))
    def off(t):
        flat = torch.zeros(t.numel() + offset, device="cuda", dtype=t.dtype)
        flat[offset:] = t.flatten()
        return flat[offset:].view(t.shape)
    for dtype in (torch.float32, torch.bfloat16):
        table, w = randn(3, 136, seed=3, dtype=dtype), randn(136, seed=4, dtype=dtype)
        want = native.block_norm(x, branch, gate=table, post_norm="rms", post_weight=w, weight=w, mod_shift=table)
        got = native.block_norm(x, branch, gate=off(table), post_norm="rms", post_weight=off(w), weight=off(w), mod_shift=off(table))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        q, w = randn(1, 6, 2, 64, seed=5, dtype=torch.bfloat16), randn(128, seed=6, dtype=dtype)
        turn = lambda w: native.rotary(q, None, torch.arange(6, device="cuda", dtype=torch.int32)[:, None], torch.ones(32, device="cuda", dtype=torch.float64),
                                       sections=(32,), norm="token", q_weight=w)[0]
        assert torch.equal(turn(off(w)), turn(w))


@gpu
def test_binding_and_python_way_give_the_same(native, quant, rope):
    """The ordinary calls that the binding takes, against the Python way on the same inputs; that it takes them, and leaves
    what is not ordinary."""
    module = native._lib.load_binding()
    assert module is not None, "sq_binding.so is not built"
    x, codes, scales, weight, weight_scales, bias = fp8_case(quant, 48, 264, 512, torch.bfloat16)
    branch = randn(48, 512, seed=9, dtype=torch.bfloat16)
    table = randn(4, 3, 512, seed=10, dtype=torch.bfloat16)
    w32 = randn(512, seed=11)
    qkv = randn(2, 24, 12, 64, seed=12, dtype=torch.bfloat16)
    positions = rope.grid_positions(2, 3, 4, device="cuda")
    freq = rope.rotary_frequencies((12, 10, 10), device="cuda")
    calls = [
        lambda: native.fp8_gemm(codes, scales, weight, weight_scales, bias, out_dtype=torch.bfloat16),
        lambda: native.fp8_gemm(codes.view(2, 24, 512), scales.contiguous(), weight, weight_scales, out_dtype=torch.float16),
        lambda: native.fp8_linear(x, weight, weight_scales, bias, input_activation="gelu"),
        lambda: native.block_norm(x.view(4, 12, 512), norm="layer", mod_scale=table[:, 1], mod_shift=table[:, 0], quantize=True),
        lambda: native.block_norm(x, branch, gate=w32, norm=None, post_norm="rms", post_weight=w32, post_bias=table[0, 0]),
        lambda: native.block_norm(x, branch, gate=table[:, 2:3], residual_scale=0.5, weight=w32, bias=w32, eps=1e-3),
        lambda: native.rotary(qkv[:, :, :6], qkv[:, :, 6:8], positions, freq, sections=(12, 10, 10), layout="half", norm="head", q_weight=w32[:64]),
        lambda: native.rotary(qkv, None, positions.long()[None], freq, sections=(12, 10, 10)),
    ]
    flat = lambda t: [] if t is None else [t] if isinstance(t, torch.Tensor) else [u for v in t for u in flat(v)]
    for call in calls:
        fast = flat(call())
        native._binding.enabled = False
        try:
            slow = flat(call())
        finally:
            native._binding.enabled = True
        assert len(fast) == len(slow)
        for a, b in zip(fast, slow):
            assert a.shape == b.shape and a.dtype == b.dtype and a.stride() == b.stride()
            assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
    assert module.fp8_linear(x, weight, weight_scales, bias, None) is not None
    for odd in (x.t().contiguous().t(), x.cpu(), x.float(), x[:0], x.clone().requires_grad_(), x[:, :508], "x"):
        assert module.fp8_linear(odd, weight, weight_scales, bias, None) is None
    assert module.fp8_linear(x, weight, weight_scales) is None  # another number of arguments
    assert module.fp8_linear(x, weight, weight_scales, bias, "relu") is None
    assert module.rotary(qkv, None, positions, freq, [12, 10, 10], "interleaved", None, None, None, 1e-6) is None  # sections: a tuple
    assert module.rotary(qkv, None, positions, freq, (33,), "interleaved", None, None, None, 1e-6) is None
    assert native.rotary(qkv, None, positions, freq, sections=[12, 10, 10])[1] is None


@gpu
def test_offsets_past_32_bits(native, quant, rope):
    """The last rows of tensors of more than 2^31 elements, against the same rows alone."""
    rows, last = 530000, 200
    x = torch.empty(rows, 4096, device="cuda", dtype=torch.bfloat16).normal_()
    end = x[-last:].clone()
    h, (codes, scales) = native.block_norm(x, x, norm="rms", quantize=True)
    want_h, (want_codes, want_scales) = native.block_norm(end, end, norm="rms", quantize=True)
    assert torch.equal(h[-last:], want_h) and torch.equal(scales[-last:], want_scales)
    assert torch.equal(codes[-last:].view(torch.uint8), want_codes.view(torch.uint8))
    del h, codes, scales
    positions = torch.arange(rows, device="cuda")[:, None]
    turn = lambda t, p: native.rotary(t, None, p, rope.rotary_frequencies((64,), device="cuda"), sections=(64,), norm="head")[0]
    assert torch.equal(turn(x.view(1, rows, 32, 128), positions)[:, -last:], turn(end.view(1, last, 32, 128), positions[-last:]))
    weight, weight_scales = quant.quantize_weight_block(randn(4096, 128, scale=0.1))
    narrow = x[:, :128].contiguous()
    y = native.fp8_linear(narrow, weight, weight_scales)[-last:].double()
    want = native.fp8_linear(narrow[-last:].clone(), weight, weight_scales).double()
    # other tiles, other order of a run's 128 products: 128 U of their magnitudes on either side, and a rounding each
    size = (narrow[-last:].float().abs() * 1.07) @ quant.dequantize_weight_block(weight, weight_scales).float().abs().t()
    assert ((y - want).abs() <= 2 * 128 * U * size.double() + 2.0 ** -7 * want.abs()).all()


@gpu
def test_two_streams_at_once(native, quant):
    """Calls on two streams, unordered: each has its own outputs and workspaces."""
    x, _, _, weight, weight_scales, bias = fp8_case(quant, 512, 1024, 1024, torch.bfloat16)
    want = native.fp8_linear(x, weight, weight_scales, bias)
    want_h, want_z = native.block_norm(x, x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            got.append((native.fp8_linear(x, weight, weight_scales, bias), *native.block_norm(x, x)))
    torch.cuda.synchronize()
    for y, h, z in got:
        assert torch.equal(y, want) and torch.equal(h, want_h) and torch.equal(z, want_z)


# ---------------------------------------------------------------------------------------------------- refusals
def test_c_abi_refuses_before_any_launch(pkg):
    """Host-side checks of the C entry points: no GPU needed, the pointers are never read."""
    lib_mod = importlib.import_module(P + "_lib")
    lib = lib_mod.load_library()
    ok, off = 4096, 4096 + 4
    gemm = lambda codes=ok, scales=ok, w=ok, ws=ok, bias=None, out=ok, dt=0, m=4, n=16, k=128, rs=1: lib.sq_fp8_gemm(
        codes, scales, rs, 4, w, ws, bias, out, dt, m, n, k, None)
    for kw in ({"codes": None}, {"scales": None}, {"w": None}, {"ws": None}, {"out": None}):
        assert gemm(**kw) == lib_mod.ERR_NULL
    for kw in ({"codes": off}, {"w": off}, {"out": off}, {"scales": 4097}, {"ws": 4098}, {"bias": 4097}, {"m": -1}, {"n": 12}, {"n": 0},
               {"k": 0}, {"k": 24}, {"k": 131088}, {"rs": -1}):
        assert gemm(**kw) == lib_mod.ERR_SHAPE
    assert gemm(dt=2) == lib_mod.ERR_ENUM and gemm(m=0) == lib_mod.OK
    quantize = lambda x=ok, dt=0, rows=4, k=128, act=0, codes=ok, scales=ok: lib.sq_fp8_quantize(x, dt, rows, k, act, codes, scales, 1, 4, None)
    assert quantize(x=None) == lib_mod.ERR_NULL and quantize(scales=None) == lib_mod.ERR_NULL
    assert quantize(x=off) == lib_mod.ERR_SHAPE and quantize(k=120) == lib_mod.ERR_SHAPE and quantize(rows=-1) == lib_mod.ERR_SHAPE
    assert quantize(rows=1 << 40) == lib_mod.ERR_SHAPE
    assert quantize(dt=3) == lib_mod.ERR_ENUM and quantize(act=2) == lib_mod.ERR_ENUM and quantize(rows=0) == lib_mod.OK
    linear = lambda x=ok, n=16, ws=ok, nbytes=1 << 20, rows=4, out=ok: lib.sq_fp8_linear(x, 0, rows, 128, n, 0, ok, ok, None, out, ws, nbytes, None)
    assert lib.sq_fp8_workspace_bytes(3, 272) == 1024 + 256 and lib.sq_fp8_workspace_bytes(-1, 16) == 0
    assert linear(ws=None) == lib_mod.ERR_NULL and linear(nbytes=16) == lib_mod.ERR_WORKSPACE
    assert linear(n=12) == lib_mod.ERR_SHAPE and linear(ws=off) == lib_mod.ERR_SHAPE and linear(out=None) == lib_mod.ERR_NULL
    assert linear(rows=0) == lib_mod.OK

    def norm(**kw):
        base = {"x": ok, "branch": ok, "h_out": ok, "z_out": ok, "rows": 4, "width": 64, "residual_scale": 1.0, "eps": 1e-6,
                "norm_kind": lib_mod.NORM_RMS}
        return lib.sq_block_norm(lib_mod.ctypes.byref(lib_mod.BlockNorm(**{**base, **kw})), None)

    assert lib.sq_block_norm(None, None) == lib_mod.ERR_NULL
    for kw in ({"x": None}, {"h_out": None}, {"z_out": None}, {"branch": None, "norm_kind": 0}):
        assert norm(**kw) == lib_mod.ERR_NULL
    for kw in ({"dtype": 2}, {"norm_kind": 3}, {"post_kind": -1}, {"norm_kind": 0, "scales": ok}, {"post_weight": lib_mod.Param(ok)},
               {"branch": None, "gate": lib_mod.Param(ok, 0, 4)}, {"norm_kind": 0, "mod_scale": lib_mod.Param(ok, 0, 4)}):
        assert norm(**kw) == lib_mod.ERR_ENUM
    for kw in ({"x": off}, {"branch": off}, {"h_out": off}, {"z_out": off}, {"width": 60}, {"width": 16392}, {"rows": -1}, {"rows": 1 << 31},
               {"width": 72, "scales": ok}, {"scales": 4097}, {"gate": lib_mod.Param(off, 0, 4)}, {"gate": lib_mod.Param(ok, 0, 0)},
               {"gate": lib_mod.Param(ok, 4, 1)}, {"weight": lib_mod.Param(off)}, {"weight": lib_mod.Param(ok + 16, 0, 0, 1)}):
        assert norm(**kw) == lib_mod.ERR_SHAPE
    assert norm(rows=0) == lib_mod.OK

    def rotary(sections=(8, 8), **kw):
        strides = (lib_mod.c_int64 * 3)(512, 64, 32)
        base = {"q": ok, "k": ok, "q_out": ok, "k_out": ok, "positions": ok, "inv_freq": ok, "batch": 1, "length": 8, "heads": 2,
                "kv_heads": 2, "dim": 32, "axes": 2, "q_strides": strides, "k_strides": strides, "q_out_strides": strides,
                "k_out_strides": strides, "position_token_stride": 2}
        args = lib_mod.Rotary(**{**base, **kw})
        args.sections[:len(sections)] = sections
        return lib.sq_rotary(lib_mod.ctypes.byref(args), None)

    assert lib.sq_rotary(None, None) == lib_mod.ERR_NULL
    for kw in ({"q": None}, {"k": None}, {"q_out": None}, {"k_out": None}, {"positions": None}, {"inv_freq": None}):
        assert rotary(**kw) == lib_mod.ERR_NULL
    for kw in ({"dtype": 2}, {"layout": 2}, {"norm": 3}, {"position_type": 3}, {"q_weight": ok}):
        assert rotary(**kw) == lib_mod.ERR_ENUM
    for kw in ({"heads": 1023, "kv_heads": 2}, {"heads": 1 << 30}, {"heads": 2049, "kv_heads": 0, "dim": 16, "sections": (8,), "axes": 1}):
        assert rotary(**kw) == lib_mod.ERR_SHAPE
    odd = (lib_mod.c_int64 * 3)(512, 64, 36)
    for kw in ({"dim": 36}, {"dim": 264}, {"heads": 0}, {"axes": 0}, {"axes": 5}, {"q": off}, {"k_out": off}, {"q_strides": odd},
               {"k_out_strides": odd}, {"positions": 4097}, {"inv_freq": 4100}, {"sections": (8, 9)}, {"sections": (0, 0)},
               {"sections": (-1, 8)}, {"batch": -1}):
        assert rotary(**kw) == lib_mod.ERR_SHAPE
    assert rotary(length=0) == lib_mod.OK


def test_host_helpers(quant, rope):
    with pytest.raises(ValueError):
        quant.quantize_weight_block(torch.zeros(4))
    with pytest.raises(ValueError):
        rope.rotary_frequencies(())
    with pytest.raises(ValueError):
        rope.grid_positions()
    w = torch.randn(130, 272, generator=torch.Generator().manual_seed(0))
    codes, scales = quant.quantize_weight_block(w)
    assert codes.shape == w.shape and scales.shape == (2, 3)
    back = quant.dequantize_weight_block(codes, scales)
    s = scales.repeat_interleave(128, 0)[:130].repeat_interleave(128, 1)[:, :272]
    assert ((back - w).abs() <= w.abs() * 2.0 ** -4 * (1 + 8 * U) + s * 2.0 ** -10).all()
    values = torch.randn(5, 272, generator=torch.Generator().manual_seed(1))
    run_codes, run_scales = quant.quantize_token_runs(values)
    assert run_codes.shape == values.shape and run_scales.shape == (5, 3)
    assert torch.equal(quant.fake_quant_token_runs(values), run_codes.float() * run_scales.repeat_interleave(128, 1)[:, :272])
    freq = rope.rotary_frequencies((2, 0, 3))
    assert freq.dtype == torch.float64 and torch.allclose(freq, torch.tensor([1, 1e-2, 1, 10000 ** (-1 / 3), 10000 ** (-2 / 3)], dtype=torch.float64))
    assert torch.allclose(rope.rotary_frequencies((2, 2), per_axis=False), 10000.0 ** (-torch.arange(4, dtype=torch.float64) / 4))
    assert rope.even_sections(128) == (22, 21, 21) and rope.even_sections(64, 1) == (32,)
    # the plain form turns a pair by the angle: 64-bit complex products
    x = torch.randn(1, 6, 2, 8, generator=torch.Generator().manual_seed(2))
    positions, f = rope.grid_positions(2, 3), rope.rotary_frequencies((1, 2))
    got = rope.rotary_reference(x, positions, f, sections=(1, 2))
    want, _ = plain_rotary(x, positions, f, (1, 2), "interleaved", None, None)
    assert (got.double() - want).abs().max() <= 16 * U * x.abs().max()


def test_extended_dit_on_the_cpu(dit):
    """The plain-torch backend needs no GPU; what a configuration refuses."""
    cfg = small_dit(dit, hidden=64, heads=2, ffn=128, latent_tokens=12, action_tokens=4, grid=(2, 2, 3))
    model = dit.SyntheticDiT(cfg, device="cpu", backend="reference")
    x = torch.randn(1, 16, 64, generator=torch.Generator().manual_seed(0)).bfloat16()
    y = model(x)
    assert y.shape == x.shape and y.isfinite().all()
    assert (y.float().square().mean(-1) - 1).abs().max() < 0.02  # the final norm, rounded to bf16
    assert not torch.equal(model(x.flip(1)), y.flip(1))  # the positions count
    with pytest.raises(ValueError, match="grid"):
        small_dit(dit, grid=(3, 7, 7))
    with pytest.raises(ValueError, match="linear"):
        small_dit(dit, linear="int3")
    with pytest.raises(RuntimeError, match="step"):
        model.blocks[0](x)
    with pytest.raises(ValueError, match="extended_parity"):
        dit.stack_parity(model, x)
    assert dit.DiTConfig().plain


def test_operators_need_the_gpu(native):
    """No CPU fallback, as everywhere in this package."""
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    for call in (lambda: native.fp8_quantize(x), lambda: native.block_norm(x),
                 lambda: native.fp8_linear(x, x.to(torch.float8_e4m3fn), torch.ones(1, 1)),
                 lambda: native.rotary(x.view(1, 1, 4, 128), None, torch.zeros(1, 1), torch.ones(1), sections=(1,))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@gpu
def test_python_refusals(native, quant):
    x = randn(4, 128, dtype=torch.bfloat16)
    w, ws = quant.quantize_weight_block(randn(16, 128))
    codes, scales = native.fp8_quantize(x)
    good = dict(weight=w, weight_scales=ws)

    def refused(error, match, fn, *args, **kw):
        with pytest.raises(error, match=match):
            fn(*args, **kw)

    grad = x.clone().requires_grad_()
    refused(RuntimeError, "no backward", native.fp8_quantize, grad)
    refused(RuntimeError, "no backward", native.fp8_linear, grad, **good)
    refused(RuntimeError, "no backward", native.block_norm, x, grad)
    refused(RuntimeError, "no backward", native.block_norm, x, x, gate=torch.ones(128, device="cuda", requires_grad=True))
    with torch.no_grad():
        native.block_norm(grad)
    refused(ValueError, "multiple of 16", native.fp8_quantize, x[:, :120])
    refused(ValueError, "bf16 or fp16", native.fp8_quantize, x.float())
    refused(ValueError, "input_activation", native.fp8_quantize, x, input_activation="relu")
    refused(ValueError, "weight must be", native.fp8_linear, x, w.float(), ws)
    refused(ValueError, "shape", native.fp8_linear, x, w[:12], ws)
    refused(ValueError, "weight_scales", native.fp8_linear, x, w, ws[:, :0])
    refused(ValueError, "weight_scales", native.fp8_linear, x, w, ws.half())
    refused(ValueError, "device", native.fp8_linear, x, w, ws.cpu())
    refused(ValueError, "bias", native.fp8_linear, x, w, ws, x[0, :8])
    refused(ValueError, "bias", native.fp8_linear, x, w, ws, torch.zeros(16, device="cuda"))
    refused(ValueError, "out must", native.fp8_linear, x, w, ws, out=torch.empty(4, 15, device="cuda", dtype=torch.bfloat16))
    refused(RuntimeError, "workspace", native.fp8_linear, x, w, ws, workspace=torch.empty(16, device="cuda", dtype=torch.uint8))
    refused(ValueError, "scales must", native.fp8_gemm, codes, scales[:3], w, ws, out_dtype=torch.bfloat16)
    refused(ValueError, "codes must", native.fp8_gemm, x, scales, w, ws, out_dtype=torch.bfloat16)
    refused(ValueError, "out_dtype", native.fp8_gemm, codes, scales, w, ws, out_dtype=torch.float32)
    refused(ValueError, "norm", native.block_norm, x, norm="batch")
    refused(ValueError, "without a branch", native.block_norm, x, norm=None)
    refused(ValueError, "without a branch", native.block_norm, x, gate=x[0])
    refused(ValueError, "without a norm", native.block_norm, x, x, norm=None, quantize=True)
    refused(ValueError, "post_norm", native.block_norm, x, x, post_weight=x[0])
    refused(ValueError, "branch must", native.block_norm, x, x[:2])
    refused(ValueError, "branch must", native.block_norm, x, x.half())
    refused(ValueError, "rows must cover", native.block_norm, x, x, gate=randn(3, 128))
    refused(ValueError, "dtype or float32", native.block_norm, x, x, gate=x[0].half())
    refused(ValueError, r"must be \[128\]", native.block_norm, x, weight=x[:1])
    refused(ValueError, "multiple of 8", native.block_norm, x[:, :100])
    refused(ValueError, "multiple of 8", native.block_norm, x[:, :120], quantize=True)
    refused(ValueError, "out must", native.block_norm, x, x, out=x[:, :64])
    q = randn(1, 4, 2, 64, dtype=torch.bfloat16)
    pos = torch.zeros(4, 1, device="cuda", dtype=torch.int32)
    f = torch.ones(32, device="cuda", dtype=torch.float64)
    refused(RuntimeError, "no backward", native.rotary, q.clone().requires_grad_(), None, pos, f, sections=(32,))
    refused(ValueError, "batch, tokens", native.rotary, q[0], None, pos, f, sections=(32,))
    refused(ValueError, "sections", native.rotary, q, None, pos, f, sections=(33,))
    refused(ValueError, "sections", native.rotary, q, None, pos, f, sections=(8,) * 5)
    refused(ValueError, "inv_freq", native.rotary, q, None, pos, f.float(), sections=(32,))
    refused(ValueError, "inv_freq", native.rotary, q, None, pos, f[:31], sections=(32,))
    refused(ValueError, "positions", native.rotary, q, None, pos[:3], f, sections=(32,))
    refused(ValueError, "positions", native.rotary, q, None, pos.half(), f, sections=(32,))
    refused(ValueError, "device", native.rotary, q, None, pos.cpu(), f, sections=(32,))
    refused(ValueError, "layout", native.rotary, q, None, pos, f, sections=(32,), layout="neox")
    refused(ValueError, "belong to a norm", native.rotary, q, None, pos, f, sections=(32,), q_weight=q[0, 0, 0])
    refused(ValueError, "q_weight", native.rotary, q, None, pos, f, sections=(32,), norm="token", q_weight=q[0, 0, 0])
    refused(ValueError, "k must match", native.rotary, q, q[:, :3], pos, f, sections=(32,))
    refused(ValueError, "head shape", native.rotary, q[..., :60], None, pos, f[:30], sections=(30,))
    refused(ValueError, "head shape", native.rotary, q.expand(1, 4, 2, 64).repeat(1, 1, 600, 1), None, pos, f, sections=(32,))
    refused(ValueError, "out for q", native.rotary, q, None, pos, f, sections=(32,), out=(q[:, :1].expand(1, 4, 2, 64), None))
