"""The block operators where they can go wrong: the order in which the e4m3 product's warps hand memory to one another, calls
at the border of what the entry points take, and what they refuse.  Formulas, tolerances and helpers are test_block_ops'."""
import ctypes
import importlib
import random
import re
import subprocess
import threading
import time
from pathlib import Path

import pytest
import torch

from test_block_ops import DTYPES, P, check_block_norm, fp8_case, fp8_product, fp8_slack, gpu, half_step, no_device_timeouts, randn, within  # noqa: F401

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def native(pkg):
    return importlib.import_module(P + "native")


@pytest.fixture(scope="module")
def quant(pkg):
    return importlib.import_module(P + "quant")


# ------------------------------------------------------------------------- warps of the e4m3 product for many tokens
class Barrier:
    """An mbarrier: a phase ends when `count` arrivals are in; a wait names the parity of the phase it waits for."""

    def __init__(self, count):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1

    def passed(self, parity):
        return (self.phase & 1) != parity


def pair_kernel(stages, parts, runs, rng, free_by_readers):
    """One pair of thread blocks of ``sq_fp8_pair_kernel`` at the grain of its barriers, its warps stepped in random order:
    the first operand, accumulator or factor that a warp found in place of its own run's, every warp
    waiting, or None.  ``stages``: of the operand ring; ``parts``: products a
    run (1: 128 channels, 2: 256).  ``free_by_readers``: a place for factors is free when its readers say so; otherwise
    when the MMAs of a later run are done."""
    blocks, depth, drains = (0, 1), 4 // parts, 2
    full = [Barrier(2) for _ in range(stages)]
    acc_empty = [Barrier(2 * drains // parts) for _ in range(4)]
    empty = [[Barrier(parts) for _ in range(stages)] for _ in blocks]
    acc_full = [[Barrier(1) for _ in range(4)] for _ in blocks]
    ready = [[Barrier(1) for _ in range(2)] for _ in blocks]
    free = [[Barrier(drains) for _ in range(2)] for _ in blocks]
    slots = [[None] * 8 for _ in blocks]
    operands = [[None] * stages for _ in blocks]
    accumulators = [[None] * 4 for _ in blocks]
    wrong = []

    def producer(block):
        for run in range(runs):
            yield lambda: empty[block][run % stages].passed((run // stages & 1) ^ 1)
            operands[block][run % stages] = run
            yield lambda: True
            full[run % stages].arrive()

    def issuer(mine):
        for product in range(mine, runs * parts, 2):
            run, acc = product // parts, product % 4
            yield lambda: full[run % stages].passed(run // stages & 1)
            yield lambda: acc_empty[acc].passed((product // 4 & 1) ^ 1)
            for block in blocks:
                accumulators[block][acc] = None
            yield lambda: True  # the MMAs end some time after
            for block in blocks:
                if operands[block][run % stages] != run:
                    wrong.append(("operand", run, operands[block][run % stages]))
                accumulators[block][acc] = product
                acc_full[block][acc].arrive()
                empty[block][run % stages].arrive()

    def factors(block):
        for batch in range(-(-runs // 4)):
            if free_by_readers:
                if batch >= 2:
                    yield lambda: free[block][batch & 1].passed((batch >> 1 & 1) ^ 1)
            elif batch:
                run = 2 if batch == 1 else 4 * batch - 5 + depth
                yield lambda: empty[block][run % stages].passed(run // stages & 1)
            for run in range(4 * batch, 4 * batch + 4):
                slots[block][run & 7] = run
                yield lambda: True
            ready[block][batch & 1].arrive()

    def drain(block, share):
        for run in range(runs):
            acc = run % 4 if parts == 1 else run * 2 % 4 + share
            turn = run // 4 if parts == 1 else run // 2
            yield lambda: acc_full[block][acc].passed(turn & 1)
            if run % 4 == 0:
                yield lambda: ready[block][run >> 2 & 1].passed(run >> 3 & 1)
            if accumulators[block][acc] != (run if parts == 1 else 2 * run + share):
                wrong.append(("accumulator", run, accumulators[block][acc]))
            if slots[block][run & 7] != run:
                wrong.append(("factor", run, slots[block][run & 7]))
            acc_empty[acc].arrive()
            yield lambda: True
            if run % 4 == 3:
                free[block][run >> 2 & 1].arrive()

    warps = [producer(0), producer(1), issuer(0), issuer(1), factors(0), factors(1)]
    warps += [drain(block, share) for block in blocks for share in range(drains)]
    waiting = {warp: next(warp, None) for warp in warps}
    pace = {warp: rng.choice((1, 1, 1, 40)) for warp in warps}
    while any(wait is not None for wait in waiting.values()):
        able = [warp for warp, wait in waiting.items() if wait is not None and wait()]
        if not able:
            return "every warp waits"
        warp = rng.choices(able, [1 / pace[warp] for warp in able])[0]
        waiting[warp] = next(warp, None)
        if wrong:
            return wrong[0]
    return None


@pytest.mark.parametrize("stages,parts", [(7, 1), (5, 2)])
def test_factors_stay_until_they_are_read(stages, parts):
    rng = random.Random(stages)
    for runs in (1, 3, 4, 5, 8, 9, 12, 13, 16, 17, 29, 40, 41):
        for _ in range(40):
            assert pair_kernel(stages, parts, runs, rng, free_by_readers=True) is None


def test_done_products_do_not_free_factors():
    """With one product a run, "the MMAs of a later run are done" lets a batch overwrite factors not yet read: the two issuers
    are not ordered, and a barrier one round behind has the parity waited for.  The stepping above finds it."""
    rng = random.Random(0)
    assert any(pair_kernel(7, 1, 40, rng, free_by_readers=False) for _ in range(2000))


@gpu
@pytest.mark.parametrize("m,n,k", [(1001, 1480, 2000), (1024, 1408, 14336), (2048, 1024, 4096), (700, 1408, 8208)])
def test_fp8_gemm_of_128_channel_tiles_and_many_runs(native, quant, m, n, k):
    """Shapes of the pair kernel with 128 channels a tile and more runs than two batches of factors, back to back."""
    _, codes, scales, weight, weight_scales, bias = fp8_case(quant, m, n, k, torch.bfloat16)
    scales = scales * torch.exp2(randn(*scales.shape, seed=9).round())  # every run's factor is another
    want, size = fp8_product(codes, scales, weight, weight_scales, bias)
    outs = [native.fp8_gemm(codes, scales, weight, weight_scales, bias, out_dtype=torch.bfloat16) for _ in range(20)]
    within(outs[0], want, fp8_slack(size, k), torch.bfloat16)
    assert all(torch.equal(out, outs[0]) for out in outs[1:])


# ---------------------------------------------------------------------------------------------- inputs autograd tracks
def operator_calls(native, quant, rope):
    """(name, call, its tensors by name) of each operator on small inputs."""
    x, codes, scales, weight, weight_scales, bias = fp8_case(quant, 6, 64, 128, torch.bfloat16)
    linear = dict(weight=weight, weight_scales=weight_scales, bias=bias)
    vector, rows = randn(128, seed=5), randn(3, 128, seed=6, dtype=torch.bfloat16)
    norm = dict(x=x, branch=x + 1, gate=rows, post_weight=vector, post_bias=vector, weight=vector, bias=vector, mod_scale=rows, mod_shift=rows)
    q, k = (randn(1, 6, 2, 64, seed=s, dtype=torch.bfloat16) for s in (7, 8))
    head = randn(64, seed=9)
    turn = dict(q=q, k=k, positions=torch.arange(6.0, device="cuda")[:, None], inv_freq=rope.rotary_frequencies((32,), device="cuda"),
                q_weight=head, k_weight=head)
    return [("fp8_quantize", lambda t: native.fp8_quantize(t["x"]), dict(x=x)),
            ("fp8_gemm", lambda t: native.fp8_gemm(**t, out_dtype=torch.bfloat16), dict(codes=codes, scales=scales, **linear)),
            ("fp8_linear", lambda t: native.fp8_linear(**t), dict(x=x, **linear)),
            ("block_norm", lambda t: native.block_norm(**t, post_norm="rms"), norm),
            ("rotary", lambda t: native.rotary(**t, sections=(32,), norm="head"), turn)]


@pytest.fixture(scope="module")
def rope(pkg):
    return importlib.import_module(P + "rotary")


@gpu
@pytest.mark.parametrize("binding", [True, False])
def test_every_tracked_input_is_refused(native, quant, rope, binding):
    native._binding.enabled = binding
    try:
        for name, call, tensors in operator_calls(native, quant, rope):
            call(tensors)
            for key, tensor in tensors.items():
                tracked = {**tensors, key: torch.nn.Parameter(tensor)}
                with pytest.raises(RuntimeError, match="no backward"):
                    call(tracked)
                with torch.no_grad():
                    call(tracked)
                with torch.autograd.forward_ad.dual_level():
                    dual = torch.autograd.forward_ad.make_dual(tensor, tensor.clone())
                    with pytest.raises(RuntimeError, match="no forward-mode"), torch.no_grad():
                        call({**tensors, key: dual})
                    call(tensors)
    finally:
        native._binding.enabled = True


# ----------------------------------------------------------------------------------------------- the stack's linears
@pytest.fixture(scope="module")
def dit(pkg):
    return importlib.import_module(P + "dit")


def test_configurations_that_users_are_shown(dit):
    """Every ``DiTConfig(...)`` of the introduction is one."""
    shown = re.findall(r"DiTConfig\(([^()]*)\)", (ROOT / "README.md").read_text())
    assert any("rotary=True" in call for call in shown)
    for call in shown:
        assert not dit.DiTConfig(**eval(f"dict({call})")).plain


def test_a_quantized_input_takes_no_activation(dit):
    linear = dit.BlockScaledLinear(torch.ones(16, 128), backend="native")
    pair = (torch.zeros(2, 128).to(torch.float8_e4m3fn), torch.ones(2, 1))
    with pytest.raises(ValueError, match="no input_activation"):
        linear(pair, input_activation="gelu")
    for backend in ("native", "reference"):
        linear.backend = backend
        with pytest.raises(ValueError, match="'gelu'"):
            linear(torch.zeros(2, 128), input_activation="relu")
    with pytest.raises(ValueError, match="native backend"):
        linear(pair)


def small_stack(dit, device, **kw):
    cfg = dit.DiTConfig(**{**dict(blocks=2, hidden=256, heads=2, ffn=256, latent_tokens=12, action_tokens=4, grid=(2, 2, 3), linear="fp8",
                                  modulated=True, rotary=True), **kw})
    return dit.SyntheticDiT(cfg, device=device, backend="native" if device == "cuda" else "reference")


@pytest.mark.parametrize("move", [lambda m: m.half(), lambda m: m.to(torch.float16), lambda m: m.to("cpu", torch.float16)])
def test_moving_to_a_dtype_leaves_codes_and_scales(dit, move):
    linear = dit.BlockScaledLinear(torch.randn(16, 144).bfloat16(), bias=torch.ones(16, dtype=torch.bfloat16), backend="reference")
    codes, scales, keys = linear.weight.clone(), linear.weight_scales.clone(), list(linear.state_dict())
    assert move(linear) is linear
    assert linear.weight.dtype is torch.float8_e4m3fn and torch.equal(linear.weight.view(torch.uint8), codes.view(torch.uint8))
    assert linear.weight_scales.dtype is torch.float32 and torch.equal(linear.weight_scales, scales)
    assert list(linear.state_dict()) == keys and linear.bias.dtype is torch.float16
    assert linear(torch.ones(2, 144)).dtype is torch.float16
    meta = linear.to("meta")
    assert meta.weight.is_meta and meta.weight.dtype is torch.float8_e4m3fn and meta.weight_scales.dtype is torch.float32
    stack = small_stack(dit, "cpu")
    freq = stack.inv_freq.clone()
    move(stack)
    assert torch.equal(stack.inv_freq, freq) and stack.positions.dtype is torch.int32


@gpu
def test_stack_in_half_precision(dit):
    stack = small_stack(dit, "cuda")
    x = randn(1, 16, 256)
    with torch.no_grad():
        want = stack(x.bfloat16())
        got = stack.half()(x.half())
    assert got.dtype is torch.float16
    # the same weights on inputs and activations rounded to 2^-11 instead of 2^-8: apart by roundings of bf16 and the codes
    # they flip (the bar of a block's branch in test_block_ops, 4e-2, for each of the two blocks)
    assert float((got.float() - want.float()).norm() / want.float().norm()) < 8e-2


def test_weights_quantized_under_another_default_dtype(quant):
    weight = torch.randn(130, 144)
    want = quant.quantize_weight_block(weight)
    torch.set_default_dtype(torch.bfloat16)
    try:
        got = quant.quantize_weight_block(weight)
    finally:
        torch.set_default_dtype(torch.float32)
    assert got[1].dtype is torch.float32 and torch.equal(got[1], want[1])
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8))


# -------------------------------------------------------------------------------------------- the binding is optional
def test_building_without_a_host_compiler_or_pytorch(pkg, monkeypatch):
    build = importlib.import_module(P + "build")
    monkeypatch.setattr(build, "stale", lambda: False)
    which = build.shutil.which
    monkeypatch.setattr(build.shutil, "which", lambda name: None if name == "g++" else which(name))
    with pytest.warns(UserWarning, match="needs PyTorch and g"):
        assert build.build() == build.LIB
    monkeypatch.setattr(build.shutil, "which", which)
    monkeypatch.setattr(build, "binding_path", lambda: None)
    with pytest.warns(UserWarning, match="needs PyTorch and g"):
        assert build.build() == build.LIB


def test_binding_of_another_release_or_broken(pkg, monkeypatch, tmp_path):
    lib, build = importlib.import_module(P + "_lib"), importlib.import_module(P + "build")
    assert f"torch-{torch.__version__}.so" in build.binding_path().name and "cpython" in build.binding_path().name
    load = lib.load_binding.__wrapped__
    monkeypatch.setattr(lib, "binding_path", lambda: tmp_path / "sq_binding.of-another-release.so")
    assert load() is None
    (tmp_path / "sq_binding.of-another-release.so").write_bytes(b"not a shared object")
    with pytest.warns(UserWarning, match="does not load"):
        assert load() is None
    monkeypatch.setattr(lib, "binding_path", lambda: None)
    assert load() is None


# ------------------------------------------------------------------------------------------------------ host threads
@gpu
def test_other_threads_run_while_a_call_waits(native):
    """A call that waits for room in the launch queue does not hold the interpreter: a thread that ticks every millisecond
    goes on while the device is busy for about half a second and more launches are asked for than its queue holds."""
    x = randn(64, 1024, dtype=torch.bfloat16)
    native.block_norm(x)
    torch.cuda.synchronize()
    ticks, done = [], threading.Event()

    def tick():
        while not done.wait(0.001):
            ticks.append(time.perf_counter())

    thread = threading.Thread(target=tick)
    thread.start()
    try:
        torch.cuda._sleep(10 ** 9)
        begin = time.perf_counter()
        for _ in range(3000):
            native.block_norm(x)
        waited = time.perf_counter() - begin
    finally:
        done.set()
        thread.join()
    torch.cuda.synchronize()
    assert waited > 0.2, "the launches did not wait for the device"
    longest = max(b - a for a, b in zip(ticks, ticks[1:]))
    assert longest < waited / 2


@gpu
def test_calls_from_two_threads(native, quant):
    x, _, _, weight, weight_scales, bias = fp8_case(quant, 300, 512, 1024, torch.bfloat16)
    want, want_norm = native.fp8_linear(x, weight, weight_scales, bias), native.block_norm(x, x)
    torch.cuda.synchronize()
    wrong = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                y, (h, z) = native.fp8_linear(x, weight, weight_scales, bias), native.block_norm(x, x)
                torch.cuda.current_stream().synchronize()
                if not (torch.equal(y, want) and torch.equal(h, want_norm[0]) and torch.equal(z, want_norm[1])):
                    wrong.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not wrong


# ----------------------------------------------------------------------------------------- outputs that share memory
OVERLAP_HARNESS = """
#include "sq_overlap.h"
static sq::View view(const long long* v) {
  return sq::View(reinterpret_cast<const void*>(v[0]), v[1], v[2], v[3], v[4], v[5], v[6], v[7]);
}
extern "C" int overlaps(const long long* a, const long long* b) { return sq::overlaps(view(a), view(b)); }
extern "C" int overlaps_itself(const long long* a) { return sq::overlaps_itself(view(a)); }
"""


def test_overlap_of_views_against_their_bytes(pkg, tmp_path):
    source, library = tmp_path / "harness.cpp", tmp_path / "harness.so"
    source.write_text(OVERLAP_HARNESS)
    csrc = ROOT / "fastwamjoint-quantization_b200" / "csrc"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", f"-I{csrc}", str(source), "-o", str(library)], check=True)
    harness = ctypes.CDLL(str(library))
    rng = random.Random(0)
    pack = lambda v: (ctypes.c_longlong * 8)(*v)

    def some_view():
        nested = rng.random() < 0.5
        counts = [rng.choice((1, 1, 2, 3, 5)) for _ in range(3)]
        run = rng.choice((1, 2, 4, 8))
        if nested:
            inner = run + rng.choice((0, 0, 2))
            middle = inner * counts[2] + rng.choice((0, 4))
            strides = [middle * counts[1] + rng.choice((0, 16)), middle, inner]
            if rng.random() < 0.3:
                strides[0], strides[1], counts[0], counts[1] = strides[1], strides[0], counts[1], counts[0]
        else:
            strides = [rng.randrange(0, 24) for _ in range(3)]
        return [rng.randrange(1, 160), run, counts[0], strides[0], counts[1], strides[1], counts[2], strides[2]]

    def runs(v):
        return [v[0] + i * v[3] + j * v[5] + k * v[7] for i in range(v[2]) for j in range(v[4]) for k in range(v[6])]

    seen = {True: 0, False: 0}
    for _ in range(4000):
        a, b = some_view(), some_view()
        if rng.random() < 0.4:  # neighbours in one packed row
            b[1:] = a[1:]
            b[0] = a[0] + rng.randrange(0, 40)
        bytes_a = [x + i for x in runs(a) for i in range(a[1])]
        bytes_b = {x + i for x in runs(b) for i in range(b[1])}
        want = not bytes_b.isdisjoint(bytes_a)
        seen[want] += 1
        assert bool(harness.overlaps(pack(a), pack(b))) is want and bool(harness.overlaps(pack(b), pack(a))) is want
        assert bool(harness.overlaps_itself(pack(a))) is (len(set(bytes_a)) < len(bytes_a))
    assert min(seen.values()) > 500
    for empty in ([0, 8, 1, 0, 1, 0, 1, 0], [64, 0, 1, 0, 1, 0, 1, 0], [64, 8, 0, 8, 1, 0, 1, 0]):
        assert not harness.overlaps(pack(empty), pack([1, 200, 1, 0, 1, 0, 1, 0])) and not harness.overlaps_itself(pack(empty))


def test_c_abi_refuses_overlap(pkg):
    """Shared memory is found on the host; the pointers are never read (every call here is refused)."""
    lib_mod = importlib.import_module(P + "_lib")
    lib, refused = lib_mod.load_library(), lib_mod.ERR_OVERLAP
    at = lambda kib: 1 << 20 | kib << 10  # tensors far apart
    gemm = dict(codes=at(0), scales=at(64), rs=1, gs=4, w=at(128), ws=at(192), bias=at(256), out=at(320))

    def product(**kw):
        c = {**gemm, **kw}
        return lib.sq_fp8_gemm(c["codes"], c["scales"], c["rs"], c["gs"], c["w"], c["ws"], c["bias"], c["out"], 0, 4, 16, 256, None)

    for key in ("codes", "scales", "w", "ws", "bias"):
        assert product(out=gemm[key]) == refused
        assert product(**{key: gemm["out"] + 2 * 4 * 16 - 16}) == refused
    quantize = lambda x, codes, scales, rs=1, gs=4: lib.sq_fp8_quantize(x, 0, 4, 256, 0, codes, scales, rs, gs, None)
    assert quantize(at(0), at(0), at(64)) == refused and quantize(at(0), at(64), at(1)) == refused
    assert quantize(at(0), at(64), at(64)) == refused and quantize(at(0), at(64), at(128), 1, 2) == refused
    assert quantize(at(0), at(64), at(128), -1, 4) == lib_mod.ERR_SHAPE
    linear = lambda x, w, ws, bias, out, work: lib.sq_fp8_linear(x, 0, 4, 256, 16, 0, w, ws, bias, out, work, 1 << 14, None)
    apart = [at(64 * i) for i in range(6)]
    for other in range(5):
        assert linear(*[apart[other] if i == 5 else a for i, a in enumerate(apart)]) == refused
    for other in (1, 2, 3):
        assert linear(*[apart[other] if i == 4 else a for i, a in enumerate(apart)]) == refused

    def norm(**kw):
        base = dict(x=at(0), branch=at(64), h_out=at(128), z_out=at(192), rows=4, width=64, residual_scale=1.0, eps=1e-6,
                    norm_kind=lib_mod.NORM_RMS)
        return lib.sq_block_norm(lib_mod.ctypes.byref(lib_mod.BlockNorm(**{**base, **kw})), None)

    row = lambda p: lib_mod.Param(p, 64, 1, 0)
    for kw in (dict(h_out=at(0) + 128), dict(h_out=at(64) + 16), dict(z_out=at(128)), dict(z_out=at(0) + 16), dict(gate=row(at(128))),
               dict(mod_shift=row(at(192))), dict(weight=lib_mod.Param(at(128) + 384)), dict(z_out=at(0), scales=at(256), scales_row_stride=1,
                                                                                         scales_group_stride=4),
               dict(scales=at(128), scales_row_stride=1, scales_group_stride=4), dict(scales=at(256))):
        assert norm(**kw) == refused

    def rotary(**kw):
        strides = (lib_mod.c_int64 * 3)(512, 64, 32)
        base = dict(q=at(0), k=at(64), q_out=at(128), k_out=at(192), positions=at(256), inv_freq=at(320), batch=1, length=8, heads=2, kv_heads=2,
                    dim=32, axes=1, q_strides=strides, k_strides=strides, q_out_strides=strides, k_out_strides=strides, position_token_stride=1)
        args = lib_mod.Rotary(**{**base, **{n: (lib_mod.c_int64 * 3)(*v) if isinstance(v, tuple) else v for n, v in kw.items()}})
        args.sections[0] = 16
        return lib.sq_rotary(lib_mod.ctypes.byref(args), None)

    for kw in (dict(q_out=at(64)), dict(k_out=at(0)), dict(q_out=at(192)), dict(q_out=at(0) + 64), dict(q_out=at(0), q_out_strides=(512, 32, 256)),
               dict(q_out_strides=(512, 32, 32)), dict(k_out_strides=(512, 32, 16)), dict(q_out=at(256)), dict(k_out=at(320)),
               dict(norm=1, q_weight=at(128)), dict(norm=1, k_weight=at(128))):
        assert rotary(**kw) == refused


@gpu
def test_outputs_that_share_memory_are_refused(native, quant, rope):
    x, codes, scales, weight, weight_scales, bias = fp8_case(quant, 128, 128, 128, torch.bfloat16)
    gemm = lambda out: native.fp8_gemm(codes, scales, weight, weight_scales, bias, out_dtype=torch.bfloat16, out=out)
    room = torch.empty(128, 128, device="cuda", dtype=torch.bfloat16)
    want = gemm(None)
    assert torch.equal(gemm(room), want)
    double = torch.zeros(2 * 128 * 128, device="cuda", dtype=torch.uint8)
    codes_in = double[: 128 * 128].view(torch.float8_e4m3fn).view(128, 128)
    with pytest.raises(ValueError, match="share no memory"):
        native.fp8_gemm(codes_in, scales, weight, weight_scales, out_dtype=torch.bfloat16, out=double.view(torch.bfloat16).view(128, 128))
    work = torch.empty(1 << 16, device="cuda", dtype=torch.uint8)
    with pytest.raises(ValueError, match="share no memory"):
        native.fp8_linear(x, weight, weight_scales, bias, workspace=work, out=work[: 2 * 128 * 128].view(torch.bfloat16).view(128, 128))
    inside = x.clone()
    want = native.fp8_linear(x, weight, weight_scales, bias)  # the quantizer has read x before the product writes
    assert torch.equal(native.fp8_linear(inside, weight, weight_scales, bias, out=inside), want)

    qkv = randn(2, 9, 6, 64, dtype=torch.bfloat16)
    q, k = qkv[:, :, :4], qkv[:, :, 4:]
    positions, freq = torch.arange(9, device="cuda", dtype=torch.int32)[:, None], rope.rotary_frequencies((32,), device="cuda")
    turn = lambda q, k, out=None: native.rotary(q, k, positions, freq, sections=(32,), out=out)
    spare = torch.empty(2, 9, 4, 64, device="cuda", dtype=torch.bfloat16)
    late = torch.empty(2, 10, 6, 64, device="cuda", dtype=torch.bfloat16)
    late[:, :9] = qkv
    for inputs, out in (((q, k), (qkv[:, :, 1:5], None)), ((q, k), (spare, spare[:, :, :2])), ((q, k), (None, q[:, :, :2])),
                        ((late[:, :9, :4], None), (late[:, 1:, :4], None)),
                        ((q, None), (spare.flatten()[: 2 * 9 * 4 * 64].as_strided((2, 9, 4, 64), (2304, 64, 64, 1)), None))):
        with pytest.raises(ValueError, match="share no memory"):
            turn(*inputs, out=out)
    want = turn(q, k)
    turn(q, k, out=(q, k))  # neighbours in one packed tensor, each its own input
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


# ---------------------------------------------------------------------------------------------------------- rotary
@gpu
@pytest.mark.parametrize("shape", [(1, 1, 1, 64), (1, 1, 3, 64), (2, 1, 1, 64), (1, 5, 1, 64), (3, 1, 2, 64)])
def test_rotary_strides_of_axes_with_one_index(native, rope, shape):
    """An axis of one index may have any stride: a single token or head cut out of a wider tensor."""
    x = randn(*shape, dtype=torch.bfloat16)
    batch, tokens, heads, dim = shape
    positions, freq = torch.arange(3, 3 + tokens, device="cuda", dtype=torch.int32)[:, None], rope.rotary_frequencies((32,), device="cuda")
    turn = lambda t, out=None: native.rotary(t, None, positions, freq, sections=(32,), out=out)[0]
    want = turn(x)
    strides = [67 if n == 1 else s for n, s in zip(shape[:3], x.stride())]
    odd = torch.zeros(batch * tokens * heads * dim, device="cuda", dtype=torch.bfloat16).as_strided(shape, (*strides, 1))
    odd.copy_(x)
    assert torch.equal(turn(odd), want)
    room = torch.zeros_like(x).as_strided(shape, (*strides, 1))
    assert turn(x, (room, None)) is room and torch.equal(room, want)
    assert torch.equal(turn(odd, (odd, None)), want) and torch.equal(odd, want)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dim,pairs", [(16, 3), (64, 5), (64, 8), (72, 14), (128, 62), (128, 63)])
def test_rotary_passes_the_rest_of_a_head_through(native, rope, dim, pairs, layout, dtype):
    """Elements past the turned pairs come out bit for bit, infinities and negative zeros too, and disturb nothing."""
    x = randn(2, 7, 3, dim, dtype=dtype)
    rest = x[..., 2 * pairs:]
    rest[..., 0::3], rest[..., 1::4], rest[0, 0, 0, -1] = float("inf"), -0.0, float("nan")
    positions, freq = torch.arange(1, 8, device="cuda", dtype=torch.int32)[:, None], rope.rotary_frequencies((pairs,), device="cuda")
    got = native.rotary(x, None, positions, freq, sections=(pairs,), layout=layout)[0]
    nan = rest.isnan()
    assert torch.equal(got[..., 2 * pairs:].isnan(), nan)
    assert torch.equal(got[..., 2 * pairs:].view(torch.int16)[~nan], rest.view(torch.int16)[~nan])
    alone = x.clone()
    alone[..., 2 * pairs:] = 0
    alone = native.rotary(alone, None, positions, freq, sections=(pairs,), layout=layout)[0]
    assert torch.equal(got[..., :2 * pairs], alone[..., :2 * pairs]) and alone.isfinite().all()


# -------------------------------------------------------------------------------------------------------- block norms
@gpu
@pytest.mark.parametrize("eps", [0.0, 1e-35, 1e-12])
@pytest.mark.parametrize("width", [64, 1000, 2048, 4096, 6144, 14336])
def test_block_norm_of_tiny_and_huge_rows(native, width, eps):
    """Rows whose squares leave the range of fp32 on either side, with an eps that does not cover the small ones."""
    x = randn(7, width) * torch.tensor([1e-30, 1e-25, 1e-19, 1e-15, 1.0, 1e19, 1e30], device="cuda")[:, None]
    x, branch = x.bfloat16(), x.flip(1).bfloat16()
    check_block_norm(native, x, norm="rms", eps=eps)
    check_block_norm(native, x, norm="layer", eps=eps)
    check_block_norm(native, torch.zeros_like(x), branch, post_norm="rms", norm="layer", eps=eps)
    _, z = native.block_norm(torch.zeros_like(x), norm="rms", eps=max(eps, 1e-35))
    assert not z.any()
