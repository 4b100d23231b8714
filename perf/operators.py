"""Timed cases of the block operators of the video / action transformer: the 8-bit floating-point linear with a scale for
each block of 128, the norms before and after a block with its gate and residual scale, and rotary positions on several
axes.  ``run`` computes them in elementary torch operations, or - where ``own`` is true - through the framework's calls."""
import functools
import importlib
import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@functools.lru_cache(maxsize=1)
def _native():
    entry = importlib.import_module("__graft_entry__")
    entry.load_package()
    return importlib.import_module("fastwamjoint_quantization_b200.native")


# ---------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one chunk of 32 action tokens through the action expert's FFN: the smallest product, latency counts
        {"name": "gemm_action_chunk", "kind": "gemm", "m": 32, "n": 4096, "k": 1024, "dtype": "bf16", "bias": True},
        # nothing is a multiple of a tile: tokens left over after padding is dropped, a narrow adapter
        {"name": "gemm_ragged", "kind": "gemm", "m": 1001, "n": 1480, "k": 2000, "dtype": "fp16", "bias": True},
        # a long clip through the widest layer: the largest product
        {"name": "gemm_long_clip", "kind": "gemm", "m": 8192, "n": 14336, "k": 4096, "dtype": "bf16", "bias": False},
        # one token (a modulation / time embedding projection): weight bytes and latency
        {"name": "linear_one_token", "kind": "linear", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16", "bias": True, "gelu": False},
        # three latent frames of the video expert, long K with the activation in front
        {"name": "linear_three_frames", "kind": "linear", "m": 294, "n": 1024, "k": 14336, "dtype": "bf16", "bias": True, "gelu": True},
        # the benchmark stack's 1560 latent + 32 action tokens through the FFN's second linear
        {"name": "linear_stack_down", "kind": "linear", "m": 1592, "n": 4096, "k": 12288, "dtype": "bf16", "bias": False, "gelu": True},
        # 32 action tokens, LayerNorm + AdaLN in front of a block (no branch yet): the smallest norm
        {"name": "norm_action_front", "kind": "norm", "m": 32, "h": 1024, "groups": 2, "dtype": "bf16", "branch": False,
         "post": "none", "norm": "layer", "quantize": False, "fp32_mod": False},
        # between attention and FFN of the stack: normed branch, gate, residual, next norm, e4m3 codes for the next linear;
        # every token has a modulation row of its own (per-token timesteps)
        {"name": "norm_stack_between", "kind": "norm", "m": 1592, "h": 4096, "groups": 1592, "dtype": "bf16", "branch": True,
         "post": "rms", "norm": "rms", "quantize": True, "fp32_mod": False},
        # a long clip, fp16, one modulation row for each of 16 frames: the largest norm
        {"name": "norm_long_clip", "kind": "norm", "m": 32768, "h": 4096, "groups": 16, "dtype": "fp16", "branch": True,
         "post": "none", "norm": "layer", "quantize": False, "fp32_mod": True},
        # 32 action tokens, norm over all heads: the smallest rotation
        {"name": "rotary_action_chunk", "kind": "rotary", "batch": 1, "tokens": 32, "heads": 8, "kv_heads": 8, "dim": 128,
         "axes": 3, "layout": "interleaved", "norm": "token", "dtype": "bf16", "far": 0},
        # image tokens with a head length off the vector sizes, pairs half a head apart, far positions
        {"name": "rotary_odd_heads", "kind": "rotary", "batch": 2, "tokens": 1003, "heads": 10, "kv_heads": 5, "dim": 72,
         "axes": 2, "layout": "half", "norm": "none", "dtype": "fp16", "far": 1000000},
        # two long clips, shared key heads, norm of each head: the largest rotation
        {"name": "rotary_long_clip", "kind": "rotary", "batch": 2, "tokens": 16384, "heads": 32, "kv_heads": 8, "dim": 128,
         "axes": 3, "layout": "interleaved", "norm": "head", "dtype": "bf16", "far": 0},
    ]


def _log(rng, lo, hi, step=1):
    return max(lo, min(hi, step * round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)))


def draw(rng):
    kind = rng.choice(["gemm", "linear", "norm", "rotary"])
    dtype = rng.choice(["bf16", "fp16"])
    if kind in ("gemm", "linear"):
        while True:
            m, n, k = _log(rng, 1, 8192), _log(rng, 64, 14336, 8), _log(rng, 128, 14336, 16)
            if m * n * k <= 8192 * 14336 * 4096:
                break
        case = {"kind": kind, "m": m, "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.5}
        if kind == "linear":
            case["gelu"] = rng.random() < 0.5
        return case
    if kind == "norm":
        while True:
            span, groups, h = _log(rng, 1, 4096), _log(rng, 1, 512), _log(rng, 64, 14336, 16)
            if span * groups * h <= 32768 * 4096:
                break
        branch = rng.random() < 0.7
        return {"kind": kind, "m": span * groups, "h": h, "groups": groups, "dtype": dtype, "branch": branch,
                "post": rng.choice(["none", "rms", "layer"]) if branch else "none", "norm": rng.choice(["rms", "layer"]),
                "quantize": rng.random() < 0.4, "fp32_mod": rng.random() < 0.5}
    while True:
        batch, tokens, dim = rng.randint(1, 4), _log(rng, 1, 32768), rng.choice([40, 64, 72, 80, 96, 112, 128, 160, 192, 256])
        kv_heads = _log(rng, 1, 24)
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        if batch * tokens * (heads + kv_heads) * dim <= 2 * 16384 * 40 * 128 and (heads + kv_heads) * dim <= 8192:
            break
    return {"kind": kind, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "axes": rng.choice([1, 2, 3]), "layout": rng.choice(["interleaved", "half"]),
            "norm": rng.choice(["none", "head", "token"]), "dtype": dtype, "far": rng.choice([0, 0, 1000000])}


# --------------------------------------------------------------------------------------------------------- inputs
def _sections(case):
    """Rotated pairs of each axis: an even share of the head, the remainder on the first axis (time)."""
    pairs, axes = case["dim"] // 2, case["axes"]
    share = pairs // axes
    return (pairs - share * (axes - 1),) + (share,) * (axes - 1)


def _activations(gen, rows, width):
    """Unit rows with one channel in a hundred twenty times as large, as the stack's activations have."""
    x = torch.randn(rows, width, generator=gen, device="cuda")
    loud = torch.rand(width, generator=gen, device="cuda") < 0.01
    return x * torch.where(loud, 20.0, 1.0)


def _weight(gen, n, k):
    """e4m3 weights with fp32 scales of 128 x 128 blocks, as a checkpoint holds them."""
    w = torch.randn(n, k, generator=gen, device="cuda") * 0.02
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    padded = torch.zeros(nb * BLOCK, kb * BLOCK, device="cuda")
    padded[:n, :k] = w
    blocks = padded.view(nb, BLOCK, kb, BLOCK)
    scales = blocks.abs().amax(dim=(1, 3)).clamp_min(1e-12) / E4M3_MAX
    codes = (blocks / scales[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).view(nb * BLOCK, kb * BLOCK)[:n, :k]
    return codes.to(torch.float8_e4m3fn).contiguous(), scales.contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    rand = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    state = {"case": dict(case)}
    if case["kind"] in ("gemm", "linear"):
        m, n, k = case["m"], case["n"], case["k"]
        state["weight"], state["weight_scales"] = _weight(gen, n, k)
        state["bias"] = (rand(n) * 0.1).to(dtype) if case["bias"] else None
        x = _activations(gen, m, k)
        if case["kind"] == "linear":
            state["x"] = x.to(dtype)
        else:
            kb = -(-k // BLOCK)
            groups = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).view(m, kb, BLOCK)
            scales = groups.abs().amax(dim=2).clamp_min(1e-6) / E4M3_MAX
            codes = (groups / scales[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).view(m, kb * BLOCK)[:, :k]
            state["codes"] = codes.to(torch.float8_e4m3fn).contiguous()
            # the layout the framework's quantizer leaves: the tokens of one block next to each other
            state["scales"] = scales.t().contiguous().t()
        return state
    if case["kind"] == "norm":
        m, h, groups = case["m"], case["h"], case["groups"]
        mod = torch.float32 if case["fp32_mod"] else dtype
        state["x"] = _activations(gen, m, h).to(dtype)
        table = rand(groups, 3, h) * 0.3  # one row of shift, scale, gate for each group, sliced as models slice it
        table = table.to(mod)
        state["shift"], state["scale"], state["gate"] = table[:, 0], table[:, 1], table[:, 2]
        state["weight"] = (1.0 + 0.1 * rand(h)).to(dtype)
        if case["branch"]:
            state["branch"] = (rand(m, h) * 2.0).to(dtype)
            state["post_weight"] = None if case["post"] == "none" else (1.0 + 0.1 * rand(h)).to(dtype)
        return state
    b, t, heads, kv, dim = (case[x] for x in ("batch", "tokens", "heads", "kv_heads", "dim"))
    # one packed projection, as the attention's linear writes it; q and k are strided views
    qkv = rand(b, t, heads + 2 * kv, dim).to(dtype)
    state["q"], state["k"] = qkv[:, :, :heads], qkv[:, :, heads:heads + kv]
    sections = _sections(case)
    state["sections"] = sections
    state["axis"] = torch.tensor([a for a, count in enumerate(sections) for _ in range(count)], device="cuda")
    state["inv_freq"] = torch.cat([10000.0 ** (-torch.arange(s, dtype=torch.float64) / s) for s in sections]).cuda()
    # tokens in raster order of a clip: time x height x width (as many axes as there are), at an offset in time
    side = [26, 20][: case["axes"] - 1]
    index = torch.arange(t, device="cuda", dtype=torch.int64)
    columns = []
    for extent in side:
        columns.insert(0, index % extent)
        index = index // extent
    columns.insert(0, index + case["far"])
    start = torch.randint(0, 64, (b, 1, 1), generator=gen, device="cuda")
    state["positions"] = (torch.stack(columns, dim=-1)[None] + start).to(torch.int32).contiguous()
    if case["norm"] != "none":
        width = dim if case["norm"] == "head" else None
        state["q_weight"] = (1.0 + 0.1 * rand(width or heads * dim)).to(dtype)
        state["k_weight"] = (1.0 + 0.1 * rand(width or kv * dim)).to(dtype)
    return state


# ------------------------------------------------------------------------------------------------------ plain form
def _plain_quantize(x):
    """fp32 [m, k] -> e4m3 codes and the fp32 scale of each run of 128."""
    m, k = x.shape
    kb = -(-k // BLOCK)
    runs = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).view(m, kb, BLOCK)
    amax = runs.abs().amax(dim=2)
    scales = (amax / torch.full_like(amax, E4M3_MAX)).clamp_min(1e-8)
    codes = (runs * (1.0 / scales)[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    return codes.to(torch.float8_e4m3fn).view(m, kb * BLOCK)[:, :k], scales


def _plain_product(codes, scales, weight, weight_scales, bias, dtype):
    n, k = weight.shape
    a = codes.float() * scales.repeat_interleave(BLOCK, dim=1)[:, :k]
    w = weight.float() * weight_scales.repeat_interleave(BLOCK, dim=0)[:n].repeat_interleave(BLOCK, dim=1)[:, :k]
    y = a @ w.t()
    if bias is not None:
        y = y + bias.float()
    return y.to(dtype)


def _plain_gelu(x):
    return 0.5 * x * (1.0 + torch.erf(x * (1.0 / math.sqrt(2.0))))


def _plain_norm(v, kind, weight):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(dim=-1, keepdim=True)
    v = v * torch.rsqrt(v.square().mean(dim=-1, keepdim=True) + 1e-6)
    return v if weight is None else v * weight.float()


def _plain_rotary(x, cos, sin, layout, norm, weight):
    b, t, heads, dim = x.shape
    v = x.float()
    if norm == "head":
        v = _plain_norm(v, "rms", weight)
    elif norm == "token":
        v = _plain_norm(v.reshape(b, t, heads * dim), "rms", weight).view(b, t, heads, dim)
    pairs = cos.shape[-1]
    cos, sin = cos[:, :, None], sin[:, :, None]
    if layout == "interleaved":
        first, second = v[..., 0:2 * pairs:2], v[..., 1:2 * pairs:2]
        turned = torch.stack((first * cos - second * sin, first * sin + second * cos), dim=-1).flatten(-2)
    else:
        first, second = v[..., :pairs], v[..., pairs:2 * pairs]
        turned = torch.cat((first * cos - second * sin, first * sin + second * cos), dim=-1)
    return torch.cat((turned, v[..., 2 * pairs:]), dim=-1).to(x.dtype)


def _run_plain(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "gemm":
        return _plain_product(state["codes"], state["scales"], state["weight"], state["weight_scales"], state["bias"], dtype)
    if case["kind"] == "linear":
        x = state["x"].float()
        if case["gelu"]:
            x = _plain_gelu(x)
        codes, scales = _plain_quantize(x)
        return _plain_product(codes, scales, state["weight"], state["weight_scales"], state["bias"], dtype)
    if case["kind"] == "norm":
        span = case["m"] // case["groups"]
        rows = lambda v: v.float().repeat_interleave(span, dim=0)
        h = state["x"].float()
        out = []
        if case["branch"]:
            h = 0.5 * h + rows(state["gate"]) * _plain_norm(state["branch"].float(), case["post"], state["post_weight"])
            out.append(h.to(dtype))
        z = _plain_norm(h, case["norm"], state["weight"]) * (1.0 + rows(state["scale"])) + rows(state["shift"])
        return out + (list(_plain_quantize(z)) if case["quantize"] else [z.to(dtype)])
    angles = state["positions"].double()[..., state["axis"]] * state["inv_freq"]
    cos, sin = angles.cos().float(), angles.sin().float()
    args = (cos, sin, case["layout"], case["norm"])
    return [_plain_rotary(state["q"], *args, state.get("q_weight")), _plain_rotary(state["k"], *args, state.get("k_weight"))]


# ------------------------------------------------------------------------------------------------ the framework's calls
def _run_own(state):
    native = _native()
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "gemm":
        return native.fp8_gemm(state["codes"], state["scales"], state["weight"], state["weight_scales"], state["bias"],
                               out_dtype=dtype)
    if case["kind"] == "linear":
        return native.fp8_linear(state["x"], state["weight"], state["weight_scales"], state["bias"],
                                 input_activation="gelu" if case["gelu"] else None)
    if case["kind"] == "norm":
        fused = {}
        if case["branch"]:
            fused = {"branch": state["branch"], "gate": state["gate"], "residual_scale": 0.5,
                     "post_norm": None if case["post"] == "none" else case["post"], "post_weight": state["post_weight"]}
        h, z = native.block_norm(state["x"], norm=case["norm"], weight=state["weight"], mod_scale=state["scale"],
                                 mod_shift=state["shift"], eps=1e-6, quantize=case["quantize"], **fused)
        return ([h] if case["branch"] else []) + (list(z) if case["quantize"] else [z])
    q, k = native.rotary(state["q"], state["k"], state["positions"], state["inv_freq"], sections=state["sections"],
                         layout=case["layout"], norm=None if case["norm"] == "none" else case["norm"],
                         q_weight=state.get("q_weight"), k_weight=state.get("k_weight"), eps=1e-6)
    return [q, k]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------------------------------------------------------- in 64 bits
def _exact_codes(x):
    m, k = x.shape
    codes, scales = torch.empty_like(x), []
    for g in range(0, k, BLOCK):
        part = x[:, g:g + BLOCK]
        s = torch.clamp(part.abs().max(dim=1).values / E4M3_MAX, min=1e-8)
        codes[:, g:g + BLOCK] = (part / s[:, None]).float().to(torch.float8_e4m3fn).double()
        scales.append(s)
    return codes, torch.stack(scales, dim=1)


def _exact_standardised(v, kind):
    if kind == "none":
        return v
    if kind == "layer":
        return (v - v.mean(-1, keepdim=True)) / (v.var(-1, unbiased=False, keepdim=True) + 1e-6).sqrt()
    return v / ((v * v).sum(-1, keepdim=True) / v.shape[-1] + 1e-6).sqrt()


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("gemm", "linear"):
        if case["kind"] == "linear":
            x = s["x"].double()
            if case["gelu"]:
                x = x * torch.special.ndtr(x)
            codes, scales = _exact_codes(x)
        else:
            codes, scales = s["codes"].double(), s["scales"].double()
        n, k = s["weight"].shape
        w = s["weight"].double()
        t = s["weight_scales"].double()
        y = torch.zeros(codes.shape[0], n, dtype=torch.float64, device="cuda")
        for g in range(t.shape[1]):
            cut = slice(g * BLOCK, min(k, (g + 1) * BLOCK))
            column = t[:, g].repeat_interleave(BLOCK)[:n]
            y.addmm_(codes[:, cut] * scales[:, g:g + 1], (w[:, cut] * column[:, None]).t())
        return y if s["bias"] is None else y + s["bias"].double()
    if case["kind"] == "norm":
        group = torch.arange(case["m"], device="cuda") // (case["m"] // case["groups"])
        h, out = s["x"].double(), []
        if case["branch"]:
            b = _exact_standardised(s["branch"].double(), case["post"])
            if s["post_weight"] is not None:
                b = b * s["post_weight"].double()
            h = h / 2 + s["gate"].double()[group] * b
            out.append(h)
        z = _exact_standardised(h, case["norm"]) * s["weight"].double()
        z = z + z * s["scale"].double()[group] + s["shift"].double()[group]
        return out + (list(_exact_codes(z)) if case["quantize"] else [z])
    pairs = sum(s["sections"])
    phase, first = [], 0
    for a, count in enumerate(s["sections"]):
        phase.append(s["positions"][..., a].double()[..., None] * s["inv_freq"][first:first + count])
        first += count
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.cat(phase, dim=-1))[:, :, None]
    out = []
    for name in ("q", "k"):
        v = s[name].double()
        if case["norm"] == "head":
            v = _exact_standardised(v, "rms") * s[name + "_weight"].double()
        elif case["norm"] == "token":
            flat = v.flatten(2)
            v = (_exact_standardised(flat, "rms") * s[name + "_weight"].double()).unflatten(2, v.shape[2:])
        if case["layout"] == "interleaved":
            z = torch.view_as_complex(v[..., :2 * pairs].unflatten(-1, (pairs, 2)).contiguous()) * turn
            head = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(v[..., :pairs], v[..., pairs:2 * pairs]) * turn
            head = torch.cat((z.real, z.imag), dim=-1)
        out.append(torch.cat((head, v[..., 2 * pairs:]), dim=-1))
    return out


# ------------------------------------------------------------------------------------------- what cannot be done without
def work(case):
    if case["kind"] in ("gemm", "linear"):
        m, n, k = case["m"], case["n"], case["k"]
        kb, nb = -(-k // BLOCK), -(-n // BLOCK)
        activations = m * k * 2 if case["kind"] == "linear" else m * k + 4 * m * kb
        return {"bytes": activations + n * k + 4 * nb * kb + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if case["kind"] == "norm":
        m, h = case["m"], case["h"]
        vectors = (3 if case["branch"] else 2) * case["groups"] * h * (4 if case["fp32_mod"] else 2)
        vectors += (1 if case["post"] == "none" else 2) * h * 2
        written = (m * h + 4 * m * -(-h // BLOCK)) if case["quantize"] else 2 * m * h
        read = (2 if case["branch"] else 1) * 2 * m * h
        return {"bytes": read + vectors + written + (2 * m * h if case["branch"] else 0), "flops": (16 if case["branch"] else 9) * m * h}
    tokens = case["batch"] * case["tokens"]
    heads = case["heads"] + case["kv_heads"]
    elements = tokens * heads * case["dim"]
    weights = {"none": 0, "head": 4 * case["dim"], "token": 2 * heads * case["dim"]}[case["norm"]]
    return {"bytes": 4 * elements + 4 * tokens * case["axes"] + 4 * case["dim"] + weights,
            "flops": elements * (3 if case["norm"] == "none" else 7)}
