"""Tensor-level wrappers over the C ABI: they allocate outputs and scratch with
``torch.empty`` on the current device (so CUDA-graph capture uses PyTorch's
graph-private pool, as the reference's ``torch::empty`` calls do,
``kernels/w4a8/csrc/w4a8.cu:1358-1360``) and launch on the current stream."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16}


def _require_cuda(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor: the B200 path has no CPU fallback.")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def prepass(x: torch.Tensor, *, abits: int, mode: str, inverse=None, signs=None, rht_block: int = 128,
            act_scale=None, gains=None, span: int = 1, streams: int = 1, seq_tokens: int | None = None,
            codes_layout: int = _lib.CODES_EVEN_ODD, pack_int4: bool = False, out=None, mix=None):
    """Run the fused activation pre-pass.  ``x`` is [..., tokens, K] bf16/fp16.
    Returns ``(codes, row_scales)``: int8 [rows, K] (or uint8 [rows, K/2] when
    ``pack_int4``) and fp32 [rows].  ``mix`` (fp32 [order, order] of +-1) selects the composite rotation
    ``order x power of two`` instead of the block rotation of length ``rht_block``."""
    _require_cuda(x, "x")
    x = x.contiguous()
    k = x.shape[-1]
    rows = x.numel() // k
    if out is not None:
        codes, row_scales = out
    else:
        codes = torch.empty((rows, k // 2) if pack_int4 else (rows, k), device=x.device,
                            dtype=torch.uint8 if pack_int4 else torch.int8)
        row_scales = torch.empty((rows,), device=x.device, dtype=torch.float32)
    if mix is not None:
        mix = _mix_matrix(mix, x)
        with torch.cuda.device(x.device):
            status = _lib.load_library().sq_prepass_composite(
                x.data_ptr(), _DTYPES[x.dtype], rows, k, int(abits),
                _lib.ACT_TOKEN if mode == "token" else _lib.ACT_STATIC,
                _ptr(inverse), _ptr(signs), mix.data_ptr(), int(mix.shape[0]), _ptr(act_scale), _ptr(gains),
                int(span), int(streams), int(seq_tokens if seq_tokens is not None else x.shape[-2]),
                int(codes_layout), int(bool(pack_int4)), codes.data_ptr(), row_scales.data_ptr(), _stream())
        _lib.check(status, "sq_prepass_composite")
        return codes, row_scales
    with torch.cuda.device(x.device):
        status = _lib.load_library().sq_prepass(
            x.data_ptr(), _DTYPES[x.dtype], rows, k, int(abits),
            _lib.ACT_TOKEN if mode == "token" else _lib.ACT_STATIC,
            _ptr(inverse), _ptr(signs), int(rht_block), _ptr(act_scale), _ptr(gains),
            int(span), int(streams), int(seq_tokens if seq_tokens is not None else x.shape[-2]),
            int(codes_layout), int(bool(pack_int4)), codes.data_ptr(), row_scales.data_ptr(), _stream())
    _lib.check(status, "sq_prepass")
    return codes, row_scales


def prepack_weights(packed: torch.Tensor) -> torch.Tensor:
    """uint8 [N, K/2] packed int4 weights -> int8 [N, K] in the GEMM's own operand form (``sq_prepack_weights``).
    Pass the result wherever ``packed`` goes: ``gemm`` and ``linear`` tell the two forms apart by dtype."""
    _require_cuda(packed, "packed")
    if packed.dtype != torch.uint8 or packed.ndim != 2 or not packed.is_contiguous():
        raise ValueError("packed must be a contiguous uint8 [N, K/2] tensor.")
    n, half = packed.shape
    tiled = torch.empty((n, 2 * half), device=packed.device, dtype=torch.int8)
    with torch.cuda.device(packed.device):
        status = _lib.load_library().sq_prepack_weights(packed.data_ptr(), n, 2 * half, tiled.data_ptr(), _stream())
    _lib.check(status, "sq_prepack_weights")
    return tiled


def _wscale_mode(packed: torch.Tensor, w_scales: torch.Tensor) -> int:
    mode = _lib.WSCALE_GROUP_F16 if w_scales.dtype == torch.float16 else _lib.WSCALE_CHANNEL_F32
    return mode | (_lib.WEIGHTS_PREPACKED if packed.dtype == torch.int8 else 0)


def _mix_matrix(mix: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    if mix.ndim != 2 or mix.shape[0] != mix.shape[1] or mix.dtype != torch.float32 or mix.device != x.device:
        raise ValueError("mix must be a square fp32 matrix on the input's device.")
    return mix.contiguous()


def gemm(codes: torch.Tensor, packed: torch.Tensor, w_scales: torch.Tensor, row_scales: torch.Tensor, bias,
         *, out_dtype: torch.dtype, codes_layout: int = _lib.CODES_EVEN_ODD, want_accumulators: bool = False,
         check_kernel: bool = False, out: torch.Tensor | None = None, int4_range: bool = False,
         split: bool = True):
    """codes int8 [M, K] x packed uint8 [N, K/2] -> [M, N] in ``out_dtype``.
    ``w_scales`` fp32 [N] selects the per-channel form, fp16 [N, K/128] the group form.
    ``int4_range`` promises that every code lies in [-8, 7] (SQ_CODES_INT4_RANGE): faster group form.
    ``check_kernel`` runs the CUDA-core cross-check kernel instead of the tensor-core one (tests only).
    ``split`` lends the kernel scratch for tiles split along K (``sq_gemm_split``); without it only whole
    tiles are scheduled."""
    _require_cuda(codes, "codes")
    m, k = codes.shape
    n = packed.shape[0]
    group = w_scales.dtype == torch.float16
    if out is None:
        out = torch.empty((m, n), device=codes.device, dtype=out_dtype)
    acc = None
    if want_accumulators:
        acc = torch.empty((m, n, k // 128 if group else 1), device=codes.device, dtype=torch.int32)
    lib = _lib.load_library()
    layout = int(codes_layout) | (_lib.CODES_INT4_RANGE if int4_range else 0)
    with torch.cuda.device(codes.device):
        if check_kernel or not split:
            fn = lib.sq_gemm_check if check_kernel else lib.sq_gemm
            status = fn(codes.data_ptr(), layout, packed.data_ptr(), w_scales.data_ptr(),
                        _wscale_mode(packed, w_scales), row_scales.data_ptr(), _ptr(bias),
                        out.data_ptr(), _DTYPES[out_dtype], m, n, k, _ptr(acc), _stream())
        else:
            scratch = torch.empty((max(lib.sq_split_workspace_bytes(m), 16),), device=codes.device, dtype=torch.uint8)
            status = lib.sq_gemm_split(codes.data_ptr(), layout, packed.data_ptr(), w_scales.data_ptr(),
                                       _wscale_mode(packed, w_scales), row_scales.data_ptr(), _ptr(bias),
                                       out.data_ptr(), _DTYPES[out_dtype], m, n, k, _ptr(acc),
                                       scratch.data_ptr(), scratch.numel(), _stream())
    _lib.check(status, "sq_gemm_check" if check_kernel else "sq_gemm")
    return (out, acc) if want_accumulators else out


def gemm_scatter(codes: torch.Tensor, packed: torch.Tensor, w_scales: torch.Tensor, row_scales: torch.Tensor, bias,
                 out_pointers, out_ld: int, out_col0: int, *, out_dtype: torch.dtype, int4_range: bool = False):
    """Channel-split GEMM (``sq_gemm_scatter``): this GPU's [M, N] block is stored into columns
    ``[out_col0, out_col0 + N)`` of the row-major [M, out_ld] matrices at ``out_pointers`` - raw device addresses,
    the first one local, the others the same matrix on the other GPUs of the split (peer pointers)."""
    import ctypes
    _require_cuda(codes, "codes")
    m, k = codes.shape
    n = packed.shape[0]
    pointers = (ctypes.c_void_p * len(out_pointers))(*[int(ptr) for ptr in out_pointers])
    layout = int(_lib.CODES_EVEN_ODD) | (_lib.CODES_INT4_RANGE if int4_range else 0)
    with torch.cuda.device(codes.device):
        status = _lib.load_library().sq_gemm_scatter(
            codes.data_ptr(), layout, packed.data_ptr(), w_scales.data_ptr(), _wscale_mode(packed, w_scales),
            row_scales.data_ptr(), _ptr(bias), ctypes.cast(pointers, ctypes.c_void_p), len(out_pointers), int(out_ld),
            int(out_col0), _DTYPES[out_dtype], m, n, k, _stream())
    _lib.check(status, "sq_gemm_scatter")


def _rows_view(t: torch.Tensor, width: int, name: str):
    """(data pointer, row stride in elements, rows) of a tensor whose last axis is contiguous and whose leading
    axes collapse to evenly strided rows - e.g. the strided slice ``modulation[:, 0]`` of a [groups, 6, width] tensor."""
    if t.shape[-1] != width or t.stride(-1) != 1:
        raise ValueError(f"{name} must have a contiguous last axis of {width} elements.")
    flat = t.reshape(-1, width) if t.is_contiguous() else t
    if flat.ndim != 2:
        raise ValueError(f"{name} must be viewable as evenly strided rows.")
    return flat.data_ptr(), (flat.stride(0) if flat.shape[0] > 1 else width), flat.shape[0]


def linear(x: torch.Tensor, packed: torch.Tensor, w_scales: torch.Tensor, bias, *, abits: int, mode: str,
           inverse=None, signs=None, rht_block: int = 128, act_scales=None, gains=None, call: int = 0,
           span: int = 1, streams: int = 1, out: torch.Tensor | None = None,
           workspace: torch.Tensor | None = None, norm: str | None = None, norm_eps: float = 1e-6, norm_weight=None,
           mod_scale=None, mod_shift=None, round_after_norm: bool = False, activation: str | None = None,
           gate=None, residual=None, input_activation: str | None = None, mix=None,
           call_index: torch.Tensor | None = None) -> torch.Tensor:
    """One whole quantized linear (pre-pass + GEMM) through ``sq_linear_fused``.  ``out`` and ``workspace``
    (uint8, at least ``sq_workspace_bytes(rows, K)``) may be passed to reuse buffers across calls.

    Optional fused work: ``input_activation="gelu"`` applied to x first (rounded to x's dtype); ``norm`` ("layer" without affine, or "rms" with optional ``norm_weight``) and AdaLN
    modulation ``(1 + mod_scale) * y + mod_shift`` in front of the quantizer (one modulation row per equal
    share of the input rows), optionally rounded to x's dtype (``round_after_norm``); ``activation="gelu"``,
    ``gate`` (one row per equal share of the output rows) and ``residual`` behind the GEMM:
    ``out = residual + gate * act(linear(x))``.

    ``call_index`` (a CUDA int32 tensor of one element) makes static mode read its schedule entry from device
    memory when the kernel runs instead of taking ``call`` on the host: one captured graph then serves every
    denoise call."""
    _require_cuda(x, "x")
    x = x.contiguous()
    k = x.shape[-1]
    rows = x.numel() // k
    n = packed.shape[0]
    lib = _lib.load_library()
    nbytes = lib.sq_workspace_bytes(rows, k)
    if workspace is None:
        # room for the K-split scratch too (the kernel uses it when the tile count does not fill the SMs evenly)
        nbytes += lib.sq_split_workspace_bytes(rows)
        workspace = torch.empty((max(nbytes, 1),), device=x.device, dtype=torch.uint8)
    elif workspace.numel() < nbytes or workspace.dtype != torch.uint8 or not workspace.is_cuda:
        raise RuntimeError("workspace must be a CUDA uint8 tensor of at least sq_workspace_bytes(rows, K) bytes.")
    else:
        nbytes = workspace.numel()
    if out is None:
        out = torch.empty((*x.shape[:-1], n), device=x.device, dtype=x.dtype)
    elif out.shape != (*x.shape[:-1], n) or out.dtype != x.dtype or not out.is_contiguous():
        raise RuntimeError("out must be a contiguous tensor of shape x.shape[:-1] + (N,) in x's dtype.")
    group = w_scales.dtype == torch.float16
    calls = 0 if act_scales is None else act_scales.numel()
    if call_index is not None and (call_index.dtype != torch.int32 or call_index.numel() != 1
                                   or call_index.device != x.device):
        raise ValueError("call_index must be a one-element int32 tensor on the input's device.")
    if mix is not None:
        # composite rotation (order x power of two); a rotated site takes no block fusion (runtime.py:75-78)
        if (norm is not None or mod_scale is not None or gate is not None or residual is not None
                or activation is not None or input_activation is not None):
            raise ValueError("the composite rotation cannot be combined with fused block work.")
        mix = _mix_matrix(mix, x)
        with torch.cuda.device(x.device):
            status = lib.sq_linear_composite(
                x.data_ptr(), _DTYPES[x.dtype], rows, k, n, int(abits),
                _lib.ACT_TOKEN if mode == "token" else _lib.ACT_STATIC,
                _ptr(inverse), _ptr(signs), mix.data_ptr(), int(mix.shape[0]), _ptr(act_scales), _ptr(gains),
                int(calls), int(call), _ptr(call_index), int(span), int(streams), int(x.shape[-2]),
                packed.data_ptr(), w_scales.data_ptr(), _wscale_mode(packed, w_scales),
                _ptr(bias), out.data_ptr(), workspace.data_ptr(), nbytes, _stream())
        _lib.check(status, "sq_linear_composite")
        return out
    norm_kind = {None: _lib.NORM_NONE, "layer": _lib.NORM_LAYER, "rms": _lib.NORM_RMS}[norm]
    mod_ptr = shift_ptr = gate_ptr = None
    mod_span = gate_span = 1
    mod_stride = gate_stride = 0
    if mod_scale is not None:
        mod_ptr, mod_stride, mod_rows = _rows_view(mod_scale, k, "mod_scale")
        shift_ptr, shift_stride, shift_rows = _rows_view(mod_shift, k, "mod_shift")
        if shift_stride != mod_stride or shift_rows != mod_rows or rows % mod_rows:
            raise ValueError("AdaLN scale and shift must share a layout and cover complete input rows.")
        mod_span = rows // mod_rows
    if gate is not None:
        gate_ptr, gate_stride, gate_rows = _rows_view(gate, n, "gate")
        if rows % gate_rows:
            raise ValueError("Gate groups must cover complete output rows.")
        gate_span = rows // gate_rows
    if residual is not None:
        residual = residual.contiguous()
    with torch.cuda.device(x.device):
        status = lib.sq_linear_scheduled(
            x.data_ptr(), _DTYPES[x.dtype], rows, k, n, int(abits),
            _lib.ACT_TOKEN if mode == "token" else _lib.ACT_STATIC,
            _ptr(inverse), _ptr(signs), int(rht_block), _ptr(act_scales), _ptr(gains), int(calls), int(call),
            _ptr(call_index), int(span), int(streams), int(x.shape[-2]),
            packed.data_ptr(), w_scales.data_ptr(), _wscale_mode(packed, w_scales),
            _ptr(bias), _lib.ACT_FN_GELU if input_activation == "gelu" else _lib.ACT_FN_NONE, norm_kind, float(norm_eps), _ptr(norm_weight), mod_ptr, shift_ptr, int(mod_span),
            int(mod_stride), int(bool(round_after_norm)),
            _lib.ACT_FN_NONE, gate_ptr, int(gate_span), int(gate_stride),
            _ptr(residual), out.data_ptr(), workspace.data_ptr(), nbytes, _stream())
    _lib.check(status, "sq_linear_scheduled")
    if activation == "gelu":  # an output activation is not fused into the GEMM (it measured slower there)
        if gate is not None or residual is not None:
            raise ValueError("an output activation cannot be combined with a fused gate or residual.")
        out = torch.nn.functional.gelu(out)
    return out


# ---------------------------------------------------------------------------------------- operators of a block
# The smallest calls of these operators take 2 to 5 us on the device, so what the host does per call is their cost.  Each
# wrapper offers its call to the binding first (``csrc/sq_binding.cpp``), which launches it if it is an ordinary one and answers
# None if not; the Python below takes those - views to copy, outputs given, refusals - and everything where the binding is not
# built.  There properties are read once, arguments go to C packed by position, the stream is asked for by device index.
RUN = 128  # k that share a scale in the e4m3 product, and the rows of a weight block
_E4M3 = torch.float8_e4m3fn


def _no_gradient(*tensors) -> None:
    """The operators below are forward only.  An input that autograd tracks is refused - an e4m3 weight held as a parameter,
    a forward-mode tangent: its gradient would be lost without a word."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("the B200 operators have no backward pass: call them under torch.no_grad() or detach the inputs.")
    if forward_ad._current_level >= 0:  # a dual level is open; no_grad() does not stop tangents
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("the B200 operators have no forward-mode derivative: detach the inputs.")


class _Binding:
    """The binding's functions as attributes, looked up at the first call of any; ``enabled = False`` sends every call the
    Python way."""
    NAMES = ("fp8_gemm", "fp8_linear", "block_norm", "rotary")

    def __init__(self):
        for name in self.NAMES:
            setattr(self, name, self._first_call(name))

    def _first_call(self, name: str):
        def call(*args):
            self.enabled = True
            return getattr(self, name)(*args)
        return call

    @property
    def enabled(self) -> bool:
        return self.fp8_gemm is not self._decline

    @enabled.setter
    def enabled(self, on: bool) -> None:
        module = _lib.load_binding() if on else None
        for name in self.NAMES:
            setattr(self, name, self._decline if module is None else getattr(module, name))

    @staticmethod
    def _decline(*args) -> None:
        return None


_binding = _Binding()


def _call(name: str, device: torch.device, *args) -> None:
    """One C entry point on ``device`` and its current stream."""
    fn = getattr(_lib.load_library(), name)
    index = device.index
    if index == torch.cuda.current_device():
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status, name)


def _vectors(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous and 16-byte aligned (a copy where it is not): what the kernels read as vectors."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _require_rows(x: torch.Tensor, name: str = "x") -> None:
    if not x.is_cuda:
        _require_cuda(x, name)
    if x.dtype not in _DTYPES or x.ndim < 2:
        raise ValueError(f"{name} must be a bf16 or fp16 tensor with token and channel axes.")


def _round256(n: int) -> int:
    return (n + 255) & ~255


_ACTIVATIONS = {None: _lib.ACT_FN_NONE, "gelu": _lib.ACT_FN_GELU}


def _input_activation(name: str | None) -> int:
    if name not in _ACTIVATIONS:
        raise ValueError("input_activation must be None or 'gelu'.")
    return _ACTIVATIONS[name]


def _scales_for(rows: int, width: int, device) -> torch.Tensor:
    """fp32 [rows, runs] with the rows of a run next to each other, as the product reads them."""
    return torch.empty_strided((rows, -(-width // RUN)), (1, max(rows, 1)), dtype=torch.float32, device=device)


def fp8_quantize(x: torch.Tensor, *, input_activation: str | None = None):
    """``x`` [..., tokens, K] bf16/fp16 -> ``(codes, scales)``: float8_e4m3fn of x's shape and fp32 [rows, ceil(K / 128)],
    one scale per token and run of 128 channels (``max(amax / 448, 1e-8)``; codes are ``x * (1 / scale)`` rounded to
    nearest even).  ``input_activation="gelu"`` applies the erf GELU first, in fp32.  K must be a multiple of 16."""
    _require_rows(x)
    _no_gradient(x)
    activation = _input_activation(input_activation)
    k = x.shape[-1]
    if k == 0 or k % 16:
        raise ValueError("the channel axis must be a positive multiple of 16.")
    x = _vectors(x)
    device = x.device
    rows = x.numel() // k
    codes = torch.empty_like(x, dtype=_E4M3)
    scales = _scales_for(rows, k, device)
    _call("sq_fp8_quantize", device, x.data_ptr(), _DTYPES[x.dtype], rows, k, activation, codes.data_ptr(),
          scales.data_ptr(), 1, max(rows, 1))
    return codes, scales


def _check_fp8_weight(device, k: int, weight, weight_scales, bias, dtype) -> int:
    if weight.device != device or weight_scales.device != device or (bias is not None and bias.device != device):
        raise ValueError("weight, weight_scales and bias must be on the input's device.")
    if weight.dtype is not _E4M3 or weight.ndim != 2 or not weight.is_contiguous() or weight.data_ptr() % 16:
        raise ValueError("weight must be a contiguous, 16-byte aligned float8_e4m3fn [N, K] tensor.")
    n, width = weight.shape
    if width != k or k == 0 or k % 16 or n == 0 or n % 8:
        raise ValueError(f"Unsupported e4m3 linear shape: K={k} (a multiple of 16), N={n} (a multiple of 8), weight {(n, width)}.")
    if weight_scales.dtype is not torch.float32 or weight_scales.shape != (-(-n // RUN), -(-k // RUN)) or not weight_scales.is_contiguous():
        raise ValueError("weight_scales must be contiguous float32 [ceil(N / 128), ceil(K / 128)].")
    if bias is not None and (bias.dtype is not dtype or bias.shape != (n,) or not bias.is_contiguous()):
        raise ValueError("bias must be contiguous, [N], in the output's dtype.")
    return n


def _checked_output(out, shape, dtype, device) -> torch.Tensor:
    if out.shape != shape or out.dtype != dtype or out.device != device or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"out must be a contiguous, 16-byte aligned {dtype} tensor of shape {tuple(shape)} on the input's device.")
    return out


def fp8_gemm(codes: torch.Tensor, scales: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, bias=None, *,
             out_dtype: torch.dtype, out: torch.Tensor | None = None) -> torch.Tensor:
    """e4m3 codes [..., K] (with fp32 ``scales`` [rows, ceil(K / 128)], any strides) x e4m3 weight [N, K] (with fp32
    ``weight_scales`` [ceil(N / 128), ceil(K / 128)], one per 128 x 128 block) + bias -> [..., N] in ``out_dtype``.  Sums in
    fp32, one rounding.  ``quant.quantize_weight_block`` makes the weight's form, ``fp8_quantize`` the codes'.  ``out`` shares no
    memory with an input (refused)."""
    if out is None and (y := _binding.fp8_gemm(codes, scales, weight, weight_scales, bias, out_dtype)) is not None:
        return y
    if not codes.is_cuda:
        _require_cuda(codes, "codes")
    _no_gradient(codes, scales, weight, weight_scales, bias, out)
    if codes.dtype is not _E4M3 or codes.ndim < 2:
        raise ValueError("codes must be a float8_e4m3fn tensor with token and channel axes.")
    if out_dtype not in _DTYPES:
        raise ValueError("out_dtype must be torch.bfloat16 or torch.float16.")
    device = codes.device
    shape = codes.shape
    k = shape[-1]
    n = _check_fp8_weight(device, k, weight, weight_scales, bias, out_dtype)
    codes = _vectors(codes)
    rows = codes.numel() // k
    if scales.dtype is not torch.float32 or scales.device != device or scales.shape != (rows, -(-k // RUN)):
        raise ValueError("scales must be float32 [rows, ceil(K / 128)] on the codes' device.")
    out_shape = (*shape[:-1], n)
    out = codes.new_empty(out_shape, dtype=out_dtype) if out is None else _checked_output(out, out_shape, out_dtype, device)
    if rows:
        row_stride, run_stride = scales.stride()
        _call("sq_fp8_gemm", device, codes.data_ptr(), scales.data_ptr(), row_stride, run_stride, weight.data_ptr(),
              weight_scales.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), _DTYPES[out_dtype], rows, n, k)
    return out


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, bias=None, *,
               input_activation: str | None = None, out: torch.Tensor | None = None,
               workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``linear([gelu](x))`` in e4m3: ``fp8_quantize`` and ``fp8_gemm`` as one call, the product's set-up and first weight
    loads running under the quantizer.  ``workspace`` (uint8, at least ``sq_fp8_workspace_bytes(rows, K)``) may be passed
    to reuse a buffer across calls that are ordered on the device; ``out`` may be x's memory, but share none with the others."""
    if out is None and workspace is None and (y := _binding.fp8_linear(x, weight, weight_scales, bias, input_activation)) is not None:
        return y
    _require_rows(x)
    _no_gradient(x, weight, weight_scales, bias, out)
    activation = _input_activation(input_activation)
    device, shape, dtype = x.device, x.shape, x.dtype
    k = shape[-1]
    n = _check_fp8_weight(device, k, weight, weight_scales, bias, dtype)
    x = _vectors(x)
    rows = x.numel() // k
    nbytes = _round256(rows * k) + _round256(rows * -(-k // RUN) * 4)  # sq_fp8_workspace_bytes
    if workspace is None:
        workspace = x.new_empty((nbytes,), dtype=torch.uint8)
    elif (workspace.dtype != torch.uint8 or workspace.device != device or workspace.numel() < nbytes
          or not workspace.is_contiguous() or workspace.data_ptr() % 16):
        raise RuntimeError("workspace must be a contiguous, 16-byte aligned uint8 tensor on the input's device of at least "
                           "sq_fp8_workspace_bytes(rows, K) bytes.")
    out_shape = (*shape[:-1], n)
    out = x.new_empty(out_shape) if out is None else _checked_output(out, out_shape, dtype, device)
    if rows:
        _call("sq_fp8_linear", device, x.data_ptr(), _DTYPES[dtype], rows, k, n, activation, weight.data_ptr(),
              weight_scales.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), workspace.data_ptr(), nbytes)
    return out


_ABSENT = (0, 0, 0, 0, 0)


def _channel_param(t, kept: list, width: int, dtype, device, name: str):
    """Fields of an ``SqParam`` for a [width] vector in the rows' dtype or fp32."""
    if t is None:
        return _ABSENT
    f32 = t.dtype is torch.float32
    if t.device != device or not (f32 or t.dtype is dtype):
        raise ValueError(f"{name} must be on the input's device, in its dtype or float32.")
    if t.shape != (width,):
        raise ValueError(f"{name} must be [{width}].")
    pointer = t.data_ptr()
    if pointer % (32 if f32 else 16) or not t.is_contiguous():  # 8 parameters are one load
        t = t.clone(memory_format=torch.contiguous_format)
        kept.append(t)
        pointer = t.data_ptr()
    return (pointer, 0, 0, f32, 0)


def _row_param(t, kept: list, rows: int, width: int, dtype, device, name: str):
    """The same for rows of parameters, each for an equal share of the input rows."""
    if t is None:
        return _ABSENT
    f32 = t.dtype is torch.float32
    if t.device != device or not (f32 or t.dtype is dtype):
        raise ValueError(f"{name} must be on the input's device, in its dtype or float32.")
    if t.ndim < 1 or t.shape[-1] != width:
        raise ValueError(f"{name} must have a last axis of {width} elements.")
    if t.ndim != 2:
        t = t.reshape(-1, width)  # a view where the leading axes collapse to evenly spaced rows
        kept.append(t)
    groups = t.shape[0]
    if rows and (groups == 0 or rows % groups):
        raise ValueError(f"{name} rows must cover complete input rows: {groups} rows for {rows}.")
    stride, step = t.stride()
    pointer = t.data_ptr()
    if step != 1 or stride % 8 or pointer % (32 if f32 else 16):
        t = t.clone(memory_format=torch.contiguous_format)
        kept.append(t)
        pointer, stride = t.data_ptr(), width
    return (pointer, stride, rows // groups if rows else 1, f32, 0)


_NORMS = {None: _lib.NORM_NONE, "layer": _lib.NORM_LAYER, "rms": _lib.NORM_RMS}


def block_norm(x: torch.Tensor, branch: torch.Tensor | None = None, *, gate=None, residual_scale: float = 1.0,
               post_norm: str | None = None, post_weight=None, post_bias=None, norm: str | None = "rms", weight=None,
               bias=None, mod_scale=None, mod_shift=None, eps: float = 1e-6, quantize: bool = False,
               out: torch.Tensor | None = None):
    """The norms around a block in one pass over its rows, returned as ``(h, z)``::

        h = residual_scale * x + gate * (post_norm(branch) * post_weight + post_bias)
        z = (norm(h) * weight + bias) * (1 + mod_scale) + mod_shift

    ``x`` and ``branch`` are [..., width] bf16/fp16.  Without a ``branch`` h is x itself; with ``norm=None`` z is None.
    Norms are "rms" or "layer", their statistics in fp32 from the unrounded h, both with ``eps``.  Weights and biases are
    [width]; gate, mod_scale and mod_shift [..., width], each row for an equal share of x's rows (a strided slice of a
    modulation table is read in place), all in x's dtype or fp32.  ``quantize`` gives z as ``(codes, scales)`` for
    ``fp8_gemm`` (``fp8_quantize``'s rule, no rounding to x's dtype between).  ``out`` takes h; it may be x or branch itself,
    and shares no memory with an input otherwise (refused)."""
    if out is None and (pair := _binding.block_norm(x, branch, gate, residual_scale, post_norm, post_weight, post_bias, norm,
                                                         weight, bias, mod_scale, mod_shift, eps, quantize)) is not None:
        return pair
    _require_rows(x)
    _no_gradient(x, branch, gate, post_weight, post_bias, weight, bias, mod_scale, mod_shift, out)
    if norm not in _NORMS or post_norm not in _NORMS:
        raise ValueError("norm and post_norm must be None, 'rms' or 'layer'.")
    if branch is None and (norm is None or gate is not None or post_norm is not None or residual_scale != 1.0 or out is not None):
        raise ValueError("without a branch there is a norm alone: no gate, post_norm, residual_scale or out.")
    if norm is None and (quantize or any(t is not None for t in (weight, bias, mod_scale, mod_shift))):
        raise ValueError("without a norm there is nothing to weigh, modulate or quantize.")
    if post_norm is None and (post_weight is not None or post_bias is not None):
        raise ValueError("post_weight and post_bias belong to a post_norm.")
    device, shape, dtype = x.device, x.shape, x.dtype
    width = shape[-1]
    if width == 0 or width % (16 if quantize else 8) or width > 16384:
        raise ValueError("the channel axis must be a multiple of 8 (16 with quantize) up to 16384.")
    x_rows = _vectors(x)
    rows = x.numel() // width
    kept = []  # copies made for alignment live until the launch
    gate, mod_scale, mod_shift = (_row_param(t, kept, rows, width, dtype, device, name) for t, name in (
        (gate, "gate"), (mod_scale, "mod_scale"), (mod_shift, "mod_shift")))
    post_weight, post_bias, weight, bias = (_channel_param(t, kept, width, dtype, device, name) for t, name in (
        (post_weight, "post_weight"), (post_bias, "post_bias"), (weight, "weight"), (bias, "bias")))
    h, z = x, None
    branch_ptr = h_ptr = z_ptr = scales_ptr = 0
    if branch is not None:
        if branch.shape != shape or branch.dtype is not dtype or branch.device != device:
            raise ValueError("branch must match x's shape, dtype and device.")
        branch = _vectors(branch)
        if out is None:
            h = torch.empty_like(x_rows)
        else:
            h = _checked_output(out, shape, dtype, device)
        branch_ptr, h_ptr = branch.data_ptr(), h.data_ptr()
    if norm is not None:
        z = torch.empty_like(x_rows, dtype=_E4M3) if quantize else torch.empty_like(x_rows)
        z_ptr = z.data_ptr()
        if quantize:
            scales = _scales_for(rows, width, device)
            scales_ptr = scales.data_ptr()
            z = (z, scales)
    if rows:
        _call("sq_block_norm", device,
              _lib.BLOCK_NORM.pack(x_rows.data_ptr(), branch_ptr, *gate, *post_weight, *post_bias, *weight, *bias, *mod_scale,
                                   *mod_shift, h_ptr, z_ptr, scales_ptr, 1, rows, rows, width, residual_scale, eps,
                                   _DTYPES[dtype], _NORMS[post_norm], _NORMS[norm], 0))
    return h, z


_NO_SECTIONS = (0,) * _lib.ROTARY_AXES
_POSITIONS = {torch.int32: _lib.POS_INT32, torch.int64: _lib.POS_INT64, torch.float32: _lib.POS_FP32}
_ROTARY_LAYOUTS = {"interleaved": _lib.ROTARY_INTERLEAVED, "half": _lib.ROTARY_HALF}
_ROTARY_NORMS = {None: _lib.ROTARY_NORM_NONE, "head": _lib.ROTARY_NORM_HEAD, "token": _lib.ROTARY_NORM_TOKEN}


def _heads_strides(t: torch.Tensor):
    """Batch, token and head strides of [batch, tokens, heads, dim]; an axis of one index has none of its own and gets one
    on the vector grid."""
    (b, s, h, _), (batch, tokens, heads, dim) = t.stride(), t.shape
    if heads == 1:
        h = dim
    if batch == 1 and b % 8:
        b = 0
    if tokens == 1 and s % 8:
        s = b
    return b, s, h


def _heads_input(t: torch.Tensor):
    """(tensor, pointer, batch / token / head strides) with vectors the kernel can read in place, or a copy that has them."""
    b, s, h = _heads_strides(t)
    if t.stride(3) != 1 or (b | s | h) % 8 or t.data_ptr() % 16:
        t = _vectors(t)
        b, s, h = _heads_strides(t)
    return t, t.data_ptr(), (b, s, h)


def _heads_output(out, like, shape, dtype, device, name: str):
    if out is None:
        out = like.new_empty(shape)
        return out, out.data_ptr(), (shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3])
    fits = out.shape == shape and out.dtype is dtype and out.device == device and out.stride(3) == 1 and out.data_ptr() % 16 == 0
    strides = _heads_strides(out) if fits else None
    fits = fits and all(s % 8 == 0 and (s > 0 or n == 1) for s, n in zip(strides, shape))
    if not fits:
        raise ValueError(f"out for {name} must match it, with a contiguous last axis, strides that are multiples of 8 "
                         "elements and 16-byte alignment.")
    return out, out.data_ptr(), strides


def _rotary_weight(t, kept: list, count: int, dim: int, norm, dtype, device, name: str):
    if t is None:
        return 0, False
    if norm is None:
        raise ValueError("q_weight and k_weight belong to a norm.")
    f32 = t.dtype is torch.float32
    if t.device != device or not (f32 or t.dtype is dtype) or t.shape != ((count * dim,) if norm == "token" else (dim,)):
        raise ValueError(f"{name} must be [dim] (head norm) or [heads * dim] (token norm), in q's dtype or float32, on its device.")
    pointer = t.data_ptr()
    if pointer % (32 if f32 else 16) or not t.is_contiguous():  # 8 parameters are one load
        t = t.clone(memory_format=torch.contiguous_format)
        kept.append(t)
        pointer = t.data_ptr()
    return pointer, f32


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *, sections,
           layout: str = "interleaved", norm: str | None = None, q_weight=None, k_weight=None, eps: float = 1e-6, out=None):
    """Rotary positions on several axes, with the q/k norm in front: returns ``(q, k)`` rotated.

    ``q`` [batch, tokens, heads, dim] and ``k`` [batch, tokens, kv_heads, dim] (or None) bf16/fp16, strided views of a
    packed projection read in place.  Pair j of every head turns by ``positions[..., axis] * inv_freq[j]`` radians;
    ``sections`` are the pairs of each axis, in order (``rotary.rotary_frequencies`` makes inv_freq, float64 [pairs],
    ``rotary.grid_positions`` the positions of a clip).  ``positions`` is [tokens, axes] or [batch, tokens, axes], int32,
    int64 or float32, any value, however far or negative: angles are reduced in 64 bits (the rotation by
    ``-positions`` undoes it).  ``layout``: pairs are neighbours ("interleaved") or half the rotated length apart
    ("half"); elements past 2 * pairs pass through.  ``norm``: RMS of each head ("head", weights [dim]) or over all
    heads of a token ("token", weights [heads * dim]), statistics in fp32 (values up to 2^56, and from 2^-56 where eps is
    zero).  ``out`` is a pair (q, k) of tensors to write, strided as a cache or a transposed view may be; they may be the
    inputs themselves, and share no memory with an input, each other or themselves otherwise (refused)."""
    if out is None and (pair := _binding.rotary(q, k, positions, inv_freq, sections, layout, norm, q_weight, k_weight, eps)) is not None:
        return pair
    if not q.is_cuda:
        _require_cuda(q, "q")
    if q.ndim != 4 or q.dtype not in _DTYPES:
        raise ValueError("q must be a bf16 or fp16 tensor [batch, tokens, heads, dim].")
    out_q, out_k = out if out is not None else (None, None)
    _no_gradient(q, k, q_weight, k_weight, inv_freq, positions, out_q, out_k)
    device, shape, dtype = q.device, q.shape, q.dtype
    batch, tokens, heads, dim = shape
    kv_heads = 0
    if k is not None:
        k_shape = k.shape
        if k.ndim != 4 or k.dtype is not dtype or k.device != device or (k_shape[0], k_shape[1], k_shape[3]) != (batch, tokens, dim):
            raise ValueError("k must match q in dtype, device, batch, tokens and dim.")
        kv_heads = k_shape[2]
    elif k_weight is not None or out_k is not None:
        raise ValueError("there is no k to weigh or to write.")
    axes, pairs = len(sections), sum(sections)
    if not 1 <= axes <= _lib.ROTARY_AXES or min(sections) < 0 or pairs < 1 or 2 * pairs > dim:
        raise ValueError(f"sections must be the pairs of 1 to {_lib.ROTARY_AXES} axes, at most dim / 2 together.")
    lanes = 1 << (dim // 8 - 1).bit_length() if dim >= 8 else 0
    if dim % 8 or not 8 <= dim <= 256 or heads == 0 or (k is not None and kv_heads == 0) or (heads + kv_heads) * lanes > 4096:
        raise ValueError(f"Unsupported head shape: {heads} + {kv_heads} heads of {dim}.")
    if layout not in _ROTARY_LAYOUTS or norm not in _ROTARY_NORMS:
        raise ValueError("layout must be 'interleaved' or 'half', norm None, 'head' or 'token'.")
    if inv_freq.dtype is not torch.float64 or inv_freq.shape != (pairs,) or not inv_freq.is_contiguous() or inv_freq.device != device:
        raise ValueError("inv_freq must be contiguous float64 [pairs] on the input's device.")
    p_shape = positions.shape
    if (positions.dtype not in _POSITIONS or len(p_shape) not in (2, 3) or p_shape[-2:] != (tokens, axes)
            or (len(p_shape) == 3 and p_shape[0] not in (1, batch)) or positions.device != device):
        raise ValueError("positions must be int32, int64 or float32 [tokens, axes] or [batch, tokens, axes] on the input's device.")
    if positions.stride(-1) != 1:
        positions = positions.contiguous()
    p_strides = positions.stride()
    kept = []  # copies made for alignment live until the launch
    q_weight, q_f32 = _rotary_weight(q_weight, kept, heads, dim, norm, dtype, device, "q_weight")
    k_weight, k_f32 = _rotary_weight(k_weight, kept, kv_heads, dim, norm, dtype, device, "k_weight")
    q, q_ptr, q_strides = _heads_input(q)
    q_out, q_to, q_out_strides = _heads_output(out_q, q, shape, dtype, device, "q")
    k_out, k_ptr, k_to = None, 0, 0
    k_strides = k_out_strides = (0, 0, 0)
    if k is not None:
        k, k_ptr, k_strides = _heads_input(k)
        k_out, k_to, k_out_strides = _heads_output(out_k, k, k_shape, dtype, device, "k")
    if batch * tokens:
        _call("sq_rotary", device,
              _lib.ROTARY.pack(q_ptr, k_ptr, q_to, k_to, *q_strides, *k_strides, *q_out_strides, *k_out_strides, q_weight, k_weight,
                               positions.data_ptr(), p_strides[0] if len(p_shape) == 3 and p_shape[0] > 1 else 0, p_strides[-2],
                               inv_freq.data_ptr(), batch, tokens, heads, kv_heads, dim, axes, *sections, *_NO_SECTIONS[axes:],
                               _DTYPES[dtype], _ROTARY_LAYOUTS[layout], _ROTARY_NORMS[norm], _POSITIONS[positions.dtype],
                               q_f32, k_f32, eps, 0))
    return q_out, k_out


TIMELINE_ROLES = ("tma_issue", "unpack_start", "unpack_done", "acc_free", "mma_issue", "drain_start",
                  "acc_released", "drain_done", "mma_committed", "drain_top", "acc_loaded", "item_end")


def gemm_timeline(codes, packed, w_scales, row_scales, bias):
    """``gemm`` for the group-scale bf16 case plus the pipeline timeline of thread block 0: returns
    ``(out, stamps)`` with ``stamps`` an int64 [12, 512] tensor of SM clock values (0 = slot not reached);
    rows are named by ``TIMELINE_ROLES``."""
    _require_cuda(codes, "codes")
    m, k = codes.shape
    n = packed.shape[0]
    out = torch.empty((m, n), device=codes.device, dtype=torch.bfloat16)
    stamps = torch.zeros((len(TIMELINE_ROLES), 512), device=codes.device, dtype=torch.int64)
    with torch.cuda.device(codes.device):
        status = _lib.load_library().sq_gemm_timeline(codes.data_ptr(), packed.data_ptr(), w_scales.data_ptr(),
                                                      row_scales.data_ptr(), _ptr(bias), out.data_ptr(), m, n, k,
                                                      stamps.data_ptr(), _stream())
    _lib.check(status, "sq_gemm_timeline")
    return out, stamps


def mma_rate(n_cols: int = 128, iterations: int = 2000) -> float:
    """SM cycles the tensor pipe takes per ``kind::i8`` MMA of M = 128, N = ``n_cols``, K = 32 when one thread
    issues them back to back (``sq_mma_rate``; synchronises)."""
    cycles = torch.zeros(1, device="cuda", dtype=torch.int64)
    status = _lib.load_library().sq_mma_rate(int(n_cols), int(iterations), cycles.data_ptr(), _stream())
    _lib.check(status, "sq_mma_rate")
    torch.cuda.synchronize()
    return cycles.item() / (4.0 * iterations)


def wait_probe(limit_us: int = 1000) -> int:
    """Run ``sq_wait_probe``: a thread block waits ``limit_us`` microseconds for a barrier nobody arrives at and
    gives up.  Returns the nanoseconds it waited (synchronises); ``device_status()`` afterwards reports 9190 once."""
    waited = torch.zeros(1, device="cuda", dtype=torch.int64)
    _lib.check(_lib.load_library().sq_wait_probe(int(limit_us), waited.data_ptr(), _stream()), "sq_wait_probe")
    torch.cuda.synchronize()
    return int(waited.item())


def device_status() -> int:
    """Read and clear the device-side status word (synchronises)."""
    return int(_lib.load_library().sq_device_status())
