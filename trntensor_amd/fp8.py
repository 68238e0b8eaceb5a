"""The 8-bit chain of a language model's layer on fused HIP kernels: activations
and weights in 8-bit floats (e4m3) with a scale for each block of 128.

The reference has no counterpart. Products take both operands in 8 bits, at
the matrix units' full rate, and what runs between them writes rows in 8 bits::

    w_qkv = trntensor.Fp8Matrix(codes, scales)              # or Fp8Matrix.quantize(weights)

    h, x = trntensor.rms_norm(y, w_norm, residual=x, fp8=True)      # x += y, and its norm in 8 bits
    h = trntensor.fp8_gated_matmul(h, w_gate, w_up)                 # silu(h Wg^T) * (h Wu^T), in 8 bits
    y = trntensor.fp8_matmul(h, w_down)

All run on torch's current stream and never wait for the device. They have no
backward pass, and refuse tensors that ask for one. Activations are float32,
bfloat16 or float16; norms are held in 32 bits, and results rounded once, to the
activations' dtype or to 8 bits. Products of codes are summed in 32 bits for
results in float32; for results of 16 and 8 bits by the 8-bit matrix
instructions, which align eight products at a time to the largest and drop what
lies below 2^-13 of its power of two: about 2^-16 of a sum of random terms, and at
most 2^-10 of the largest product for each eight. Operands on the host are staged
to the others' device (the current one if all are), and results in the
activations' dtype go back to the first one's; rows in 8 bits stay on the device.
"""

from __future__ import annotations

import math
import struct

import torch

from . import serving
from .hip import _fastpath, _lib, dispatch
from .serving import FP8, _check_dtype, _check_grad, _CODES, _Fixed

E8M0 = torch.float8_e8m0fnu
BLOCK = 128

# The argument structs of include/trntensor_hip.h, eight bytes a field.
_QUANTIZE_ARGS = struct.Struct("=7q")
_NORM_ARGS = struct.Struct("=6qd7q")
_MATMUL_ARGS = struct.Struct("=10q")
_GATED_ARGS = struct.Struct("=17q")

_ACTIVATIONS = {"silu": 0, "gelu_tanh": 1}


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _home(what: str, *tensors) -> torch.device:
    """The device that a call runs on: its operands' one HIP device, or the current one."""
    device = None
    for t in tensors:
        if t is not None and t.device.type == "cuda":
            if device is not None and t.device != device:
                raise RuntimeError(f"{what} has operands on {device} and {t.device}")
            device = t.device
    return dispatch._device() if device is None else device


def _rows(t: torch.Tensor, device: torch.device) -> torch.Tensor:
    """`t` as (rows, elements) on the device, its elements of unit stride."""
    t = t.to(device).resolve_neg()
    t = t if t.dim() == 2 else t.reshape(math.prod(t.shape[:-1]), t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _shaped(t: torch.Tensor, shape, last: int) -> torch.Tensor:
    """Two-dimensional rows, of which `last` elements count, in their own shape."""
    if t.shape[1] != last:
        t = t.narrow(1, 0, last)
    return t.unflatten(0, shape[:-1]) if len(shape) > 1 else t[0]


class Fp8Rows(_Fixed):
    """Activations (..., features) in 8-bit floats, with one power of two for
    each row and block of 128 features: a value is its code times its scale.

    ``codes`` is float8_e4m3fn (..., features) and ``scales`` float8_e8m0fnu
    (..., ceil(features / 128)), both on one device; :func:`fp8_quantize`,
    :func:`rms_norm` and :func:`fp8_gated_matmul` make them. The constructor
    copies what a program holds, to the current HIP device if that is on the
    host. ``dtype`` (float32, bfloat16 or float16) is what products of the
    rows are given in.
    """

    __slots__ = ("shape", "dtype", "device", "_codes", "_scales")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
        if codes.dtype != FP8 or codes.dim() < 1 or codes.shape[-1] < 1:
            raise ValueError(f"codes must be float8_e4m3fn (..., features); got {codes.dtype} {tuple(codes.shape)}")
        want = (*codes.shape[:-1], _blocks(codes.shape[-1]))
        if scales.dtype != E8M0 or tuple(scales.shape) != want:
            raise ValueError(f"scales must be float8_e8m0fnu {want}; got {scales.dtype} {tuple(scales.shape)}")
        if dtype not in _CODES:
            raise NotImplementedError(f"dtype must be float32, bfloat16 or float16, not {dtype}")
        _check_grad("Fp8Rows", codes, scales)
        dispatch.require_hip()
        device = _home("Fp8Rows", codes, scales)
        self.shape = codes.shape
        self.dtype = dtype
        self.device = device
        self._codes, self._scales = _room(codes.shape, device, torch.zeros)
        features = codes.shape[-1]
        self._codes.view(torch.uint8)[:, :features] = codes.to(device).view(torch.uint8).reshape(-1, features)
        self._scales.view(torch.uint8)[:, : want[-1]] = scales.to(device).view(torch.uint8).reshape(-1, want[-1])

    @staticmethod
    def _of(shape, dtype, codes, scales) -> "Fp8Rows":
        rows = _new(Fp8Rows)
        _put_shape(rows, shape)
        _put_dtype(rows, dtype)
        _put_device(rows, codes.device)
        _put_codes(rows, codes)
        _put_scales(rows, scales)
        return rows

    def _check_memory(self):
        """Tensors that were resized or given other memory since are not what products would read."""
        count, blocks = math.prod(self.shape[:-1]), _blocks(self.shape[-1])
        for t, width in ((self._codes, blocks * BLOCK), (self._scales, -(-blocks // 4) * 4)):
            if (t.device != self.device or tuple(t.shape) != (count, width) or not t.is_contiguous()
                    or t.untyped_storage().nbytes() < t.storage_offset() + count * width):
                raise RuntimeError("the tensors of an Fp8Rows were given other memory: make another one of them")

    @property
    def codes(self) -> torch.Tensor:
        """float8_e4m3fn (..., features); rows start every multiple of 128 codes."""
        shape = self.shape
        n = shape[-1]
        return self._codes if len(shape) == 2 and n % BLOCK == 0 else _shaped(self._codes, shape, n)

    @property
    def scales(self) -> torch.Tensor:
        """float8_e8m0fnu (..., ceil(features / 128)); rows start every multiple of 4 scales."""
        shape = self.shape
        n = shape[-1]
        return self._scales if len(shape) == 2 and n % (4 * BLOCK) == 0 else _shaped(self._scales, shape, _blocks(n))

    def dequantize(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The rows' values, in ``dtype`` (the rows' one if None)."""
        scales = self.scales.float().repeat_interleave(BLOCK, dim=-1)[..., : self.shape[-1]]
        return (self.codes.float() * scales).to(self.dtype if dtype is None else dtype)

    def __repr__(self) -> str:
        return f"Fp8Rows({tuple(self.shape)}, dtype={self.dtype}, device={self.device})"


# What sets the attributes of rows that an operator has made (no check in between).
_new = Fp8Rows.__new__
_put_shape, _put_dtype, _put_device, _put_codes, _put_scales = (getattr(Fp8Rows, name).__set__ for name in Fp8Rows.__slots__)


def _room(shape, device: torch.device, make=torch.empty):
    """Codes and scales of rows of this shape as the kernels lay them out."""
    count, blocks = math.prod(shape[:-1]), _blocks(shape[-1])
    return (make((count, blocks * BLOCK), dtype=torch.uint8, device=device).view(FP8),
            make((count, -(-blocks // 4) * 4), dtype=torch.uint8, device=device).view(E8M0))


class Fp8Matrix(_Fixed):
    """A weight matrix (out_features, in_features) in 8-bit floats with a scale
    for each block of 128 x 128: ``W[n, k] = scales[n // 128, k // 128] * codes[n, k]``.

    ``codes`` is float8_e4m3fn (out_features, in_features) and ``scales``
    (ceil(out_features / 128), ceil(in_features / 128)), float32 or, where they
    are powers of two, float8_e8m0fnu, which the matrix units apply by themselves.

    The weights are laid out once, here, in copies on ``codes``' device (the
    current GPU if that is the host), codes in the tiles that the matrix units
    take. Operands that ask for a gradient are refused.
    """

    __slots__ = ("shape", "device", "scale_dtype", "_packed", "_scales", "_host")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype != FP8 or codes.dim() != 2 or codes.shape[1] < 1:
            raise ValueError(f"codes must be float8_e4m3fn (out_features, in_features); got {codes.dtype} {tuple(codes.shape)}")
        n, k = codes.shape
        want = (_blocks(n), _blocks(k))
        if scales.dtype not in (torch.float32, E8M0) or tuple(scales.shape) != want:
            raise ValueError(f"scales must be float32 or float8_e8m0fnu {want}; got {scales.dtype} {tuple(scales.shape)}")
        _check_grad("Fp8Matrix", codes, scales)
        dispatch.require_hip()
        device = _home("Fp8Matrix", codes, scales)
        codes = codes.to(device).contiguous()
        lib = _lib.load()
        self._packed = torch.empty(lib.tt_fp8_packed_bytes(n, k), dtype=torch.uint8, device=device)
        serving._launch("tt_fp8_pack", device, n, k, codes.data_ptr(), k, self._packed.data_ptr())
        if scales.dtype == torch.float32:
            self._scales = scales.detach().to(device, copy=True).contiguous()
        else:
            self._scales = torch.zeros((want[0], -(-want[1] // 4) * 4), dtype=torch.uint8, device=device)
            self._scales[:, : want[1]] = scales.to(device).view(torch.uint8)
        self.shape = (n, k)
        self.device = device
        self.scale_dtype = scales.dtype
        host = _fastpath.module()
        self._host = None if host is None else host.Fp8Host(_fastpath.serving_entries(), self._packed, self._scales, n, k,
                                                            scales.dtype == E8M0)

    @classmethod
    def quantize(cls, weights: torch.Tensor) -> "Fp8Matrix":
        """Weights (out_features, in_features) in float32, bfloat16 or float16,
        rounded to 8 bits: a block's scale is the smallest power of two, 2^-127
        at least, that brings its largest finite magnitude to 448 or below.
        Infinities become NaN, and NaN stays NaN."""
        if weights.dim() != 2 or weights.shape[1] < 1:
            raise ValueError(f"weights must be (out_features, in_features); got {tuple(weights.shape)}")
        _check_dtype("weights", weights)
        _check_grad("Fp8Matrix.quantize", weights)
        dispatch.require_hip()
        device = _home("Fp8Matrix.quantize", weights)
        n, k = weights.shape
        codes = torch.empty((n, k), dtype=FP8, device=device)
        scales = torch.empty((_blocks(n), _blocks(k)), dtype=torch.uint8, device=device)
        for i in range(_blocks(n)):  # 128 rows at a time: no 32-bit copy of it all
            part = weights[i * BLOCK: (i + 1) * BLOCK].to(device).float()
            rows = part.shape[0]
            part = torch.nn.functional.pad(part, (0, -k % BLOCK)).view(rows, -1, BLOCK)
            size = torch.where(part.isfinite(), part.abs(), 0.0).amax(dim=(0, 2))
            fraction, e = torch.frexp(size)
            e = torch.where(size > 0, e - 9 + (fraction > 0.875).int(), -127).clamp(min=-127)
            # 2^-e from its bits: powers that a GPU computes are a unit off for some exponents
            # (halfway weights would go to the odd code), and have the default dtype's range.
            inverse = (127 - e).bitwise_left_shift(23).view(torch.float32)
            part = torch.where(part.isfinite(), part * inverse[:, None], math.nan).to(FP8)
            codes[i * BLOCK: i * BLOCK + rows] = part.view(rows, -1)[:, :k]
            scales[i] = (e + 127).to(torch.uint8)
        return cls(codes, scales.view(E8M0))

    def __repr__(self) -> str:
        return f"Fp8Matrix({self.shape[0]}, {self.shape[1]}, scales {self.scale_dtype}, device={self.device})"


def fp8_quantize(x: torch.Tensor) -> Fp8Rows:
    """Rows (..., features) of float32, bfloat16 or float16 rounded to 8 bits.

    A block's scale is the smallest power of two, 2^-127 at least, that brings
    its largest finite magnitude to 448 or below; codes are rounded to nearest
    even. Infinities become NaN (the format has none), and NaN stays NaN. Rows
    need a unit stride and one row pitch, else they are copied.
    """
    host = _fastpath.rows_host()
    if host is not None and dispatch._use_hip() and isinstance(x, torch.Tensor):
        out = host.quantize(x)
        if out is not None:
            return Fp8Rows._of(x.shape, x.dtype, *out)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be (..., features); got {tuple(x.shape)}")
    code = _check_dtype("x", x)
    _check_grad("fp8_quantize", x)
    dispatch.require_hip()
    device = _home("fp8_quantize", x)
    x2 = _rows(x, device)
    codes, scales = _room(x.shape, device)
    serving._launch("tt_fp8_quantize", device, _QUANTIZE_ARGS.pack(
        code, x2.shape[0], x2.shape[1], x2.stride(0), x2.data_ptr(), codes.data_ptr(), scales.data_ptr()))
    return Fp8Rows._of(x.shape, x.dtype, codes, scales)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
             eps: float = 1e-6, fp8: bool = False):
    """Rows over their root mean square: ``h / sqrt(mean(h^2) + eps) * weight``,
    h being x or, with ``residual``, their sum.

    ``x`` is (..., features) in float32, bfloat16 or float16, ``residual`` alike,
    ``weight`` (features,) in any of the three (ones if None). Returns the norm
    in x's dtype or, with ``fp8``, as :class:`Fp8Rows`; with a residual, a pair
    of the norm and h in x's dtype. The norm follows from h before that
    rounding. Squares are summed in 32 bits, those of rows that would overflow or
    vanish there again with a power of two taken out: any magnitudes below 2^63 are
    taken, whatever the width. Larger ones may overflow, and the row's norm is zeros
    then. Rows need a unit stride and one row pitch, else they are copied.
    """
    host = _fastpath.rows_host()
    if host is not None and dispatch._use_hip() and isinstance(x, torch.Tensor):
        out = host.norm(x, weight, residual, eps, fp8)
        if out is not None:
            y = Fp8Rows._of(x.shape, x.dtype, out[0], out[1]) if fp8 else out[0]
            return y if residual is None else (y, out[2])
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be (..., features); got {tuple(x.shape)}")
    dim = x.shape[-1]
    code = _check_dtype("x", x)
    wcode = 0
    if weight is not None:
        if tuple(weight.shape) != (dim,):
            raise ValueError(f"weight must have shape ({dim},); got {tuple(weight.shape)}")
        wcode = _check_dtype("weight", weight)
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must be {x.dtype} {tuple(x.shape)}; got {residual.dtype} {tuple(residual.shape)}")
    if not 0.0 <= eps < 1e38:
        raise ValueError(f"eps must be finite and not negative; got {eps}")
    _check_grad("rms_norm", x, weight, residual)
    dispatch.require_hip()
    device = _home("rms_norm", x, weight, residual)
    x2 = _rows(x, device)
    r2 = total = None
    if residual is not None:
        r2 = _rows(residual, device)
        total = torch.empty(x.shape, dtype=x.dtype, device=device)
    if weight is not None:
        weight = weight.to(device).resolve_neg().contiguous()
    y = codes = scales = None
    if fp8:
        codes, scales = _room(x.shape, device)
    else:
        y = torch.empty(x.shape, dtype=x.dtype, device=device)
    serving._launch("tt_rms_norm", device, _NORM_ARGS.pack(
        code, wcode, x2.shape[0], dim, x2.stride(0), 0 if r2 is None else r2.stride(0), eps, x2.data_ptr(), *map(_ptr, (r2, weight)),
        *map(_ptr, (total, y, codes, scales))))
    y = Fp8Rows._of(x.shape, x.dtype, codes, scales) if fp8 else y.to(x.device)
    return y if residual is None else (y, total.to(x.device))


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _operand(what: str, x, w: Fp8Matrix) -> Fp8Rows:
    """`x` as rows in 8 bits on the weights' device."""
    if not isinstance(x, Fp8Rows):
        if x.dim() < 1 or x.shape[-1] != w.shape[1]:
            raise ValueError(f"x must be (..., {w.shape[1]}); got {tuple(x.shape)}")
        if x.device.type == "cuda" and x.device != w.device:
            raise RuntimeError(f"x is on {x.device}, the weights on {w.device}")
        _check_dtype("x", x)
        _check_grad(what, x)
        dispatch.require_hip()
        x = fp8_quantize(x.to(w.device))
    if x.shape[-1] != w.shape[1]:
        raise ValueError(f"x must be (..., {w.shape[1]}); got {tuple(x.shape)}")
    if x.device != w.device:
        raise RuntimeError(f"x is on {x.device}, the weights on {w.device}")
    x._check_memory()
    return x


def _scale_code(w: Fp8Matrix) -> int:
    return _lib.TT_F32 if w.scale_dtype == torch.float32 else _lib.TT_E8M0


def fp8_matmul(x: Fp8Rows | torch.Tensor, w: Fp8Matrix, *, dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ W.T`` for rows and weights in 8 bits: (..., in_features) to (..., out_features).

    ``x`` is :class:`Fp8Rows`, or a tensor that is quantized first, as by
    :func:`fp8_quantize`. The result is rounded once to ``dtype`` (that of x if
    None); how products are summed follows from that dtype, as at the top of this
    module: in 32 bits for float32. With float32 scales a block of 128 is summed,
    times its row's scale, before its weights' scale multiplies it. Sums that pass
    float32's range on the way are infinite. A row's scale times a weight's has to
    be a float32 (2^-126 to 2^127) for float32 results. NaN in a row gives NaN in the
    row's result, and so do its block's codes under a scale of NaN (byte 255).
    """
    if w._host is not None and isinstance(x, Fp8Rows) and dispatch._use_hip():
        y = w._host.run(x._codes, x._scales, x.shape, x.dtype if dtype is None else dtype)
        if y is not None:
            return y
    home = None if isinstance(x, Fp8Rows) else x.device
    x = _operand("fp8_matmul", x, w)
    code = _CODES.get(x.dtype if dtype is None else dtype)
    if code is None:
        raise NotImplementedError(f"dtype must be float32, bfloat16 or float16, not {dtype}")
    dispatch.require_hip()
    n, k = w.shape
    y = torch.empty((*x.shape[:-1], n), dtype=x.dtype if dtype is None else dtype, device=w.device)
    serving._launch("tt_fp8_matmul", w.device, _MATMUL_ARGS.pack(
        code, _scale_code(w), x._codes.shape[0], n, k, x._codes.data_ptr(), x._scales.data_ptr(), w._packed.data_ptr(),
        w._scales.data_ptr(), y.data_ptr()))
    return y if home is None or home == w.device else y.to(home)


def fp8_gated_matmul(x: Fp8Rows | torch.Tensor, gate: Fp8Matrix, up: Fp8Matrix, *, activation: str = "silu",
                     fp8: bool = True) -> Fp8Rows | torch.Tensor:
    """``act(x @ gate.T) * (x @ up.T)``, the first half of a gated feed-forward block.

    ``x`` is as :func:`fp8_matmul` takes it; ``gate`` and ``up`` are weights of
    one shape, with scales of one dtype. ``activation`` is "silu", a / (1 + exp(-a)), or
    "gelu_tanh", a (1 + tanh(sqrt(2 / pi) (a + 0.044715 a^3))) / 2; what is below 10^-36 of
    it counts as 0. The result is rounded once: to 8 bits as :func:`fp8_quantize` does, or
    without ``fp8`` to x's dtype; sums are as in :func:`fp8_matmul`. A block's scale follows
    sums in 32 bits where the other ones leave it open, within 2^-12 of a power of two's
    border (unless many values share it). Returns :class:`Fp8Rows` or a tensor (...,
    out_features).
    """
    if gate.shape != up.shape or gate.scale_dtype != up.scale_dtype:
        raise ValueError(f"gate and up must be alike; got {gate} and {up}")
    if gate.device != up.device:
        raise RuntimeError(f"gate is on {gate.device}, up on {up.device}")
    kind = _ACTIVATIONS.get(activation)
    if kind is None:
        raise ValueError(f"activation must be one of {tuple(_ACTIVATIONS)}; got {activation!r}")
    if gate._host is not None and up._host is not None and isinstance(x, Fp8Rows) and dispatch._use_hip():
        out = gate._host.gated(up._host, x._codes, x._scales, x.shape, x.dtype, kind, fp8)
        if out is not None:
            return Fp8Rows._of(torch.Size((*x.shape[:-1], gate.shape[0])), x.dtype, *out) if fp8 else out[0]
    home = None if isinstance(x, Fp8Rows) else x.device
    x = _operand("fp8_gated_matmul", x, gate)
    dispatch.require_hip()
    n, k = gate.shape
    device = gate.device
    shape = torch.Size((*x.shape[:-1], n))
    y = codes = scales = None
    if fp8:
        codes, scales = _room(shape, device)
    else:
        y = torch.empty(shape, dtype=x.dtype, device=device)
    head = (_CODES[x.dtype], _scale_code(gate), kind, x._codes.shape[0], n, k, x._codes.data_ptr(), x._scales.data_ptr(),
            gate._packed.data_ptr(), gate._scales.data_ptr(), up._packed.data_ptr(), up._scales.data_ptr(),
            *map(_ptr, (y, codes, scales)))
    need = _lib.load().tt_fp8_gated_workspace_bytes(_GATED_ARGS.pack(*head, 0, 0)) if fp8 else 0
    room = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    serving._launch("tt_fp8_gated_matmul", device, _GATED_ARGS.pack(*head, _ptr(room), need))
    if fp8:
        return Fp8Rows._of(shape, x.dtype, codes, scales)
    return y if home is None or home == device else y.to(home)
