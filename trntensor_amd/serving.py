"""Serving operators of language models on fused HIP kernels: products with
4-bit weights, appending to a paged cache of 8-bit keys and values, and
attention over that cache.

The reference has no counterpart. One decode step of a layer is a chain of
contractions around a cache, and these are its links::

    w_qkv = trntensor.Q4Matrix(codes, scales, hidden, 128, zeros=zeros)
    cache = trntensor.KVCache.empty(pages, kv_heads, head_dim)

    q, k, v = trntensor.q4_matmul(x, w_qkv).view(B, T, -1, D).split([HQ, H, H], dim=2)
    q = trntensor.kv_append(cache, k, v, table, held, q=q, cos=cos, sin=sin)
    o = trntensor.kv_attention(q, cache, table, held + T)
    y = trntensor.q4_matmul(o.flatten(2), w_out)

All three run on torch's current stream and never wait for the device: how
many tokens each sequence holds, and in which pages, is read there. They have
no backward pass, and refuse tensors that ask for one. Activations are
float32, bfloat16 or float16; sums, softmax statistics and rotations are held
in 32 bits, and results rounded once to the activations' dtype. Two steps
before that round too: attention's weights enter the product with the values
in 8 bits for bfloat16, 16 for float16 and 24 for float32, and 4-bit products
keep about 22 of the 24 bits. Operands on the host are staged to the weights'
or cache's device, and the result goes back to the first one's.
"""

from __future__ import annotations

import math
import struct

import torch
from torch.autograd import forward_ad

from .hip import _fastpath, _lib, dispatch, engine

_CODES = {torch.float32: _lib.TT_F32, torch.bfloat16: _lib.TT_BF16, torch.float16: _lib.TT_F16}
FP8 = torch.float8_e4m3fn

# The argument structs of include/trntensor_hip.h, eight bytes a field.
_Q4_ARGS = struct.Struct("=13q")
_CACHE = struct.Struct("=8q")
_APPEND_ARGS = struct.Struct("=26q")
_ATTENTION_ARGS = struct.Struct("=11qd5q")
_WORKSPACE = struct.Struct("=2q")


def _check_dtype(what: str, t: torch.Tensor) -> int:
    code = _CODES.get(t.dtype)
    if code is None:
        raise NotImplementedError(f"{what} must be float32, bfloat16 or float16, not {t.dtype}")
    return code


def _check_grad(what: str, *tensors) -> None:
    for t in tensors:
        if t is None:
            continue
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad() or detach its operands")
        if torch._C._is_fwd_grad_enabled() and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} has no forward-mode derivative: take its operands' primals")


def _launch(name: str, device: torch.device, *args) -> None:
    """One library call on torch's current stream of `device`."""
    fn = getattr(_lib.load(), name)
    if device.index == torch.cuda.current_device():
        st = fn(*args, engine._stream_ptr(device))
    else:
        with torch.cuda.device(device):
            st = fn(*args, engine._stream_ptr(device))
    if st:
        _lib.check(st, name)


class _Fixed:
    """Attributes are set once: calls go by the memory and sizes found at construction."""

    __slots__ = ()

    def __setattr__(self, name, value):
        if not name.startswith("_") and hasattr(self, name):
            raise AttributeError(f"{type(self).__name__}.{name} is fixed at construction: make another {type(self).__name__}")
        object.__setattr__(self, name, value)

    def _check_memory(self):
        """Tensors given other memory since (``t.data = ...``, a resized storage) are not what calls would work on."""
        if self._memory != tuple(0 if t is None else t.data_ptr() for t in self._tensors()):
            raise RuntimeError(f"the tensors of a {type(self).__name__} were given other memory: make another one of them")


# ---------------------------------------------------------------------------
# 4-bit weights
# ---------------------------------------------------------------------------
class Q4Matrix(_Fixed):
    """A weight matrix (out_features, in_features) held in 4 bits:
    ``W[n, k] = scales[n, k // group_size] * (code[n, k] - zeros[n, k // group_size])``.

    ``codes`` is uint8 (out_features, ceil(in_features / 2)): byte j of a row
    holds column 2j in its low half and column 2j + 1 in its high half.
    ``scales`` and ``zeros`` are (out_features, ceil(in_features /
    group_size)) in one of float32, bfloat16, float16; without ``zeros`` every
    zero point is 8. ``group_size`` is 32, 64 or a multiple of 128.

    The weights are laid out once, here, in copies on ``codes``' device (the
    current GPU if that is the host): codes in the tiles that the matrix units
    take, scales with the output features contiguous. Scales and zero points
    that ask for a gradient are refused.
    """

    __slots__ = ("packed", "scales", "zeros", "shape", "group_size", "device", "_code", "_host", "_memory")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, in_features: int, group_size: int,
                 zeros: torch.Tensor | None = None):
        if codes.dtype != torch.uint8 or codes.dim() != 2:
            raise ValueError(f"codes must be uint8 (out_features, in_features / 2); got {codes.dtype} {tuple(codes.shape)}")
        n, k = codes.shape[0], int(in_features)
        if k < 1 or codes.shape[1] != (k + 1) // 2:
            raise ValueError(f"codes of {k} columns must be {(k + 1) // 2} bytes wide; got {codes.shape[1]}")
        if group_size not in (32, 64) and (group_size < 128 or group_size % 128):
            raise ValueError(f"group_size must be 32, 64 or a multiple of 128; got {group_size}")
        groups = -(-k // group_size)
        self._code = _check_dtype("scales", scales)
        for name, t in (("scales", scales), ("zeros", zeros)):
            if t is not None and (tuple(t.shape) != (n, groups) or t.dtype != scales.dtype):
                raise ValueError(f"{name} must be {scales.dtype} ({n}, {groups}); got {t.dtype} {tuple(t.shape)}")
        _check_grad("Q4Matrix", scales, zeros)
        dispatch.require_hip()
        device = codes.device if codes.device.type == "cuda" else dispatch._device()
        codes = codes.to(device).contiguous()
        lib = _lib.load()
        self.packed = torch.empty(lib.tt_q4_packed_bytes(n, k), dtype=torch.uint8, device=device)
        _launch("tt_q4_pack", device, n, k, codes.data_ptr(), codes.shape[1], self.packed.data_ptr())
        self.scales, self.zeros = (None if t is None else self._by_group(t.detach().to(device)) for t in (scales, zeros))
        self.shape = (n, k)
        self.group_size = int(group_size)
        self.device = device
        self._memory = tuple(0 if t is None else t.data_ptr() for t in self._tensors())
        host = _fastpath.module()
        self._host = None if host is None else host.Q4Host(_fastpath.serving_entries(), self.packed, self.scales, self.zeros,
                                                           n, k, self.group_size, self._code)

    def _tensors(self):
        return self.packed, self.scales, self.zeros

    @staticmethod
    def _by_group(t: torch.Tensor) -> torch.Tensor:
        """(out_features, groups) as (groups, out_features rounded up to a multiple of 16)."""
        out = torch.zeros((t.shape[1], -(-t.shape[0] // 16) * 16), dtype=t.dtype, device=t.device)
        out[:, : t.shape[0]] = t.t()
        return out

    def __repr__(self) -> str:
        return f"Q4Matrix({self.shape[0]}, {self.shape[1]}, group_size={self.group_size}, device={self.device})"


def q4_matmul(x: torch.Tensor, w: Q4Matrix) -> torch.Tensor:
    """``x @ W.T`` for weights in 4 bits: (..., in_features) to (..., out_features).

    Codes are widened in registers on their way into the matrix units, so the
    weights cross memory at half a byte each; products are summed in 32 bits
    and the result is rounded once to x's dtype. Summed are x times 1 + code /
    16, and the share of the offset is taken off, which costs about two of the
    24 bits: codes that equal their zero point give 2^-22 of sum |x| s 16, not
    always 0. Rows of x need a unit stride and one row pitch, else they are
    copied. A row of x that holds an infinity gives infinities or NaN, one that
    holds NaN gives NaN; sums of x beyond float32's range overflow however small
    the scales, and so do scales of 2^124 and more.
    """
    if w._host is not None and dispatch._use_hip() and isinstance(x, torch.Tensor):
        y = w._host.run(x)
        if y is not None:
            return y
    n, k = w.shape
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"x must be (..., {k}); got {tuple(x.shape)}")
    code = _check_dtype("x", x)
    _check_grad("q4_matmul", x)
    dispatch.require_hip()
    home = x.device
    if home != w.device:
        if home.type == "cuda":
            raise RuntimeError(f"x is on {home}, the weights on {w.device}")
        x = x.to(w.device)
    x2 = x if x.dim() == 2 else x.reshape(-1, k)
    m = x2.shape[0]
    if (x2.stride(1) != 1 and k > 1) or (m > 1 and x2.stride(0) < k):
        x2 = x2.contiguous()
    y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=w.device)
    zeros = w.zeros
    w._check_memory()
    _launch("tt_q4_matmul", w.device, _Q4_ARGS.pack(
        code, w._code, m, n, k, w.group_size, max(x2.stride(0), k), n, x2.data_ptr(), w.packed.data_ptr(),
        w.scales.data_ptr(), 0 if zeros is None else zeros.data_ptr(), y.data_ptr()))
    return y if home == w.device else y.to(home)


# ---------------------------------------------------------------------------
# the paged cache
# ---------------------------------------------------------------------------
class KVCache(_Fixed):
    """Pages of keys and values in 8-bit floats (e4m3), with one power-of-two
    scale for each page and head: a value is its code times its page's scale.

    ``k`` is (pages, heads, page_size, width) and ``v`` (pages, heads, width,
    page_size), both ``torch.float8_e4m3fn`` with width = head_dim rounded up
    to a multiple of 64 (keys' codes past head_dim are zeros); ``k_scale`` and
    ``v_scale`` are float32 (pages, heads), 2^-64 to 2^120. page_size is a multiple of 16,
    head_dim at most 256. The constructor takes tensors a program holds;
    :meth:`empty` makes a cache. Its attributes are fixed, what the tensors
    hold is not. Which pages are whose is the program's business: calls take a
    page table.
    """

    __slots__ = ("k", "v", "k_scale", "v_scale", "head_dim", "page_size", "num_pages", "num_heads", "device", "_packed",
                 "_scale", "_host", "_memory")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, head_dim: int):
        if k.dim() != 4:
            raise ValueError(f"k must be 4D (pages, heads, page_size, width); got shape {tuple(k.shape)}")
        pages, heads, page, width = k.shape
        if head_dim < 1 or head_dim > 256:
            raise NotImplementedError(f"head_dim {head_dim} (1 to 256)")
        if width != -(-head_dim // 64) * 64:
            raise ValueError(f"k's rows hold head_dim {head_dim} rounded up to a multiple of 64; got {width}")
        if page < 16 or page % 16 or page > 65536:
            raise ValueError(f"page_size must be a multiple of 16, at most 65536; got {page}")
        if heads < 1:
            raise ValueError("a cache has at least one head")
        for name, t, shape, dtype in (("k", k, (pages, heads, page, width), FP8), ("v", v, (pages, heads, width, page), FP8),
                                      ("k_scale", k_scale, (pages, heads), torch.float32),
                                      ("v_scale", v_scale, (pages, heads), torch.float32)):
            if tuple(t.shape) != shape or t.dtype != dtype:
                raise ValueError(f"{name} must be {dtype} {shape}; got {t.dtype} {tuple(t.shape)}")
            if t.device.type != "cuda" or t.device != k.device:
                raise RuntimeError(f"a cache's tensors are on one HIP device; {name} is on {t.device}")
            if not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name} must be contiguous and 16-byte aligned")
        _check_grad("KVCache", k, v, k_scale, v_scale)
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            mantissa, exponent = torch.frexp(t)
            if not ((mantissa == 0.5) & (exponent > -64) & (exponent <= 121)).all():
                raise ValueError(f"{name} must be powers of two from 2^-64 to 2^120, those that kv_append takes")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.head_dim, self.page_size, self.num_pages, self.num_heads = int(head_dim), page, pages, heads
        self.device = k.device
        self._scale = 1.0 / math.sqrt(self.head_dim)
        self._memory = tuple(t.data_ptr() for t in self._tensors())
        self._packed = _CACHE.pack(*self._memory, pages, heads, page, self.head_dim)
        host = _fastpath.module()
        self._host = None if host is None else host.CacheHost(_fastpath.serving_entries(), k, v, k_scale, v_scale,
                                                              self.head_dim)

    def _tensors(self):
        return self.k, self.v, self.k_scale, self.v_scale

    @classmethod
    def empty(cls, num_pages: int, num_heads: int, head_dim: int, page_size: int = 64,
              device: torch.device | None = None) -> "KVCache":
        """A cache of zeros on `device` (the current HIP device if None)."""
        dispatch.require_hip()
        device = dispatch._device() if device is None else torch.device(device)
        width = -(-head_dim // 64) * 64
        k = torch.zeros((num_pages, num_heads, page_size, width), dtype=torch.uint8, device=device).view(FP8)
        v = torch.zeros((num_pages, num_heads, width, page_size), dtype=torch.uint8, device=device).view(FP8)
        scale = torch.ones((2, num_pages, num_heads), dtype=torch.float32, device=device)
        return cls(k, v, scale[0].clone(), scale[1].clone(), head_dim)

    @property
    def nbytes(self) -> int:
        """Bytes of its codes and scales."""
        return 2 * (self.k.numel() + 4 * self.k_scale.numel())

    def __repr__(self) -> str:
        return (f"KVCache({self.num_pages} pages of {self.page_size} tokens, {self.num_heads} heads of {self.head_dim}, "
                f"device={self.device})")


def _place(cache: KVCache, t: torch.Tensor, what: str) -> torch.Tensor:
    if t.device == cache.device:
        return t
    if t.device.type == "cuda":
        raise RuntimeError(f"{what} is on {t.device}, the cache on {cache.device}")
    return t.to(cache.device)


def _rows(cache: KVCache, t: torch.Tensor, what: str, batch: int, tokens: int, heads: int | None) -> torch.Tensor:
    """`t` as (batch, tokens, heads, head_dim) on the cache's device, its last dim of unit stride."""
    s = t.shape
    if len(s) != 4 or s[0] != batch or s[1] != tokens or s[3] != cache.head_dim or (heads is not None and s[2] != heads):
        want = f"({batch}, {tokens}, {'heads' if heads is None else heads}, {cache.head_dim})"
        raise ValueError(f"{what} must have shape {want}; got {tuple(s)}")
    if t.device != cache.device:
        t = _place(cache, t, what)
    return t if t.stride(3) == 1 or s[3] == 1 else t.contiguous()


def _schedule(cache: KVCache, batch: int, table, lengths, counts):
    """The page table, lengths and counts as the kernels read them: int32 on the cache's device."""
    if table.dim() != 2 or table.shape[0] != batch:
        raise ValueError(f"page_table must have shape ({batch}, pages a sequence); got {tuple(table.shape)}")
    for name, t in (("page_table", table), ("lengths", lengths), ("counts", counts)):
        if t is None:
            continue
        if t.dtype != torch.int32:
            raise ValueError(f"{name} must be int32; got {t.dtype}")
        if t is not table and tuple(t.shape) != (batch,):
            raise ValueError(f"{name} must have shape ({batch},); got {tuple(t.shape)}")
    dev = cache.device
    if table.device != dev:
        table = _place(cache, table, "page_table")
    if table.stride(1) != 1 and table.shape[1] > 1:
        table = table.contiguous()
    if lengths.device != dev:
        lengths = _place(cache, lengths, "lengths")
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    if counts is not None:
        if counts.device != dev:
            counts = _place(cache, counts, "counts")
        if not counts.is_contiguous():
            counts = counts.contiguous()
    return table, lengths, counts


def kv_append(cache: KVCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, *,
              counts: torch.Tensor | None = None, q: torch.Tensor | None = None, cos: torch.Tensor | None = None,
              sin: torch.Tensor | None = None, interleaved: bool = False) -> torch.Tensor | None:
    """Append keys and values to a paged cache, rotating keys (and queries) by position.

    ``k`` and ``v`` are (batch, tokens, heads, head_dim), any strides with the
    last dim contiguous; sequence b's first ``counts[b]`` tokens (all, without
    counts) go behind the ``lengths[b]`` it holds. ``page_table`` (batch,
    pages a sequence) names the page of each run of page_size tokens. Table,
    lengths and counts are int32. The caller adds the counts to its lengths.

    With ``cos`` and ``sin`` (float32, (positions, r / 2), positions no fewer
    than the table covers) the first r elements of every key, and of ``q``
    (batch, tokens, q_heads, head_dim) if given, are rotated in pairs: element
    i with i + r / 2, or neighbours if ``interleaved``. Returns the rotated
    queries (zeros in rows past a sequence's count), or None without q.

    A page's scale follows its largest magnitude: it is the power of two that
    just brings it into the format's range, and when a later token needs a
    larger one the page's earlier codes are rounded to it, which loses only
    bits below the format's smallest step at the new scale. Magnitudes too
    large for any scale (infinities) saturate; NaN stays NaN. Tokens past the
    table's end, or whose page number is none of the cache's, are dropped. A
    page that is written to must belong to one sequence.
    """
    if cache._host is not None and dispatch._use_hip():
        done, out = cache._host.append(k, v, page_table, lengths, counts, q, cos, sin, interleaved)
        if done:
            return out
    if k.dim() != 4:
        raise ValueError(f"k must be 4D (batch, tokens, heads, head_dim); got shape {tuple(k.shape)}")
    batch, tokens = k.shape[0], k.shape[1]
    code = _check_dtype("k", k)
    k = _rows(cache, k, "k", batch, tokens, cache.num_heads)
    home = None
    if v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
        raise RuntimeError("k, v and q must share one dtype")
    v = _rows(cache, v, "v", batch, tokens, cache.num_heads)
    _check_grad("kv_append", k, v, q, cos, sin)
    dispatch.require_hip()
    table, lengths, counts = _schedule(cache, batch, page_table, lengths, counts)
    rot = 0
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is not None:
        if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
            raise ValueError(f"cos and sin must be float32 (positions, pairs) alike; got {cos.dtype} {tuple(cos.shape)}, "
                             f"{sin.dtype} {tuple(sin.shape)}")
        rot = 2 * cos.shape[1]
        if rot < 2 or rot > cache.head_dim:
            raise ValueError(f"{cos.shape[1]} pairs do not fit head_dim {cache.head_dim}")
        if cos.shape[0] < table.shape[1] * cache.page_size:
            raise ValueError(f"cos and sin cover {cos.shape[0]} positions, the page table {table.shape[1] * cache.page_size}")
        cos, sin = _place(cache, cos, "cos").contiguous(), _place(cache, sin, "sin").contiguous()
    out, heads = None, 0
    if q is not None:
        if cos is None:
            raise ValueError("q is taken to be rotated: it needs cos and sin")
        home = q.device
        q = _rows(cache, q, "q", batch, tokens, None)
        heads = q.shape[2]
        out = torch.empty((batch, tokens, heads, cache.head_dim), dtype=q.dtype, device=cache.device)
    sk, sv, sq = k.stride(), v.stride(), k.stride() if q is None else q.stride()
    if batch and tokens:
        cache._check_memory()
        _launch("tt_kv_append", cache.device, _APPEND_ARGS.pack(
            code, batch, tokens, heads, rot, bool(interleaved), table.shape[1], table.stride(0), sk[0], sk[1], sk[2],
            sv[0], sv[1], sv[2], sq[0], sq[1], sq[2], k.data_ptr(), v.data_ptr(), q.data_ptr() if heads else 0,
            out.data_ptr() if heads else 0, 0 if cos is None else cos.data_ptr(), 0 if sin is None else sin.data_ptr(),
            table.data_ptr(), lengths.data_ptr(), 0 if counts is None else counts.data_ptr()) + cache._packed)
    return out if out is None or home == cache.device else out.to(home)


def kv_attention(q: torch.Tensor, cache: KVCache, page_table: torch.Tensor, lengths: torch.Tensor, *,
                 counts: torch.Tensor | None = None, scale: float | None = None, window: int | None = None,
                 sinks: int = 0) -> torch.Tensor:
    """Causal attention of each sequence's last tokens over its cached ones.

    ``q`` is (batch, tokens, q_heads, head_dim), q_heads a multiple of the
    cache's heads (neighbouring query heads share one). ``lengths`` (int32)
    counts the tokens each sequence holds, the queries' own among them; its
    first ``counts[b]`` rows of q (all, without counts) are its last tokens.
    The token at position p sees every token up to p or, with ``window``, the
    last ``window`` of those and the first ``sinks`` of the sequence.
    ``scale`` multiplies the products (1 / sqrt(head_dim) by default; finite).

    Returns q's shape and dtype; queries that see nothing (empty sequences,
    rows past their count) give zeros. No masked slot has any influence,
    whatever its page holds. The products of a query and a key's codes, and
    weighted sums before they are divided, are held in 32 bits: queries of 2^110
    and values of 2^100 and more may overflow them. bfloat16 calls round the
    weights to 8 bits before they are summed and applied (float16 16, float32
    24): a result errs by up to 2^-8 of its values' distance from it.
    """
    if cache._host is not None and dispatch._use_hip():
        out = cache._host.attention(q, page_table, lengths, counts, cache._scale if scale is None else scale,
                                    0 if window is None else window or -1, sinks)
        if out is not None:
            return out
    if q.dim() != 4:
        raise ValueError(f"q must be 4D (batch, tokens, heads, head_dim); got shape {tuple(q.shape)}")
    batch, tokens, heads, dim = q.shape
    code = _check_dtype("q", q)
    if heads < 1 or heads % cache.num_heads:
        raise ValueError(f"{heads} query heads do not share {cache.num_heads} cache heads evenly")
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1; got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative; got {sinks}")
    _check_grad("kv_attention", q)
    dispatch.require_hip()
    home = q.device
    q = _rows(cache, q, "q", batch, tokens, heads)
    table, lengths, counts = _schedule(cache, batch, page_table, lengths, counts)
    out = torch.empty((batch, tokens, heads, dim), dtype=q.dtype, device=cache.device)
    if batch and tokens:
        cache._check_memory()
        sq = q.stride()
        head = (code, batch, tokens, heads, window or 0, sinks, table.shape[1], table.stride(0), sq[0], sq[1], sq[2],
                cache._scale if scale is None else float(scale), q.data_ptr(), out.data_ptr(), table.data_ptr(),
                lengths.data_ptr(), 0 if counts is None else counts.data_ptr())
        packed = _ATTENTION_ARGS.pack(*head) + cache._packed
        need = _lib.load().tt_kv_attention_workspace_bytes(packed + _WORKSPACE.pack(0, 0))
        ws = torch.empty(need, dtype=torch.uint8, device=cache.device) if need else None
        _launch("tt_kv_attention", cache.device, packed + _WORKSPACE.pack(0 if ws is None else ws.data_ptr(), need))
    return out if home == cache.device else out.to(home)
