"""What the 8-bit chain refuses, and how it checks its arguments, without a
GPU; the oracle's rounding against torch's."""

import struct

import pytest
import torch

import trntensor_amd as tt
from oracle import fp8 as ref
from trntensor_amd import serving
from trntensor_amd.hip import _lib, dispatch

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


@pytest.fixture
def lib():
    handle = _lib.load()
    assert handle is not None, _lib.load_error()
    return handle


@pytest.fixture
def no_gpu(monkeypatch):
    monkeypatch.setattr(dispatch, "require_hip", lambda: None)

    def refuse(*a):
        raise AssertionError("a launch was reached")

    monkeypatch.setattr(serving, "_launch", refuse)


class _Matrix:
    """What the checks before a launch read of weights."""

    _host = None

    def __init__(self, n=64, k=256, scale_dtype=torch.float32):
        self.shape, self.scale_dtype, self.device = (n, k), scale_dtype, torch.device("cpu")


def test_oracle_exponents():
    for amax, e in ((448.0, 0), (448.1, 1), (224.0, -1), (0.0, -127), (1e-45, -127), (1.75, -8), (1.76, -7), (3e38, 120)):
        assert ref.exponent(amax) == e
    x = torch.tensor([[float("inf"), 448.0, float("nan")] + [0.0] * 126 + [1.75]])
    assert ref.exponents(x).tolist() == [[0, -8]]


def test_rows_and_matrix_checks():
    codes, scales = torch.zeros((3, 200), dtype=E4M3), torch.zeros((3, 2), dtype=torch.uint8).view(E8M0)
    for bad in ((codes.float(), scales), (codes[:, :0], scales), (torch.zeros((), dtype=E4M3), scales)):
        with pytest.raises(ValueError, match="codes must be"):
            tt.Fp8Rows(*bad)
    for bad in (scales[:, :1], scales.float(), scales[:2], scales[0]):
        with pytest.raises(ValueError, match="scales must be"):
            tt.Fp8Rows(codes, bad)
    with pytest.raises(NotImplementedError, match="float64"):
        tt.Fp8Rows(codes, scales, dtype=torch.float64)
    wide = torch.zeros((1, 2))
    for bad in (codes.float(), codes[0], codes[:, :0]):
        with pytest.raises(ValueError, match="codes must be"):
            tt.Fp8Matrix(bad, wide)
    for bad in (wide[:, :1], wide.half(), wide.to(torch.uint8), wide[0], torch.zeros((3, 2))):
        with pytest.raises(ValueError, match="scales must be"):
            tt.Fp8Matrix(codes, bad)
    with pytest.raises(RuntimeError, match="no backward"):
        tt.Fp8Matrix(codes, wide.requires_grad_())
    for bad, kind in ((torch.zeros(4), ValueError), (torch.zeros((4, 0)), ValueError), (torch.zeros((4, 4), dtype=torch.float64), NotImplementedError),
                      (torch.zeros((4, 4), requires_grad=True), RuntimeError)):
        with pytest.raises(kind):
            tt.Fp8Matrix.quantize(bad)


def test_norm_and_quantize_checks(no_gpu):
    x, w = torch.zeros((2, 5, 96)), torch.ones(96)
    for call, kind, match in (
        (dict(x=x.double()), NotImplementedError, "float64"),
        (dict(x=torch.zeros(())), ValueError, "features"),
        (dict(x=x[..., :0]), ValueError, "features"),
        (dict(weight=w[:95]), ValueError, "weight must have shape"),
        (dict(weight=w[None]), ValueError, "weight must have shape"),
        (dict(weight=w.double()), NotImplementedError, "float64"),
        (dict(residual=x[:1]), ValueError, "residual"),
        (dict(residual=x.half()), ValueError, "residual"),
        (dict(eps=-1e-6), ValueError, "eps"),
        (dict(eps=float("nan")), ValueError, "eps"),
        (dict(eps=float("inf")), ValueError, "eps"),
        (dict(weight=w.clone().requires_grad_()), RuntimeError, "no backward"),
        (dict(residual=x.clone().requires_grad_()), RuntimeError, "no backward"),
    ):
        with pytest.raises(kind, match=match):
            kw = dict(x=x, weight=w) | call
            tt.rms_norm(kw.pop("x"), kw.pop("weight"), **kw)
    for bad, kind in ((x.long(), NotImplementedError), (torch.zeros(()), ValueError), (x[..., :0], ValueError),
                      (x.clone().requires_grad_(), RuntimeError)):
        with pytest.raises(kind):
            tt.fp8_quantize(bad)


def test_product_checks(no_gpu):
    w, x = _Matrix(), torch.zeros((2, 256))
    for call in (tt.fp8_matmul, lambda a, b: tt.fp8_gated_matmul(a, b, b)):
        for bad, kind in ((x[:, :255], ValueError), (x.double(), NotImplementedError), (torch.zeros(()), ValueError),
                          (x.clone().requires_grad_(), RuntimeError)):
            with pytest.raises(kind):
                call(bad, w)
    with pytest.raises(ValueError, match="alike"):
        tt.fp8_gated_matmul(x, w, _Matrix(n=65))
    with pytest.raises(ValueError, match="alike"):
        tt.fp8_gated_matmul(x, w, _Matrix(scale_dtype=E8M0))
    with pytest.raises(ValueError, match="activation"):
        tt.fp8_gated_matmul(x, w, w, activation="relu")


def test_fixed_attributes():
    rows = tt.Fp8Rows._of((2, 3), torch.float32, torch.zeros((2, 128), dtype=torch.uint8).view(E4M3),
                          torch.zeros((2, 4), dtype=torch.uint8).view(E8M0))
    with pytest.raises(AttributeError, match="fixed"):
        rows.dtype = torch.float16
    with pytest.raises(AttributeError):
        rows.codes = rows.codes
    assert rows.codes.shape == (2, 3) and rows.scales.shape == (2, 1)
    assert "Fp8Rows((2, 3)" in repr(rows)


# ---------------------------------------------------------------------------
# the C entry points refuse before any HIP call
# ---------------------------------------------------------------------------
def _quantize(lib, **kw):
    f = dict(dtype=0, rows=2, dim=96, stride=96, x=256, codes=256, scales=256) | kw
    return lib.tt_fp8_quantize(struct.pack("=7q", *f.values()), None)


def _norm(lib, **kw):
    f = dict(dtype=0, wdtype=0, rows=2, dim=96, stride=96, rstride=96, eps=1e-6, x=256, residual=0, weight=0, sum=0, y=256, codes=0,
             scales=0) | kw
    return lib.tt_rms_norm(struct.pack("=6qd7q", *f.values()), None)


def _product(lib, **kw):
    f = dict(dtype=0, sdtype=0, M=2, N=16, K=128, x=256, xs=256, w=256, ws=256, y=256) | kw
    return lib.tt_fp8_matmul(struct.pack("=10q", *f.values()), None)


def _gated(lib, query=False, **kw):
    f = dict(dtype=0, sdtype=0, act=0, M=2, N=16, K=128, x=256, xs=256, g=256, gs=256, u=256, us=256, y=0, codes=256, scales=256, ws=256,
             ws_bytes=1 << 30) | kw
    packed = struct.pack("=17q", *f.values())
    return lib.tt_fp8_gated_workspace_bytes(packed) if query else lib.tt_fp8_gated_matmul(packed, None)


def test_c_refusals(lib):
    for fn, name in ((lib.tt_fp8_quantize, b"tt_fp8_quantize"), (lib.tt_rms_norm, b"tt_rms_norm"), (lib.tt_fp8_matmul, b"tt_fp8_matmul"),
                     (lib.tt_fp8_gated_matmul, b"tt_fp8_gated_matmul")):
        assert fn(None, None) == _lib.TT_INVALID
        assert lib.tt_last_error().startswith(name)
    assert lib.tt_fp8_gated_workspace_bytes(None) == 0
    for kw in (dict(rows=-1), dict(dim=0), dict(x=0), dict(codes=0), dict(scales=0), dict(codes=264), dict(scales=258)):
        assert _quantize(lib, **kw) == _lib.TT_INVALID, kw
    for kw in (dict(dtype=1), dict(dim=1 << 31), dict(rows=1 << 40)):
        assert _quantize(lib, **kw) == _lib.TT_UNSUPPORTED, kw
    assert _quantize(lib, rows=0, x=0) == _lib.TT_OK
    for kw in (dict(rows=-1), dict(dim=0), dict(x=0), dict(y=0), dict(codes=256, scales=256), dict(y=0, codes=256), dict(y=0, scales=256),
               dict(residual=256), dict(sum=256), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=1e39), dict(y=0, codes=264, scales=256),
               dict(y=0, codes=256, scales=257)):
        assert _norm(lib, **kw) == _lib.TT_INVALID, kw
    for kw in (dict(dtype=1), dict(weight=256, wdtype=6), dict(dim=1 << 31)):
        assert _norm(lib, **kw) == _lib.TT_UNSUPPORTED, kw
    assert _norm(lib, rows=0) == _lib.TT_OK
    for kw in (dict(M=-1), dict(N=-1), dict(K=0), dict(x=0), dict(xs=0), dict(w=0), dict(ws=0), dict(y=0), dict(x=264), dict(w=264),
               dict(xs=258), dict(ws=257)):
        assert _product(lib, **kw) == _lib.TT_INVALID, kw
    for kw in (dict(dtype=1), dict(sdtype=3), dict(sdtype=4), dict(M=1 << 40), dict(N=1 << 31), dict(K=1 << 31)):
        assert _product(lib, **kw) == _lib.TT_UNSUPPORTED, kw
    assert _product(lib, M=0) == _lib.TT_OK and _product(lib, N=0, w=0) == _lib.TT_OK
    for kw in (dict(M=-1), dict(act=2), dict(act=-1), dict(x=0), dict(gs=0), dict(u=0), dict(y=256), dict(codes=0), dict(scales=0),
               dict(y=0, codes=0, scales=0), dict(g=264), dict(us=258), dict(codes=264), dict(scales=258)):
        assert _gated(lib, **kw) == _lib.TT_INVALID, kw
    for kw in (dict(dtype=1), dict(sdtype=3), dict(M=1 << 40)):
        assert _gated(lib, **kw) == _lib.TT_UNSUPPORTED, kw
    assert _gated(lib, M=0) == _lib.TT_OK
    need = _gated(lib, query=True)
    if need:
        assert _gated(lib, ws=0) == _lib.TT_INVALID and _gated(lib, ws_bytes=need - 1) == _lib.TT_INVALID


def test_c_refusals_of_calls_beyond_the_grid(lib):
    """Calls whose extents are allowed one by one, but not together."""
    big = 1 << 30
    for dtype in (_lib.TT_F32, _lib.TT_BF16):
        for kind in (_lib.TT_F32, _lib.TT_E8M0):
            for k in (128, big):  # on tiles, and where their offsets do not reach
                assert _product(lib, dtype=dtype, sdtype=kind, M=big, N=big, K=k) == _lib.TT_UNSUPPORTED
                for out in (dict(y=256, codes=0, scales=0), dict(y=0, codes=256, scales=256, ws_bytes=1 << 62)):
                    assert _gated(lib, dtype=dtype, sdtype=kind, M=big, N=big, K=k, **out) == _lib.TT_UNSUPPORTED
    assert _gated(lib, query=True, M=3, N=200, K=(1 << 23) + 1) == 3 * 200 * 4  # no tiles: 32-bit products in between
    assert _quantize(lib, rows=(1 << 31) - 1, dim=big, stride=big) == _lib.TT_UNSUPPORTED


def test_rows_given_other_memory_are_refused(no_gpu):
    def rows(count=2, codes=256, scales=4):
        return tt.Fp8Rows._of((2, 256), torch.float32, torch.zeros((count, codes), dtype=torch.uint8).view(E4M3),
                              torch.zeros((count, scales), dtype=torch.uint8).view(E8M0))

    rows()._check_memory()
    for bad in (rows(count=1), rows(codes=128), rows(scales=8)):
        for call in (lambda: tt.fp8_matmul(bad, _Matrix()), lambda: tt.fp8_gated_matmul(bad, _Matrix(), _Matrix())):
            with pytest.raises(RuntimeError, match="other memory"):
                call()
    short = rows()
    short._codes.untyped_storage().resize_(500)
    with pytest.raises(RuntimeError, match="other memory"):
        tt.fp8_matmul(short, _Matrix())


def test_c_pack_refusals(lib):
    assert lib.tt_fp8_packed_bytes(17, 129) == 2 * 2 * 2048 and lib.tt_fp8_packed_bytes(0, 5) == 0
    for args in ((-1, 8, 256, 8, 256), (4, 0, 256, 4, 256), (4, 8, 0, 8, 256), (4, 8, 256, 8, 0), (4, 9, 256, 8, 256), (4, 8, 256, 8, 264)):
        assert lib.tt_fp8_pack(*args, None) == _lib.TT_INVALID, args
        assert lib.tt_last_error().startswith(b"tt_fp8_pack")
    assert lib.tt_fp8_pack(1 << 31, 8, 256, 8, 256, None) == _lib.TT_UNSUPPORTED
    assert lib.tt_fp8_pack(0, 8, 0, 8, 0, None) == _lib.TT_OK
