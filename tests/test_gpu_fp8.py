"""The 8-bit chain on the GPU against its definitions in float64
(oracle/fp8.py): rows in 8 bits, the root-mean-square norm, products and the
gated block.

Tolerances, fixed before the first run. u is the unit roundoff of the result's
dtype (2^-24, 2^-8, 2^-11 for float32, bfloat16, float16); a value in 8 bits
is off by 2^-4 of itself or, below the format's smallest normal, by 2^-10 of its
block's scale.
  fp8_quantize: none. A scale is a power of two and dividing by it is exact.
  rms_norm: squares round once, and a thread adds at most K / 256 + 8 of them,
    then 10 partial sums: (K / 256 + 19) 2^-24 of a sum of positive terms, half
    of it through the root; x + residual, the mean, its sum with eps, the root,
    the reciprocal and two products round once each, the reciprocal and the root
    by up to two units: (K / 512 + 20) 2^-24 in all.
  fp8_matmul: u |y| for the final rounding, plus the 32-bit sums' of K terms of
    A = sum |x w| in all: they err like a random walk, 2^-24 (16 + sqrt K) A.
    Results that are not float32 come from matrix instructions that align each
    eight products to the one of the largest power of two and drop what lies
    below 2^-13 of it: seven of the eight, 7 2^-13 max |x w| for each eight, and
    2^-23 A a block of 128 more for accumulators that may be cut off, not rounded.
    Which eight meet is the kernels' business, so that the sum over any eights'
    maxima is bounded by that of the largest of each 128: 7 2^-13 16 max |x w|.
  fp8_gated_matmul: the products' errors da and db as above; neither activation
    is steeper than 1.13, so |b| 1.13 da + |act(a)| db; exp(-z) errs by 2^-22 |z|
    (z takes four roundings) and a unit, which a / (1 + exp(-z)) passes on at
    most whole, and four roundings follow: |h| (2^-21 + 2^-22 |z|).
"""

import math

import pytest
import torch

import trntensor_amd as tt
from oracle import fp8 as ref

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = list(U)
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _randn(shape, seed, dtype=torch.float32, size=1.0):
    return (size * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(dtype)


def _values(rows):
    """(codes' values, scales, values) of Fp8Rows as two-dimensional float64 tensors."""
    k = rows.shape[-1]
    codes, scales = rows.codes.cpu().double().reshape(-1, k), rows.scales.cpu().double()
    scales = scales.reshape(-1, scales.shape[-1])
    return codes, scales, codes * ref.spread(scales, k)


def _bytes(t):
    return t.view(torch.uint8)


def _check_padding(rows):
    """What lies past the features and blocks is zeros: the products read it."""
    k = rows.shape[-1]
    assert not _bytes(rows._codes)[:, k:].any()
    assert not _bytes(rows._scales)[:, -(-k // 128):].any()


def _check_quantized(x, rows):
    codes, scales, _ = _values(rows)
    want, e = ref.quantize(x)
    assert torch.equal(scales, torch.exp2(e.double()))
    assert torch.equal(codes.isnan(), want.isnan())
    assert torch.equal(codes.nan_to_num(), want.nan_to_num())
    _check_padding(rows)


def _check_rows8(rows, want, rel):
    """Rows in 8 bits of values `want`, known to `rel` (of them, or a tensor of absolute errors)."""
    _, scales, got = _values(rows)
    err = rel if isinstance(rel, torch.Tensor) else rel * want.abs()
    low = ref.exponents((want.abs() - err).clamp(min=0.0))
    high = ref.exponents(want.abs() + err)
    e = torch.log2(scales)
    assert ((e >= low) & (e <= high)).all()
    tol = err + 2.0 ** -4 * (want.abs() + err) + 2.0 ** -10 * ref.spread(scales, want.shape[1])
    assert ((got - want).abs() <= tol).all()
    _check_padding(rows)


# ---------------------------------------------------------------------------
# rows into 8 bits
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 127), (3, 128), (2, 129), (5, 8), (1, 511), (2, 513), (4, 1000), (1, 2048),
                                 (3, 2049), (2, 4100), (1, 16383), (300, 40), (2, 20000)])
def test_quantize(hip, m, k, dtype):
    x = _randn((m, k), m + k, dtype) * torch.exp2(torch.randint(-6, 6, (m, k), generator=torch.Generator().manual_seed(k))).to(dtype)
    rows = tt.fp8_quantize(x.cuda())
    assert rows.shape == (m, k) and rows.dtype == dtype
    _check_quantized(x, rows)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_ends_of_the_types(hip, dtype):
    """Blocks of zeros, of the smallest and largest values, at and around the scale's steps, with infinities and NaN."""
    info = torch.finfo(dtype)
    inf, nan = math.inf, math.nan
    firsts = [0.0, -0.0, info.tiny, info.smallest_normal * 2.0 ** -3, info.max, -info.max, 448.0, 449.0, 450.0, 1.75, 1.75 * (1 + info.eps),
              2.0 ** -10, inf, -inf, nan, 2.0 ** -118, 2.0 ** -120]
    x = torch.zeros((len(firsts), 256), dtype=dtype)
    x[:, 3] = torch.tensor(firsts, dtype=torch.float64).to(dtype)
    x[:, 130] = x[:, 3] / 3
    x[:, 255] = 1.0
    x[5, 7], x[6, 8], x[7, 9] = inf, nan, -inf  # beside finite values
    _check_quantized(x, tt.fp8_quantize(x.cuda()))


def test_quantize_every_value_of_the_format(hip):
    """Codes come back as they are, beside 448 in their block, and halfway values go to the even neighbour."""
    codes = torch.arange(256, dtype=torch.uint8).view(E4M3).float()
    codes = codes[codes.isfinite()]
    mids = torch.sort(codes.abs().unique()).values
    mids = (mids[1:] + mids[:-1]) / 2
    x = torch.zeros((4, 128))
    x[:, 0] = 448.0
    x[0, 1:128], x[1, 1:128] = codes[:127], codes[127:]
    x[2, 1:127], x[3, 1:127] = mids, -mids
    _check_quantized(x, tt.fp8_quantize(x.cuda()))


def test_quantize_strides_shapes_and_host(hip):
    wide = _randn((6, 3, 700), 4, torch.bfloat16).cuda()
    for x in (wide[:, 0, 5:205], wide[:, :, 8:200], wide[:, 1, 16:400:2], wide[0, 0, :192], wide[:0, 0, :192],
              wide[:1, :1, :192].expand(6, 3, 192), wide.permute(1, 2, 0)[0, :192].t(), wide[0, 0, 1:2], wide[:, 0, ::700]):
        rows = tt.fp8_quantize(x)
        assert rows.shape == x.shape and rows.codes.shape == x.shape
        assert rows.scales.shape == (*x.shape[:-1], -(-x.shape[-1] // 128))
        _check_quantized(x.cpu().reshape(-1, x.shape[-1]), rows)
    host = tt.fp8_quantize(wide[:, 0, :192].cpu())
    assert host.device.type == "cuda"
    _check_quantized(wide[:, 0, :192].cpu(), host)
    rows = tt.Fp8Rows(host.codes, host.scales, dtype=torch.float32)
    assert torch.equal(_bytes(rows._codes), _bytes(host._codes)) and torch.equal(_bytes(rows._scales), _bytes(host._scales)) and rows.dtype == torch.float32
    _, _, values = _values(host)
    assert torch.equal(rows.dequantize().cpu().double(), values)
    one = tt.fp8_quantize(wide[0, 0, :130])
    rows = tt.Fp8Rows(one.codes.cpu(), one.scales.cpu())
    assert rows.shape == (130,) and torch.equal(_bytes(rows._codes), _bytes(one._codes)) and torch.equal(_bytes(rows._scales), _bytes(one._scales))


# ---------------------------------------------------------------------------
# the norm
# ---------------------------------------------------------------------------
def _check_norm(x, weight, residual, eps, fp8):
    dev = [None if t is None else t.cuda() for t in (x, weight, residual)]
    got = tt.rms_norm(dev[0], dev[1], residual=dev[2], eps=eps, fp8=fp8)
    k = x.shape[-1]
    want, h = ref.rms_norm(x, weight, residual, eps)
    if residual is not None:
        got, total = got
        assert total.dtype == x.dtype
        # One 32-bit sum, rounded to the dtype: both roundings at most.
        assert ((total.cpu().double() - h).abs() <= (U[x.dtype] + 2.0 ** -24) * (1 + 2.0 ** -8) * h.abs()).all()
    rel = (k / 512 + 20) * 2.0 ** -24
    if fp8:
        assert got.dtype == x.dtype and got.shape == x.shape
        _check_rows8(got, want, rel)
    else:
        assert got.dtype == x.dtype and got.shape == x.shape
        # float16 results below its normal range are off by half of its smallest step.
        small = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
        assert ((got.cpu().double() - want).abs() <= (rel + U[x.dtype]) * (1 + 2.0 ** -8) * want.abs() + small).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("m,k,residual,weight", [
    (1, 1, False, None), (1, 127, True, torch.float32), (3, 128, False, torch.bfloat16), (2, 129, True, None),
    (5, 511, False, torch.float16), (1, 512, True, torch.bfloat16), (2, 513, False, None), (333, 199, True, torch.float16),
    (4, 1000, True, torch.float32), (1, 2048, True, torch.bfloat16), (3, 2049, False, torch.float16), (2, 4096, True, None),
    (2, 4099, True, torch.float32), (3, 8192, True, torch.bfloat16), (2, 8200, False, None), (2, 16384, True, torch.float16),
    (1, 16385, True, torch.bfloat16), (2, 40000, True, None),
])
def test_rms_norm(hip, m, k, residual, weight, fp8, dtype):
    x = _randn((m, k), k, dtype)
    r = _randn((m, k), k + 1, dtype, 3.0) if residual else None
    w = None if weight is None else (1.0 + 0.1 * _randn((k,), k + 2)).to(weight)
    _check_norm(x, w, r, 1e-6, fp8)


@pytest.mark.parametrize("fp8", [False, True])
def test_rms_norm_eps_and_empty_rows(hip, fp8):
    x = _randn((5, 300), 1, torch.bfloat16)
    x[1] = 0.0
    x[2] *= 2.0 ** -30  # eps counts
    x[3] *= 2.0 ** 50
    _check_norm(x, None, None, 1e-5, fp8)
    _check_norm(x[2:], None, None, 0.0, fp8)
    y = tt.rms_norm(x[:0].cuda(), residual=x[:0].cuda(), fp8=fp8)
    assert y[0].shape == (0, 300) and y[1].shape == (0, 300)


def test_rms_norm_strides_host_and_values_that_are_not_finite(hip):
    wide = _randn((4, 3, 500), 7, torch.float16)
    w = _randn((500,), 8, torch.float32)
    for x, r in ((wide[:, 0, :200], wide[:, 1, 100:300]), (wide[:, 0, 5:205], wide[:, 1, 100:500:2]), (wide[:1, :1, :200].expand(4, 3, 200), wide[..., :200])):
        for weight in (w[:200], w[::2][:200]):
            y, h = tt.rms_norm(x.cuda(), weight.cuda(), residual=r.cuda())
            y2, h2 = tt.rms_norm(x.cuda().contiguous(), weight.cuda().contiguous(), residual=r.cuda().contiguous())
            assert y.shape == x.shape and torch.equal(y, y2) and torch.equal(h, h2)
            host, hh = tt.rms_norm(x, weight, residual=r)
            assert host.device.type == "cpu" and hh.device.type == "cpu" and torch.equal(host, y.cpu()) and torch.equal(hh, h.cpu())
    x = _randn((3, 260), 9)
    x[0, 5], x[1, 6], x[2, 7] = math.nan, math.inf, 1e30
    y = tt.rms_norm(x.cuda()).cpu()
    assert y[0].isnan().all()
    assert y[1, 6].isnan() and not y[1, :6].any()  # a row over an infinite mean
    assert not y[2].any()
    rows = tt.rms_norm(x.cuda(), fp8=True)
    codes, scales, _ = _values(rows)
    assert codes[0].isnan().all() and codes[1, 6].isnan() and not codes[1, :6].any()


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
def _rows8(m, k, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    codes = (90.0 * torch.randn((m, k), generator=g)).clamp(-448.0, 448.0).to(E4M3)
    scales = torch.randint(114, 122, (m, -(-k // 128)), generator=g, dtype=torch.uint8).view(E8M0)
    return tt.Fp8Rows(codes, scales, dtype=dtype), codes.double() * ref.spread(scales, k)


def _weights8(n, k, seed, e8m0):
    g = torch.Generator().manual_seed(seed)
    codes = (100.0 * torch.randn((n, k), generator=g)).clamp(-448.0, 448.0).to(E4M3)
    shape = (-(-n // 128), -(-k // 128))
    if e8m0:
        scales = torch.randint(108, 116, shape, generator=g, dtype=torch.uint8).view(E8M0)
    else:
        scales = 2.0 ** -16 * (0.5 + torch.rand(shape, generator=g))
    return tt.Fp8Matrix(codes, scales), ref.weights(codes, scales)


def _sum_error(x, w, exact):
    """What sums of x w^T in 32 bits (`exact`) or of the 8-bit matrix instructions may be off by."""
    size = x.abs() @ w.abs().t()
    err = 2.0 ** -24 * (16 + math.sqrt(x.shape[1])) * size
    if exact:
        return err
    xd, wd = x.abs().float().cuda(), w.abs().float().cuda()
    top = torch.zeros(size.shape, device="cuda")
    for i in range(0, x.shape[1], 128):
        step = max(1, (1 << 27) // (wd.shape[0] * 128))
        for j in range(0, x.shape[0], step):
            top[j: j + step] += (xd[j: j + step, None, i: i + 128] * wd[None, :, i: i + 128]).amax(dim=2)
    return err + 7 * 2.0 ** -13 * 16 * top.cpu().double() + 2.0 ** -23 * -(-x.shape[1] // 128) * size


def _check_product(x, w, y):
    want = x @ w.t()
    assert y.shape == want.shape
    tol = U[y.dtype] * want.abs() + (1 + U[y.dtype]) * _sum_error(x, w, y.dtype == torch.float32)
    err = (y.cpu().double() - want).abs()
    assert (err <= tol).all(), f"{(err / tol.clamp(min=1e-300)).max():.3g} times the tolerance"


SHAPES = [(1, 1, 1), (1, 7, 31), (1, 16, 128), (2, 17, 129), (1, 64, 256), (3, 33, 95), (15, 48, 384), (16, 80, 512), (17, 96, 300),
          (1, 130, 1000), (31, 200, 640), (32, 128, 1024), (33, 129, 1100), (48, 257, 513), (64, 131, 1024), (65, 300, 200), (100, 100, 2000),
          (127, 255, 500), (128, 256, 512), (129, 257, 640), (200, 384, 129), (255, 511, 128), (256, 256, 1024), (257, 300, 1152),
          (300, 513, 1500), (511, 129, 700), (513, 640, 384), (600, 100, 2048), (1, 2000, 4100), (8, 600, 8192), (700, 1030, 100)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("e8m0", [True, False])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul(hip, m, n, k, e8m0, dtype):
    rows, x = _rows8(m, k, m + n, dtype)
    mat, w = _weights8(n, k, k, e8m0)
    y = tt.fp8_matmul(rows, mat)
    assert y.dtype == dtype
    _check_product(x, w, y)


# Many rows and columns, for every tile.
LARGE = [(4000, 4096, 300), (3900, 4100, 129), (2048, 4000, 640), (1000, 4100, 256), (520, 4096, 700), (250, 4080, 1100), (64, 16400, 513),
         (30, 16384, 300), (16, 20000, 128), (8200, 257, 200)]


@pytest.mark.parametrize("e8m0", [True, False])
@pytest.mark.parametrize("m,n,k", LARGE)
def test_matmul_many_rows_and_columns(hip, m, n, k, e8m0):
    rows, x = _rows8(m, k, m + n)
    mat, w = _weights8(n, k, k, e8m0)
    for dtype in DTYPES:
        _check_product(x, w, tt.fp8_matmul(rows, mat, dtype=dtype))


@pytest.mark.parametrize("e8m0", [True, False])
@pytest.mark.parametrize("m", [128, 300])
def test_matmul_every_code_and_column(hip, m, e8m0):
    """x the unit vectors: row k of the result is column k of the weights, exactly."""
    n, k = 200, m
    codes = torch.arange(n * k).reshape(n, k) % 256
    codes = torch.where(codes % 128 == 127, 0, codes).to(torch.uint8).view(E4M3)
    scales = torch.randint(120, 134, (2, -(-k // 128)), generator=torch.Generator().manual_seed(3), dtype=torch.uint8).view(E8M0)
    mat = tt.Fp8Matrix(codes, scales if e8m0 else scales.float())
    y = tt.fp8_matmul(torch.eye(k).cuda(), mat)
    assert torch.equal(y.cpu().double(), ref.weights(codes, scales).t())


def test_matmul_operands_results_and_dtypes(hip):
    mat, w = _weights8(70, 300, 1, True)
    x = _randn((4, 3, 300), 2, torch.bfloat16)
    rows = tt.fp8_quantize(x.cuda())
    y = tt.fp8_matmul(rows, mat)
    assert y.shape == (4, 3, 70) and y.dtype == torch.bfloat16
    assert torch.equal(y, tt.fp8_matmul(x.cuda(), mat))
    host = tt.fp8_matmul(x, mat)
    assert host.device.type == "cpu" and torch.equal(host, y.cpu())
    for dtype in DTYPES:
        z = tt.fp8_matmul(rows, mat, dtype=dtype)
        assert z.dtype == dtype
        _check_product(_values(rows)[2], w, z.reshape(12, 70))
    assert tt.fp8_matmul(x[:0].cuda(), mat).shape == (0, 3, 70)
    assert tt.fp8_matmul(x[0, 0].cuda(), mat).shape == (70,)
    none = tt.Fp8Matrix(torch.zeros((0, 300), dtype=E4M3), torch.zeros((0, 3)))
    assert tt.fp8_matmul(rows, none).shape == (4, 3, 0)
    with pytest.raises(ValueError, match="300"):
        tt.fp8_matmul(x[..., :299].cuda(), mat)
    with pytest.raises(NotImplementedError, match="float64"):
        tt.fp8_matmul(rows, mat, dtype=torch.float64)


@pytest.mark.parametrize("m", [5, 200, 400])
@pytest.mark.parametrize("e8m0", [True, False])
def test_matmul_nan_stays_in_its_row(hip, m, e8m0):
    n, k = 150, 300
    rows, x = _rows8(m, k, 5)
    mat, w = _weights8(n, k, 6, e8m0)
    clean = tt.fp8_matmul(rows, mat)
    _bytes(rows._codes)[m // 2, 170] = 0x7F
    y = tt.fp8_matmul(rows, mat)
    assert y[m // 2].isnan().all()
    keep = torch.arange(m) != m // 2
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (129, 300), (300, 129), (40, 1000)])
def test_matrix_quantize(hip, shape):
    for dtype in DTYPES:
        w = _randn(shape, 11, dtype, 0.05)
        w[0, 0] = 448.0
        mat = tt.Fp8Matrix.quantize(w.cuda())
        n, k = shape
        e = torch.tensor([[ref.exponent(w[i: i + 128, j: j + 128].double().abs().max().item()) for j in range(0, k, 128)]
                          for i in range(0, n, 128)])
        codes = ref.round_e4m3(w.double() / ref.weights(torch.ones(shape), torch.exp2(e.double())))
        want = ref.weights(codes, torch.exp2(e.double()))
        eye = torch.eye(k)
        assert torch.equal(tt.fp8_matmul(eye.cuda(), mat).cpu().double(), want.t())
    w[0, 0], w[-1, -1] = math.inf, 1.0
    y = tt.fp8_matmul(torch.eye(shape[1]).cuda(), tt.Fp8Matrix.quantize(w)).cpu()
    assert y[0, 0].isnan() or shape == (1, 1)


# ---------------------------------------------------------------------------
# the gated block
# ---------------------------------------------------------------------------
def _gated(x, wg, wu, activation, exact):
    """(h, what it may be off by) before its rounding."""
    a, b = x @ wg.t(), x @ wu.t()
    da, db = _sum_error(x, wg, exact), _sum_error(x, wu, exact)
    h = ref.act(a, activation) * b
    z = a if activation == "silu" else 1.6 * (a.abs() + 0.045 * a.abs() ** 3)
    return h, 1.13 * b.abs() * da + ref.act(a, activation).abs() * db + 1.13 * da * db + h.abs() * (2.0 ** -21 + 2.0 ** -22 * z.abs())


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("e8m0", [True, False])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gated_matmul(hip, m, n, k, e8m0, activation):
    dtype = DTYPES[(m + n) % 3]
    rows, x = _rows8(m, k, m + n, dtype)
    gate, wg = _weights8(n, k, k, e8m0)
    up, wu = _weights8(n, k, k + 1, e8m0)
    want, err = _gated(x, wg, wu, activation, False)
    got = tt.fp8_gated_matmul(rows, gate, up, activation=activation)
    assert got.shape == (m, n) and got.dtype == dtype
    _check_rows8(got, want, err)
    plain = tt.fp8_gated_matmul(rows, gate, up, activation=activation, fp8=False)
    assert plain.dtype == dtype
    if dtype == torch.float32:
        err = _gated(x, wg, wu, activation, True)[1]
    small = 2.0 ** -25 if dtype == torch.float16 else 0.0
    assert ((plain.cpu().double() - want).abs() <= U[dtype] * want.abs() + (1 + U[dtype]) * err + small).all()


@pytest.mark.parametrize("e8m0", [True, False])
@pytest.mark.parametrize("m,n,k", [(m, n // 2 + 3, k) for m, n, k in LARGE])
def test_gated_matmul_many_rows_and_columns(hip, m, n, k, e8m0):
    rows, x = _rows8(m, k, m + n)
    gate, wg = _weights8(n, k, k, e8m0)
    up, wu = _weights8(n, k, k + 1, e8m0)
    want, err = _gated(x, wg, wu, "silu", False)
    _check_rows8(tt.fp8_gated_matmul(rows, gate, up), want, err)
    for dtype in (torch.bfloat16, torch.float32):
        plain = tt.fp8_gated_matmul(tt.Fp8Rows(rows.codes, rows.scales, dtype), gate, up, fp8=False)
        if dtype == torch.float32:
            err = _gated(x, wg, wu, "silu", True)[1]
        assert ((plain.cpu().double() - want).abs() <= U[dtype] * want.abs() + (1 + U[dtype]) * err).all()


@pytest.mark.parametrize("e8m0", [True, False])
@pytest.mark.parametrize("m,n,k", [(1, 4096, 128), (40, 1024, 500), (300, 2048, 256), (512, 8192, 128)])
def test_gated_scales_next_to_a_border(hip, m, n, k, e8m0):
    """Scales are those of 32-bit sums where the largest value is next to 448 times a
    power of two. All products are positive, so that a sum errs by its roundings
    relative to itself: in 32 bits 15 of a lane's 16 terms, two of its scale, and six
    and seven where lanes and wavefronts are joined, 31 2^-24 with what is of second
    order. silu passes 1.3 of that on, and the activation adds 8 2^-24: 80 2^-24
    in all. With float scales the blocks of 128 columns have, for one row each,
    their largest value 160 2^-24 above or below the border."""
    band = 80 * 2.0 ** -24
    blocks, kb = -(-n // 128), -(-k // 128)
    rand = torch.Generator().manual_seed(m + n)

    def positive(rows, cols):
        return torch.randn((rows, cols), generator=rand).abs().to(E4M3)

    x, g, u = positive(m, k), positive(n, k), positive(n, k)
    gs = torch.full((blocks, kb), 4.0 / k)
    us = 0.5 + torch.rand((blocks, kb), generator=rand)
    if e8m0:
        gs, us = torch.full((blocks, kb), 2.0 ** (2 - k.bit_length())), torch.ones((blocks, kb))
    else:
        us[:] = us[:, :1]  # one factor for all of a block's columns

    def exact():
        def product(w, s):
            return x.double() @ ref.weights(w.double(), s.double()).t()

        a = product(g, gs)
        return (a / (1.0 + torch.exp(-a)) * product(u, us)).view(m, blocks, 128).amax(dim=2)

    if not e8m0:
        top = exact()
        for b in range(blocks):
            value = top[17 * b % m, b].item()
            border = 448.0 * 2.0 ** round(math.log2(value / 448.0))
            us[b] *= border * (1.0 + (2 * band if b % 2 else -2 * band)) / value
    want = exact()
    e = torch.ceil(torch.log2(want / 448.0))
    border = want / (448.0 * 2.0 ** torch.round(torch.log2(want / 448.0))) - 1.0
    sure = border.abs() > band
    assert sure.sum() > 0.99 * sure.numel()
    if not e8m0:
        assert (sure & (border.abs() < 3 * band)).sum() >= blocks
        to_w = [tt.Fp8Matrix(w.cuda(), s.cuda()) for w, s in ((g, gs), (u, us))]
    else:
        to_w = [tt.Fp8Matrix(w.cuda(), (torch.log2(s) + 127).to(torch.uint8).view(E8M0).cuda()) for w, s in ((g, gs), (u, us))]
    rows = tt.Fp8Rows(x.cuda(), torch.full((m, kb), 127, dtype=torch.uint8).view(E8M0).cuda())
    got = tt.fp8_gated_matmul(rows, *to_w)
    assert torch.equal(got.scales.float().log2().cpu()[sure], e.float()[sure])
    codes = got.codes.float().view(m, blocks, 128).amax(dim=2)
    assert (codes >= 224.0).all() and (codes <= 448.0).all()


@pytest.mark.parametrize("m", [1, 300])
def test_scale_of_255_is_nan(hip, m):
    x, scales = torch.ones((m, 256)).to(E4M3), torch.full((m, 2), 127, dtype=torch.uint8)
    scales[m // 2, 1] = 255
    w = tt.Fp8Matrix(torch.ones((256, 256)).to(E4M3).cuda(), torch.ones((2, 2)).cuda())
    for dtype in DTYPES:
        y = tt.fp8_matmul(tt.Fp8Rows(x.cuda(), scales.view(E8M0).cuda(), dtype), w).cpu()
        assert y[m // 2].isnan().all() and (y[torch.arange(m) != m // 2] == 256.0).all()
    byte = torch.tensor([[127, 255], [127, 127]], dtype=torch.uint8)
    w = tt.Fp8Matrix(torch.ones((256, 256)).to(E4M3).cuda(), byte.view(E8M0).cuda())
    for dtype in DTYPES:
        y = tt.fp8_matmul(torch.ones((m, 256), dtype=dtype).cuda(), w).cpu()
        assert y[:, :128].isnan().all() and (y[:, 128:] == 256.0).all()


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("m,n,k", [(1, 300, 200), (17, 300, 512), (70, 1030, 256), (300, 2048, 256), (513, 4100, 128)])
def test_gated_values_that_are_not_finite(hip, m, n, k, activation):
    """NaN stays in its row; what passes float32's range is NaN in 8 bits and has no part in its block's scale.

    A sum is surely finite where the magnitudes of its blocks' sums add up to less
    than 2^128, since running sums in any order stay below that, and surely not
    where itself is beyond it: its last addition, if not one before. Where only
    running sums or a block's pass it (a multiply-add may hold one that does),
    either is right."""
    rows, x = _rows8(m, k, m + n)
    gate, wg = _weights8(n, k, k, False)
    g = torch.Generator().manual_seed(n)
    codes = (100.0 * torch.randn((n, k), generator=g)).clamp(-448.0, 448.0).to(E4M3)
    scales = 2.0 ** -16 * (0.5 + torch.rand((-(-n // 128), -(-k // 128)), generator=g))
    scales[1] = 2.0 ** 121  # the second block of columns: values on both sides of the range's end
    up, wu = tt.Fp8Matrix(codes, scales), ref.weights(codes, scales)[128:256]
    clean = tt.fp8_gated_matmul(rows, gate, up, activation=activation)
    got = clean.codes[:, 128:256].float().cpu()

    h, err = _gated(x, wg[128:256], wu * 2.0 ** -100, activation, False)
    end, off = 2.0 ** 28, _sum_error(x, wu * 2.0 ** -100, False)
    parts = torch.stack([(x[:, i: i + 128] @ wu[:, i: i + 128].t()).abs() * 2.0 ** -100 for i in range(0, k, 128)])
    b = (x @ wu.t()).abs() * 2.0 ** -100
    fine = (parts.sum(dim=0) + off < end) & (h.abs() + err < end)
    bad = (b - off >= end) | (h.abs() - err >= end)
    assert not (fine & bad).any() and fine.any() and bad.any() and (fine | bad).float().mean() > 0.5
    assert got[fine].isfinite().all() and got[bad].isnan().all()
    low = torch.where(fine, h.abs() - err, torch.zeros_like(h)).amax(dim=1)
    high = torch.where(fine, h.abs() + err, torch.zeros_like(h)).amax(dim=1)
    sure = (fine | bad).all(dim=1) & (low > 0)
    e = torch.ceil(torch.log2(low.clamp(min=1e-300) / 448.0))
    sure &= e == torch.ceil(torch.log2(high.clamp(min=1e-300) / 448.0))
    assert torch.equal(clean.scales[:, 1].float().log2().cpu()[sure], (e + 100)[sure].float())

    rest = torch.cat((clean.codes[:, :128], clean.codes[:, 256:]), dim=1).float()
    assert rest.isfinite().all()
    row = m // 2
    _bytes(rows._codes)[row, k // 2] = 0x7F
    got = tt.fp8_gated_matmul(rows, gate, up, activation=activation)
    assert got.codes[row].float().isnan().all() and (_bytes(got.scales)[row] == 0).all()
    keep = torch.arange(m) != row
    assert torch.equal(_bytes(got.codes)[keep], _bytes(clean.codes)[keep]) and torch.equal(_bytes(got.scales)[keep], _bytes(clean.scales)[keep])
