"""Serving operators on the GPU against their definitions in float64
(oracle/serving.py): 4-bit products, the append to a paged 8-bit cache, and
attention over it.

Tolerances, fixed before the first run. u is the unit roundoff of the result's
dtype (2^-24, 2^-8, 2^-11 for float32, bfloat16, float16).
  q4_matmul: u |y| for the final rounding, plus the 32-bit sums': K additions
    of terms no larger than A = sum |x| s (|c - z| + 24) (codes pass the matrix
    units as 16 + c, and 16 + z is taken off) err like a random walk,
    2^-24 (16 + sqrt K) A.
  kv_append: none. Rotations are float32 products and sums, rounded one by one,
    and codes, scales and rotated queries follow from them without choice.
  kv_attention: u |o|, plus the rounding of probabilities times sum p |v|
    (2^-8 in bfloat16, which holds them in 8 bits, else 2^-15), plus what an
    error ds of the scores does, 2 ds max|v| with ds = 2^-24 (16 + sqrt D)
    (sum |q k| scale), and 2^-24 (16 + sqrt L) max |v| for the sums over L keys.
"""

import math

import pytest
import torch

import trntensor_amd as tt
from oracle import serving as ref

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = list(U)
F8 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------
# 4-bit products
# ---------------------------------------------------------------------------
def _q4(n, k, group, dtype, zeros, seed):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, dtype=torch.uint8)
    groups = -(-k // group)
    scales = (0.02 * (0.5 + torch.rand((n, groups), generator=g))).to(dtype)
    z = (15 * torch.rand((n, groups), generator=g)).to(dtype) if zeros else None
    return codes, scales, z


def _check_q4(x, codes, scales, z, k, group, y):
    w = ref.q4_weights(codes, scales, k, group, z)
    want = x.double() @ w.t()
    ones = w.abs()
    s = scales.double()[:, torch.arange(k) // group]
    size = x.double().abs() @ (ones + 24.0 * s.abs()).t()
    tol = U[y.dtype] * want.abs() + 2.0 ** -24 * (16 + math.sqrt(k)) * size
    assert y.shape == want.shape
    err = (y.cpu().double() - want).abs()
    assert (err <= tol).all(), f"{(err / tol.clamp(min=1e-300)).max():.3g} times the tolerance"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize(
    "m,n,k,group",
    [
        (1, 1, 1, 32),
        (1, 7, 31, 32),  # half a byte left over
        (1, 16, 128, 128),
        (1, 64, 256, 64),
        (3, 33, 95, 32),
        (1, 257, 1000, 128),  # last group short
        (2, 100, 129, 64),
        (5, 130, 640, 32),
        (15, 48, 384, 128),
        (16, 80, 512, 64),
        (17, 96, 300, 32),
        (33, 70, 257, 128),
        (64, 131, 1024, 256),
        (65, 40, 200, 64),
        (130, 72, 512, 512),
        (1, 520, 4224, 128),
        (4, 24, 8192, 64),
        # many rows on both sides
        (17, 8200, 130, 128),
        (32, 8320, 1024, 128),
        (33, 8193, 1290, 256),
        (64, 8448, 900, 128),
        (100, 8209, 640, 128),
        (20, 8288, 250, 32),
        (2, 8300, 300, 128),
        (9, 8250, 300, 128),
        (12, 5000, 390, 128),
        (20, 4200, 270, 128),
        (40, 2200, 200, 64),
    ],
)
def test_q4_matmul(hip, m, n, k, group, zeros, dtype):
    codes, scales, z = _q4(n, k, group, dtype, zeros, m + n + k)
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(k)).to(dtype)
    w = tt.Q4Matrix(codes, scales, k, group, zeros=z)
    _check_q4(x, codes, scales, z, k, group, tt.q4_matmul(x.cuda(), w))


@pytest.mark.parametrize("scale_dtype", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_q4_matmul_scales_of_another_dtype(hip, dtype, scale_dtype):
    codes, scales, z = _q4(50, 256, 64, scale_dtype, True, 4)
    x = torch.randn((3, 256), generator=torch.Generator().manual_seed(5)).to(dtype)
    _check_q4(x, codes, scales, z, 256, 64, tt.q4_matmul(x.cuda(), tt.Q4Matrix(codes.cuda(), scales.cuda(), 256, 64, zeros=z.cuda())))


@pytest.mark.parametrize("dtype,scale_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32),
                                               (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("m,n,k,group", [(9, 8250, 300, 128), (20, 4200, 270, 128), (20, 8288, 250, 32), (40, 2200, 200, 64)])
def test_q4_matmul_many_rows_and_scales_of_another_dtype(hip, m, n, k, group, dtype, scale_dtype):
    codes, scales, z = _q4(n, k, group, scale_dtype, True, m + n)
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(9)).to(dtype)
    w = tt.Q4Matrix(codes.cuda(), scales.cuda(), k, group, zeros=z.cuda())
    _check_q4(x, codes, scales, z, k, group, tt.q4_matmul(x.cuda(), w))


def test_q4_matmul_every_code_and_column(hip):
    """x the unit vectors: row k of the result is column k of the weights, exactly."""
    n, k = 48, 160
    codes, scales, _ = _q4(n, k, 32, torch.float32, False, 6)
    codes[:, :8] = torch.arange(8, dtype=torch.uint8) * 0x22 + 0x10  # every code, in both halves
    scales = torch.exp2(torch.randint(-4, 5, scales.shape, generator=torch.Generator().manual_seed(7)).float())
    want = ref.q4_weights(codes, scales, k, 32, None)
    got = tt.q4_matmul(torch.eye(k).cuda(), tt.Q4Matrix(codes, scales, k, 32))
    assert torch.equal(got.cpu().double(), want.t())


def test_q4_matmul_strided_rows_shapes_and_host_operands(hip):
    codes, scales, z = _q4(40, 192, 64, torch.bfloat16, True, 8)
    w = tt.Q4Matrix(codes, scales, 192, 64, zeros=z)
    wide = torch.randn((6, 3, 400), generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).cuda()
    for x in (wide[:, 0, 5:197], wide[:, :, 8:200], wide[:, 1, 16:400:2], wide[0, 0, :192], wide[:0, 0, :192],
              wide[:1, :1, :192].expand(6, 3, 192), wide.permute(1, 2, 0)[0, :192].t()):
        y = tt.q4_matmul(x, w)
        assert y.shape == (*x.shape[:-1], 40)
        _check_q4(x.cpu().reshape(-1, 192), codes, scales, z, 192, 64, y.reshape(-1, 40))
    host = tt.q4_matmul(wide[:, 0, :192].cpu(), w)
    assert host.device.type == "cpu" and torch.equal(host, tt.q4_matmul(wide[:, 0, :192].contiguous(), w).cpu())


@pytest.mark.parametrize("dtype", DTYPES)
def test_q4_matmul_keeps_nan_and_infinity_to_their_rows(hip, dtype):
    codes, scales, z = _q4(80, 512, 128, dtype, True, 10)
    x = torch.randn((20, 512), generator=torch.Generator().manual_seed(11)).to(dtype)
    w = tt.Q4Matrix(codes, scales, 512, 128, zeros=z)
    clean = tt.q4_matmul(x.cuda(), w).cpu()
    x[3, 100], x[7, 511] = math.nan, math.inf
    got = tt.q4_matmul(x.cuda(), w).cpu()
    bad = torch.zeros(20, dtype=torch.bool)
    bad[[3, 7]] = True
    assert torch.equal(got[~bad], clean[~bad])
    assert got[3].isnan().all() and not got[7].isfinite().any()


# ---------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------
def _width(dim):
    return -(-dim // 64) * 64


def _cache(pages, heads, page, dim, seed, fill=None):
    """A cache of random codes (or of one byte) and scales, on the device, and
    the same as float64 values for the oracle."""
    g = torch.Generator().manual_seed(seed)
    w = _width(dim)

    def codes(*shape):
        if fill is not None:
            return torch.full(shape, fill, dtype=torch.uint8).view(F8)
        return (torch.randn(shape, generator=g) * 90).clamp(-448, 448).to(F8)

    k, v = codes(pages, heads, page, w), codes(pages, heads, w, page)
    if fill is None:
        k.view(torch.uint8)[..., dim:] = 0
    ks, vs = (torch.exp2(torch.randint(-9, -5, (pages, heads), generator=g).float()) for _ in range(2))
    dev = tt.KVCache(k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), head_dim=dim)
    return dev, {"k": k.double(), "v": v.double(), "k_scale": ks.double(), "v_scale": vs.double()}


def _same(dev, want, dim):
    """Every code and scale of the cache is the oracle's (compared as values, NaN equal to NaN)."""
    for name in ("k", "v", "k_scale", "v_scale"):
        got, exp = getattr(dev, name).cpu().double(), want[name]
        if name == "v":
            got, exp = got[:, :, :dim], exp[:, :, :dim]
        assert torch.equal(got.isnan(), exp.isnan()), name
        assert torch.equal(got.nan_to_num(), exp.nan_to_num()), f"{name}: {(got != exp).sum()} of {got.numel()} differ"


def _turns(positions, rot):
    angle = torch.arange(positions).double()[:, None] * torch.exp(torch.arange(rot // 2).double() * (-9.2 * 2 / rot))
    return angle.cos().float(), angle.sin().float()


def _qkv(batch, tokens, heads, share, dim, dtype, seed):
    """Queries, keys and values as views of one projection's output."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((batch, tokens, (share + 2) * heads, dim), generator=g) * 3).to(dtype)
    return x.split([share * heads, heads, heads], dim=2), x.cuda().split([share * heads, heads, heads], dim=2)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    "heads,share,dim,rot,page,tokens,lengths,counts,interleaved",
    [
        (1, 1, 64, 64, 16, 1, [0], None, False),
        (2, 4, 128, 128, 64, 1, [0, 1, 63, 64, 100, 127], None, False),
        (3, 1, 80, 32, 16, 1, [5, 15, 16, 47], [1, 0, 1, 1], True),
        (2, 2, 64, 64, 32, 7, [0, 30, 31, 32], [7, 7, 0, 5], False),
        (1, 3, 96, 96, 16, 50, [0, 9, 16], [50, 33, 1], True),
        (2, 1, 256, 64, 128, 130, [0, 127], None, False),
        (1, 2, 40, 10, 48, 60, [3, 47], None, True),
        (2, 1, 33, 2, 16, 20, [0, 14], None, False),
        (1, 8, 128, 128, 64, 200, [1, 64], [200, 64], False),
        (2, 1, 200, 200, 64, 65, [10], None, True),
    ],
)
def test_kv_append(hip, heads, share, dim, rot, page, tokens, lengths, counts, interleaved, dtype):
    batch = len(lengths)
    width = -(-(max(lengths) + tokens) // page)
    dev, want = _cache(batch * width + 2, heads, page, dim, 1)
    table = torch.randperm(batch * width + 2, generator=torch.Generator().manual_seed(2))[: batch * width]
    table = table.to(torch.int32).reshape(batch, width)
    cos, sin = _turns(width * page, rot)
    (q, k, v), (dq, dk, dv) = _qkv(batch, tokens, heads, share, dim, dtype, 3)
    n = None if counts is None else _i32(counts)
    out = ref.append(want, k, v, table, lengths, n, q, cos, sin, interleaved)
    got = tt.kv_append(dev, dk, dv, table.cuda(), _i32(lengths).cuda(), counts=None if n is None else n.cuda(), q=dq,
                       cos=cos.cuda(), sin=sin.cuda(), interleaved=interleaved)
    assert got.dtype == dtype and torch.equal(got.cpu(), out.to(dtype))
    _same(dev, want, dim)


@pytest.mark.parametrize("dtype", DTYPES)
def test_kv_append_token_by_token_with_growing_values(hip, dtype):
    """A page whose tokens grow (its older codes are rounded again and again),
    one whose tokens shrink, zeros, and values that no scale reaches."""
    heads, dim, page, steps = 2, 64, 16, 24
    dev, want = _cache(6, heads, page, dim, 4, fill=0x7F)  # whatever lay there before
    table = _i32([[4, 1], [0, 5], [2, 3]])
    g = torch.Generator().manual_seed(5)
    most = 6e4 if dtype == torch.float16 else 3e38
    for step in range(steps):
        k = torch.randn((3, 1, heads, dim), generator=g)
        v = torch.randn((3, 1, heads, dim), generator=g)
        k[0] *= 1.7 ** step
        v[1] *= 0.6 ** step
        k[2, :, 1] = 0.0
        if step == 20:
            v[2, 0, 0, 3], v[2, 0, 0, 4], k[1, 0, 1, 5], k[1, 0, 0, 0] = math.inf, -math.inf, math.nan, most
        k, v = k.clamp(-most, most).to(dtype) if step != 20 else k.to(dtype), v.to(dtype)
        held = _i32([step] * 3)
        ref.append(want, k, v, table, held, None, None, None, None, False)
        assert tt.kv_append(dev, k.cuda(), v.cuda(), table.cuda(), held.cuda()) is None
    # Codes past the tokens appended are what they were (NaN); those before agree.
    _same(dev, want, dim)


def test_kv_append_rounds_every_value_as_defined(hip):
    """All bfloat16 values of a block at a scale of one: ties, subnormal codes, saturation."""
    x = torch.arange(0, 65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = x[x.float().abs() <= 448]  # 2^8 codes' range at scale 1 (the largest magnitude is 448)
    x = torch.cat([x, torch.zeros((-x.numel()) % (64 * 64), dtype=torch.bfloat16)]).reshape(-1, 64, 1, 64)
    x[:, 0, 0, 0] = 448.0
    pages = x.shape[0]
    dev = tt.KVCache.empty(pages, 1, 64, 64)
    table = torch.arange(pages, dtype=torch.int32).reshape(pages, 1).cuda()
    tt.kv_append(dev, x.cuda(), x.cuda(), table, torch.zeros(pages, dtype=torch.int32).cuda())
    assert (dev.k_scale == 1).all() and (dev.v_scale == 1).all()
    want = ref.round_e4m3(x[:, :, 0])
    assert torch.equal(dev.k[:, 0].cpu().double(), want)
    assert torch.equal(dev.v[:, 0].cpu().double(), want.transpose(1, 2))


def test_kv_append_drops_what_has_no_page(hip):
    """Page numbers outside the cache, tokens past the table's end, negative
    lengths and counts: nothing is written for them, the rest as usual."""
    heads, dim, page = 2, 64, 16
    dev, want = _cache(5, heads, page, dim, 6)
    table = _i32([[3, -1, 0], [7, 1, 1 << 30], [2, 4, -5], [4, 4, 4]])
    lengths, counts = [10, 5, 40, -3], [20, 40, 30, 5]
    (q, k, v), (dq, dk, dv) = _qkv(4, 40, heads, 1, dim, torch.bfloat16, 7)
    cos, sin = _turns(48, 64)
    ref.append(want, k[:3], v[:3], table[:3], lengths[:3], _i32(counts[:3]), q[:3], cos, sin, False)
    before = {n: getattr(dev, n).clone() for n in ("k", "v", "k_scale", "v_scale")}
    got = tt.kv_append(dev, dk, dv, table.cuda(), _i32(lengths).cuda(), counts=_i32(counts).cuda(), q=dq, cos=cos.cuda(),
                       sin=sin.cuda())
    _same(dev, want, dim)
    assert torch.isfinite(got).all()
    for n, t in before.items():
        getattr(dev, n).copy_(t)
    tt.kv_append(dev, dk, dv, table.cuda(), _i32(lengths).cuda(), counts=_i32([0, -1, 0, -7]).cuda())
    for n, t in before.items():
        assert torch.equal(getattr(dev, n).view(torch.uint8), t.view(torch.uint8)), n


def test_kv_append_strides_and_host_operands(hip):
    heads, dim, page = 2, 80, 32
    table = _i32([[1, 0], [2, 3]])
    cos, sin = _turns(64, 80)
    g = torch.Generator().manual_seed(8)
    base = torch.randn((2, heads, 9, dim), generator=g)  # [batch][head][token][dim]
    forms = []
    for dev in ("cuda", "cpu"):
        x = base.to(dev)
        tr = x.transpose(1, 2)
        forms += [(tr, tr.contiguous()), (tr.contiguous(), tr), (x.transpose(2, 3).contiguous().permute(0, 3, 1, 2), tr)]
    first = None
    for k, v in forms:
        cache, _ = _cache(4, heads, page, dim, 9)
        q = tt.kv_append(cache, k, v, table.to(k.device), _i32([3, 30]).to(k.device), q=k, cos=cos, sin=sin)
        assert q.device.type == k.device.type and q.is_contiguous()
        got = [t.cpu() for t in (q, cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _check_attention(got, q, want_cache, table, lengths, counts, scale, window, sinks):
    dtype, dim = q.dtype, q.shape[3]
    out, spread = ref.attention(q, want_cache, table, lengths, counts, scale, window, sinks)
    longest = max([1, *[int(x) for x in lengths]])
    ds = 2.0 ** -24 * (16 + math.sqrt(dim)) * spread[..., 0:1]
    tol = (U[dtype] * out.abs() + (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -15) * spread[..., 2:3]
           + (2 * ds + 2.0 ** -24 * (16 + math.sqrt(longest))) * spread[..., 1:2])
    assert got.shape == q.shape and got.dtype == dtype
    err = (got.cpu().double() - out).abs()
    assert not got.isnan().any()
    assert (err <= tol).all(), f"{(err / tol.clamp(min=1e-300)).max():.3g} times the tolerance"
    empty = spread[..., 1] == 0
    assert (got.cpu()[empty] == 0).all()


def _attention_case(heads, share, dim, page, tokens, lengths, counts, window, sinks, dtype, scale=None, seed=11):
    batch = len(lengths)
    width = max(1, -(-max(lengths) // page))
    dev, want = _cache(batch * width + 1, heads, page, dim, seed)
    table = torch.randperm(batch * width + 1, generator=torch.Generator().manual_seed(seed + 1))[: batch * width]
    table = table.to(torch.int32).reshape(batch, width)
    # The slots past each sequence's end hold NaN codes, or lie in no page.
    for b, n in enumerate(lengths):
        for block in range(width):
            at, live = int(table[b, block]), min(max(n - block * page, 0), page)
            if live == 0:
                table[b, block] = -1
            else:
                dev.k.view(torch.uint8)[at, :, live:] = 0x7F
                dev.v.view(torch.uint8)[at, :, :, live:] = 0xFF
    q = torch.randn((batch, tokens, heads * share, dim), generator=torch.Generator().manual_seed(seed + 2)).to(dtype)
    n = None if counts is None else _i32(counts)
    got = tt.kv_attention(q.cuda(), dev, table.cuda(), _i32(lengths).cuda(), counts=None if n is None else n.cuda(),
                          scale=scale, window=window, sinks=sinks)
    _check_attention(got, q, want, table, lengths, n, 1 / math.sqrt(dim) if scale is None else scale, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    "heads,share,dim,page,tokens,lengths,counts,window,sinks",
    [
        (1, 1, 64, 16, 1, [1], None, None, 0),
        (2, 4, 128, 64, 1, [0, 1, 15, 16, 17, 63, 64, 65, 200], None, None, 0),
        (1, 8, 128, 16, 1, [257, 300], None, None, 0),
        (2, 5, 80, 32, 1, [33, 500], None, None, 0),
        (3, 1, 96, 128, 1, [129, 1000, 0], None, None, 0),
        (1, 3, 256, 64, 1, [70, 900], None, None, 0),
        (1, 2, 200, 16, 2, [40], None, None, 0),
        (2, 1, 1, 16, 1, [20], None, None, 0),
        (1, 1, 40, 48, 1, [100, 47, 48], None, None, 0),
        # several queries a sequence, ragged
        (2, 4, 128, 64, 3, [3, 64, 130], None, None, 0),
        (1, 1, 64, 16, 5, [5, 9, 2, 0], [5, 0, 2, 0], None, 0),
        (1, 3, 64, 32, 17, [17, 100], [17, 3], None, 0),
        (2, 2, 128, 64, 70, [70, 200, 90], [70, 64, 1], None, 0),
        (1, 4, 80, 16, 130, [150], None, None, 0),
        # windows and sinks
        (2, 4, 64, 16, 1, [10, 100, 300], None, 16, 0),
        (1, 2, 128, 64, 1, [700, 65, 64], None, 100, 4),
        (2, 1, 96, 32, 3, [400, 129, 3], None, 1, 1),
        (1, 2, 64, 16, 40, [300, 41], None, 33, 7),
        (1, 1, 128, 64, 80, [80, 500], [80, 70], 64, 70),
        (2, 2, 64, 128, 2, [1000], None, 2000, 4),
        (1, 5, 128, 32, 1, [600], None, 50, 1000),
    ],
)
def test_kv_attention(hip, heads, share, dim, page, tokens, lengths, counts, window, sinks, dtype):
    _attention_case(heads, share, dim, page, tokens, lengths, counts, window, sinks, dtype)


@pytest.mark.parametrize(
    "dtype,heads,share,dim,page,tokens,lengths,counts,window,sinks",
    [
        # every block of rows that is taken, whole and with its keys split
        (torch.bfloat16, 8, 4, 128, 64, 1024, [3000, 2500], None, None, 0),
        (torch.float16, 8, 4, 96, 32, 1024, [3000, 1100], [1024, 700], None, 0),
        (torch.bfloat16, 2, 4, 128, 64, 512, [32768], None, None, 0),
        (torch.float16, 2, 4, 64, 64, 512, [20000], None, None, 0),
        (torch.bfloat16, 8, 4, 64, 16, 128, [1000] * 8, None, None, 0),
        (torch.bfloat16, 1, 4, 128, 64, 200, [5000, 0], None, None, 0),
        (torch.float32, 8, 4, 128, 16, 256, [1500, 900], None, None, 0),
        (torch.float32, 2, 2, 256, 32, 300, [5000], None, None, 0),
        (torch.bfloat16, 4, 3, 200, 32, 400, [4000, 100, 0], [400, 30, 0], None, 0),
        (torch.bfloat16, 8, 4, 128, 64, 1024, [3000, 2500], None, 700, 5),
        (torch.float16, 8, 4, 128, 64, 600, [600, 2001], None, 100, 130),
    ],
)
def test_kv_attention_many_rows(hip, dtype, heads, share, dim, page, tokens, lengths, counts, window, sinks):
    """Some tokens of calls too large to check whole; the others are finite."""
    batch, width, g = len(lengths), -(-max(lengths) // page), torch.Generator().manual_seed(17)
    dev, want = _cache(batch * width, heads, page, dim, 16)
    table = torch.randperm(batch * width, generator=g).to(torch.int32).reshape(batch, width)
    for b, n in enumerate(lengths):
        for block in range(width):
            live = min(max(n - block * page, 0), page)
            dev.k.view(torch.uint8)[int(table[b, block]), :, live:] = 0x7F
            dev.v.view(torch.uint8)[int(table[b, block]), :, :, live:] = 0xFF
    q = torch.randn((batch, tokens, heads * share, dim), generator=g).to(dtype)
    n = None if counts is None else _i32(counts)
    got = tt.kv_attention(q.cuda(), dev, table.cuda(), _i32(lengths).cuda(), counts=None if n is None else n.cuda(),
                          window=window, sinks=sinks).cpu()
    assert got.isfinite().all()
    for b, held in enumerate(lengths):
        live = tokens if counts is None else counts[b]
        picked = {0, 1, 15, 16, 63, 64, live // 2, live - 1, *torch.randint(0, tokens, (6,), generator=g).tolist()}
        for t in sorted(x for x in picked if 0 <= x < tokens):
            if t >= live or held - live + t < 0:
                assert (got[b, t] == 0).all()
                continue
            # A token sees what a single query behind its position sees.
            _check_attention(got[b : b + 1, t : t + 1], q[b : b + 1, t : t + 1], want, table[b : b + 1],
                             _i32([held - live + t + 1]), None, 1 / math.sqrt(dim), window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, 2.0, -0.5])
def test_kv_attention_scale(hip, scale, dtype):
    """Scores that pick single keys, none at all (a mean), and reversed ones."""
    _attention_case(2, 3, 64, 16, 2, [150, 64], None, None, 0, dtype, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 20])
def test_kv_attention_every_code(hip, tokens, dtype):
    """Sequence c holds code c: as the only value seen it comes back as it is
    (every code times a power of two is exact in each type here); as a key
    beside a zero key it weighs as its value says."""
    codes = torch.arange(256, dtype=torch.uint8)
    table, lengths = torch.arange(256, dtype=torch.int32)[:, None].cuda(), _i32([tokens] * 256).cuda()
    value = codes.view(F8).double()
    finite = value.isfinite()
    cache = tt.KVCache.empty(256, 1, 64, page_size=32)
    cache.v.view(torch.uint8)[:, 0, :, :] = codes.cuda()[:, None, None]
    cache.v_scale.fill_(2.0 ** -3)
    q = torch.zeros((256, tokens, 1, 64), dtype=dtype)
    got = tt.kv_attention(q.cuda(), cache, table, lengths).cpu().double()
    tol = (U[dtype] + 2.0 ** -24 * 32 + (2.0 ** -8 if tokens > 1 and dtype == torch.bfloat16 else 2.0 ** -15 if tokens > 1 else 0))
    want = (value / 8)[:, None, None, None].expand(got.shape)
    if tokens == 1:
        assert torch.equal(got[finite], want[finite])
    assert ((got - want)[finite].abs() <= tol * want[finite].abs()).all()
    assert got[~finite].isnan().all() and not got[finite].isnan().any()

    cache.k.view(torch.uint8)[:, 0, tokens - 1, 5] = codes.cuda()
    cache.k_scale.fill_(2.0 ** -5)
    cache.v.view(torch.uint8).zero_()
    cache.v.view(torch.uint8)[:, 0, :, tokens - 1] = 0x38  # 1.0
    cache.v_scale.fill_(1.0)
    q[..., 5] = 1
    got = tt.kv_attention(q.cuda(), cache, table, lengths, scale=0.5).cpu().double()[finite][:, -1, 0]
    e = torch.exp(value[finite] / 64)
    want = (e / (e + tokens - 1))[:, None].expand(got.shape)
    tol = U[dtype] + (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -15) + 2 * 2.0 ** -24 * 24 * 7 + 2.0 ** -24 * 24
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_kv_attention_long(hip, dtype):
    """A long sequence beside short ones, for which the work is split and joined."""
    _attention_case(1, 2, 64, 64, 1, [9000, 3, 0, 4097], None, None, 0, dtype)


@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 2)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_kv_attention_keeps_nan_to_who_sees_it(hip, dtype, window, sinks):
    """NaN among a chunk's own keys and values: only queries that see the token
    get it (values: only in that element)."""
    heads, dim, page, tokens, held = 1, 64, 16, 30, 75
    dev, want = _cache(6, heads, page, dim, 21)
    table = _i32([[5, 0, 3, 1, 2]])
    q = torch.randn((1, tokens, 2, dim), generator=torch.Generator().manual_seed(22)).to(dtype)
    clean, _ = ref.attention(q, want, table, [held], None, 0.125, window, sinks)
    key, value = 60, 52
    dev.k.view(torch.uint8)[int(table[0, key // page]), 0, key % page, 7] = 0x7F
    dev.v.view(torch.uint8)[int(table[0, value // page]), 0, 9, value % page] = 0xFF
    got = tt.kv_attention(q.cuda(), dev, table.cuda(), _i32([held]).cuda(), scale=0.125, window=window, sinks=sinks).cpu()
    for t in range(tokens):
        pos = held - tokens + t
        sees = [j <= pos and (window is None or j > pos - window or j < sinks) for j in (key, value)]
        bad = torch.zeros(dim, dtype=torch.bool)
        bad[9] = sees[1]
        if sees[0]:
            bad[:] = True
        assert torch.equal(got[0, t].isnan(), bad.expand(2, dim)), (t, sees)
        assert (got[0, t][:, ~bad].double() - clean[0, t][:, ~bad]).abs().max().nan_to_num() < 0.1 if (~bad).any() else True


def test_kv_attention_skips_pages_that_are_not(hip):
    heads, dim, page = 2, 64, 16
    dev, want = _cache(4, heads, page, dim, 23)
    table = _i32([[0, -1, 2], [9, 1 << 30, -7], [3, 1, 77]])
    lengths = [48, 30, 100]  # the last is past what its table covers
    q = torch.randn((3, 2, 4, dim), generator=torch.Generator().manual_seed(24))
    got = tt.kv_attention(q.cuda(), dev, table.cuda(), _i32(lengths).cuda())
    _check_attention(got, q, want, table, lengths, None, 0.125, None, 0)
    assert (got[1] == 0).all()
    got = tt.kv_attention(q.cuda(), dev, table.cuda(), _i32([0, -4, 1]).cuda(), counts=_i32([2, 1, 2]).cuda())
    _check_attention(got, q, want, table, [0, 0, 1], _i32([2, 1, 2]), 0.125, None, 0)


def test_kv_attention_infinite_and_huge_queries(hip):
    """Scores of thousands choose their key without overflow; infinities give what the formula gives."""
    dev, want = _cache(4, 1, 64, 64, 25)
    table = _i32([[2, 0, 3, 1]])
    q = torch.randn((1, 1, 2, 64), generator=torch.Generator().manual_seed(26)) * 1e4
    got = tt.kv_attention(q.cuda(), dev, table.cuda(), _i32([250]).cuda())
    out, _ = ref.attention(q, want, table, [250], None, 0.125, None, 0)
    assert (got.cpu().double() - out).abs().max() <= 1e-3 * out.abs().max()
    q[0, 0, 1] = math.nan
    got = tt.kv_attention(q.cuda(), dev, table.cuda(), _i32([250]).cuda())
    assert got[0, 0, 1].isnan().all() and not got[0, 0, 0].isnan().any()


def test_kv_attention_strides_and_host_operands(hip):
    dev, _ = _cache(9, 2, 32, 80, 27)
    table, lengths = _i32([[3, 1, 8, 0], [2, 4, 5, 6]]), _i32([100, 77])
    base = torch.randn((2, 4, 3, 200), generator=torch.Generator().manual_seed(28)).to(torch.bfloat16)
    q = base.transpose(1, 2)[..., 40:120]  # tokens and heads exchanged, rows at an odd place
    wide = torch.full((2, 9), -1, dtype=torch.int32)
    wide[:, 3:7] = table
    want = tt.kv_attention(q.contiguous().cuda(), dev, table.cuda(), lengths.cuda())
    assert torch.equal(tt.kv_attention(base.cuda().transpose(1, 2)[..., 40:120], dev, wide.cuda()[:, 3:7], lengths.cuda()), want)
    assert torch.equal(tt.kv_attention(q[..., :].cuda(), dev, table.t().contiguous().t().cuda(), lengths.cuda()), want)
    host = tt.kv_attention(q, dev, table, lengths)
    assert host.device.type == "cpu" and torch.equal(host, want.cpu())


# ---------------------------------------------------------------------------
# streams, graphs, offsets
# ---------------------------------------------------------------------------
def _step(x, w_in, w_out, cache, table, held, cos, sin, heads, share, dim):
    batch, tokens = x.shape[:2]
    q, k, v = tt.q4_matmul(x, w_in).view(batch, tokens, -1, dim).split([heads * share, heads, heads], dim=2)
    q = tt.kv_append(cache, k, v, table, held, q=q, cos=cos, sin=sin)
    return tt.q4_matmul(tt.kv_attention(q, cache, table, held + tokens).flatten(2), w_out)


def _step_parts(seed=31, heads=2, share=4, dim=64):
    hidden = heads * share * dim
    mats = []
    for n, k, s in (((share + 2) * heads * dim, hidden, 1), (hidden, hidden, 2)):
        codes, scales, _ = _q4(n, k, 128, torch.bfloat16, False, seed + s)
        mats.append(tt.Q4Matrix(codes, scales * 0.1, k, 128))
    cos, sin = (t.cuda() for t in _turns(8 * 64, dim))
    table = torch.arange(24, dtype=torch.int32).reshape(3, 8).flip(1).contiguous().cuda()
    x = torch.randn((3, 1, hidden), generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()
    return (x, *mats), (table, _i32([0, 63, 300]).cuda(), cos, sin, heads, share, dim)


def test_a_step_on_another_stream(hip):
    """The whole step queued behind a slow producer on a side stream, without waiting, gives the default stream's result."""
    (x, w_in, w_out), rest = _step_parts()
    want = _step(x, w_in, w_out, tt.KVCache.empty(24, 2, 64), *rest)
    cache = tt.KVCache.empty(24, 2, 64)
    big = torch.randn((4096, 4096), device="cuda")
    slow = torch.zeros_like(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(20):
            big = big @ big * 1e-4
        slow.copy_(x)
        got = _step(slow, w_in, w_out, cache, *rest)
    side.synchronize()
    assert torch.equal(got, want)


def test_a_step_in_a_graph(hip):
    """Captured once and replayed with other inputs, eager work in between."""
    (x, w_in, w_out), rest = _step_parts()
    cache = tt.KVCache.empty(24, 2, 64)
    inputs = x.clone()
    _step(inputs, w_in, w_out, cache, *rest)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(inputs, w_in, w_out, cache, *rest)
    for i in range(4):
        inputs.copy_(x * (1 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        want = _step(x * (1 + i), w_in, w_out, cache, *rest)  # the same slots: written alike
        assert torch.equal(got, want), i


def test_calls_without_the_host_path(hip):
    """What the compiled host path launches is what Python launches."""
    g = torch.Generator().manual_seed(31)
    codes, scales, z = _q4(6 * 64, 256, 64, torch.bfloat16, True, 32)
    w = tt.Q4Matrix(codes.cuda(), scales.cuda(), 256, 64, zeros=z.cuda())
    angles = torch.rand((128, 32), generator=g)
    cos, sin = torch.cos(angles).cuda(), torch.sin(angles).cuda()
    x = torch.randn((3, 40, 256), generator=g).to(torch.bfloat16).cuda()
    table = torch.arange(6, dtype=torch.int32).view(3, 2).cuda()
    held, counts = _i32([0, 30, 64]).cuda(), _i32([40, 0, 13]).cuda()
    found = []
    for direct in (True, False):
        cache = tt.KVCache.empty(6, 2, 64, 64)
        assert w._host is not None and cache._host is not None
        host = w._host
        if not direct:
            w._host = cache._host = None
        q, k, v = tt.q4_matmul(x, w).view(3, 40, 6, 64).split([2, 2, 2], dim=2)
        q = tt.kv_append(cache, k, v, table, held, counts=counts, q=q, cos=cos, sin=sin, interleaved=True)
        o = tt.kv_attention(q, cache, table, held + counts, counts=counts, window=50, sinks=2)
        found.append([q, o, cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale])
        w._host = host
    for a, b in zip(*found):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bad", [0.0, -1.0, 3.0, 2.0 ** -65, 2.0 ** 121, float("inf"), float("nan")])
def test_a_cache_takes_powers_of_two_in_range(hip, bad):
    c = tt.KVCache.empty(2, 1, 64, 16)
    for ok in (2.0 ** -64, 2.0 ** 120):
        tt.KVCache(c.k, c.v, torch.full_like(c.k_scale, ok), torch.full_like(c.v_scale, ok), 64)
    scale = c.v_scale.clone()
    scale[1, 0] = bad
    with pytest.raises(ValueError, match="powers of two"):
        tt.KVCache(c.k, c.v, c.k_scale, scale, 64)


def test_results_repeat_bit_for_bit(hip):
    (x, w_in, w_out), rest = _step_parts(seed=41)
    first = _step(x, w_in, w_out, tt.KVCache.empty(24, 2, 64), *rest)
    for _ in range(5):
        assert torch.equal(_step(x, w_in, w_out, tt.KVCache.empty(24, 2, 64), *rest), first)


def test_offsets_beyond_32_bits(hip):
    """A cache of over 2^32 codes: its first and last pages hold a sequence's tokens."""
    heads, dim, page = 8, 128, 64
    pages = (1 << 32) // (heads * dim * page) + 20
    cache = tt.KVCache.empty(pages, heads, dim, page)
    small = tt.KVCache.empty(3, heads, dim, page)
    g = torch.Generator().manual_seed(33)
    k, v = (torch.randn((1, 150, heads, dim), generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    q = torch.randn((1, 1, heads, dim), generator=g).to(torch.bfloat16).cuda()
    held, zero = _i32([150]).cuda(), _i32([0]).cuda()
    outs = []
    for c, t in ((cache, [[pages - 1, 0, pages - 7]]), (small, [[1, 0, 2]])):
        tt.kv_append(c, k, v, _i32(t).cuda(), zero)
        outs.append(tt.kv_attention(q, c, _i32(t).cuda(), held))
    assert torch.equal(outs[0], outs[1])
    assert torch.equal(cache.v.view(torch.uint8)[pages - 1], small.v.view(torch.uint8)[1])
    assert (outs[0] != 0).any()
