"""Serving operators on the GPU where their precision and their ranges end,
against their definitions in float64 (oracle/serving.py). Every tolerance is
derived at its test, before its first run; u is the unit roundoff of a result's
dtype (2^-24, 2^-8, 2^-11 for float32, bfloat16, float16).
"""

import math

import pytest
import torch
from torch.autograd import forward_ad

import trntensor_amd as tt
from oracle import serving as ref
from tests import test_gpu_serving as base
from tests.test_gpu_serving import F8, _cache, _i32

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = list(U)


@pytest.mark.parametrize("tokens", [1, 18])
@pytest.mark.parametrize("low", [-64, -60, -8, 100])
def test_kv_attention_float32_weights_do_not_depend_on_value_scales(hip, low, tokens):
    """Two keys of nearly equal weight, in pages whose value scales lie far
    apart: the values of one page outweigh the other's, so that the result is a
    weight times that page's value.

    Tolerance: scores are at most 2^-4, so their errors are below 2^-24 of the
    result. Each of two exponentials errs by a unit in the last place (2^-23)
    and moves the result p by p (1 - p) <= 1/4 of it; their sum, its reciprocal,
    the product and the result round by 2^-24 each, the split into parts by
    2^-24, the product's sums by 2^-24: below 2^-21 of the value in all.
    """
    batch, heads, share, dim, page = 16, 4, 4 if tokens == 1 else 1, 64, 16
    dev, want = _cache(2 * batch, heads, page, dim, 1)
    # Token 0 in one page, the last in the other: a window of one and one sink.
    value = torch.tensor(1.0)
    dev.v.copy_(value.to(F8).expand(dev.v.shape))
    want["v"].fill_(1.0)
    scales = torch.exp2(torch.tensor([0.0, low])).repeat(batch)[:, None].expand(2 * batch, heads)
    dev.v_scale.copy_(scales)
    want["v_scale"].copy_(scales)
    table = torch.arange(2 * batch, dtype=torch.int32).reshape(batch, 2)
    table[1::2] = table[1::2].flip(1)
    held = 17
    q = torch.randn((batch, 1, heads * share, dim), generator=torch.Generator().manual_seed(2)) * 2.0 ** -6
    # More rows than one tile's: the last token's, behind rows that are before the sequence's start.
    rows = q.expand(batch, tokens, heads * share, dim).contiguous()
    got = tt.kv_attention(rows.cuda(), dev, table.cuda(), _i32([held] * batch).cuda(), window=1, sinks=1)[:, -1:]
    out, spread = ref.attention(q, want, table, [held] * batch, None, dim ** -0.5, 1, 1)
    err = (got.cpu().double() - out).abs() / spread[..., 1:2]
    assert err.max() <= 2.0 ** -21, f"2^{math.log2(err.max()):.1f} of the values"


@pytest.mark.parametrize("heads,share,dim,page,tokens,lengths", [(2, 4, 128, 64, 1, [5, 40, 64, 130]), (1, 3, 64, 16, 5, [70, 5]),
                                                                 (2, 1, 192, 32, 40, [90, 300]), (1, 2, 256, 16, 1, [1500])])
def test_kv_attention_float32_keeps_its_bits(hip, heads, share, dim, page, tokens, lengths):
    """Queries and weights enter the matrix units as three parts, 24 bits together.

    Tolerance: u |o|; 2^-22 sum p |v| for the exponentials (a unit in the last
    place), the split and its products; 2 ds max |v| with ds = 2^-24 (16 +
    sqrt D) sum |q k| scale, small here since the queries are; and 2^-24 (16 +
    sqrt L) max |v| for the sums over L keys. Two parts would err by 2^-16 p |v|.
    """
    batch, width = len(lengths), -(-max(lengths) // page)
    dev, want = _cache(batch * width, heads, page, dim, 18)
    table = torch.arange(batch * width, dtype=torch.int32).reshape(batch, width).flip(1).contiguous()
    q = 0.05 * torch.randn((batch, tokens, heads * share, dim), generator=torch.Generator().manual_seed(19))
    got = tt.kv_attention(q.cuda(), dev, table.cuda(), _i32(lengths).cuda()).cpu().double()
    out, spread = ref.attention(q, want, table, lengths, None, dim ** -0.5, None, 0)
    ds = 2.0 ** -24 * (16 + math.sqrt(dim)) * spread[..., 0:1]
    tol = (2.0 ** -24 * out.abs() + 2.0 ** -22 * spread[..., 2:3]
           + (2 * ds + 2.0 ** -24 * (16 + math.sqrt(max(lengths)))) * spread[..., 1:2])
    err = (got - out).abs()
    assert (err <= tol).all(), f"{(err / tol.clamp(min=1e-300)).max():.3g} times the tolerance"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,held", [(1, 5), (1, 40), (3, 200), (40, 200), (1, 3000)])
def test_kv_attention_sums_the_weights_that_it_applies(hip, tokens, held, dtype):
    """Values that lie close together far from zero: rounding a weight may move
    a result by its share of the values' distance from the result, not of the
    values, because the weights' sum is that of the rounded ones.

    Tolerance: the result's rounding, u |o|; the weights' (2^-8 in bfloat16,
    2^-16 in two parts), times sum p |v - o|; an error ds of the scores, 2 ds
    max |v - o| with ds = 2^-24 (16 + sqrt D) sum |q k| scale; and for sums in
    32 bits over L keys, and the exponentials, 2^-24 (16 + sqrt L) max |v|.
    """
    batch, heads, share, dim, page = 6, 2, 4, 64, 16
    width = -(-held // page)
    dev, want = _cache(batch * width, heads, page, dim, 3)
    v = (1.0 + 0.125 * torch.randint(0, 2, dev.v.shape, generator=torch.Generator().manual_seed(4))).to(F8)
    dev.v.copy_(v.cuda())
    dev.v_scale.fill_(1.0)
    want["v"], want["v_scale"] = v.double(), torch.ones_like(want["v_scale"])
    table = torch.arange(batch * width, dtype=torch.int32).reshape(batch, width).flip(1).contiguous()
    q = torch.randn((batch, tokens, heads * share, dim), generator=torch.Generator().manual_seed(5)).to(dtype)
    lengths = [held] * batch
    got = tt.kv_attention(q.cuda(), dev, table.cuda(), _i32(lengths).cuda()).cpu().double()
    out, spread = ref.attention(q, want, table, lengths, None, dim ** -0.5, None, 0)
    # sum p |v - o| is at most twice p (1 - p) times the values' step, p being the larger ones' weight.
    p = (out - 1.0) / 0.125
    apart = 0.25 * p * (1 - p)
    ds = 2.0 ** -24 * (16 + math.sqrt(dim)) * spread[..., 0:1]
    tol = (U[dtype] * out.abs() + (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -16) * apart + 2 * ds * 0.125
           + 2.0 ** -24 * (16 + math.sqrt(held)) * 1.125)
    err = (got - out).abs()
    assert (err <= tol).all(), f"{(err / tol).max():.3g} times the tolerance, {(err > tol).sum()} of {err.numel()}"


def test_kv_attention_of_more_row_blocks_than_a_join_would_take(hip):
    """A million sequences of more than 16 query rows: one launch, whose
    workgroups need no others to join what they find."""
    batch, tokens, dim, page = 1_100_000, 17, 16, 32
    dev, _ = _cache(5, 1, page, dim, 6)
    table = _i32([[3], [0], [4], [1], [2]]).repeat(batch // 5, 1)
    q = torch.randn((5, tokens, 1, dim), generator=torch.Generator().manual_seed(7)).to(torch.bfloat16).cuda()
    lengths = _i32([17, 32, 20, 0, 25])
    want = tt.kv_attention(q, dev, table[:5].cuda(), lengths.cuda())
    got = tt.kv_attention(q.repeat(batch // 5, 1, 1, 1), dev, table.cuda(), lengths.repeat(batch // 5).cuda())
    assert torch.equal(got.view(batch // 5, 5, tokens, 1, dim), want.expand(batch // 5, -1, -1, -1, -1))


def test_kv_append_of_more_query_rows_than_a_launch_has_workgroups(hip):
    """2^24 rows of queries, four a workgroup; most lie past the table's end and give zeros."""
    tokens, dim, page = 1 << 23, 16, 65536
    dev = tt.KVCache.empty(2, 1, dim, page)
    angle = torch.rand((page, dim // 2), generator=torch.Generator().manual_seed(8)).cuda()
    row = torch.randn((2, 1, 1, dim), generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).cuda()
    args = (_i32([[0], [1]]).cuda(), _i32([page - 70, page - 20]).cuda())
    kw = dict(cos=angle.cos(), sin=angle.sin())
    want = tt.kv_append(dev, *(row.expand(2, 100, 1, dim),) * 2, *args, q=row.expand(2, 100, 1, dim), **kw)
    got = tt.kv_append(dev, *(row.expand(2, tokens, 1, dim),) * 2, *args, q=row.expand(2, tokens, 1, dim), **kw)
    assert want[0, :70].ne(0).any() and not want[0, 70:].any() and not want[1, 20:].any()
    assert torch.equal(got[:, :100], want) and not got[:, 100:].any()


@pytest.mark.parametrize("name", ["x", "attention q", "k", "v", "q"])
def test_calls_on_the_device_refuse_tangents(hip, name):
    """The compiled path of ordinary calls does not lose them either."""
    table, held = _i32([[0, 1], [2, 3]]).cuda(), _i32([3, 0]).cuda()
    dev, _ = _cache(4, 2, 16, 64, 10)
    kw = {n: torch.zeros((2, 1, 2, 64), device="cuda") for n in ("k", "v", "q", "attention q", "x")}
    w = tt.Q4Matrix(torch.zeros((8, 32), dtype=torch.uint8), torch.ones((8, 1)), 64, 64)
    cos = torch.zeros((32, 32), device="cuda")
    with forward_ad.dual_level():
        kw[name] = forward_ad.make_dual(kw[name], torch.ones_like(kw[name]))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            tt.kv_append(dev, kw["k"], kw["v"], table, held, q=kw["q"], cos=cos, sin=cos)
            tt.kv_attention(kw["attention q"], dev, table, held)
            tt.q4_matmul(kw["x"], w)


def test_weights_and_caches_that_ask_for_a_gradient(hip):
    """Refused while gradients are on; taken as numbers under no_grad."""
    codes = torch.randint(0, 256, (8, 32), generator=torch.Generator().manual_seed(11), dtype=torch.uint8)
    scales, x = torch.ones((8, 1)), torch.ones((1, 64)).cuda()
    want = tt.q4_matmul(x, tt.Q4Matrix(codes, scales, 64, 64))
    with torch.no_grad():
        assert torch.equal(tt.q4_matmul(x, tt.Q4Matrix(codes, scales.clone().requires_grad_(), 64, 64)), want)
    c = tt.KVCache.empty(2, 1, 64, 16)
    ask = c.v_scale.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="KVCache has no backward"):
        tt.KVCache(c.k, c.v, c.k_scale, ask, 64)
    with torch.no_grad():
        tt.KVCache(c.k, c.v, c.k_scale, ask, 64)


@pytest.mark.parametrize("k", [1, 7, 127, 129, 1001])
def test_laid_out_codes_past_the_columns_are_zeros(hip, k):
    """An odd number of columns leaves half a byte, which may hold anything."""
    n = 35
    codes = torch.randint(0, 256, (n, (k + 1) // 2), generator=torch.Generator().manual_seed(k), dtype=torch.uint8)
    cleared = codes.clone()
    codes[:, -1] |= 0xF0
    cleared[:, -1] &= 0x0F
    scales = torch.ones((n, -(-k // 32)))
    a, b = (tt.Q4Matrix(c, scales, k, 32) for c in (codes, cleared))
    assert torch.equal(a.packed, b.packed)
    x = torch.randn((3, k), generator=torch.Generator().manual_seed(1)).cuda()
    assert torch.equal(tt.q4_matmul(x, a), tt.q4_matmul(x, b))


def test_weights_and_caches_keep_their_attributes(hip):
    """Calls go by the memory found at construction: what would change it and be ignored is refused."""
    c = tt.KVCache.empty(2, 1, 64, 16)
    w = tt.Q4Matrix(torch.zeros((8, 32), dtype=torch.uint8), torch.ones((8, 1)), 64, 64)
    for thing in (c, w):
        for name in [n for n in type(thing).__slots__ if not n.startswith("_")]:
            with pytest.raises(AttributeError, match=f"{name} is fixed"):
                setattr(thing, name, getattr(thing, name))
    c.k.view(torch.uint8).fill_(1)  # what they hold may change


@pytest.mark.parametrize("compiled", [True, False])
@pytest.mark.parametrize("name", ["k", "v", "k_scale", "v_scale", "packed", "scales", "zeros"])
def test_calls_refuse_tensors_that_were_given_other_memory(hip, name, compiled):
    c = tt.KVCache.empty(2, 1, 64, 16)
    ones = torch.ones((8, 1))
    w = tt.Q4Matrix(torch.zeros((8, 32), dtype=torch.uint8), ones, 64, 64, zeros=ones)
    if not compiled:
        c._host = w._host = None
    x, table, held = torch.zeros((1, 1, 1, 64)).cuda(), _i32([[0, 1]]).cuda(), _i32([3]).cuda()
    calls = [lambda: tt.kv_append(c, x, x, table, held), lambda: tt.kv_attention(x, c, table, held)]
    if not hasattr(c, name):
        calls = [lambda: tt.q4_matmul(x, w)]
    for call in calls:
        call()
    t = getattr(c if hasattr(c, name) else w, name)
    was = t.data
    t.data = t.data.clone()
    for call in calls:
        with pytest.raises(RuntimeError, match="other memory"):
            call()
    t.data = was
    for call in calls:
        call()


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf])
def test_kv_attention_refuses_a_scale_that_is_no_number(hip, scale):
    dev, _ = _cache(2, 1, 16, 64, 12)
    with pytest.raises(ValueError, match="scale"):
        tt.kv_attention(torch.ones((1, 1, 1, 64)).cuda(), dev, _i32([[0, 1]]).cuda(), _i32([20]).cuda(), scale=scale)


# ---------------------------------------------------------------------------
# sizes and cuts of calls that each take a kernel or a path of their own
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    "heads,share,dim,rot,page,tokens,lengths,counts,interleaved",
    [
        # rows of 192 codes, which a wavefront's lanes do not divide evenly
        (2, 2, 192, 192, 64, 70, [0, 60], [70, 33], False),
        (1, 9, 160, 64, 32, 40, [5, 31], None, True),
        (2, 1, 136, 128, 16, 33, [0, 15, 16], None, False),
        (1, 16, 192, 96, 16, 1, [0, 17, 31], [1, 0, 1], True),
        (2, 3, 136, 136, 48, 50, [3, 47], None, False),
        (1, 2, 130, 130, 32, 9, [30], None, True),
        (3, 1, 176, 16, 128, 300, [100], None, False),
    ],
)
def test_kv_append_of_heads_between_128_and_192(hip, heads, share, dim, rot, page, tokens, lengths, counts, interleaved, dtype):
    base.test_kv_append(hip, heads, share, dim, rot, page, tokens, lengths, counts, interleaved, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    "heads,share,dim,page,tokens,lengths,counts,window,sinks",
    [
        (2, 4, 136, 64, 1, [0, 1, 63, 64, 65, 200], None, None, 0),
        (1, 2, 160, 16, 3, [3, 64, 130], [3, 0, 2], None, 0),
        (1, 5, 192, 32, 1, [600], None, 50, 70),
        (2, 2, 192, 64, 30, [70, 200, 0], [30, 9, 0], None, 0),
        (1, 3, 136, 48, 70, [150], None, 33, 7),
        (1, 1, 160, 128, 130, [140, 300], None, None, 0),
    ],
)
def test_kv_attention_of_heads_between_128_and_192(hip, heads, share, dim, page, tokens, lengths, counts, window, sinks, dtype):
    base._attention_case(heads, share, dim, page, tokens, lengths, counts, window, sinks, dtype)


@pytest.mark.parametrize("dtype,tokens", [(torch.bfloat16, 500), (torch.float16, 260), (torch.float32, 130)])
def test_kv_attention_of_many_rows_and_heads_between_128_and_192(hip, dtype, tokens):
    for dim in (136, 192):
        base.test_kv_attention_many_rows(hip, dtype, 2, 3, dim, 32, tokens, [2500, 700], [tokens, 20], None, 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    "heads,share,dim,page,tokens,lengths,counts,window,sinks",
    [
        # pairs of sequence and head cut anywhere, over several heads and sequences
        (3, 2, 128, 64, 1, [5000, 3, 0, 2049], None, None, 0),
        (8, 2, 192, 32, 1, [3000, 1100], None, None, 0),
        (2, 4, 256, 16, 3, [2000, 0, 1500], [3, 1, 2], None, 0),
        (5, 1, 80, 16, 1, [1, 1300, 1, 1200], None, None, 0),
        # queries before their sequence's start, and rows past their counts
        (2, 3, 64, 64, 5, [4000, 3, 2100], [5, 5, 0], None, 0),
        # windows of more tiles than a workgroup takes, and sinks before them
        (2, 2, 96, 64, 2, [6000, 4000, 9], None, 2000, 70),
        (4, 1, 128, 128, 1, [9000, 1500], None, 1100, 1),
        # more sequences than a wavefront looks at together, most of them short or empty
        (1, 2, 64, 16, 1, [2100, *[n % 5 * 7 for n in range(75)], 700, 0, 1900], None, None, 0),
    ],
)
def test_kv_attention_of_long_tables(hip, heads, share, dim, page, tokens, lengths, counts, window, sinks, dtype):
    base._attention_case(heads, share, dim, page, tokens, lengths, counts, window, sinks, dtype)


def _wide(dtype, heads, share, dim, page, tokens, lengths, width, missing=(), counts=None, seed=51):
    """Attention through a table of `width` entries, -1 past each sequence's end and at `missing` (sequence, entry)."""
    dev, want = _cache(sum(-(-n // page) for n in lengths) + 1, heads, page, dim, seed)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lengths):
        used = -(-n // page)
        table[b, :used] = torch.arange(at, at + used, dtype=torch.int32).flip(0)
        at += used
    for b, entry in missing:
        table[b, entry] = -1
    q = torch.randn((len(lengths), tokens, heads * share, dim), generator=torch.Generator().manual_seed(seed + 1)).to(dtype)
    n = None if counts is None else _i32(counts)
    got = tt.kv_attention(q.cuda(), dev, table.cuda(), _i32(lengths).cuda(), counts=None if n is None else n.cuda())
    base._check_attention(got, q, want, table, lengths, n, 1 / math.sqrt(dim), None, 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 20, 70, 300])
def test_kv_attention_through_tables_wider_than_the_sequences(hip, tokens, dtype):
    """How a call is cut follows from the table's width, what is there from the lengths."""
    for lengths in ([300], [70, 0, 310]):
        _wide(dtype, 1, 2, 64, 16, tokens, lengths, 2000)
    _wide(dtype, 2, 1, 128, 64, tokens, [330, 90], 700, counts=[tokens, 1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 3, 40])
def test_kv_attention_of_long_sequences_that_miss_pages(hip, tokens, dtype):
    _wide(dtype, 2, 2, 64, 16, tokens, [3000, 1500], 400, missing=[(0, e) for e in (*range(40, 60), 0, 100, 187)]
          + [(1, e) for e in range(5, 90)])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k,group", [(300, 700, 520, 128), (513, 200, 390, 64), (257, 330, 640, 32), (400, 130, 1000, 256)])
def test_q4_matmul_of_hundreds_of_rows(hip, m, n, k, group, dtype):
    base.test_q4_matmul(hip, m, n, k, group, True, dtype)


# ---------------------------------------------------------------------------
# values at the ends of their types
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 40])
def test_kv_attention_of_infinite_queries(hip, tokens, dtype, value):
    """A score is then infinite or NaN, and the formula gives NaN: for that
    query head alone."""
    dev, _ = _cache(4, 2, 64, 64, 13)
    table, held = _i32([[2, 0, 3, 1]]).cuda(), _i32([250]).cuda()
    q = torch.randn((1, tokens, 6, 64), generator=torch.Generator().manual_seed(14)).to(dtype)
    clean = tt.kv_attention(q.cuda(), dev, table, held)
    q[0, tokens // 2, 4, 17] = value
    got = tt.kv_attention(q.cuda(), dev, table, held)
    bad = torch.zeros(got.shape[:3], dtype=torch.bool, device="cuda")
    bad[0, tokens // 2, 4] = True
    assert got[bad].isnan().all() and torch.equal(got[~bad], clean[~bad])


def test_float16_operands_below_the_normal_range(hip):
    """Subnormal activations and queries count as what they are."""
    g = torch.Generator().manual_seed(15)
    codes, scales, z = base._q4(70, 256, 64, torch.float32, True, 16)
    x = (torch.randint(-900, 900, (20, 256), generator=g).double() * 2.0 ** -24).to(torch.float16)
    assert x.abs().max() < 2.0 ** -14
    w = tt.Q4Matrix(codes, scales * 2.0 ** 14, 256, 64, zeros=z)
    base._check_q4(x, codes, scales * 2.0 ** 14, z, 256, 64, tt.q4_matmul(x.cuda(), w))
    for tokens in (1, 40):
        dev, want = _cache(4, 1, 64, 64, 17)
        q = (torch.randint(-900, 900, (1, tokens, 2, 64), generator=g).double() * 2.0 ** -24).to(torch.float16)
        table = _i32([[2, 0, 3, 1]])
        got = tt.kv_attention(q.cuda(), dev, table.cuda(), _i32([250]).cuda(), scale=2.0 ** 12)
        base._check_attention(got, q, want, table, [250], None, 2.0 ** 12, None, 0)
