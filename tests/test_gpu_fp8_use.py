"""The 8-bit chain as a program uses it: the operators one after the other, on
streams of their own, in captured graphs that share weights, from several
threads, and through the C interface between guard bytes.

Tolerances of the chain, fixed before its first run: each product takes operands
that are off by half a step of 8 bits (2^-4 of each value, 2^-10 of a block's scale
for the smallest) against the chain in 64 bits that rounds at the same places;
what differs there is which of two neighbouring codes a value next to their middle
gets. An operator's own result differs from the 64-bit one by at most 2^-13 of a
row's norm, so that at most about 2^-13 / 2^-4 = 2^-9 of the values change their
code, by 2^-3 each: 2^-4.5 2^-3 < 2^-7 of the norm an operator, 2^-5 for three of
them in a row with the final rounding.
"""

import ctypes
import struct
import threading

import pytest
import torch

import trntensor_amd as tt
from oracle import fp8 as ref
from trntensor_amd.hip import _fastpath, _lib

pytestmark = pytest.mark.gpu

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _randn(shape, seed, dtype=torch.float32, size=1.0):
    return (size * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(dtype)


def _bytes(t):
    return t.view(torch.uint8)


def _matrix(n, k, seed, e8m0=True):
    mat = tt.Fp8Matrix.quantize(_randn((n, k), seed, size=k ** -0.5).cuda())
    if e8m0:
        return mat
    codes = (100.0 * _randn((n, k), seed)).clamp(-448.0, 448.0).to(E4M3)
    scales = 0.01 * k ** -0.5 * (0.5 + torch.rand((-(-n // 128), -(-k // 128)), generator=torch.Generator().manual_seed(seed)))
    return tt.Fp8Matrix(codes.cuda(), scales.cuda())


def _feed_forward(x, y, w, layer):
    """A pre-norm feed-forward block with the residual stream."""
    h, x = tt.rms_norm(y, w, residual=x, fp8=True)
    h = tt.fp8_gated_matmul(h, layer["gate"], layer["up"])
    return tt.fp8_matmul(h, layer["down"]), x


def _layer(hidden, mlp, seed):
    return {"gate": _matrix(mlp, hidden, seed), "up": _matrix(mlp, hidden, seed + 1), "down": _matrix(hidden, mlp, seed + 2)}


def _values(mat):
    """The weights that a matrix stands for, through its products with the unit vectors."""
    return tt.fp8_matmul(torch.eye(mat.shape[1]).cuda(), mat).t().cpu().double()


@pytest.mark.parametrize("rows,hidden,mlp", [(1, 256, 640), (5, 192, 320), (70, 384, 1000), (300, 512, 768)])
def test_chain_against_64_bits(hip, rows, hidden, mlp):
    layer = _layer(hidden, mlp, 1)
    x, y, w = _randn((rows, hidden), 4, torch.bfloat16), _randn((rows, hidden), 5, torch.bfloat16), 1 + 0.1 * _randn((hidden,), 6)
    out, stream = _feed_forward(x.cuda(), y.cuda(), w.cuda(), layer)

    def rounded(v):
        codes, e = ref.quantize(v)
        return codes * ref.spread(torch.exp2(e.double()), v.shape[1])

    h, total = ref.rms_norm(y, w, x, 1e-6)
    h = rounded(h)
    h = rounded(ref.act(h @ _values(layer["gate"]).t(), "silu") * (h @ _values(layer["up"]).t()))
    want = h @ _values(layer["down"]).t()
    assert ((stream.cpu().double() - total).abs() <= 2.0 ** -8 * 1.01 * total.abs()).all()
    assert (out.cpu().double() - want).norm() <= 2.0 ** -5 * want.norm()


@pytest.mark.parametrize("fast", [True, False])
def test_calls_give_the_same_with_and_without_the_host_path(hip, monkeypatch, fast):
    if not fast:
        monkeypatch.setattr(_fastpath, "rows_host", lambda: None)
        monkeypatch.setattr(_fastpath, "module", lambda: None)
    layer, floats = _layer(320, 500, 10), _matrix(77, 320, 13, e8m0=False)
    for lead in ((), (3,), (2, 4), (0,), (2, 0, 3)):
        x, y = (_randn((*lead, 320), s, torch.float16).cuda() for s in (14, 15))
        w = _randn((320,), 16, torch.float32).cuda()
        rows, total = tt.rms_norm(y, w, residual=x, fp8=True)
        plain, total2 = tt.rms_norm(y, w, residual=x)
        assert torch.equal(total, total2) and plain.shape == x.shape and rows.shape == x.shape
        again = tt.fp8_quantize(y)
        assert again.codes.shape == (*lead, 320) and again.scales.shape == (*lead, 3)
        h = tt.fp8_gated_matmul(rows, layer["gate"], layer["up"], activation="gelu_tanh")
        assert h.shape == (*lead, 500) and h.dtype == torch.float16
        assert tt.fp8_gated_matmul(rows, layer["gate"], layer["up"], fp8=False).shape == (*lead, 500)
        for z in (tt.fp8_matmul(h, layer["down"]), tt.fp8_matmul(rows, layer["up"], dtype=torch.float32)):
            assert z.shape[:-1] == torch.Size(lead)
        got = (_bytes(rows._codes), _bytes(rows._scales), total, plain, _bytes(again._codes), _bytes(h._codes), _bytes(h._scales), tt.fp8_matmul(rows, floats))
        expected = _EXPECTED.setdefault(lead, got)
        for a, b in zip(got, expected):
            assert torch.equal(a, b)


_EXPECTED = {}


def test_results_repeat_bit_for_bit_and_do_not_depend_on_earlier_calls(hip):
    layer = _layer(1024, 1500, 20)
    for rows in (1, 20, 100, 600):
        x, y, w = _randn((rows, 1024), 21, torch.bfloat16).cuda(), _randn((rows, 1024), 22, torch.bfloat16).cuda(), torch.ones(1024).cuda()
        first = _feed_forward(x, y, w, layer)
        for _ in range(3):
            _feed_forward(y, x, 2 * w, layer)
            again = _feed_forward(x, y, w, layer)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_streams_that_share_weights(hip):
    """Calls on four streams at once, with no wait between them."""
    layer = _layer(512, 900, 30)
    inputs = [(_randn((m, 512), 31 + m, torch.bfloat16).cuda(), _randn((m, 512), 32 + m, torch.bfloat16).cuda()) for m in (1, 17, 130, 400)]
    w = torch.ones(512).cuda()
    want = [_feed_forward(x, y, w, layer) for x, y in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    for _ in range(5):
        got = []
        for s, (x, y) in zip(streams, inputs):
            with torch.cuda.stream(s):
                got.append(_feed_forward(x, y, w, layer))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_two_graphs_that_share_weights(hip):
    """Each captured with its own buffers, replayed in turn with eager calls between, and checked each time."""
    layer = _layer(384, 700, 40)
    w = torch.ones(384).cuda()
    buffers, graphs, outs = [], [], []
    for m in (2, 150):
        x, y = torch.zeros((m, 384), dtype=torch.bfloat16, device="cuda"), torch.zeros((m, 384), dtype=torch.bfloat16, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _feed_forward(x, y, w, layer)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_feed_forward(x, y, w, layer))
        buffers.append((x, y))
        graphs.append(graph)
    for step in range(4):
        for i in (step % 2, 1 - step % 2):
            x, y = buffers[i]
            x.copy_(_randn(x.shape, 41 + step, torch.bfloat16))
            y.copy_(_randn(x.shape, 51 + step, torch.bfloat16))
            graphs[i].replay()
            want = _feed_forward(x, y, w, layer)
            torch.cuda.synchronize()
            assert torch.equal(outs[i][0], want[0]) and torch.equal(outs[i][1], want[1])


def test_threads_that_share_weights(hip):
    layer = _layer(256, 400, 60)
    w = torch.ones(256).cuda()
    inputs = [(_randn((m, 256), 61 + m, torch.bfloat16).cuda(), _randn((m, 256), 62 + m, torch.bfloat16).cuda()) for m in (1, 33, 257)]
    want = [_feed_forward(x, y, w, layer) for x, y in inputs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = _feed_forward(*inputs[i], w, layer)
                torch.cuda.current_stream().synchronize()
                if not (torch.equal(got[0], want[i][0]) and torch.equal(got[1], want[i][1])):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(inputs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_operands_are_not_written(hip):
    layer = _layer(300, 420, 70)
    for m in (3, 260):
        x, y = _randn((m, 300), 71, torch.float16).cuda(), _randn((m, 300), 72, torch.float16).cuda()
        rows = tt.fp8_quantize(x)
        before = [t.clone() for t in (x, y, _bytes(rows._codes), _bytes(rows._scales), layer["gate"]._packed, layer["gate"]._scales)]
        tt.rms_norm(x, residual=y, fp8=True)
        tt.fp8_gated_matmul(rows, layer["gate"], layer["up"])
        tt.fp8_matmul(rows, layer["gate"])
        for a, b in zip(before, (x, y, _bytes(rows._codes), _bytes(rows._scales), layer["gate"]._packed, layer["gate"]._scales)):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# the C interface: nothing outside a result is written
# ---------------------------------------------------------------------------
class _Guarded:
    """`size` bytes on the device with 4 KiB of 0xA5 on either side."""

    def __init__(self, size):
        self.all = torch.full((size + 8192,), 0xA5, dtype=torch.uint8, device="cuda")
        self.size = size

    @property
    def ptr(self):
        return self.all.data_ptr() + 4096

    def check(self):
        assert (self.all[:4096] == 0xA5).all() and (self.all[4096 + self.size:] == 0xA5).all()
        return self.all[4096: 4096 + self.size]


def _call(name, fmt, *fields):
    lib = _lib.load()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    status = getattr(lib, name)(struct.pack(fmt, *fields), stream)
    assert status == 0, lib.tt_last_error()


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (3, 130, 257), (17, 200, 128), (100, 257, 300), (300, 129, 700), (513, 1030, 200), (4100, 4110, 129)])
@pytest.mark.parametrize("e8m0", [True, False])
def test_c_calls_stay_in_their_results(hip, m, n, k, e8m0):
    gate, up = _matrix(n, k, 80, e8m0), _matrix(n, k, 81, e8m0)
    x = _randn((m, k), 82, torch.bfloat16).cuda()
    width, per_row = -(-k // 128) * 128, -(-(-(-k // 128)) // 4) * 4
    codes, scales = _Guarded(m * width), _Guarded(m * per_row)
    _call("tt_fp8_quantize", "=7q", _lib.TT_BF16, m, k, k, x.data_ptr(), codes.ptr, scales.ptr)
    rows = tt.fp8_quantize(x)
    assert torch.equal(codes.check().view(m, width), _bytes(rows._codes)) and torch.equal(scales.check().view(m, per_row), _bytes(rows._scales))
    total, codes2, scales2 = _Guarded(m * k * 2), _Guarded(m * width), _Guarded(m * per_row)
    _call("tt_rms_norm", "=6qd7q", _lib.TT_BF16, 0, m, k, k, k, 1e-6, x.data_ptr(), x.data_ptr(), 0, total.ptr, 0, codes2.ptr, scales2.ptr)
    normed, h = tt.rms_norm(x, residual=x, fp8=True)
    assert torch.equal(codes2.check().view(m, width), _bytes(normed._codes)) and torch.equal(scales2.check().view(m, per_row), _bytes(normed._scales))
    assert torch.equal(total.check().view(torch.bfloat16).view(m, k), h)
    plain = _Guarded(m * k * 2)
    _call("tt_rms_norm", "=6qd7q", _lib.TT_BF16, 0, m, k, k, 0, 1e-6, x.data_ptr(), 0, 0, 0, plain.ptr, 0, 0)
    assert torch.equal(plain.check().view(torch.bfloat16).view(m, k), tt.rms_norm(x))
    kind = _lib.TT_E8M0 if e8m0 else _lib.TT_F32
    for dtype, code in ((torch.bfloat16, _lib.TT_BF16), (torch.float16, _lib.TT_F16), (torch.float32, _lib.TT_F32)):
        y = _Guarded(m * n * dtype.itemsize)
        _call("tt_fp8_matmul", "=10q", code, kind, m, n, k, rows._codes.data_ptr(), rows._scales.data_ptr(), gate._packed.data_ptr(),
              gate._scales.data_ptr(), y.ptr)
        assert torch.equal(y.check().view(dtype).view(m, n), tt.fp8_matmul(rows, gate, dtype=dtype))
        y = _Guarded(m * n * dtype.itemsize)
        head = (code, kind, 0, m, n, k, rows._codes.data_ptr(), rows._scales.data_ptr(), gate._packed.data_ptr(), gate._scales.data_ptr(),
                up._packed.data_ptr(), up._scales.data_ptr())
        _call("tt_fp8_gated_matmul", "=17q", *head, y.ptr, 0, 0, 0, 0)
        want = tt.fp8_gated_matmul(tt.Fp8Rows(rows.codes, rows.scales, dtype), gate, up, fp8=False)
        assert torch.equal(y.check().view(dtype).view(m, n), want)
    width, per_row = -(-n // 128) * 128, -(-(-(-n // 128)) // 4) * 4
    codes, scales = _Guarded(m * width), _Guarded(m * per_row)
    query = struct.pack("=17q", *head, 0, codes.ptr, scales.ptr, 0, 0)
    room = _Guarded(_lib.load().tt_fp8_gated_workspace_bytes(query))
    _call("tt_fp8_gated_matmul", "=17q", *head, 0, codes.ptr, scales.ptr, room.ptr, room.size)
    room.check()
    want = tt.fp8_gated_matmul(rows, gate, up)
    assert torch.equal(codes.check().view(m, width), _bytes(want._codes)) and torch.equal(scales.check().view(m, per_row), _bytes(want._scales))


# ---------------------------------------------------------------------------
# refusals that the checks of the usual form hand on
# ---------------------------------------------------------------------------
def test_refusals(hip):
    mat, other = _matrix(128, 256, 90), _matrix(128, 300, 91)
    x, w = torch.ones((4, 256), device="cuda"), torch.ones(256, device="cuda")
    rows = tt.fp8_quantize(x)

    def asks(t):
        return t.clone().requires_grad_()

    for call, kind in (
        (lambda: tt.fp8_quantize(x.double()), NotImplementedError),
        (lambda: tt.fp8_quantize(x.long()), NotImplementedError),
        (lambda: tt.fp8_quantize(x[:, :0]), ValueError),
        (lambda: tt.fp8_quantize(asks(x)), RuntimeError),
        (lambda: tt.rms_norm(asks(x), w), RuntimeError),
        (lambda: tt.rms_norm(x, asks(w)), RuntimeError),
        (lambda: tt.rms_norm(x, w, residual=asks(x)), RuntimeError),
        (lambda: tt.rms_norm(x, w[:255]), ValueError),
        (lambda: tt.rms_norm(x, w.double()), NotImplementedError),
        (lambda: tt.rms_norm(x, w, residual=x[:3]), ValueError),
        (lambda: tt.rms_norm(x, w, residual=x.half()), ValueError),
        (lambda: tt.rms_norm(x, w, eps=-1.0), ValueError),
        (lambda: tt.rms_norm(x, w, eps=float("nan")), ValueError),
        (lambda: tt.fp8_matmul(rows, other), ValueError),
        (lambda: tt.fp8_matmul(x, other), ValueError),
        (lambda: tt.fp8_matmul(asks(x), mat), RuntimeError),
        (lambda: tt.fp8_matmul(rows, mat, dtype=torch.float64), NotImplementedError),
        (lambda: tt.fp8_gated_matmul(rows, mat, other), ValueError),
        (lambda: tt.fp8_gated_matmul(rows, other, other), ValueError),
        (lambda: tt.fp8_gated_matmul(rows, mat, _matrix(128, 256, 92, e8m0=False)), ValueError),
        (lambda: tt.fp8_gated_matmul(rows, mat, mat, activation="relu"), ValueError),
    ):
        with pytest.raises(kind):
            call()
    with torch.no_grad():  # nothing asks here
        assert torch.equal(tt.rms_norm(asks(x), asks(w)), tt.rms_norm(x, w))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: tt.fp8_quantize(dual), lambda: tt.rms_norm(dual, w), lambda: tt.rms_norm(x, w, residual=dual),
                     lambda: tt.fp8_matmul(dual, mat), lambda: tt.fp8_gated_matmul(dual, mat, mat)):
            with pytest.raises(RuntimeError):
                call()


@pytest.mark.parametrize("which", ["codes", "scales"])
def test_rows_whose_tensors_were_resized_are_refused(hip, which):
    mat = _matrix(128, 512, 93)
    for change in (lambda t: t.resize_(16, t.shape[1]), lambda t: t.resize_(4, t.shape[1]), lambda t: t.resize_(t.shape[1], 8),
                   lambda t: t.untyped_storage().resize_(8), lambda t: t.untyped_storage().resize_(0)):
        rows = tt.fp8_quantize(torch.ones((8, 512), device="cuda"))
        tt.fp8_matmul(rows, mat)
        change(getattr(rows, which))
        for call in (lambda: tt.fp8_matmul(rows, mat), lambda: tt.fp8_gated_matmul(rows, mat, mat)):
            with pytest.raises(RuntimeError, match="other memory"):
                call()


def test_rows_of_other_shapes_share_a_layout(hip):
    """One, two and more dimensions, and widths that need no padding and that do."""
    for shape in ((512,), (3, 512), (2, 3, 512), (2, 3, 130), (130,), (3, 256), (0, 512), (2, 0, 130)):
        x = _randn(shape, 94).cuda()
        rows = tt.fp8_quantize(x)
        assert rows.codes.shape == shape and rows.scales.shape == (*shape[:-1], -(-shape[-1] // 128))
        flat = tt.fp8_quantize(x.reshape(-1, shape[-1]))
        assert torch.equal(_bytes(rows.codes.contiguous()).view(-1), _bytes(flat.codes.contiguous()).view(-1))
        assert torch.equal(_bytes(rows.scales.contiguous()).view(-1), _bytes(flat.scales.contiguous()).view(-1))
        mat = _matrix(96, shape[-1], 95)
        assert torch.equal(tt.fp8_matmul(rows, mat).view(-1, 96), tt.fp8_matmul(flat, mat))
        again = tt.Fp8Rows(rows.codes, rows.scales, torch.float32)
        assert torch.equal(again.dequantize(), rows.dequantize())


def test_views_that_stand_for_their_negatives(hip):
    x, w, r = (_randn(s, 96 + i).cuda() for i, s in enumerate(((5, 256), (256,), (5, 256))))
    nx, nw, nr = (torch._neg_view(-t) for t in (x, w, r))
    assert torch.equal(nx, x) and nx.is_neg()
    assert torch.equal(_bytes(tt.fp8_quantize(nx).codes), _bytes(tt.fp8_quantize(x).codes))
    for got, want in zip(tt.rms_norm(nx, nw, residual=nr), tt.rms_norm(x, w, residual=r)):
        assert torch.equal(got, want)
    assert torch.equal(tt.rms_norm(x, nw), tt.rms_norm(x, w)) and torch.equal(tt.rms_norm(x, residual=nr)[0], tt.rms_norm(x, residual=r)[0])
    mat = _matrix(64, 256, 97)
    assert torch.equal(tt.fp8_matmul(nx, mat), tt.fp8_matmul(x, mat))
    assert torch.equal(tt.fp8_matmul(x, tt.Fp8Matrix.quantize(torch._neg_view(-r.cpu()))), tt.fp8_matmul(x, tt.Fp8Matrix.quantize(r)))


# ---------------------------------------------------------------------------
# offsets past 32 bits: the last rows give what they give alone
#
# Calls of other sizes sum a block's products alike and up to 64 blocks in another
# order: 64 additions and eight joins of at most 2^-23 of a running sum each, which is
# 64 blocks' largest at most, 72 64 2^-23 < 10^-3 of it. Two roundings to bfloat16
# are 2^-8 apart, two codes next to each other 2^-3.
# ---------------------------------------------------------------------------
MANY = (1 << 31) // 8192 + 5


def _ends(k, seed):
    """MANY rows of k elements, zeros but for the last seven, and those."""
    last = _randn((7, k), seed, torch.bfloat16).cuda()
    x = torch.zeros((MANY, k), dtype=torch.bfloat16, device="cuda")
    x[-7:] = last
    return x, last


@pytest.mark.parametrize("residual", [False, True])
def test_rows_past_32_bits(hip, residual):
    x, last = _ends(8192, 98)
    w = _randn((8192,), 99).cuda()
    if not residual:
        got, want = tt.fp8_quantize(x), tt.fp8_quantize(last)
        assert torch.equal(_bytes(got.codes[-7:]), _bytes(want.codes)) and torch.equal(_bytes(got.scales[-7:]), _bytes(want.scales))
        assert not _bytes(got.codes[:-7]).any() and not _bytes(got.scales[:-7]).any()
        mat = _matrix(20, 8192, 100)
        y = tt.fp8_matmul(got, mat)
        few = tt.fp8_matmul(want, mat).double()
        assert not y[:-7].any() and ((y[-7:].double() - few).abs() <= 2.0 ** -8 * few.abs() + 1e-3 * few.abs().max()).all()
    got = tt.rms_norm(x, w, residual=x if residual else None, fp8=True)
    want = tt.rms_norm(last, w, residual=last if residual else None, fp8=True)
    if residual:
        assert torch.equal(got[1][-7:], want[1]) and not got[1][:-7].any()
        got, want = got[0], want[0]
    assert torch.equal(_bytes(got.codes[-7:]), _bytes(want.codes)) and torch.equal(_bytes(got.scales[-7:]), _bytes(want.scales))


@pytest.mark.parametrize("e8m0", [True, False])
def test_results_past_32_bits(hip, e8m0):
    n, k = 8200, 128
    x, last = _ends(k, 101)
    gate, up = _matrix(n, k, 102, e8m0), _matrix(n, k, 103, e8m0)
    rows, few = tt.fp8_quantize(x), tt.fp8_quantize(last)
    for call in (lambda r: tt.fp8_matmul(r, gate), lambda r: tt.fp8_gated_matmul(r, gate, up, fp8=False)):
        y, want = call(rows), call(few).double()
        assert not y[:-7].any() and ((y[-7:].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-3 * want.abs().max()).all()
        del y
    got, want = tt.fp8_gated_matmul(rows, gate, up), tt.fp8_gated_matmul(few, gate, up)
    assert not _bytes(got.codes[:-7]).any()
    a, b = tt.Fp8Rows(got.codes[-7:], got.scales[-7:]).dequantize().double(), want.dequantize().double()
    assert ((a - b).abs() <= 2.0 ** -3 * b.abs() + 1e-3 * b.abs().max()).all()


@pytest.mark.parametrize("m", [1, 100])
def test_weights_past_32_bits(hip, m):
    """Rows of weights that repeat give columns that repeat, in whatever half of the memory they lie."""
    k = 8192
    codes = torch.zeros((MANY, k), dtype=torch.uint8, device="cuda")
    few = (100.0 * _randn((144, k), 104)).clamp(-448.0, 448.0).to(E4M3).cuda()
    first = (MANY - 144) // 128 * 128
    codes[first: first + 144] = _bytes(few)
    scales = torch.full((-(-MANY // 128), k // 128), 0.01, device="cuda")
    mat, small = tt.Fp8Matrix(codes.view(E4M3), scales), tt.Fp8Matrix(few, scales[:2])
    del codes
    x = tt.fp8_quantize(_randn((m, k), 105, torch.bfloat16).cuda())
    for call in (tt.fp8_matmul, lambda r, w: tt.fp8_gated_matmul(r, w, w, fp8=False)):
        y, want = call(x, mat), call(x, small).double()
        part = y[:, first: first + 144].double()
        assert ((part - want).abs() <= 2.0 ** -8 * want.abs() + 1e-3 * want.abs().max()).all()
        assert not y[:, :first].any() and not y[:, first + 144:].any()


@pytest.mark.parametrize("m", [1, 20])
def test_columns_past_what_tiles_reach(hip, m):
    """More than 2^23 columns, all but some thousand zeros. A sum errs by 2^-24 for each
    of 3000 terms of either sign, and what the 8-bit instructions drop of eight products
    is at most seven times 2^-13 of the largest, 7 2^-13 of all magnitudes; the activation
    is no steeper than 1.13, and results round by 2^-9."""
    n, k = 40, (1 << 23) + 200
    g = torch.Generator().manual_seed(m)
    where = torch.cat((torch.randint(0, k, (3000,), generator=g).unique(), torch.tensor([k - 1]))).unique()
    x = torch.zeros((m, k), dtype=torch.bfloat16)
    x[:, where] = torch.randn((m, len(where)), generator=g).to(torch.bfloat16)
    rows = tt.fp8_quantize(x.cuda())
    xv = rows.dequantize(torch.float32)[:, where.cuda()].cpu().double()
    assert ((xv - x[:, where].double()).abs() <= 2.0 ** -4 * x[:, where].double().abs() + 2.0 ** -10 * 2.0 ** -6).all()
    mats, values = [], []
    for seed in (1, 2):
        codes = torch.zeros((n, k), dtype=torch.uint8, device="cuda")
        few = (50.0 * torch.randn((n, len(where)), generator=g)).clamp(-448.0, 448.0).to(E4M3)
        codes[:, where.cuda()] = _bytes(few).cuda()
        mats.append(tt.Fp8Matrix(codes.view(E4M3), torch.full((1, -(-k // 128)), 2.0 ** -11, device="cuda")))
        values.append(few.double() * 2.0 ** -11)
    (gate, up), (wg, wu) = mats, values
    a, b = xv @ wg.t(), xv @ wu.t()
    da, db = (7 * 2.0 ** -13 + 3000 * 2.0 ** -24) * (xv.abs() @ wg.abs().t()), (7 * 2.0 ** -13 + 3000 * 2.0 ** -24) * (xv.abs() @ wu.abs().t())
    assert ((tt.fp8_matmul(rows, gate).cpu().double() - a).abs() <= 2.0 ** -8 * a.abs() + 1.01 * da).all()
    exact = tt.fp8_matmul(rows, gate, dtype=torch.float32).cpu().double()
    assert ((exact - a).abs() <= 2.0 ** -23 * a.abs() + 3000 * 2.0 ** -24 * (xv.abs() @ wg.abs().t())).all()
    h, err = a / (1 + torch.exp(-a)) * b, 1.13 * b.abs() * da + a.abs() * db + 1.13 * da * db
    assert ((tt.fp8_gated_matmul(rows, gate, up, fp8=False).cpu().double() - h).abs() <= 2.0 ** -8 * h.abs() + 1.01 * err).all()
    got = tt.fp8_gated_matmul(rows, gate, up)
    step = 2.0 ** -10 * got.scales.float().cpu().double()
    assert ((got.dequantize(torch.float32).cpu().double() - h).abs() <= 2.0 ** -4 * h.abs() + 1.07 * err + step).all()
    norm = tt.rms_norm(x.cuda()).cpu().double()
    want = x.double() / torch.sqrt((x.double() ** 2).mean(dim=1, keepdim=True) + 1e-6)
    assert ((norm - want).abs() <= (2.0 ** -8 + 2.0 ** -9) * want.abs()).all()
