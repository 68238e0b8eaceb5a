"""What the serving operators refuse, and how they check their arguments,
without a GPU; the oracle's rounding against torch's."""

import struct

import pytest
import torch

import trntensor_amd as tt
from oracle import serving as ref
from trntensor_amd import serving
from trntensor_amd.hip import _lib, dispatch

F8 = torch.float8_e4m3fn


@pytest.fixture
def lib():
    handle = _lib.load()
    assert handle is not None, _lib.load_error()
    return handle


class _Cache:
    """What the checks before a launch read of a cache."""

    head_dim, num_heads, page_size = 64, 2, 16
    device = torch.device("cpu")
    _host = None


def _args(tokens=3, table=4):
    x = torch.zeros((2, tokens, 2, 64))
    return x, x, torch.zeros((2, table), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)


@pytest.fixture
def no_gpu(monkeypatch):
    monkeypatch.setattr(dispatch, "require_hip", lambda: None)

    def refuse(*a):
        raise AssertionError("a launch was reached")

    monkeypatch.setattr(serving, "_launch", refuse)


def test_oracle_rounding_is_the_formats():
    x = torch.cat([torch.linspace(-448, 448, 20001), torch.exp2(torch.linspace(-12, 8.7, 20001)),
                   torch.arange(256, dtype=torch.uint8).view(F8).float()])
    x = x[x.abs() <= 448]
    assert torch.equal(ref.round_e4m3(x), x.to(F8).double())
    assert ref.round_e4m3(torch.tensor([1e9, -1e9, float("inf")])).tolist() == [448.0, -448.0, 448.0]


@pytest.mark.parametrize("amax,scale", [(448.0, 1.0), (448.1, 2.0), (224.0, 0.5), (1.0, 2.0 ** -8), (0.0, 2.0 ** -64),
                                        (1e-30, 2.0 ** -64), (1.75, 2.0 ** -8), (1.76, 2.0 ** -7)])
def test_oracle_block_scale(amax, scale):
    assert ref.block_scale(torch.tensor([0.0, -amax])) == scale
    assert ref.block_scale(torch.tensor([float("inf"), amax, float("nan")])) == scale


def test_q4_matrix_checks():
    codes, scales = torch.zeros((8, 64), dtype=torch.uint8), torch.ones((8, 4))
    for bad in (codes.int(), codes[0], codes[:, :63]):
        with pytest.raises(ValueError, match="codes"):
            tt.Q4Matrix(bad, scales, 128, 32)
    with pytest.raises(ValueError, match="codes"):
        tt.Q4Matrix(codes, scales, 0, 32)
    for group in (0, 16, 48, 100, 160, -32):
        with pytest.raises(ValueError, match="group_size"):
            tt.Q4Matrix(codes, scales, 128, group)
    with pytest.raises(ValueError, match="scales"):
        tt.Q4Matrix(codes, scales[:, :3], 128, 32)
    with pytest.raises(ValueError, match="zeros"):
        tt.Q4Matrix(codes, scales, 128, 32, zeros=scales.half())
    with pytest.raises(NotImplementedError, match="float64"):
        tt.Q4Matrix(codes, scales.double(), 128, 32)


def test_cache_checks():
    k, v, s = torch.zeros((4, 2, 16, 64), dtype=F8), torch.zeros((4, 2, 64, 16), dtype=F8), torch.ones((4, 2))
    with pytest.raises(RuntimeError, match="HIP device"):
        tt.KVCache(k, v, s, s, head_dim=64)
    for args, kind, match in (((k[0], v, s, s, 64), ValueError, "4D"), ((k, v, s, s, 65), ValueError, "multiple of 64"),
                              ((k, v, s, s, 0), NotImplementedError, "head_dim"),
                              ((k, v, s, s, 257), NotImplementedError, "head_dim"),
                              ((k[:, :, :8], v, s, s, 64), ValueError, "page_size"),
                              ((k[:, :0], v, s, s, 64), ValueError, "head")):
        with pytest.raises(kind, match=match):
            tt.KVCache(*args)


def test_append_checks(no_gpu):
    c = _Cache()
    k, v, table, held = _args()
    cos = torch.zeros((64, 32))
    for call, kind, match in (
        (dict(k=k[0]), ValueError, "4D"),
        (dict(k=k[..., :32]), ValueError, "k must have shape"),
        (dict(v=v[:, :2]), ValueError, "v must have shape"),
        (dict(v=v[:, :, :1]), ValueError, "v must have shape"),
        (dict(k=k.double()), NotImplementedError, "float64"),
        (dict(v=v.half()), RuntimeError, "one dtype"),
        (dict(q=k.half(), cos=cos, sin=cos), RuntimeError, "one dtype"),
        (dict(q=k), ValueError, "cos and sin"),
        (dict(cos=cos), ValueError, "go together"),
        (dict(cos=cos, sin=cos[:, :3]), ValueError, "alike"),
        (dict(cos=cos.half(), sin=cos.half()), ValueError, "float32"),
        (dict(cos=cos[:63], sin=cos[:63]), ValueError, "63 positions"),
        (dict(cos=torch.zeros((64, 33)), sin=torch.zeros((64, 33))), ValueError, "33 pairs"),
        (dict(cos=cos[:, :0], sin=cos[:, :0]), ValueError, "0 pairs"),
        (dict(q=k[:1], cos=cos, sin=cos), ValueError, "q must have shape"),
        (dict(page_table=table[:1]), ValueError, "page_table"),
        (dict(page_table=table.long()), ValueError, "page_table must be int32"),
        (dict(lengths=held.long()), ValueError, "lengths must be int32"),
        (dict(lengths=held[:1]), ValueError, "lengths must have shape"),
        (dict(counts=held[None]), ValueError, "counts must have shape"),
        (dict(v=v.clone().requires_grad_()), RuntimeError, "no backward"),
    ):
        with pytest.raises(kind, match=match):
            kw = dict(k=k, v=v, page_table=table, lengths=held) | call
            tt.kv_append(c, kw.pop("k"), kw.pop("v"), kw.pop("page_table"), kw.pop("lengths"), **kw)


def test_attention_checks(no_gpu):
    c = _Cache()
    q, _, table, held = _args()
    for call, kind, match in (
        (dict(q=q[0]), ValueError, "4D"),
        (dict(q=q[:, :, :1]), ValueError, "1 query heads"),
        (dict(q=torch.zeros((2, 3, 5, 64))), ValueError, "5 query heads"),
        (dict(q=q[..., :63]), ValueError, "q must have shape"),
        (dict(q=q.double()), NotImplementedError, "float64"),
        (dict(q=q.clone().requires_grad_()), RuntimeError, "no backward"),
        (dict(window=0), ValueError, "window"),
        (dict(sinks=-1), ValueError, "sinks"),
        (dict(page_table=table[0]), ValueError, "page_table"),
        (dict(lengths=held.float()), ValueError, "lengths must be int32"),
    ):
        with pytest.raises(kind, match=match):
            kw = dict(q=q, page_table=table, lengths=held) | call
            tt.kv_attention(kw.pop("q"), c, kw.pop("page_table"), kw.pop("lengths"), **kw)
    # Nothing to do: no launch, and the result has its shape.
    assert tt.kv_attention(q[:, :0], c, table, held).shape == (2, 0, 2, 64)
    assert tt.kv_attention(q[:0], c, table[:0], held[:0]).shape == (0, 3, 2, 64)


# ---------------------------------------------------------------------------
# the C entry points refuse before any HIP call
# ---------------------------------------------------------------------------
def _cache_fields(**kw):
    f = dict(k=256, v=256, k_scale=256, v_scale=256, pages=4, heads=2, page=16, dim=64) | kw
    return list(f.values())


def _q4(lib, **kw):
    f = dict(dtype=0, scale_dtype=0, M=2, N=8, K=128, group=32, ldx=128, ldy=8, x=256, codes=256, scales=256, zeros=0, y=256,
             ws=0, ws_bytes=0) | kw
    return lib.tt_q4_matmul(struct.pack("=15q", *f.values()), None)


def test_c_q4_refusals(lib):
    assert lib.tt_q4_matmul(None, None) == _lib.TT_INVALID
    for kw in (dict(M=-1), dict(K=-1), dict(group=33), dict(group=16), dict(group=192), dict(ldx=127), dict(ldy=7), dict(codes=257),
               dict(scales=264), dict(zeros=8), dict(N=-1), dict(K=0), dict(x=0), dict(codes=0), dict(scales=0), dict(y=0)):
        assert _q4(lib, **kw) == _lib.TT_INVALID, kw
        assert lib.tt_last_error().startswith(b"tt_q4_matmul")
    for kw in (dict(dtype=1), dict(scale_dtype=1), dict(dtype=9)):
        assert _q4(lib, **kw) == _lib.TT_UNSUPPORTED, kw
    assert _q4(lib, M=0) == _lib.TT_OK and _q4(lib, N=0) == _lib.TT_OK


def test_c_q4_pack_refusals(lib):
    assert lib.tt_q4_packed_bytes(17, 129) == 2 * 2 * 1024 and lib.tt_q4_packed_bytes(0, 5) == 0
    for args in ((-1, 8, 256, 4, 256), (4, 0, 256, 4, 256), (4, 8, 0, 4, 256), (4, 8, 256, 4, 0), (4, 9, 256, 4, 256),
                 (4, 8, 256, 4, 264)):
        assert lib.tt_q4_pack(*args, None) == _lib.TT_INVALID, args
        assert lib.tt_last_error().startswith(b"tt_q4_pack")
    assert lib.tt_q4_pack(1 << 31, 8, 256, 4, 256, None) == _lib.TT_UNSUPPORTED
    assert lib.tt_q4_pack(0, 8, 0, 4, 0, None) == _lib.TT_OK


def _append(lib, cache=None, **kw):
    f = dict(dtype=0, batch=2, tokens=3, q_heads=0, rot=0, interleaved=0, width=4, stride=4, k0=1, k1=1, k2=1, v0=1, v1=1,
             v2=1, q0=1, q1=1, q2=1, k=256, v=256, q=0, q_out=0, cos=0, sin=0, table=256, lengths=256, counts=0) | kw
    return lib.tt_kv_append(struct.pack("=34q", *f.values(), *_cache_fields(**(cache or {}))), None)


def test_c_append_refusals(lib):
    assert lib.tt_kv_append(None, None) == _lib.TT_INVALID
    for kw in (dict(batch=-1), dict(tokens=-1), dict(width=-1), dict(k=0), dict(v=0), dict(lengths=0), dict(table=0),
               dict(cos=256), dict(cos=256, sin=256, rot=3), dict(cos=256, sin=256, rot=66), dict(q=256, q_out=256, q_heads=2),
               dict(q=256, cos=256, sin=256, rot=64, q_heads=2), dict(cache=dict(page=8)), dict(cache=dict(page=24)),
               dict(cache=dict(k=0)), dict(cache=dict(v=264)), dict(cache=dict(heads=0)), dict(cache=dict(dim=0))):
        assert _append(lib, **kw) == _lib.TT_INVALID, kw
        assert lib.tt_last_error().startswith(b"tt_kv_append")
    assert _append(lib, dtype=1) == _lib.TT_UNSUPPORTED
    assert _append(lib, cache=dict(dim=257)) == _lib.TT_UNSUPPORTED
    assert _append(lib, batch=1 << 40) == _lib.TT_UNSUPPORTED
    assert _append(lib, batch=0) == _lib.TT_OK and _append(lib, tokens=0) == _lib.TT_OK


def _attention(lib, cache=None, query=False, **kw):
    f = dict(dtype=0, batch=2, tokens=3, q_heads=4, window=0, sinks=0, width=4, stride=4, q0=1, q1=1, q2=1, scale=0.1, q=256,
             out=256, table=256, lengths=256, counts=0) | kw
    tail = [f.pop("ws", 0), f.pop("ws_bytes", 0)]
    packed = struct.pack("=11qd15q", *f.values(), *_cache_fields(**(cache or {})), *tail)
    return lib.tt_kv_attention_workspace_bytes(packed) if query else lib.tt_kv_attention(packed, None)


def test_c_attention_refusals(lib):
    assert lib.tt_kv_attention(None, None) == _lib.TT_INVALID
    assert lib.tt_kv_attention_workspace_bytes(None) == 0
    for kw in (dict(batch=-1), dict(tokens=-2), dict(window=-1), dict(sinks=-1), dict(q_heads=3), dict(q_heads=0), dict(q=0),
               dict(out=0), dict(table=0), dict(lengths=0), dict(cache=dict(page=0)), dict(cache=dict(k_scale=0))):
        assert _attention(lib, **kw) == _lib.TT_INVALID, kw
        assert lib.tt_last_error().startswith(b"tt_kv_attention")
    assert _attention(lib, dtype=3, cache=dict(dim=300)) == _lib.TT_UNSUPPORTED
    assert _attention(lib, dtype=5) == _lib.TT_UNSUPPORTED
    assert _attention(lib, batch=1 << 40) == _lib.TT_UNSUPPORTED
    assert _attention(lib, batch=0) == _lib.TT_OK and _attention(lib, tokens=0) == _lib.TT_OK
