"""Limits of the serving operators' calls and what they do with gradients,
without a GPU: everything here is refused before a launch."""

import struct

import pytest
import torch
from torch.autograd import forward_ad

import trntensor_amd as tt
from trntensor_amd.hip import _lib


@pytest.fixture
def lib():
    handle = _lib.load()
    assert handle is not None, _lib.load_error()
    return handle


def _attention(lib, cache=None, query=False, **kw):
    """tt_kv_attention (or its workspace) on pointers that no launch may see."""
    f = dict(dtype=3, batch=2, tokens=1, q_heads=2, window=0, sinks=0, width=4, stride=4, q0=1, q1=1, q2=1, scale=0.1, q=256,
             out=256, table=256, lengths=256, counts=0) | kw
    c = dict(k=256, v=256, k_scale=256, v_scale=256, pages=4, heads=2, page=16, dim=64) | (cache or {})
    tail = [f.pop("ws", 256), f.pop("ws_bytes", 1 << 50)]
    packed = struct.pack("=11qd15q", *f.values(), *c.values(), *tail)
    return lib.tt_kv_attention_workspace_bytes(packed) if query else lib.tt_kv_attention(packed, None)


@pytest.mark.parametrize("width", [4, 200, 4096])
def test_attention_refuses_more_pairs_than_one_launch_has_workgroups(lib, width):
    """A launch has at most 2^24 - 1 workgroups: whether a pair of sequence and
    head is one (short tables) or is joined by one (long tables)."""
    assert _attention(lib, batch=1 << 23, width=width) == _lib.TT_UNSUPPORTED
    assert lib.tt_last_error() == b"tt_kv_attention: 16777216 workgroups"


def test_attention_refuses_row_blocks_that_no_launch_holds(lib):
    """Workgroups of eight wavefronts count twice: 2^23 - 1 of them."""
    kw = dict(batch=1 << 20, cache=dict(heads=1), q_heads=1, width=1)
    assert _attention(lib, tokens=10 * 256, **kw) == _lib.TT_UNSUPPORTED
    assert lib.tt_last_error().startswith(b"tt_kv_attention: ")


class _Cache:
    """What the checks before a launch read of a cache."""

    head_dim, num_heads, page_size = 64, 2, 16
    device = torch.device("cpu")
    _host = None


class _Weights:
    shape = (8, 64)
    device = torch.device("cpu")
    _host = None


def _append(mark, name):
    x, cos = torch.zeros((2, 3, 2, 64)), torch.zeros((64, 32))
    kw = dict(k=x, v=x, q=x, cos=cos, sin=cos)
    kw[name] = mark(kw[name])
    table, held = torch.zeros((2, 4), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    return tt.kv_append(_Cache(), kw.pop("k"), kw.pop("v"), table, held, **kw)


def _attend(mark, name):
    q = mark(torch.zeros((2, 3, 2, 64)))
    return tt.kv_attention(q, _Cache(), torch.zeros((2, 4), dtype=torch.int32), torch.zeros(2, dtype=torch.int32))


def _multiply(mark, name):
    return tt.q4_matmul(mark(torch.zeros((3, 64))), _Weights())


def _dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


ROWS = [(_multiply, "x"), (_attend, "q"), (_append, "k"), (_append, "v"), (_append, "q")]


@pytest.mark.parametrize("context", [torch.enable_grad, torch.no_grad])
@pytest.mark.parametrize("call,name", ROWS)
def test_calls_refuse_tangents(call, name, context):
    """A dual tensor does not require grad, and no_grad leaves forward mode on."""
    with forward_ad.dual_level(), context(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
        call(_dual, name)


@pytest.mark.parametrize("name", ["cos", "sin"])
def test_append_refuses_derivatives_of_angles(name):
    with pytest.raises(RuntimeError, match="no backward"):
        _append(lambda t: t.clone().requires_grad_(), name)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
        _append(_dual, name)


@pytest.mark.parametrize("name", ["scales", "zeros"])
def test_weights_refuse_scales_that_ask_for_a_derivative(name):
    """The copies that are laid out would not be theirs any more."""
    kw = dict(scales=torch.ones((8, 1)), zeros=torch.ones((8, 1)))
    codes, plain = torch.zeros((8, 32), dtype=torch.uint8), kw[name]
    kw[name] = plain.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        tt.Q4Matrix(codes, kw["scales"], 64, 64, zeros=kw["zeros"])
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
        kw[name] = _dual(plain)
        tt.Q4Matrix(codes, kw["scales"], 64, 64, zeros=kw["zeros"])


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39])
def test_attention_refuses_a_scale_that_is_no_number(lib, scale):
    assert _attention(lib, scale=scale) == _lib.TT_INVALID
    assert lib.tt_last_error().startswith(b"tt_kv_attention: scale")
