"""Limits of the serving operators' calls and what they do with gradients,
without a GPU: everything here is refused before a launch."""

import struct

import pytest
import torch

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
