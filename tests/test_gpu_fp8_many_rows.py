"""More rows than a launch has workgroups (2^24 of 256 threads), where one takes several:
heads of a long batch, say."""

import struct

import pytest
import torch

import trntensor_amd as tt
from trntensor_amd.hip import _lib

MANY = (1 << 24) + 5


def _bytes(t):
    return t.view(torch.uint8)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [8, 200])
def test_more_rows_than_workgroups(hip, k):
    g = torch.Generator().manual_seed(k)
    few = torch.randn((3, 7, k), generator=g).to(torch.bfloat16).cuda()
    at = (0, MANY // 2 + 1, MANY - 7)
    x = torch.zeros((MANY, k), dtype=torch.bfloat16, device="cuda")
    for i, rows in zip(at, few):
        x[i: i + 7] = rows
    other = torch.ones(MANY, dtype=torch.bool, device="cuda")
    for i in at:
        other[i: i + 7] = False
    got = tt.fp8_quantize(x)
    assert not (_bytes(got._codes).amax(dim=1) > 0)[other].any()
    for i, rows in zip(at, few):
        want = tt.fp8_quantize(rows)
        assert torch.equal(_bytes(got._codes)[i: i + 7], _bytes(want._codes))
        assert torch.equal(_bytes(got._scales)[i: i + 7], _bytes(want._scales))
    del got
    y, h = tt.rms_norm(x, residual=x)
    assert not (y.abs().amax(dim=1) > 0)[other].any()
    for i, rows in zip(at, few):
        for a, b in zip((y, h), tt.rms_norm(rows, residual=rows)):
            assert torch.equal(a[i: i + 7], b)


def test_calls_past_a_launch_are_refused():
    lib = _lib.load()
    most = (1 << 24) - 1
    for dim, each in ((1, 4), (1024, 4), (1025, 1), (1 << 30, 1)):
        for rows in (most * each + 1, 1 << 40, 1 << 62):
            args = struct.pack("=6qd7q", 0, 0, rows, dim, dim, dim, 1e-6, 256, 0, 0, 0, 256, 0, 0)
            assert lib.tt_rms_norm(args, None) == _lib.TT_UNSUPPORTED
    for dim, each in ((128, 16), (129, 8), (512, 4), (1024, 2), (2048, 1)):
        for rows in (most * each + 1, 1 << 40, 1 << 62):
            assert lib.tt_fp8_quantize(struct.pack("=7q", 0, rows, dim, dim, 256, 256, 256), None) == _lib.TT_UNSUPPORTED
