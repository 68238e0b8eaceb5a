"""The decoder of examples/decode.py on the GPU: its prompt pass against the
same layers from the operators' definitions in float64, and its steps in a
graph against its steps without one.

Tolerance of the prompt pass, fixed before its first run: a layer rounds about
ten intermediate results to bfloat16, an error of at most 2^-9 of each element
and independent, so that two layers give about sqrt(20) 2^-9 < 0.9% of the
result. Keys and values that those errors carry over the middle between two
codes move by a whole step, 1/8 of them at most: one in 2^9 * 2^-3 steps, an
error of sqrt(2^-6) / 8 < 1.6%. Both, for an unlucky case doubled: 5%.
"""

import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

from oracle import serving as ref

pytestmark = pytest.mark.gpu

SMALL = dict(layers=2, hidden=192, q_heads=4, kv_heads=2, head_dim=64, mlp=320, vocab=500, group=64, max_tokens=256,
             pages=40, page_size=16)


@pytest.fixture
def decode(hip):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode.py")
    spec = importlib.util.spec_from_file_location("decode_example", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _from_definitions(model, weights, tokens, table, lengths):
    """Hidden states of the prompt pass in float64."""
    B, T = tokens.shape
    HQ, H, D, P = model.q_heads, model.kv_heads, model.head_dim, model.page_size
    cos, sin = model.cos.cpu(), model.sin.cpu()
    held = torch.zeros_like(lengths)
    x = model.embed.cpu().double()[tokens]
    norm = x.shape[-1:]
    for w in weights:
        qkv = (F.rms_norm(x, norm) @ w["qkv"].t()).view(B, T, HQ + 2 * H, D)
        q, k, v = qkv.split([HQ, H, H], dim=2)
        pages = int(table.max()) + 1
        cache = {"k": torch.zeros((pages, H, P, D), dtype=torch.float64), "v": torch.zeros((pages, H, D, P), dtype=torch.float64),
                 "k_scale": torch.ones((pages, H), dtype=torch.float64), "v_scale": torch.ones((pages, H), dtype=torch.float64)}
        q = ref.append(cache, k, v, table, held, lengths, q, cos, sin, False)
        # Rows of unequal prompts: each sequence by itself, its own rows its last.
        o = torch.zeros((B, T, HQ, D), dtype=torch.float64)
        for b in range(B):
            n = int(lengths[b])
            o[b, :n] = ref.attention(q[b : b + 1, :n], cache, table[b : b + 1], lengths[b : b + 1], None, D ** -0.5, None, 0)[0][0]
        x = x + o.flatten(2) @ w["out"].t()
        gate, up = (F.rms_norm(x, norm) @ w["up"].t()).chunk(2, dim=-1)
        x = x + (F.silu(gate) * up) @ w["down"].t()
    return F.rms_norm(x, norm)


def test_prompt_pass(decode, monkeypatch):
    kept = []
    made = decode.tt.Q4Matrix

    def keep(codes, scales, k, group):
        w = made(codes, scales, k, group)
        kept.append(ref.q4_weights(codes.cpu(), scales.cpu(), k, group, None))
        return w

    monkeypatch.setattr(decode.tt, "Q4Matrix", keep)
    model = decode.Decoder(**SMALL)
    weights = [dict(zip(("qkv", "out", "up", "down"), kept[4 * i : 4 * i + 4])) for i in range(SMALL["layers"])]
    g = torch.Generator().manual_seed(3)
    tokens = torch.randint(0, 500, (3, 21), generator=g)
    lengths = torch.tensor([21, 1, 14], dtype=torch.int32)
    table = torch.arange(6, dtype=torch.int32).view(2, 3).t().contiguous()
    with torch.no_grad():
        got = model.forward(tokens.cuda(), table.cuda(), torch.zeros(3, dtype=torch.int32).cuda(), lengths.cuda(),
                            counts=lengths.cuda()).cpu().double()
    want = _from_definitions(model, weights, tokens, table, lengths)
    for b in range(3):
        n = int(lengths[b])
        err = ((got[b, :n] - want[b, :n]).norm() / want[b, :n].norm()).item()
        assert err < 0.05, (b, err)


def test_steps_in_a_graph(decode):
    model = decode.Decoder(**SMALL)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 500, (n,), generator=g) for n in (40, 1, 17)]
    eager, _ = decode.answer(model, prompts, 24, graph=False)
    tokens, _ = decode.answer(model, prompts, 24)
    assert eager.shape == (3, 24) and torch.equal(eager, tokens)
