"""The decoder of examples/decode.py with 8-bit weights on the GPU: its prompt pass
against the same layers from the operators' definitions in float64, and its steps
in a graph against its steps without one.

Tolerance of the prompt pass, fixed before its first run: the definitions round at
the same places, to 8 bits in front of each product and in the cache. What differs
are the results rounded to bfloat16 between operators, about ten a layer of at most
2^-9 of each element: sqrt(20) 2^-9 < 0.9% for two layers. Those errors carry a
value over the middle between two codes once in 2^-9 / 2^-4 = 2^-5 cases, by 2^-3 of
it: 2^-2.5 2^-3 < 2.3% of what a product reads, at four places a layer and two
in the cache, of independent signs: sqrt(12) 2.3% < 8% at the end of two layers,
of which the residual stream, several times as large as what a layer adds,
shows a part: 8% in all.
"""

import importlib.util
import os

import pytest
import torch

from oracle import fp8 as ref8
from oracle import serving as ref

pytestmark = pytest.mark.gpu

SMALL = dict(layers=2, hidden=192, q_heads=4, kv_heads=2, head_dim=64, mlp=320, vocab=500, max_tokens=256, pages=40, page_size=16, fp8=True)


@pytest.fixture
def decode(hip):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode.py")
    spec = importlib.util.spec_from_file_location("decode_example", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _weights(tt, mat):
    return tt.fp8_matmul(torch.eye(mat.shape[1]).cuda(), mat).t().cpu().double()


def _rounded(x):
    flat = x.reshape(-1, x.shape[-1])
    codes, e = ref8.quantize(flat)
    return (codes * ref8.spread(torch.exp2(e.double()), flat.shape[1])).view(x.shape)


def _norm(x):
    return ref8.rms_norm(x.reshape(-1, x.shape[-1]), None, None, 1e-6)[0].view(x.shape)


def _from_definitions(model, weights, tokens, table, lengths):
    """Hidden states of the prompt pass in float64."""
    B, T = tokens.shape
    HQ, H, D, P = model.q_heads, model.kv_heads, model.head_dim, model.page_size
    cos, sin = model.cos.cpu(), model.sin.cpu()
    held = torch.zeros_like(lengths)
    x = model.embed.cpu().double()[tokens]
    for w in weights:
        qkv = (_rounded(_norm(x)) @ w["qkv"].t()).view(B, T, HQ + 2 * H, D)
        q, k, v = qkv.split([HQ, H, H], dim=2)
        pages = int(table.max()) + 1
        cache = {"k": torch.zeros((pages, H, P, D), dtype=torch.float64), "v": torch.zeros((pages, H, D, P), dtype=torch.float64),
                 "k_scale": torch.ones((pages, H), dtype=torch.float64), "v_scale": torch.ones((pages, H), dtype=torch.float64)}
        q = ref.append(cache, k, v, table, held, lengths, q, cos, sin, False)
        o = torch.zeros((B, T, HQ, D), dtype=torch.float64)
        for b in range(B):
            n = int(lengths[b])
            o[b, :n] = ref.attention(q[b: b + 1, :n], cache, table[b: b + 1], lengths[b: b + 1], None, D ** -0.5, None, 0)[0][0]
        x = x + _rounded(o.flatten(2)) @ w["out"].t()
        h = _rounded(_norm(x))
        x = x + _rounded(ref8.act(h @ w["gate"].t(), "silu") * (h @ w["up"].t())) @ w["down"].t()
    return _norm(x)


def test_prompt_pass(decode):
    model = decode.Decoder(**SMALL)
    weights = [{k: _weights(decode.tt, m) for k, m in layer.items() if k != "cache"} for layer in model.layers]
    lengths = torch.tensor([37, 5, 20], dtype=torch.int32)
    tokens = torch.randint(0, 500, (3, 37), generator=torch.Generator().manual_seed(3))
    table = torch.randperm(12, generator=torch.Generator().manual_seed(4)).to(torch.int32).view(3, 4)
    with torch.no_grad():
        got = model.forward(tokens.cuda(), table.cuda(), torch.zeros(3, dtype=torch.int32).cuda(), lengths.cuda(), counts=lengths.cuda())
    want = _from_definitions(model, weights, tokens, table, lengths)
    for b, n in enumerate(lengths.tolist()):
        err = (got[b, :n].cpu().double() - want[b, :n]).norm() / want[b, :n].norm()
        assert err <= 0.08, f"{err:.3g}"


def test_graph_steps_are_the_eager_ones(decode):
    model = decode.Decoder(**SMALL)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, 500, (n,), generator=g) for n in (30, 7, 16)]
    eager, _ = decode.answer(model, prompts, 12, graph=False)
    tokens, _ = decode.answer(model, prompts, 12)
    assert eager.shape == (3, 12) and torch.equal(eager, tokens)
