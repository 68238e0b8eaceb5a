"""A small decoder with 4-bit weights and a paged 8-bit cache, answering several
prompts at once: one ragged pass over the prompts, then one token of every
sequence at a time, the step captured in a HIP graph.

    python examples/decode.py [--layers 4] [--batch 8] [--prompt 500] [--tokens 64]

Weights are random: what it shows is how q4_matmul, kv_append and kv_attention
run together, and what a step costs.
"""

import argparse
import math
import os
import sys
import time

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import trntensor_amd as tt  # noqa: E402


def random_q4(out_features: int, in_features: int, group: int, g: torch.Generator) -> tt.Q4Matrix:
    """Random codes around zero point 8, scaled so that products keep their operand's size."""
    codes = torch.randint(0, 256, (out_features, (in_features + 1) // 2), generator=g, dtype=torch.uint8)
    groups = -(-in_features // group)
    scales = (0.5 + torch.rand((out_features, groups), generator=g)) / (4.6 * math.sqrt(in_features))
    return tt.Q4Matrix(codes.cuda(), scales.to(torch.bfloat16).cuda(), in_features, group)


class Decoder:
    """Pre-norm layers of grouped-query attention and a gated MLP."""

    def __init__(self, layers=4, hidden=1024, q_heads=8, kv_heads=2, head_dim=128, mlp=2816, vocab=4096, group=128,
                 max_tokens=2048, pages=512, page_size=64, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.page_size = page_size
        self.embed = torch.randn((vocab, hidden), generator=g).to(torch.bfloat16).cuda()
        width = (q_heads + 2 * kv_heads) * head_dim
        self.layers = [{"qkv": random_q4(width, hidden, group, g), "out": random_q4(hidden, q_heads * head_dim, group, g),
                        "up": random_q4(2 * mlp, hidden, group, g), "down": random_q4(hidden, mlp, group, g),
                        "cache": tt.KVCache.empty(pages, kv_heads, head_dim, page_size)} for _ in range(layers)]
        self.head = random_q4(vocab, hidden, group, g)
        angles = torch.arange(max_tokens)[:, None] * 10000.0 ** (-torch.arange(0, head_dim, 2) / head_dim)
        self.cos, self.sin = torch.cos(angles).float().cuda(), torch.sin(angles).float().cuda()

    def forward(self, tokens, table, held, total, counts=None):
        """Hidden states (batch, T, hidden) of T new tokens of every sequence, of
        which counts count; `held` and `total` are the lengths before and after."""
        B, T = tokens.shape
        HQ, H, D = self.q_heads, self.kv_heads, self.head_dim
        x = self.embed[tokens]
        norm = x.shape[-1:]
        for layer in self.layers:
            qkv = tt.q4_matmul(F.rms_norm(x, norm), layer["qkv"]).view(B, T, HQ + 2 * H, D)
            q, k, v = qkv.split([HQ, H, H], dim=2)
            q = tt.kv_append(layer["cache"], k, v, table, held, counts=counts, q=q, cos=self.cos, sin=self.sin)
            o = tt.kv_attention(q, layer["cache"], table, total, counts=counts)
            x = x + tt.q4_matmul(o.flatten(2), layer["out"])
            gate, up = tt.q4_matmul(F.rms_norm(x, norm), layer["up"]).chunk(2, dim=-1)
            x = x + tt.q4_matmul(F.silu(gate) * up, layer["down"])
        return F.rms_norm(x, norm)

    def next_token(self, x):
        """The likeliest next token after hidden states (batch, hidden)."""
        return tt.q4_matmul(x, self.head).argmax(-1)


@torch.no_grad()
def answer(model: Decoder, prompts: list[torch.Tensor], new_tokens: int, graph: bool = True):
    """Continues each prompt by `new_tokens` tokens; returns them (batch,
    new_tokens) and the seconds a step took."""
    B, longest = len(prompts), max(len(p) for p in prompts)
    lengths = torch.tensor([len(p) for p in prompts], dtype=torch.int32).cuda()
    padded = torch.zeros((B, longest), dtype=torch.int64)
    for row, p in zip(padded, prompts):
        row[: len(p)] = p
    per = -(-(longest + new_tokens) // model.page_size)
    # Any pages do; sequences' own lie apart here.
    table = torch.arange(B * per, dtype=torch.int32).view(per, B).t().contiguous().cuda()
    x = model.forward(padded.cuda(), table, torch.zeros_like(lengths), lengths, counts=lengths)
    token = model.next_token(x[torch.arange(B, device="cuda"), (lengths - 1).long()])
    held = lengths.clone()

    def step():
        total = held + 1
        y = model.forward(token[:, None], table, held, total)
        token.copy_(model.next_token(y[:, 0]))
        held.copy_(total)

    out = [token.clone()]
    run = step
    if graph and new_tokens > 2:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # one step outside the graph, so that everything is loaded
            step()
        torch.cuda.current_stream().wait_stream(side)
        out.append(token.clone())
        recorded = torch.cuda.CUDAGraph()
        with torch.cuda.graph(recorded):
            step()
        run = recorded.replay
    torch.cuda.synchronize()
    start, first = time.perf_counter(), len(out)
    while len(out) < new_tokens:
        run()
        out.append(token.clone())
    torch.cuda.synchronize()
    return torch.stack(out, 1), (time.perf_counter() - start) / max(1, new_tokens - first)


def main():
    a = argparse.ArgumentParser()
    for name, value in (("layers", 4), ("batch", 8), ("prompt", 500), ("tokens", 64)):
        a.add_argument(f"--{name}", type=int, default=value)
    a = a.parse_args()
    model = Decoder(layers=a.layers, max_tokens=(a.prompt + a.tokens + 64) // 64 * 64,
                    pages=a.batch * ((a.prompt + a.tokens) // 64 + 1))
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 4096, (max(1, a.prompt - 37 * i % a.prompt),), generator=g) for i in range(a.batch)]
    eager, slow = answer(model, prompts, a.tokens, graph=False)
    tokens, fast = answer(model, prompts, a.tokens)
    assert torch.equal(eager, tokens)
    print(f"{a.batch} sequences, {a.layers} layers: {slow * 1e6:.0f} us a step, {fast * 1e6:.0f} us as a graph "
          f"({a.batch / fast:.0f} tokens/s)")


if __name__ == "__main__":
    main()
