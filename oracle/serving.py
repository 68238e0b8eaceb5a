"""The serving operators from their definitions, in float64 on the CPU (test
infrastructure only): products with 4-bit weights, the append to a paged cache
of 8-bit floats, and attention over that cache. One sequence, head and block
at a time; nothing is shared with the product or its plain forms.
"""

from __future__ import annotations

import torch

E4M3 = torch.float8_e4m3fn


def q4_weights(codes: torch.Tensor, scales: torch.Tensor, k: int, group: int, zeros: torch.Tensor | None) -> torch.Tensor:
    """(n, k) float64 weights: scale * (code - zero)."""
    n = codes.shape[0]
    w = torch.empty((n, k), dtype=torch.float64)
    wide = codes.to(torch.int64)
    for j in range(k):
        c = wide[:, j // 2]
        c = c // 16 if j % 2 else c % 16
        z = 8.0 if zeros is None else zeros[:, j // group].double()
        w[:, j] = scales[:, j // group].double() * (c.double() - z)
    return w


def round_e4m3(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 values (steps of 2^(e-3), e no lower than -6), ties to
    even, saturated at 448; NaN stays NaN."""
    x = x.double().clamp(-448.0, 448.0)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -40))).clamp(min=-6.0)
    step = torch.exp2(e - 3.0)
    return torch.round(x / step) * step


def block_scale(x: torch.Tensor) -> float:
    """The smallest power of two >= 2^-64 that brings x's finite values to 448 or below."""
    x = x.double().abs()
    amax = x[x.isfinite()].max().item() if x.isfinite().any() else 0.0
    e = -64
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """x (heads, dim) rotated by one position's cos and sin (pairs,): float32
    products and sums, each rounded, as the operator defines them."""
    y = x.float().clone()
    half = cos.shape[0]
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        xa, xb = x[:, a].float(), x[:, b].float()
        y[:, a] = xa * cos[i] - xb * sin[i]
        y[:, b] = xb * cos[i] + xa * sin[i]
    return y


def append(cache: dict, k, v, table, lengths, counts, q, cos, sin, interleaved: bool) -> torch.Tensor | None:
    """Append in place to `cache` = {"k" [pages][heads][page][width], "v"
    [pages][heads][width][page], "k_scale", "v_scale"}: float64 code values and
    scales. Returns the rotated queries (float32, zeros past the counts)."""
    batch, tokens, heads, dim = k.shape
    pages, _, page, width = cache["k"].shape
    out = None if q is None else torch.zeros(q.shape)
    for b in range(batch):
        n = tokens if counts is None else min(int(counts[b]), tokens)
        held = int(lengths[b])
        new_k, new_v = {}, {}
        for t in range(n):
            p = held + t
            if p >= table.shape[1] * page:
                continue
            rk = k[b, t].float() if cos is None else rotate(k[b, t], cos[p], sin[p], interleaved)
            new_k[p], new_v[p] = rk.double(), v[b, t].double()
            if q is not None:
                out[b, t] = rotate(q[b, t], cos[p], sin[p], interleaved)
        for block in sorted({p // page for p in new_k}):
            at = int(table[b, block])
            if not 0 <= at < pages:
                continue
            slots = [p for p in new_k if p // page == block]
            older = min(slots) % page
            for h in range(heads):
                for name, new in (("k", new_k), ("v", new_v)):
                    codes = cache[name][at, h] if name == "k" else cache[name][at, h].t()  # (page, width) view
                    scale = block_scale(torch.stack([new[p][h] for p in slots]))
                    was = float(cache[name + "_scale"][at, h])
                    if older and was > scale:
                        scale = was
                    if older and scale > was:
                        codes[:older] = round_e4m3(codes[:older] * (was / scale))
                    for p in slots:
                        codes[p % page, :dim] = round_e4m3(new[p][h] / scale)
                        codes[p % page, dim:] = 0.0
                    cache[name + "_scale"][at, h] = scale
    return out


def attention(q, cache: dict, table, lengths, counts, scale: float, window: int | None, sinks: int):
    """(out, spread): float64 results, and for each row the largest sum over
    |q_d k_d| * |scale|, the largest |v| and the largest sum of p |v| among its
    keys, which bound what rounding may do to it. `cache` as in append."""
    batch, tokens, heads, dim = q.shape
    pages, kv_heads, page, _ = cache["k"].shape
    share = heads // kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64)
    spread = torch.zeros((batch, tokens, heads, 3), dtype=torch.float64)
    for b in range(batch):
        held = int(lengths[b])
        n = tokens if counts is None else int(counts[b])
        for kh in range(kv_heads):
            keys, values, place = [], [], []
            for block in range(min(-(-held // page), table.shape[1])):
                at = int(table[b, block])
                if not 0 <= at < pages:
                    continue
                m = min(page, held - block * page)
                keys.append(cache["k"][at, kh, :m, :dim] * cache["k_scale"][at, kh])
                values.append(cache["v"][at, kh, :dim, :m].t() * cache["v_scale"][at, kh])
                place += range(block * page, block * page + m)
            if not place:
                continue
            keys, values, place = torch.cat(keys), torch.cat(values), torch.tensor(place)
            for t in range(min(n, tokens)):
                pos = held - n + t
                seen = place <= pos
                if window is not None:
                    seen &= (place > pos - window) | (place < sinks)
                if pos < 0 or not seen.any():
                    continue
                for h in range(kh * share, (kh + 1) * share):
                    x = q[b, t, h].double()
                    score = (keys[seen] * x).sum(dim=1) * scale
                    prob = torch.softmax(score, dim=0)
                    out[b, t, h] = (prob[:, None] * values[seen]).sum(dim=0)
                    spread[b, t, h, 0] = (keys[seen] * x).abs().sum(dim=1).max() * abs(scale)
                    spread[b, t, h, 1] = values[seen].abs().max()
                    spread[b, t, h, 2] = (prob[:, None] * values[seen].abs()).sum(dim=0).max()
    return out, spread
