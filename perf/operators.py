"""The language-model serving operators as they are measured, beside their
plain forms.

One decode step of a transformer layer is a chain of contractions: project
with compressed weights, put the new keys and values into the cache, contract
queries with keys and probabilities with values, project again. Each case is
one pass through one of the three operators that make up the chain:

  q4       q4_matmul: activations times weights held in 4 bits, with a scale
           (and a zero point, or 8) for each group along the summed axis
  append   kv_append: new keys and values, rotated by their positions, into a
           paged cache of 8-bit floats with one scale per page and head; the
           queries are rotated on the way
  attend   kv_attention: queries against that cache, causal, optionally with
           a sliding window and some first tokens that stay visible

`run` computes the plain form (elementary torch operations in 32 bits, rounded
once) unless `own` is set, in which case it makes the framework's calls.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_FP8 = torch.float8_e4m3fn


def listed() -> list[dict]:
    return [
        # One token through a small projection: latency is all there is.
        {"name": "q4_token_small", "kind": "q4", "dtype": "f16", "m": 1, "n": 1024, "k": 1024, "group": 64,
         "zeros": True},
        # One token through an ordinary projection.
        {"name": "q4_token", "kind": "q4", "dtype": "bf16", "m": 1, "n": 4096, "k": 4096, "group": 128,
         "zeros": False},
        # A few rows, every extent odd, in 32 bits (checking a model's layers).
        {"name": "q4_ragged_f32", "kind": "q4", "dtype": "f32", "m": 5, "n": 3001, "k": 1999, "group": 32,
         "zeros": True},
        # A decode batch of 32 sequences through a wide projection (67 MB of codes).
        {"name": "q4_batch", "kind": "q4", "dtype": "bf16", "m": 32, "n": 16384, "k": 8192, "group": 128,
         "zeros": True},
        # One new token for each of 8 sequences.
        {"name": "append_token", "kind": "append", "dtype": "bf16", "batch": 8, "tokens": 1, "heads": 8, "share": 4,
         "dim": 128, "rot": 128, "interleaved": False, "page": 64, "length": 500, "ragged": 60},
        # Short drafts of unequal length, small pages, a head size that is no
        # power of two and rotated in part, neighbouring pairs.
        {"name": "append_draft_f16", "kind": "append", "dtype": "f16", "batch": 13, "tokens": 37, "heads": 5,
         "share": 3, "dim": 80, "rot": 32, "interleaved": True, "page": 16, "length": 333, "ragged": 100},
        # Four long prompts going into an empty cache.
        {"name": "append_prompt", "kind": "append", "dtype": "bf16", "batch": 4, "tokens": 4096, "heads": 8,
         "share": 4, "dim": 128, "rot": 128, "interleaved": False, "page": 64, "length": 0, "ragged": 0},
        # One sequence at the start of its answer.
        {"name": "attend_short", "kind": "attend", "dtype": "bf16", "batch": 1, "tokens": 1, "heads": 8, "share": 4,
         "dim": 128, "page": 64, "length": 200, "ragged": 0, "window": 0, "sinks": 0},
        # A decode batch of unequal contexts, the last slot of it unused.
        {"name": "attend_batch", "kind": "attend", "dtype": "bf16", "batch": 48, "tokens": 1, "heads": 8, "share": 4,
         "dim": 128, "page": 16, "length": 4096, "ragged": 100, "window": 0, "sinks": 0},
        # Two long documents (537 MB of cache).
        {"name": "attend_long", "kind": "attend", "dtype": "bf16", "batch": 2, "tokens": 1, "heads": 8, "share": 4,
         "dim": 128, "page": 64, "length": 131071, "ragged": 1, "window": 0, "sinks": 0},
        # Three drafted tokens a sequence in a model whose layer sees the last
        # thousand tokens and the first four, one key head per query head.
        {"name": "attend_window_f16", "kind": "attend", "dtype": "f16", "batch": 16, "tokens": 3, "heads": 16,
         "share": 1, "dim": 96, "page": 32, "length": 8001, "ragged": 90, "window": 1000, "sinks": 4},
        # A prompt's last chunk of 2048 tokens against 8192.
        {"name": "attend_chunk", "kind": "attend", "dtype": "bf16", "batch": 1, "tokens": 2048, "heads": 8,
         "share": 4, "dim": 128, "page": 64, "length": 8192, "ragged": 0, "window": 0, "sinks": 0},
    ]


# The most that a drawn case may cost: its kind's largest listed cases.
_MOST_Q4 = 16384 * 8192
_MOST_APPEND = 4 * 4096 * 8 * 128
_MOST_CACHE = 2 * 131071 * 8 * 128
_MOST_SCORES = 2048 * 8192 * 32


def _log_int(rng, lo: int, hi: int) -> int:
    """An integer in [lo, hi], its logarithm uniform."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    """One more case of the listed ranges."""
    kind = rng.choice(("q4", "append", "attend"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    while True:
        if kind == "q4":
            case = {"kind": "q4", "dtype": dtype, "m": _log_int(rng, 1, 64), "n": _log_int(rng, 200, 16384),
                    "k": _log_int(rng, 200, 8192), "group": rng.choice((32, 64, 128)), "zeros": rng.random() < 0.5}
            if rng.random() < 0.5:  # most layers are multiples of 128, not all
                case["n"], case["k"] = -(-case["n"] // 128) * 128, -(-case["k"] // 128) * 128
            if case["n"] * case["k"] <= _MOST_Q4 and case["m"] * case["n"] * case["k"] <= 32 * _MOST_Q4:
                return case
            continue
        heads = {"dtype": dtype, "heads": rng.choice((1, 2, 4, 5, 8, 16)), "share": rng.choice((1, 2, 3, 4, 5, 8)),
                 "dim": rng.choice((64, 80, 96, 128, 128, 256)), "page": rng.choice((16, 32, 64, 128)),
                 "ragged": rng.randint(0, 100)}
        if kind == "append":
            tokens = 1 if rng.random() < 0.4 else _log_int(rng, 2, 4096)
            length = rng.choice((0, _log_int(rng, 1, 4096)))
            case = {"kind": "append", "batch": _log_int(rng, 1, 64), "tokens": tokens, "length": length,
                    "rot": rng.choice((32, 64, heads["dim"])), "interleaved": rng.random() < 0.5, **heads}
            size = case["heads"] * case["dim"] * case["batch"]
            if size * tokens * (2 + case["share"]) <= 6 * _MOST_APPEND and size * (length + tokens) <= 8 * _MOST_APPEND:
                return case
        else:
            length = _log_int(rng, 1, 131071)
            tokens = 1 if rng.random() < 0.5 else min(length, _log_int(rng, 2, 2048))
            window, sinks = (0, 0) if rng.random() < 0.6 else (_log_int(rng, 16, 4096), rng.choice((0, 1, 4, 7)))
            case = {"kind": "attend", "batch": _log_int(rng, 1, 64), "tokens": tokens, "length": length,
                    "window": window, "sinks": sinks, **heads}
            cache = case["batch"] * length * case["heads"] * case["dim"]
            scores = case["batch"] * length * case["heads"] * case["share"] * tokens
            most = _MOST_SCORES if dtype != "f32" else _MOST_SCORES // 4
            if cache <= _MOST_CACHE and scores * max(128, case["dim"]) <= most * 128:
                return case


def _lengths(case: dict) -> list[int]:
    """Tokens held for each sequence: from `length` down by `ragged` percent."""
    b, n = case["batch"], case["length"]
    return [n - n * case["ragged"] * i // (100 * max(1, b - 1)) for i in range(b)]


def _counts(case: dict) -> list[int]:
    """New tokens of each sequence: from `tokens` down by half of `ragged`
    percent, and in `attend` no more than it holds."""
    b, t = case["batch"], case["tokens"]
    some = [t - t * case["ragged"] * i // (200 * max(1, b - 1)) for i in range(b)]
    return [min(c, n) for c, n in zip(some, _lengths(case))] if case["kind"] == "attend" else some


def _pages(case: dict) -> int:
    """Entries of the page table that each sequence has."""
    most = case["length"] + (case["tokens"] if case["kind"] == "append" else 0)
    return max(1, -(-most // case["page"]))


def _pad(dim: int) -> int:
    """A cache row holds its head size rounded up to a multiple of 64."""
    return -(-dim // 64) * 64


def _cache(g, case: dict, total: int) -> dict:
    """Codes as a block with its largest magnitude near the format's largest
    has them, and power-of-two scales: keys [page][head][token][dim], values
    [page][head][dim][token], both padded along dim."""
    h, p, d = case["heads"], case["page"], case["dim"]

    def codes(*shape):
        # A few heads' worth at a time, so that no 32-bit copy of it all is held.
        out = torch.empty(shape, dtype=_FP8, device="cuda")
        for part in out.split(max(1, (1 << 26) // math.prod(shape[1:]))):
            part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(90.0).clamp_(-448.0, 448.0))
        return out

    k, v = codes(total, h, p, _pad(d)), codes(total, h, _pad(d), p)
    k.view(torch.uint8)[..., d:] = 0
    v.view(torch.uint8)[..., d:, :] = 0
    scale = [torch.exp2(torch.randint(-8, -5, (total, h), generator=g, device="cuda").float()) for _ in range(2)]
    return {"k": k, "v": v, "k_scale": scale[0], "v_scale": scale[1]}


def _table(g, case: dict, total: int, held: list[int]) -> torch.Tensor:
    """A page table over shuffled pages; -1 past the end of a sequence."""
    b, n = case["batch"], _pages(case)
    table = torch.randperm(total, generator=g, device="cuda")[: b * n].to(torch.int32).reshape(b, n)
    used = torch.tensor([-(-t // case["page"]) for t in held], device="cuda")
    return torch.where(torch.arange(n, device="cuda") < used[:, None], table, -1)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    state = {"case": case}
    if case["kind"] == "q4":
        n, k, groups = case["n"], case["k"], -(-case["k"] // case["group"])
        state["x"] = torch.randn((case["m"], k), generator=g, device="cuda").to(dt)
        codes = torch.randint(0, 256, (n, -(-k // 2)), generator=g, device="cuda", dtype=torch.uint8)
        scales = (0.02 * (0.5 + torch.rand((n, groups), generator=g, device="cuda"))).to(dt)
        zeros = torch.randint(5, 11, (n, groups), generator=g, device="cuda").to(dt) if case["zeros"] else None
        if own:  # the program's weights: laid out once
            import trntensor_amd as tt

            state["w"] = tt.Q4Matrix(codes, scales, k, case["group"], zeros=zeros)
        else:
            state["codes"], state["scales"], state["zeros"] = codes, scales, zeros
        return state
    b, t, h, s, d = case["batch"], case["tokens"], case["heads"], case["share"], case["dim"]
    lengths, counts = _lengths(case), _counts(case)
    total = b * _pages(case) + 3
    cache = _cache(g, case, total)
    held = [n + c for n, c in zip(lengths, counts)] if case["kind"] == "append" else lengths
    state["table"] = _table(g, case, total, held)
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    state["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
    if case["kind"] == "append":
        # One projection's output, of which queries, keys and values are views.
        qkv = torch.randn((b, t, (s + 2) * h, d), generator=g, device="cuda").to(dt)
        state["q"], state["k"], state["v"] = qkv.split([s * h, h, h], dim=2)
        place = torch.arange(_pages(case) * case["page"], device="cuda", dtype=torch.float64)
        turn = torch.exp(torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64)
                         * (-2.0 * math.log(10000.0) / case["rot"]))
        angle = place[:, None] * turn
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    else:
        state["q"] = torch.randn((b, t, s * h, d), generator=g, device="cuda").to(dt)
    if own:
        import trntensor_amd as tt

        state["cache"] = tt.KVCache(cache["k"], cache["v"], cache["k_scale"], cache["v_scale"], head_dim=d)
    else:
        state["cache"] = cache
    return state


def run(state: dict):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["kind"] == "q4":
        return _plain_q4(case, state)
    return _plain_append(case, state) if case["kind"] == "append" else _plain_attend(case, state)


def _run_own(case: dict, st: dict):
    import trntensor_amd as tt

    if case["kind"] == "q4":
        return tt.q4_matmul(st["x"], st["w"])
    cache = st["cache"]
    if case["kind"] == "append":
        q = tt.kv_append(cache, st["k"], st["v"], st["table"], st["lengths"], counts=st["counts"], q=st["q"],
                         cos=st["cos"], sin=st["sin"], interleaved=case["interleaved"])
        return {"q": q, "k": cache.k, "v": cache.v, "k_scale": cache.k_scale, "v_scale": cache.v_scale}
    return tt.kv_attention(st["q"], cache, st["table"], st["lengths"], counts=st["counts"],
                           window=case["window"] or None, sinks=case["sinks"])


def _plain_q4(case: dict, st: dict) -> torch.Tensor:
    n, k = case["n"], case["k"]
    codes = torch.stack((st["codes"] & 15, st["codes"] >> 4), dim=2).reshape(n, -1)[:, :k].float()
    group = torch.arange(k, device="cuda") // case["group"]
    zeros = 8.0 if st["zeros"] is None else st["zeros"].float()[:, group]
    w = (codes - zeros) * st["scales"].float()[:, group]
    return (st["x"].float() @ w.t()).to(st["x"].dtype)


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """Pairs (a, b) of x's first dims become (a cos - b sin, b cos + a sin);
    cos and sin broadcast against [batch, token, head, pair]."""
    half = cos.shape[-1]
    turned, rest = x[..., : 2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _exponent(amax: torch.Tensor) -> torch.Tensor:
    """The smallest e with amax <= 448 * 2^e, and not below -64."""
    m, e = torch.frexp(amax)  # amax = m * 2^e with m in [0.5, 1); 448 = 0.875 * 2^9
    return torch.where(amax > 0, (e - 9 + (m > 0.875).int()), -64).clamp(min=-64)


def _stored(new, old, old_scale, is_new, is_old, had):
    """Codes and scales of the touched blocks: `new` values and `old` codes are
    [..., token, dim], `is_new`/`is_old` say which tokens are which."""
    size = torch.where(is_new & new.isfinite(), new.abs(), 0.0).amax(dim=(-2, -1))
    scale = torch.exp2(_exponent(size).float())
    scale = torch.where(had, torch.maximum(scale, old_scale), scale)
    up = (new / scale[..., None, None]).clamp(-448.0, 448.0).to(_FP8).view(torch.uint8)
    again = (old.view(_FP8).float() * (old_scale / scale)[..., None, None]).to(_FP8).view(torch.uint8)
    return torch.where(is_new, up, torch.where(is_old, again, old)), scale


def _plain_append(case: dict, st: dict) -> dict:
    cache, p, t = st["cache"], case["page"], case["tokens"]
    lengths, counts, dt = st["lengths"].long(), st["counts"].long(), st["q"].dtype
    at = (lengths[:, None] + torch.arange(t, device="cuda")).clamp(max=st["cos"].shape[0] - 1)
    cos, sin = st["cos"][at][:, :, None], st["sin"][at][:, :, None]
    valid = (torch.arange(t, device="cuda") < counts[:, None])[:, :, None, None]
    q = torch.where(valid, _rotate(st["q"].float(), cos, sin, case["interleaved"]), 0.0).to(dt)
    k = _rotate(st["k"].float(), cos, sin, case["interleaved"])
    v = st["v"].float()
    # The blocks that the new tokens may touch: [batch, block], and which token
    # of its sequence each of their slots is.
    block = (lengths // p)[:, None] + torch.arange((t + p - 2) // p + 1, device="cuda")
    slot = block[:, :, None] * p + torch.arange(p, device="cuda")
    first, last = lengths[:, None, None], (lengths + counts)[:, None, None]
    is_new, is_old = (slot >= first) & (slot < last), slot < first
    touched = is_new.any(dim=2)
    page = st["table"].long().gather(1, block.clamp(max=st["table"].shape[1] - 1))
    page, had = page[touched], is_old.any(dim=2)[touched][:, None]
    row = torch.arange(case["batch"], device="cuda")[:, None, None]
    index = (slot - first).clamp(0, t - 1)
    is_new, is_old = is_new[touched][:, None, :, None], is_old[touched][:, None, :, None]
    pad = (0, _pad(case["dim"]) - case["dim"])
    new_k, new_v = (torch.nn.functional.pad(x[row, index][touched].transpose(1, 2), pad) for x in (k, v))
    kb, ks = _stored(new_k, cache["k"].view(torch.uint8)[page], cache["k_scale"][page], is_new, is_old, had)
    old_v = cache["v"].view(torch.uint8)[page].transpose(2, 3)
    vb, vs = _stored(new_v, old_v, cache["v_scale"][page], is_new, is_old, had)
    cache["k"].view(torch.uint8)[page] = kb
    cache["v"].view(torch.uint8)[page] = vb.transpose(2, 3)
    cache["k_scale"][page], cache["v_scale"][page] = ks, vs
    return {"q": q, "k": cache["k"], "v": cache["v"], "k_scale": cache["k_scale"], "v_scale": cache["v_scale"]}


def _visible(case: dict, pos: torch.Tensor, key: torch.Tensor) -> torch.Tensor:
    """Whether the token at position `pos` sees the one at `key`."""
    seen = key <= pos
    if case["window"]:
        seen = seen & ((key > pos - case["window"]) | (key < case["sinks"]))
    return seen


def _plain_attend(case: dict, st: dict) -> torch.Tensor:
    cache, q = st["cache"], st["q"]
    b, t, h, s, d = case["batch"], case["tokens"], case["heads"], case["share"], case["dim"]
    page = st["table"].long().clamp(min=0)
    n = page.shape[1] * case["page"]
    k = cache["k"].view(torch.uint8)[page].view(_FP8)[..., :d].float() * cache["k_scale"][page][..., None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(b, h, n, d)
    q = q.float().reshape(b, t, h, s, d).permute(0, 2, 1, 3, 4).reshape(b, h, t * s, d)
    score = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(d)).reshape(b, h, t, s, n)
    pos = (st["lengths"] - st["counts"])[:, None] + torch.arange(t, device="cuda")
    seen = _visible(case, pos[:, :, None], torch.arange(n, device="cuda"))
    seen = seen & (torch.arange(t, device="cuda") < st["counts"][:, None])[:, :, None]
    score = score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    prob = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = prob.sum(dim=-1, keepdim=True)
    v = cache["v"].view(torch.uint8)[page].view(_FP8)[..., :d, :].float() * cache["v_scale"][page][..., None, None]
    v = v.permute(0, 2, 1, 4, 3).reshape(b, h, n, d)
    v = torch.where((torch.arange(n, device="cuda") < st["lengths"][:, None])[:, None, :, None], v, 0.0)
    out = (prob.reshape(b, h, t * s, n) @ v).reshape(b, h, t, s, d)
    out = torch.where(seen.any(dim=-1)[:, None, :, None, None], out / total, 0.0)
    return out.permute(0, 2, 1, 3, 4).reshape(b, t, h * s, d).to(st["q"].dtype)


def work(case: dict) -> dict:
    es = _SIZE[case["dtype"]]
    if case["kind"] == "q4":
        m, n, k, groups = case["m"], case["n"], case["k"], -(-case["k"] // case["group"])
        return {"bytes": n * k / 2 + es * (n * groups * (2 if case["zeros"] else 1) + m * k + m * n),
                "flops": 2 * m * n * k}
    h, s, d = case["heads"], case["share"], case["dim"]
    counts = _counts(case)
    if case["kind"] == "append":
        new = sum(counts)
        blocks = sum(1 if c == 1 else c // case["page"] + 1 for c in counts if c)
        return {"bytes": new * h * d * (2 * s * es + 2 * es + 2) + blocks * h * 8 + new * case["rot"] * 4,
                "flops": 3 * new * h * (s + 1) * case["rot"] + 2 * new * h * d}
    kept = rows = pairs = 0
    for n, c in zip(_lengths(case), counts):
        if not c:
            continue
        rows += c
        if case["window"]:
            start = max(0, n - c + 1 - case["window"])
            kept += n - start + min(case["sinks"], start)
            for pos in range(n - c, n):
                low = max(0, pos + 1 - case["window"])
                pairs += pos + 1 - low + min(case["sinks"], low)
        else:
            kept += n
            pairs += c * n - c * (c - 1) // 2
    return {"bytes": 2 * kept * h * d + kept // case["page"] * h * 8 + 2 * rows * h * s * d * es,
            "flops": 4 * pairs * h * s * d}


def exact(case: dict, seed: int):
    global own
    keep, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = keep
    if case["kind"] == "q4":
        return _exact_q4(case, st)
    return _exact_append(case, st) if case["kind"] == "append" else _exact_attend(case, st)


def _exact_q4(case: dict, st: dict) -> torch.Tensor:
    n, k, g = case["n"], case["k"], case["group"]
    w = torch.empty((n, 2 * st["codes"].shape[1]), dtype=torch.float64, device="cuda")
    w[:, 0::2] = (st["codes"] % 16).double()
    w[:, 1::2] = torch.div(st["codes"], 16, rounding_mode="floor").double()
    for i in range(-(-k // g)):
        zero = 8.0 if st["zeros"] is None else st["zeros"][:, i: i + 1].double()
        w[:, i * g: (i + 1) * g] = (w[:, i * g: (i + 1) * g] - zero) * st["scales"][:, i: i + 1].double()
    return torch.mm(st["x"].double(), w[:, :k].t().contiguous())


def _round_e4m3(x: torch.Tensor) -> torch.Tensor:
    """The nearest values of the 8-bit format (3 bits of mantissa, exponents
    from -6 up, ties to even), in 64 bits, saturated."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3.0)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _exact_append(case: dict, st: dict) -> dict:
    cache, p, d, half = st["cache"], case["page"], case["dim"], case["rot"] // 2
    k, v = cache["k"].double(), cache["v"].double()
    ks, vs = cache["k_scale"].double(), cache["v_scale"].double()
    q = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    first = torch.arange(half, device="cuda") * 2 if case["interleaved"] else torch.arange(half, device="cuda")
    second = first + (1 if case["interleaved"] else half)
    table = st["table"].tolist()

    def turn(x, at):
        c, s = st["cos"].double()[at][:, None], st["sin"].double()[at][:, None]
        y = x.double().clone()
        y[..., first] = x[..., first].double() * c - x[..., second].double() * s
        y[..., second] = x[..., second].double() * c + x[..., first].double() * s
        return y

    for b, (n, c) in enumerate(zip(_lengths(case), _counts(case))):
        if not c:
            continue
        at = torch.arange(n, n + c, device="cuda")
        q[b, :c] = turn(st["q"][b, :c], at)
        news = (turn(st["k"][b, :c], at).transpose(0, 1), st["v"][b, :c].double().transpose(0, 1))
        for block in range(n // p, (n + c - 1) // p + 1):
            page, lo, hi = table[b][block], max(n - block * p, 0), min(n + c - block * p, p)
            for codes, scales, new in ((k[page], ks[page], news[0]), (v[page].transpose(1, 2), vs[page], news[1])):
                x = new[:, block * p + lo - n: block * p + hi - n]
                m, e = torch.frexp(x.abs().amax(dim=(1, 2)))
                e = torch.where(m > 0, e - 9 + (m > 0.875), -64).clamp(min=-64)
                scale = torch.exp2(e.double())
                if lo:
                    scale = torch.maximum(scale, scales)
                    codes[:, :lo, :d] = _round_e4m3(codes[:, :lo, :d] * (scales / scale)[:, None, None])
                codes[:, lo:hi, :d] = _round_e4m3(x / scale[:, None, None])
                codes[:, lo:hi, d:] = 0.0
                scales[:] = scale
    return {"q": q, "k": k, "v": v, "k_scale": ks, "v_scale": vs}


def _exact_attend(case: dict, st: dict) -> torch.Tensor:
    cache, d, s = st["cache"], case["dim"], case["share"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for b, (n, c) in enumerate(zip(_lengths(case), _counts(case))):
        if not c:
            continue
        page = st["table"][b, : -(-n // case["page"])].long()
        seen = _visible(case, torch.arange(n - c, n, device="cuda")[:, None], torch.arange(n, device="cuda"))
        for h in range(case["heads"]):
            k = cache["k"].view(torch.uint8)[page, h].view(_FP8).double() * cache["k_scale"][page, h].double()[:, None, None]
            v = cache["v"].view(torch.uint8)[page, h].view(_FP8).double() * cache["v_scale"][page, h].double()[:, None, None]
            k = k.flatten(0, 1)[:n, :d]
            v = v.transpose(1, 2).flatten(0, 1)[:n, :d]
            for i in range(s):
                score = st["q"][b, :c, h * s + i].double() @ k.t().contiguous() / math.sqrt(d)
                prob = torch.softmax(score.masked_fill(~seen, -math.inf), dim=-1)
                out[b, :c, h * s + i] = prob @ v
    return out
