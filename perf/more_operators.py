"""The 8-bit chain of a language model's layer as it is measured, beside its
plain forms.

Where a layer's weights are held in 8-bit floats (e4m3), its activations pass
from one product to the next in 8 bits as well: the norm in front of a product
rounds its rows to them, a product takes both operands as they are, and the
gated half of a feed-forward block rounds what the next product reads. Each
case is one pass through one of the four operators of that chain:

  norm      rms_norm: a row over its root mean square, the residual stream's
            addition on the way, as rows in 8 bits or in the input's type
  quantize  fp8_quantize: rows in 8 bits with a power-of-two scale for each
            block of 128 elements
  product   fp8_matmul: such rows times 8-bit weights that have one scale for
            each block of 128 x 128, a power of two or any float
  gated     fp8_gated_matmul: activation(x Wg^T) * (x Wu^T), as rows in 8 bits

`run` computes the plain form (elementary torch operations in 32 bits, rounded
once) unless `own` is set, in which case it makes the framework's calls.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_EPS = 1e-6


def listed() -> list[dict]:
    return [
        # One token in front of a product: latency is all there is.
        {"name": "norm_token", "kind": "norm", "dtype": "bf16", "m": 1, "k": 4096, "residual": True, "fp8": True},
        # A small batch of odd width, in the input's type (a model's last norm).
        {"name": "norm_ragged_f16", "kind": "norm", "dtype": "f16", "m": 333, "k": 1999, "residual": False, "fp8": False},
        # A long prompt's rows, with the residual stream.
        {"name": "norm_prompt", "kind": "norm", "dtype": "bf16", "m": 8192, "k": 8192, "residual": True, "fp8": True},
        # What attention gives for a decode batch, on its way into a product.
        {"name": "quantize_batch", "kind": "quantize", "dtype": "bf16", "m": 32, "k": 4096},
        # The same of a long prompt.
        {"name": "quantize_prompt", "kind": "quantize", "dtype": "bf16", "m": 16384, "k": 8192},
        # One token through an ordinary projection.
        {"name": "product_token", "kind": "product", "dtype": "bf16", "m": 1, "n": 4096, "k": 4096, "scales": "e8m0"},
        # A decode batch through a wide projection (134 MB of codes), its scales any floats.
        {"name": "product_batch", "kind": "product", "dtype": "bf16", "m": 32, "n": 16384, "k": 8192, "scales": "f32"},
        # Some rows, every extent odd, results in 32 bits (checking a model's layers).
        {"name": "product_ragged_f32", "kind": "product", "dtype": "f32", "m": 77, "n": 3001, "k": 1999, "scales": "f32"},
        # A prompt's chunk through a large projection, both kinds of scales.
        {"name": "product_prompt", "kind": "product", "dtype": "bf16", "m": 4096, "n": 8192, "k": 8192, "scales": "e8m0"},
        {"name": "product_prompt_floats", "kind": "product", "dtype": "bf16", "m": 4096, "n": 8192, "k": 8192,
         "scales": "f32"},
        # A decode batch and a prompt's chunk through the first half of a feed-forward block.
        {"name": "gated_batch", "kind": "gated", "dtype": "bf16", "m": 16, "n": 12288, "k": 4096, "scales": "e8m0",
         "activation": "silu"},
        {"name": "gated_prompt", "kind": "gated", "dtype": "bf16", "m": 2048, "n": 16384, "k": 4096, "scales": "e8m0",
         "activation": "silu"},
    ]


# The most that a drawn case may cost: the largest listed ones.
_MOST_ROWS = 16384 * 8192
_MOST_WEIGHTS = 16384 * 8192
_MOST_PRODUCTS = 4096 * 8192 * 8192


def _log_int(rng, lo: int, hi: int) -> int:
    """An integer in [lo, hi], its logarithm uniform."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    """One more case of the listed ranges."""
    kind = rng.choice(("norm", "quantize", "product", "product", "gated"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    while True:
        case = {"kind": kind, "dtype": dtype, "m": _log_int(rng, 1, 16384), "k": _log_int(rng, 100, 16384)}
        if rng.random() < 0.5:  # most layers are multiples of 128, not all
            case["k"] = -(-case["k"] // 128) * 128
        if kind == "norm":
            case["residual"], case["fp8"] = rng.random() < 0.5, rng.random() < 0.7
        if kind in ("norm", "quantize"):
            if case["m"] * case["k"] * _SIZE[dtype] <= 2 * _MOST_ROWS // (2 if kind == "norm" else 1):
                return case
            continue
        case["n"], case["scales"] = _log_int(rng, 100, 16384), rng.choice(("e8m0", "f32"))
        if rng.random() < 0.5:
            case["n"] = -(-case["n"] // 128) * 128
        if kind == "gated":
            case["activation"] = rng.choice(("silu", "silu", "gelu_tanh"))
        weights = case["n"] * case["k"] * (2 if kind == "gated" else 1)
        if weights <= _MOST_WEIGHTS and case["m"] * weights <= _MOST_PRODUCTS:
            return case


def _blocks(n: int) -> int:
    return -(-n // 128)


def _activations(g, case: dict) -> torch.Tensor:
    """Rows with the few large features that a model's hidden states have."""
    size = torch.where(torch.rand(case["k"], generator=g, device="cuda") < 0.005, 20.0, 1.0)
    return torch.randn((case["m"], case["k"]), generator=g, device="cuda").mul_(size).to(_DTYPES[case["dtype"]])


def _rows8(g, case: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows in 8 bits as the norm or the quantizer gives them: e4m3 codes and
    their blocks' powers of two as e8m0."""
    return _quantized(_activations(g, case).float())


def _weights(g, case: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes whose blocks use the format's range, and their scales."""
    n, k = case["n"], case["k"]
    codes = torch.empty((n, k), dtype=_E4M3, device="cuda")
    for part in codes.split(max(1, (1 << 26) // k)):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(100.0).clamp_(-448.0, 448.0))
    size = 0.01 / math.sqrt(k) * (0.5 + torch.rand((_blocks(n), _blocks(k)), generator=g, device="cuda"))
    if case["scales"] == "f32":
        return codes, size
    return codes, (torch.frexp(size)[1] + 126).to(torch.uint8).view(_E8M0)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["kind"] in ("norm", "quantize"):
        state["x"] = _activations(g, case)
        if case["kind"] == "norm":
            state["weight"] = (1.0 + 0.1 * torch.randn(case["k"], generator=g, device="cuda")).to(state["x"].dtype)
            state["residual"] = _activations(g, case) if case["residual"] else None
        return state
    state["x"] = _rows8(g, case)
    names = ("gate", "up") if case["kind"] == "gated" else ("w",)
    for name in names:
        state[name] = _weights(g, case)
    if own:  # the program's weights, laid out once, and rows as an operator before gives them
        import trntensor_amd as tt

        state["x"] = tt.Fp8Rows(*state["x"], dtype=_DTYPES[case["dtype"]])
        for name in names:
            state[name] = tt.Fp8Matrix(*state[name])
    return state


def run(state: dict):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["kind"] == "norm":
        return _plain_norm(case, state)
    if case["kind"] == "quantize":
        codes, scales = _quantized(state["x"].float())
        return {"codes": codes, "scales": scales}
    return _plain_product(case, state) if case["kind"] == "product" else _plain_gated(case, state)


def _run_own(case: dict, st: dict):
    import trntensor_amd as tt

    if case["kind"] == "product":
        return tt.fp8_matmul(st["x"], st["w"])
    out = {}
    if case["kind"] == "norm":
        y = tt.rms_norm(st["x"], st["weight"], residual=st["residual"], eps=_EPS, fp8=case["fp8"])
        if case["residual"]:
            y, out["stream"] = y
        if not case["fp8"]:
            return {"y": y, **out}
    elif case["kind"] == "quantize":
        y = tt.fp8_quantize(st["x"])
    else:
        y = tt.fp8_gated_matmul(st["x"], st["gate"], st["up"], activation=case["activation"])
    return {"codes": y.codes, "scales": y.scales, **out}


def _quantized(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """float32 rows as e4m3 codes and, for each block of 128, the smallest
    power of two (2^-127 at least) that brings its values to 448 or below."""
    m, k = x.shape
    block = torch.nn.functional.pad(x, (0, -k % 128)).reshape(m, -1, 128)
    part, e = torch.frexp(block.abs().amax(dim=2))  # amax = part * 2^e with part in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(part > 0, e - 9 + (part > 0.875).int(), -127).clamp(min=-127)
    codes = torch.ldexp(block, -e[..., None]).clamp(-448.0, 448.0).to(_E4M3)
    return codes.reshape(m, -1)[:, :k].contiguous(), (e + 127).to(torch.uint8).view(_E8M0)


def _plain_norm(case: dict, st: dict) -> dict:
    x = st["x"].float()
    out = {}
    if case["residual"]:
        x = x + st["residual"].float()
        out["stream"] = x.to(st["x"].dtype)
    y = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + _EPS) * st["weight"].float()
    if not case["fp8"]:
        return {"y": y.to(st["x"].dtype), **out}
    codes, scales = _quantized(y)
    return {"codes": codes, "scales": scales, **out}


def _wide(codes: torch.Tensor, scales: torch.Tensor, rows: int) -> torch.Tensor:
    """Codes times their scales in 32 bits; a scale covers `rows` x 128."""
    n, k = codes.shape
    scales = scales.float().repeat_interleave(rows, dim=0)[:n] if rows > 1 else scales.float()
    return codes.float() * scales.repeat_interleave(128, dim=1)[:, :k]


def _plain_product(case: dict, st: dict) -> torch.Tensor:
    return (_wide(*st["x"], 1) @ _wide(*st["w"], 128).t()).to(_DTYPES[case["dtype"]])


def _plain_gated(case: dict, st: dict) -> dict:
    x = _wide(*st["x"], 1)
    gate, up = x @ _wide(*st["gate"], 128).t(), x @ _wide(*st["up"], 128).t()
    bend = gate if case["activation"] == "silu" else math.sqrt(8.0 / math.pi) * (gate + 0.044715 * gate * gate * gate)
    codes, scales = _quantized(gate / (1.0 + torch.exp(-bend)) * up)
    return {"codes": codes, "scales": scales}


def work(case: dict) -> dict:
    m, k, es = case["m"], case["k"], _SIZE[case["dtype"]]
    rows8 = m * k + m * _blocks(k)
    if case["kind"] == "quantize":
        return {"bytes": m * k * es + rows8, "flops": 3 * m * k}
    if case["kind"] == "norm":
        read, kept = (2, 1) if case["residual"] else (1, 0)
        return {"bytes": m * k * es * (read + kept) + k * es + (rows8 if case["fp8"] else m * k * es), "flops": 6 * m * k}
    n, each = case["n"], 4 if case["scales"] == "f32" else 1
    matrix = n * k + _blocks(n) * _blocks(k) * each
    if case["kind"] == "product":
        return {"bytes": rows8 + matrix + m * n * es, "flops": 2 * m * n * k}
    return {"bytes": rows8 + 2 * matrix + m * n + m * _blocks(n), "flops": 4 * m * n * k}


def exact(case: dict, seed: int):
    global own
    keep, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = keep
    if case["kind"] == "quantize":
        return _exact_rows8(st["x"].double())
    if case["kind"] == "norm":
        h = st["x"].double()
        out = {}
        if st["residual"] is not None:
            h = h + st["residual"].double()
            out["stream"] = h
        power = torch.linalg.vector_norm(h, dim=1).square() / case["k"]
        y = h / torch.sqrt(power + _EPS)[:, None] * st["weight"].double()
        return {**(_exact_rows8(y) if case["fp8"] else {"y": y}), **out}
    x = _exact_wide(*st["x"], 1)
    if case["kind"] == "product":
        return torch.mm(x, _exact_wide(*st["w"], 128).t())
    gate = torch.mm(x, _exact_wide(*st["gate"], 128).t())
    up = torch.mm(x, _exact_wide(*st["up"], 128).t())
    if case["activation"] == "silu":
        return _exact_rows8(gate * torch.sigmoid(gate) * up)
    inner = math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate ** 3)
    return _exact_rows8(0.5 * gate * (1.0 + torch.tanh(inner)) * up)


def _exact_wide(codes: torch.Tensor, scales: torch.Tensor, rows: int) -> torch.Tensor:
    out = codes.double()
    for j in range(scales.shape[1]):
        column = scales[:, j].double()
        out[:, 128 * j: 128 * (j + 1)] *= column[torch.arange(out.shape[0], device="cuda") // rows][:, None]
    return out


def _exact_rows8(y: torch.Tensor) -> dict:
    """64-bit rows over their blocks' scales, and the scales. What codes stand
    for is given unrounded, as every other output here."""
    codes, scales = torch.empty_like(y), []
    for j in range(0, y.shape[1], 128):
        part = y[:, j: j + 128]
        top = part.abs().amax(dim=1)
        e = torch.ceil(torch.log2(top / 448.0)).clamp(min=-127.0)
        e = torch.where(top > 448.0 * torch.exp2(e), e + 1.0, e)
        e = torch.where((e > -127.0) & (top <= 448.0 * torch.exp2(e - 1.0)), e - 1.0, e)
        codes[:, j: j + 128] = part / torch.exp2(e)[:, None]
        scales.append(torch.exp2(e))
    return {"codes": codes, "scales": torch.stack(scales, dim=1)}
