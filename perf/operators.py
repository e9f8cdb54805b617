"""The feed-forward and adapter operators that are measured: calls, plain forms, and the definition in 64 bits.

`mlp`: the gated feed-forward block (`fused_cpp_b200.moe.gated_mlp`), for serving (a forward pass without gradients) and for
training (output and the gradients of the input and both weights).  `lora`: a dense W8A8 projection with the low-rank
adapters of many requests beside it (`fused_cpp_b200.i8gemm.dynamic_scaled_mm_lora`).

With `own` false, `run` computes the operators from elementary torch operations in 32 bits.  `exact` computes them in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

_DEVICE = "cuda"
_OAI_ALPHA, _OAI_LIMIT = 1.702, 7.0


def _mlp(name: str, tokens: int, hidden: int, inter: int, **options) -> dict:
    case = {"name": name, "op": "mlp", "tokens": tokens, "hidden": hidden, "inter": inter, "activation": "silu", "limit": 0.0, "train": False}
    case.update(options)
    return case


def _lora(name: str, rows: int, k: int, n: int, adapters: int, rank: int, **options) -> dict:
    """order: "mixed" = every row is a request of its own, "runs" = requests of several rows one after the other.
    none: share of the requests that have no adapter."""
    case = {"name": name, "op": "lora", "rows": rows, "k": k, "n": n, "adapters": adapters, "rank": rank, "order": "mixed", "none": 0.0,
            "output": "bf16", "bias": False}
    case.update(options)
    return case


def listed() -> list:
    return [
        # One user's next token through the full-size layer's shared expert: 88 MB of weights for one row.
        _mlp("mlp_token_T1", 1, 7168, 2048, limit=10.0),
        # A decode batch of the same layer.
        _mlp("mlp_decode_T64", 64, 7168, 2048, limit=10.0),
        # A prompt's chunk through a block of ragged sizes, with the other clamped activation.
        _mlp("mlp_prompt_T1111_oai", 1111, 2880, 1416, activation="swigluoai"),
        # Prefill of the full-size layer.
        _mlp("mlp_prefill_T8192", 8192, 7168, 2048),
        # Fine-tuning on a handful of tokens: gradients of 88 MB of weights from 40 rows.
        _mlp("mlp_train_T40", 40, 7168, 2048, train=True),
        # A training micro-batch of a small model, odd token count.
        _mlp("mlp_train_T1333_gelu", 1333, 2048, 1024, train=True, activation="gelu"),
        # The largest training step: the full-size shared expert over a long batch.
        _mlp("mlp_train_T8192", 8192, 7168, 2048, train=True, limit=10.0),
        # One request with its adapter: the smallest call, latency counts.
        _lora("lora_token_M1", 1, 7168, 1536, 8, 16),
        # A decode batch in which nearly every request has another adapter, output projection of the attention.
        _lora("lora_decode_M64", 64, 16384, 7168, 32, 16, none=0.1),
        # A larger batch of few, wider adapters on the widest projection, odd row count, with a bias.
        _lora("lora_decode_M201", 201, 1536, 24576, 4, 64, none=0.25, bias=True),
        # A few prompts' chunk with 32-bit results, sizes that fit no tile.
        _lora("lora_prompt_M777_f32", 777, 2056, 1234, 5, 24, order="runs", none=0.2, output="f32"),
        # Prefill of many prompts through the output projection.
        _lora("lora_prefill_M8192", 8192, 16384, 7168, 16, 32, order="runs", none=0.1),
    ]


def _log_uniform(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    if rng.random() < 0.5:
        activation, limit = rng.choice([("silu", 0.0), ("silu", 10.0), ("gelu", 0.0), ("swigluoai", 0.0)])
        return {"op": "mlp", "tokens": _log_uniform(rng, 1, 8192), "hidden": 8 * _log_uniform(rng, 16, 896), "inter": 8 * _log_uniform(rng, 16, 256),
                "activation": activation, "limit": limit, "train": rng.random() < 0.5}
    rows, k, n = _log_uniform(rng, 1, 8192), _log_uniform(rng, 128, 16384), _log_uniform(rng, 128, 24576)
    while rows * k * n > 8192 * 16384 * 7168 // 2:
        rows = max(1, rows // 2)
    return {"op": "lora", "rows": rows, "k": k, "n": n, "adapters": _log_uniform(rng, 1, 64), "rank": _log_uniform(rng, 4, 128),
            "order": rng.choice(["mixed", "runs"]), "none": rng.choice([0.0, 0.1, 0.5]), "output": rng.choice(["bf16", "bf16", "f32"]),
            "bias": rng.random() < 0.3}


def _adapter_ids(case: dict, generator: torch.Generator) -> torch.Tensor:
    """One adapter id per row (-1: none), as a batch of requests has them."""
    rows, adapters = case["rows"], case["adapters"]
    requests = rows if case["order"] == "mixed" else max(1, min(rows, 2 * adapters))
    ids = torch.randint(adapters, (requests,), generator=generator, device=_DEVICE)
    ids = torch.where(torch.rand(requests, generator=generator, device=_DEVICE) < case["none"], torch.full_like(ids, -1), ids)
    if requests == rows:
        return ids
    # Requests of uneven lengths, one after the other.
    cuts = torch.sort(torch.randint(rows, (requests - 1,), generator=generator, device=_DEVICE)).values
    return ids[torch.searchsorted(cuts, torch.arange(rows, device=_DEVICE), right=True)]


def prepare(case: dict, seed: int) -> dict:
    generator = torch.Generator(device=_DEVICE).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=generator, device=_DEVICE) * std

    if case["op"] == "mlp":
        tokens, hidden, inter = case["tokens"], case["hidden"], case["inter"]
        # Gate and up values of a standard deviation of 3: limits of 7 and 10 are reached by some.
        state = {"case": case, "x": normal(tokens, hidden).bfloat16(), "w13": normal(2 * inter, hidden, std=3.0 / math.sqrt(hidden)).bfloat16(),
                 "w2": normal(hidden, inter, std=1.0 / math.sqrt(inter)).bfloat16()}
        if case["train"]:
            state["dy"] = normal(tokens, hidden, std=0.1).bfloat16()
            for name in ("x", "w13", "w2"):
                state[name].requires_grad_(True)
        return state
    rows, k, n, adapters, rank = case["rows"], case["k"], case["n"], case["adapters"], case["rank"]
    x = normal(rows, k)
    x[:, :: 97] *= 6.0  # channels of large activations, which set the rows' scales
    state = {"case": case, "x": x.bfloat16(), "weight": torch.randint(-127, 128, (n, k), generator=generator, device=_DEVICE, dtype=torch.int8),
             "weight_scale": (0.5 + torch.rand(n, generator=generator, device=_DEVICE)) / (73.0 * math.sqrt(k)),
             "a": normal(adapters, rank, k, std=1.0 / math.sqrt(k)).bfloat16(), "b": normal(adapters, n, rank, std=0.5 / math.sqrt(rank)).bfloat16(),
             "scaling": 0.5 + torch.rand(adapters, generator=generator, device=_DEVICE),
             "bias": normal(n, std=0.5) if case["bias"] else None, "ids": _adapter_ids(case, generator)}
    if own:
        # What a server keeps: the resident weight and the resident adapters.
        from fused_cpp_b200 import i8gemm, lora

        state["packed"] = i8gemm.prepare(state["weight"], state["weight_scale"])
        state["adapters"] = lora.prepare_adapters(state["a"], state["b"], state["scaling"])
    return state


# ---- the gated block, plain form ------------------------------------------------------------------------------------

def _gate_plain(case: dict, g: torch.Tensor, u: torch.Tensor):
    """h and its partial derivatives by g and u."""
    if case["activation"] == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        density = torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
        return g * cdf * u, u * (cdf + g * density), g * cdf
    oai = case["activation"] == "swigluoai"
    limit = _OAI_LIMIT if oai else (case["limit"] or math.inf)
    alpha, shift = (_OAI_ALPHA, 1.0) if oai else (1.0, 0.0)
    g_free, u_free = g <= limit, (u <= limit) & (u >= -limit)
    g = torch.where(g_free, g, limit)
    u = torch.where(u_free, u, limit * torch.sign(u)) + shift
    s = 1.0 / (1.0 + torch.exp(-alpha * g))
    return g * s * u, torch.where(g_free, u * s * (1.0 + alpha * g * (1.0 - s)), 0.0), torch.where(u_free, g * s, 0.0)


def _mlp_plain(state: dict):
    case = state["case"]
    inter = case["inter"]
    x, w13, w2 = (state[name].detach().float() for name in ("x", "w13", "w2"))
    gu = x @ w13.T
    h, by_g, by_u = _gate_plain(case, gu[:, :inter], gu[:, inter:])
    y = (h @ w2.T).bfloat16()
    if not case["train"]:
        return {"y": y}
    dy = state["dy"].float()
    dh = dy @ w2
    dgu = torch.cat((dh * by_g, dh * by_u), dim=1)
    return {"y": y, "dx": (dgu @ w13).bfloat16(), "dw13": (dgu.T @ x).bfloat16(), "dw2": (dy.T @ h).bfloat16()}


def _mlp_own(state: dict):
    from fused_cpp_b200 import moe

    case = state["case"]
    y = moe.gated_mlp(state["x"], state["w13"], state["w2"], activation=case["activation"], swiglu_limit=case["limit"] or None)
    if not case["train"]:
        return {"y": y}
    dx, dw13, dw2 = torch.autograd.grad(y, (state["x"], state["w13"], state["w2"]), state["dy"])
    return {"y": y, "dx": dx, "dw13": dw13, "dw2": dw2}


# ---- the projection with adapters, plain form -----------------------------------------------------------------------

def _lora_plain(state: dict):
    case = state["case"]
    x, ids = state["x"].float(), state["ids"]
    scale = x.abs().amax(dim=1, keepdim=True) / 127.0
    scale = torch.where(scale > 0, scale, 1.0)
    q = torch.clamp(torch.round(x / scale), -128, 127)
    y = (q @ state["weight"].float().T) * scale * state["weight_scale"]
    if state["bias"] is not None:
        y = y + state["bias"]
    # All adapters at once: a row's products with the others' are multiplied by nought.
    adapters, rank = case["adapters"], case["rank"]
    chosen = (ids[:, None] == torch.arange(adapters, device=ids.device)).float() * state["scaling"]
    t = (x @ state["a"].float().reshape(adapters * rank, -1).T).reshape(-1, adapters, rank) * chosen[:, :, None]
    y = y + t.reshape(-1, adapters * rank) @ state["b"].float().permute(0, 2, 1).reshape(adapters * rank, -1)
    return y if case["output"] == "f32" else y.bfloat16()


def _lora_own(state: dict):
    from fused_cpp_b200 import i8gemm

    dtype = torch.float32 if state["case"]["output"] == "f32" else torch.bfloat16
    return i8gemm.dynamic_scaled_mm_lora(state["x"], state["packed"], state["adapters"], state["ids"], bias=state["bias"], out_dtype=dtype)


def run(state: dict):
    if state["case"]["op"] == "mlp":
        return _mlp_own(state) if own else _mlp_plain(state)
    return _lora_own(state) if own else _lora_plain(state)


def work(case: dict) -> dict:
    if case["op"] == "mlp":
        tokens, hidden, inter = case["tokens"], case["hidden"], case["inter"]
        weights, rows = 6 * inter * hidden, 2 * tokens * hidden
        # Training reads x and dy, writes y and dx, reads both weights and writes both gradients.
        return {"bytes": (2 * weights + 4 * rows) if case["train"] else (weights + 2 * rows), "flops": (18 if case["train"] else 6) * tokens * inter * hidden}
    rows, k, n, adapters, rank = case["rows"], case["k"], case["n"], case["adapters"], case["rank"]
    with_adapter = rows * (1.0 - case["none"])
    requests = rows if case["order"] == "mixed" else max(1, min(rows, 2 * adapters))
    in_use = adapters * (1.0 - (1.0 - 1.0 / adapters) ** (requests * (1.0 - case["none"])))
    out = (4 if case["output"] == "f32" else 2) * rows * n
    return {"bytes": int(2 * rows * k + n * k + 4 * n + 2 * rank * (k + n) * in_use + out), "flops": int(2 * rows * n * k + 2 * rank * with_adapter * (k + n))}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def _mlp_exact(state: dict):
    case = state["case"]
    x, w2 = state["x"].detach().double(), state["w2"].detach().double()
    w_gate, w_up = state["w13"].detach().double().chunk(2, dim=0)
    gate, up = x.mm(w_gate.t()), x.mm(w_up.t())
    if case["train"]:
        gate.requires_grad_(True)
        up.requires_grad_(True)
    if case["activation"] == "gelu":
        h = gate * torch.special.ndtr(gate) * up
    elif case["activation"] == "swigluoai":
        kept = gate.clamp(max=_OAI_LIMIT)
        h = (up.clamp(-_OAI_LIMIT, _OAI_LIMIT) + 1.0) * kept * torch.sigmoid(_OAI_ALPHA * kept)
    else:
        bound = case["limit"] if case["limit"] else math.inf
        kept = gate.clamp(max=bound)
        h = kept * torch.sigmoid(kept) * up.clamp(-bound, bound)
    result = {"y": h.detach().mm(w2.t())}
    if case["train"]:
        dy = state["dy"].double()
        d_gate, d_up = torch.autograd.grad(h, (gate, up), dy.mm(w2))
        result["dx"] = d_gate.mm(w_gate) + d_up.mm(w_up)
        result["dw13"] = torch.cat((d_gate.t().mm(x), d_up.t().mm(x)))
        result["dw2"] = dy.t().mm(h.detach())
    return result


def _lora_exact(state: dict):
    x, ids = state["x"].double(), state["ids"]
    # The row scale and the quotient by it are 32-bit numbers by definition: half of a row's largest value lies on the border
    # between 63 and 64, and their roundings say to which side it falls.
    scale = state["x"].float().abs().amax(dim=1) / 127.0
    scale[scale == 0] = 1.0
    q = (state["x"].float() / scale[:, None]).double().round().clamp(-128, 127)
    scale = scale.double()
    y = q.mm(state["weight"].double().t()) * scale[:, None] * state["weight_scale"].double()[None, :]
    if state["bias"] is not None:
        y += state["bias"].double()
    for adapter in range(state["case"]["adapters"]):
        rows = torch.nonzero(ids == adapter).flatten()
        if rows.numel():
            y[rows] += state["scaling"][adapter].double() * x[rows].mm(state["a"][adapter].double().t()).mm(state["b"][adapter].double().t())
    return y


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    return _mlp_exact(state) if case["op"] == "mlp" else _lora_exact(state)
