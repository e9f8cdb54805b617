"""The gated feed-forward block and its gradients against the formulas in 64 bits.

Tolerances, element by element.  A rounding to bf16 is off by at most u = 2^-8 of the value.  Every result is a sum of products with S the sum of
their magnitudes; a product carries n roundings of its factors (y and dw2: that of h; dx and dw13: that of dh times the partial
derivative; n = 1), so n u S.  A 32-bit sum of K terms is off by at most K 2^-24 of the sum of the magnitudes, the activation's functions by less than
2^-16 of their value; with `SMALL` = K 2^-24 + 2^-15 (K the longest sum; the second-order terms of the roundings, below 2^-15, are in it) that is SMALL S, and SMALL
times the sum of the magnitudes inside dh.  gate and up are 32-bit sums too: their error enters h by its derivatives and the derivatives by theirs, which
are below 4 (1 + |gate| + |up|), or whole where a value lies so near a limit that the error may carry it across.  The result's own rounding adds u of it."""
import pytest
import torch

pytestmark = pytest.mark.gpu

STEP = torch.finfo(torch.bfloat16).eps / 2  # largest relative error of one rounding

ACTIVATIONS = [("silu", None), ("silu", 10.0), ("gelu", None), ("swigluoai", None)]


def make(tokens, hidden, inter, seed=0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(tokens, hidden, generator=g, device=device).bfloat16()
    w13 = (torch.randn(2 * inter, hidden, generator=g, device=device) * (4.0 / hidden ** 0.5)).bfloat16()
    w2 = (torch.randn(hidden, inter, generator=g, device=device) / inter ** 0.5).bfloat16()
    dy = torch.randn(tokens, hidden, generator=g, device=device).bfloat16()
    return x, w13, w2, dy


def formulas(x, w13, w2, dy, activation, limit):
    """Results in 64 bits, and the error that each may have before its own rounding."""
    x, w13, w2, dy = (t.detach().double() for t in (x, w13, w2, dy))
    gate, up = (x @ w13.T).chunk(2, dim=1)
    if activation == "gelu":
        cdf, pdf = 0.5 * torch.special.erfc(-gate * 0.5 ** 0.5), torch.exp(-gate * gate / 2) / (2 * torch.pi) ** 0.5
        h, by_gate, by_up = gate * cdf * up, up * (cdf + gate * pdf), gate * cdf
    else:
        alpha, shift, bound = (1.702, 1.0, 7.0) if activation == "swigluoai" else (1.0, 0.0, limit or float("inf"))
        cut_gate, cut_up = gate > bound, up.abs() > bound
        g, u = gate.clamp(max=bound), up.clamp(-bound, bound) + shift
        s = torch.sigmoid(alpha * g)
        h, by_gate, by_up = g * s * u, (u * s * (1 + alpha * g * (1 - s))).masked_fill(cut_gate, 0), (g * s).masked_fill(cut_up, 0)
    dh = dy @ w2
    dh_size = dy.abs() @ w2.abs()
    d = torch.cat((dh * by_gate, dh * by_up), 1)
    d_size = torch.cat((dh_size * by_gate.abs(), dh_size * by_up.abs()), 1)
    results = {"y": h @ w2.T, "dx": d @ w13, "dw13": d.T @ x, "dw2": dy.T @ h}
    sums = 2.0 ** -24 * max(x.shape[0], x.shape[1], w13.shape[0])
    small = sums + 2.0 ** -15
    slack = sums * (x.abs() @ w13.abs().T)
    gate_slack, up_slack = slack.chunk(2, dim=1)
    h_slack = by_gate.abs() * gate_slack + by_up.abs() * up_slack
    d_slack = dh_size * 4 * (1 + up.abs() + gate.abs()) * (gate_slack + up_slack)
    if activation != "gelu":
        near = ((gate - bound).abs() <= gate_slack) | ((up.abs() - bound).abs() <= up_slack)
        d_slack = d_slack + near * dh_size * 2 * (1 + up.abs()) * (1 + gate.abs())
    d_slack = torch.cat((d_slack, d_slack), 1)
    errors = {
        "y": (STEP + small) * (h.abs() @ w2.abs().T) + h_slack @ w2.abs().T,
        "dw2": (STEP + small) * (dy.abs().T @ h.abs()) + dy.abs().T @ h_slack,
        "dx": (STEP + small) * (d.abs() @ w13.abs()) + (small * d_size + d_slack) @ w13.abs(),
        "dw13": (STEP + small) * (d.abs().T @ x.abs()) + (small * d_size + d_slack).T @ x.abs(),
    }
    return results, errors


def check_all(got, x, w13, w2, dy, activation, limit):
    results, errors = formulas(x, w13, w2, dy, activation, limit)
    for name, value in got.items():
        if value is None or not value.numel():
            continue
        allowed = errors[name] * (1 + STEP) + STEP * results[name].abs() + 1e-37
        worst = ((value.double() - results[name]).abs() / allowed).max().item()
        assert worst <= 1.0, (name, worst)


def run(moe, x, w13, w2, dy, activation="silu", limit=None):
    leaves = [t.detach().requires_grad_(True) for t in (x, w13, w2)]
    y = moe.gated_mlp(*leaves, activation=activation, swiglu_limit=limit)
    dx, dw13, dw2 = torch.autograd.grad(y, leaves, dy)
    return {"y": y.detach(), "dx": dx, "dw13": dw13, "dw2": dw2}


@pytest.mark.parametrize("tokens, hidden, inter", [
    (1, 64, 64), (1, 8, 8), (2, 16, 8), (7, 72, 40), (16, 256, 128), (33, 200, 136), (64, 512, 256), (127, 264, 264), (128, 128, 384), (129, 520, 72),
    (255, 64, 1000), (256, 1024, 128), (257, 136, 520), (300, 2056, 264), (511, 384, 640), (700, 1416, 248), (1025, 320, 136)])
@pytest.mark.parametrize("activation, limit", ACTIVATIONS)
def test_block_and_gradients(cuda_device, tokens, hidden, inter, activation, limit):
    from fused_cpp_b200 import _lib, moe

    x, w13, w2, dy = make(tokens, hidden, inter, seed=tokens)
    got = run(moe, x, w13, w2, dy, activation, limit)
    check_all(got, x, w13, w2, dy, activation, limit)
    with torch.no_grad():
        assert torch.equal(moe.gated_mlp(x, w13, w2, activation=activation, swiglu_limit=limit), got["y"])
    assert _lib.dense_status() == (0, 0)
