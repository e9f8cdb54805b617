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


def test_passes_without_a_tape(cuda_device):
    from fused_cpp_b200 import moe

    for tokens, hidden, inter in ((5, 64, 40), (300, 264, 136)):
        x, w13, w2, dy = make(tokens, hidden, inter)
        want = run(moe, x, w13, w2, dy, "silu", 10.0)
        y, kept = moe.gated_mlp_forward(x, w13, w2, swiglu_limit=10.0)
        assert torch.equal(y, want["y"])
        for needs in ((True, True, True), (True, False, False), (False, True, False), (False, False, True), (False, False, False)):
            got = moe.gated_mlp_backward(dy, x, w13, w2, kept, needs=needs)
            for name, need, value in zip(("dx", "dw13", "dw2"), needs, got):
                assert (value is None) if not need else torch.equal(value, want[name]), (needs, name)


def test_gradients_of_some_inputs(cuda_device):
    from fused_cpp_b200 import moe

    x, w13, w2, dy = make(70, 128, 72)
    want = run(moe, x, w13, w2, dy)
    for chosen in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaves = [t.detach().requires_grad_(i in chosen) for i, t in enumerate((x, w13, w2))]
        y = moe.gated_mlp(*leaves)
        grads = torch.autograd.grad(y, [leaves[i] for i in chosen], dy, retain_graph=True)
        again = torch.autograd.grad(y, [leaves[i] for i in chosen], dy)
        for i, grad, second in zip(chosen, grads, again):
            assert torch.equal(grad, want[("dx", "dw13", "dw2")[i]]) and torch.equal(grad, second)


def test_leaves_accumulate_and_shared_weights(cuda_device):
    """Two uses of the same weights add their gradients; leaves take them in .grad."""
    from fused_cpp_b200 import moe

    x, w13, w2, dy = make(40, 64, 48)
    a = run(moe, x, w13, w2, dy)
    b = run(moe, x.flip(0), w13, w2, dy)
    leaves = [t.detach().requires_grad_(True) for t in (w13, w2)]
    (moe.gated_mlp(x, *leaves) * dy).sum().backward()
    (moe.gated_mlp(x.flip(0), *leaves) * dy).sum().backward()
    assert torch.equal(leaves[0].grad, a["dw13"] + b["dw13"]) and torch.equal(leaves[1].grad, a["dw2"] + b["dw2"])


def test_second_derivative_is_refused(cuda_device):
    from fused_cpp_b200 import moe

    x, w13, w2, dy = make(4, 16, 8)
    leaves = [t.requires_grad_(True) for t in (x, w13, w2)]
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(moe.gated_mlp(*leaves), leaves, dy, create_graph=True)


def test_differences(cuda_device):
    """The gradient against central differences of the block itself along random directions.  A difference of y over 2e carries two roundings of every y,
    2 u |y| / 2e at most each weighted by |dy|, of h as many inside, and a third-order term e^2 |f'''| / 6 which a small e leaves below them."""
    from fused_cpp_b200 import moe

    x, w13, w2, dy = make(64, 128, 64)
    got = run(moe, x, w13, w2, dy)
    g = torch.Generator(device="cuda").manual_seed(1)
    for name, index in (("dx", 0), ("dw13", 1), ("dw2", 2)):
        tensors = [x, w13, w2]
        direction = torch.randn(tensors[index].shape, generator=g, device="cuda")
        step = 0.25 * tensors[index].float().std() * direction
        low, high = ((tensors[index].float() + sign * step).bfloat16() for sign in (-1, 1))
        values = []
        for moved in (low, high):
            tensors[index] = moved
            values.append(moe.gated_mlp(*tensors).double())
        # Along the path from low to high the gradient changes: compare with the mean of the gradients at both ends and in the middle (Simpson).
        ends = []
        for moved in (low, high):
            tensors[index] = moved
            ends.append(run(moe, *tensors, dy)[name].double())
        mean = (ends[0] + 4 * got[name].double() + ends[1]) / 6
        moved = high.double() - low.double()
        change = ((values[1] - values[0]) * dy.double()).sum()
        predicted = (mean * moved).sum()
        # Independent roundings: the sum's standard deviation is u |dy| |y| sqrt(2) at most for y and as much for h; six of them, and 2 % for Simpson's remainder.
        noise = 6 * 2 * STEP * (2 ** 0.5) * ((values[0].abs() + values[1].abs()) / 2 * dy.double().abs()).norm() + 0.02 * (mean * moved).abs().sum().sqrt() * (mean * moved).norm().sqrt()
        assert (change - predicted).abs() <= noise, (name, change.item(), predicted.item(), noise.item())


def test_no_rows(cuda_device):
    from fused_cpp_b200 import moe

    _, w13, w2, _ = make(1, 64, 32)
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    got = run(moe, x, w13, w2, x)
    assert got["y"].shape == (0, 64) and got["dx"].shape == (0, 64)
    assert not got["dw13"].any() and not got["dw2"].any() and got["dw13"].shape == w13.shape


@pytest.mark.parametrize("tokens", [3, 300])
def test_layouts(cuda_device, tokens):
    """Rows of a wider matrix, an unaligned view, a transposed matrix, a broadcast dy, three dimensions, weights that are views: the same results."""
    from fused_cpp_b200 import moe

    x, w13, w2, dy = make(tokens, 136, 72)
    want = run(moe, x, w13, w2, dy)
    wide = torch.randn(tokens, 400, device="cuda").bfloat16()
    wide[:, 8:144] = x
    odd = torch.empty(tokens * 136 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(tokens, 136)
    odd.copy_(x)
    stacked = torch.randn(3, *w13.shape, device="cuda").bfloat16()
    stacked[1] = w13
    for form, weights in ((wide[:, 8:144], (w13, w2)), (odd, (w13, w2)), (x.t().contiguous().t(), (w13, w2)), (x, (stacked[1], w2.t().contiguous().t()))):
        got = run(moe, form, *weights, dy)
        for name in want:
            assert torch.equal(got[name], want[name]), name
    for form in (wide[:, 8:144].clone(), dy.t().contiguous().t()):
        assert torch.equal(run(moe, x, w13, w2, form)["dx"], run(moe, x, w13, w2, form.contiguous())["dx"])
    row = dy[:1].expand(tokens, -1)
    assert torch.equal(run(moe, x, w13, w2, row)["dw13"], run(moe, x, w13, w2, row.contiguous())["dw13"])
    cube = run(moe, x.view(1, tokens, 136), w13, w2, dy.view(1, tokens, 136))
    assert cube["dx"].shape == (1, tokens, 136) and torch.equal(cube["dx"][0], want["dx"]) and torch.equal(cube["dw2"], want["dw2"])
    vector = run(moe, x[0], w13, w2, dy[0])
    assert vector["y"].shape == (136,) and torch.equal(vector["y"], run(moe, x[:1], w13, w2, dy[:1])["y"][0])
    out = torch.empty(tokens * 136 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(tokens, 136)
    assert moe.gated_mlp(x, w13, w2, out=out) is out and torch.equal(out, want["y"])
    with pytest.raises(ValueError, match="out must be contiguous"):
        moe.gated_mlp(x, w13, w2, out=wide[:, 8:144])
    with pytest.raises(ValueError, match="gradients are asked for"):
        moe.gated_mlp(x.requires_grad_(True), w13, w2, out=out)


@pytest.mark.parametrize("tokens", [2, 260])
def test_not_finite(cuda_device, tokens):
    """A NaN or an infinity in one row stays in that row of y and dx; a limit does not hide a NaN."""
    from fused_cpp_b200 import moe

    x, w13, w2, dy = make(tokens, 64, 48)
    want = run(moe, x, w13, w2, dy, "silu", 10.0)
    for bad in (float("nan"), float("inf")):
        broken = x.clone()
        broken[1, 5] = bad
        got = run(moe, broken, w13, w2, dy, "silu", 10.0)
        keep = torch.arange(tokens, device="cuda") != 1
        assert torch.equal(got["y"][keep], want["y"][keep]) and torch.equal(got["dx"][keep], want["dx"][keep])
        if bad != bad:
            assert got["y"][1].isnan().all() and got["dw13"].isnan().any()


def test_streams_and_graphs(cuda_device):
    """Calls on two streams at once, and two captured graphs that are replayed in turn on new inputs, each with buffers of its own."""
    from fused_cpp_b200 import moe

    sets = [make(tokens, 256, 128, seed=tokens) for tokens in (40, 600)]
    want = [run(moe, *s, "silu", 10.0) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for stream, s in zip(streams, sets):
            with torch.cuda.stream(stream):
                got.append(run(moe, *s, "silu", 10.0))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(a[name], b[name]) for name in a)
    graphs = []
    for s in sets:
        leaves = [t.clone() for t in s]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(moe, *leaves, "silu", 10.0)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs = run(moe, *leaves, "silu", 10.0)
        graphs.append((graph, leaves, outputs))
    for round_ in range(3):
        fresh = [make(s[0].shape[0], 256, 128, seed=100 + round_) for s in sets]
        for (graph, leaves, _), new in zip(graphs, fresh):
            for to, value in zip(leaves, new):
                to.copy_(value)
            graph.replay()
        torch.cuda.synchronize()
        for (_, _, outputs), new in zip(graphs, fresh):
            expected = run(moe, *new, "silu", 10.0)
            assert all(torch.equal(outputs[name], expected[name]) for name in outputs)


def test_first_call_of_a_thread(cuda_device):
    """A thread whose first call into CUDA is the backward pass (an autograd worker's, or any other)."""
    import threading

    from fused_cpp_b200 import moe

    x, w13, w2, dy = make(20, 64, 48)
    want = run(moe, x, w13, w2, dy)
    y, kept = moe.gated_mlp_forward(x, w13, w2)
    torch.cuda.synchronize()
    found = []
    thread = threading.Thread(target=lambda: found.append(moe.gated_mlp_backward(dy, x, w13, w2, kept)))
    thread.start()
    thread.join()
    assert len(found) == 1 and torch.equal(found[0][0], want["dx"]) and torch.equal(found[0][1], want["dw13"])


def test_passes_without_a_tape_are_captured_beside_an_eager_graph(cuda_device):
    """The two passes have no leaves whose accumulators an eager graph could have tied to another stream."""
    from fused_cpp_b200 import moe

    leaves = [t.requires_grad_(True) for t in make(48, 128, 64)[:3]]
    dy = make(48, 128, 64)[3]
    alive = moe.gated_mlp(*leaves)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, kept = moe.gated_mlp_forward(*leaves)
        grads = moe.gated_mlp_backward(dy, *leaves, kept)
    graph.replay()
    assert torch.equal(y, alive.detach())
    for got, want in zip(grads, torch.autograd.grad(alive, leaves, dy)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("tokens, hidden, inter", [
    (65, 384, 384), (65, 392, 384), (66, 384, 392), (131, 192, 312), (200, 152, 904), (256, 896, 896), (80, 264, 1000), (257, 384, 384), (600, 4104, 256),
    (1333, 2048, 1024), (520, 5000, 1304), (2100, 136, 2000)])
def test_sizes_about_the_rules(cuda_device, tokens, hidden, inter):
    """Between the forms for few and for many rows, one launch or two for the gradients, and gradients whose tiles the pairs share out unevenly."""
    from fused_cpp_b200 import _lib, moe

    x, w13, w2, dy = make(tokens, hidden, inter, seed=tokens)
    want = run(moe, x, w13, w2, dy, "silu", 10.0)
    check_all(want, x, w13, w2, dy, "silu", 10.0)
    y, kept = moe.gated_mlp_forward(x, w13, w2, swiglu_limit=10.0)
    assert torch.equal(y, want["y"])
    for needs in ((True, False, False), (False, True, False), (False, False, True), (True, False, True), (False, True, True)):
        got = moe.gated_mlp_backward(dy, x, w13, w2, kept, needs=needs)
        for name, need, value in zip(("dx", "dw13", "dw2"), needs, got):
            assert (value is None) if not need else torch.equal(value, want[name]), (needs, name)
    assert _lib.dense_status() == (0, 0)


def test_refusals_of_the_library(cuda_device):
    """What only the library can see is refused as the same kind of error: a kept buffer on no boundary."""
    from fused_cpp_b200 import moe

    x, w13, w2, dy = make(5, 64, 40)
    _, kept = moe.gated_mlp_forward(x, w13, w2)
    shifted = torch.empty(kept.numel() + 2, dtype=torch.uint8, device="cuda")[2:].copy_(kept)
    with pytest.raises(ValueError, match="aligned"):
        moe.gated_mlp_backward(dy, x, w13, w2, shifted)
    with pytest.raises(ValueError, match="kept"):
        moe.gated_mlp_backward(dy, x, w13, w2, kept[:-1])
