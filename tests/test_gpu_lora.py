"""Dense W8A8 linear with low-rank adapters against the definition in 64 bits.

Tolerances, element by element.  The base product is exact up to four 32-bit roundings (accumulator, two scales, bias): 4 2^-24 of the magnitudes.  A
coefficient t_r = scaling (A x)_r is a 32-bit sum of K products (K 2^-24 of their magnitudes, the scaling's rounding in it) and is rounded to bf16 where
the result is bf16 (u = 2^-8 of it), or held as three bf16 terms (2^-24 of it) where it is fp32; the sum over ranks adds R 2^-24 of its magnitudes.
The result is rounded once: u, or 2^-24 for fp32."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24


def make(rows, k, n, count, rank, seed=0, none=0.2, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(rows, k, generator=g, device=device).bfloat16()
    w = torch.randint(-127, 128, (n, k), generator=g, device=device, dtype=torch.int8)
    s = (0.5 + torch.rand(n, generator=g, device=device)) / (73 * k ** 0.5)
    a = (torch.randn(count, rank, k, generator=g, device=device) / k ** 0.5).bfloat16()
    b = (torch.randn(count, n, rank, generator=g, device=device) / rank ** 0.5).bfloat16()
    scaling = 0.5 + torch.rand(count, generator=g, device=device)
    ids = torch.randint(count, (rows,), generator=g, device=device)
    ids[torch.rand(rows, generator=g, device=device) < none] = -1
    bias = torch.randn(n, generator=g, device=device)
    return x, w, s, a, b, scaling, ids, bias


def base_product(x, w, s, bias):
    """The quantised product by its definition, every rounding spelled out: fp32 [M, N].  Integers in 64-bit floats are exact."""
    amax = x.float().abs().amax(dim=1, keepdim=True)
    scale = torch.where(amax > 0, amax * torch.tensor(1 / 127, dtype=torch.float32, device=x.device), torch.ones_like(amax))
    q = torch.clamp(torch.round(x.float() / scale), -128, 127)
    acc = (q.double() @ w.double().T).float()
    return acc * scale * s + (0 if bias is None else bias)


def check(got, base_f32, x, a, b, scaling, ids):
    """base_f32: the fp32 base product, whose every bit is defined."""
    step = torch.finfo(got.dtype).eps / 2
    t_step = step if got.dtype == torch.bfloat16 else E32
    k, rank = x.shape[1], a.shape[1]
    want, allowed = base_f32.double(), 2 * E32 * base_f32.double().abs()
    for adapter in range(a.shape[0]):
        rows = torch.nonzero(ids == adapter).flatten()
        xr, ar, br = x[rows].double(), a[adapter].double(), b[adapter].double()
        t = scaling[adapter].double() * xr @ ar.T
        t_error = t_step * t.abs() + (k + 2) * E32 * scaling[adapter].double() * (xr.abs() @ ar.abs().T)
        want[rows] += t @ br.T
        allowed[rows] += t_error @ br.abs().T + (rank + 2) * E32 * ((t.abs() + t_error) @ br.abs().T)
    allowed = allowed * (1 + step) + step * want.abs() + 1e-30
    worst = ((got.double() - want).abs() / allowed).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("rows, k, n, count, rank", [
    (1, 16, 8, 1, 1), (1, 7168, 1536, 8, 16), (2, 130, 130, 3, 4), (3, 257, 300, 2, 8), (16, 1024, 256, 16, 16), (17, 512, 136, 5, 24), (31, 2056, 1234, 7, 40),
    (33, 384, 128, 40, 64), (64, 1536, 640, 64, 16), (65, 7168, 1536, 3, 32), (100, 336, 513, 100, 9), (128, 2048, 272, 128, 17), (129, 768, 200, 4, 128),
    (200, 1000, 24576, 6, 64), (257, 1024, 384, 200, 65), (300, 640, 129, 2, 130), (777, 2056, 1234, 5, 24), (1030, 512, 1000, 9, 200), (64, 256, 64, 2, 512)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_projection_with_adapters(cuda_device, rows, k, n, count, rank, dtype):
    from fused_cpp_b200 import i8gemm, lora

    x, w, s, a, b, scaling, ids, bias = make(rows, k, n, count, rank, seed=rows)
    packed, adapters = i8gemm.prepare(w, s), lora.prepare_adapters(a, b, scaling)
    base = base_product(x, w, s, bias)
    got = i8gemm.dynamic_scaled_mm_lora(x, packed, adapters, ids, bias=bias, out_dtype=dtype)
    check(got, base, x, a, b, scaling, ids)
    assert torch.equal(got[ids < 0], base[ids < 0].to(dtype))  # a row without an adapter is the base product, bit for bit


@pytest.mark.parametrize("rows, k, n, count, rank, none", [
    (129, 256, 25000, 3, 16, 0.0), (256, 1536, 13000, 200, 33, 0.3), (700, 130, 4504, 2, 8, 0.9), (2000, 400, 1600, 900, 16, 0.1), (3000, 272, 1288, 4, 100, 0.2),
    (5000, 129, 777, 50, 24, 0.1)])
@pytest.mark.parametrize("order", ["mixed", "runs"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_rows(cuda_device, rows, k, n, count, rank, none, order, dtype):
    """The sizes at which the two-SM kernel takes over, in wide and narrow tiles, aligned output rows and others, up to 200 adapters in 256 rows."""
    from fused_cpp_b200 import i8gemm, lora

    x, w, s, a, b, scaling, ids, bias = make(rows, k, n, count, rank, seed=rows, none=none)
    if order == "runs":
        ids = ids[torch.arange(rows, device=ids.device) // 300]
    packed, adapters = i8gemm.prepare(w, s), lora.prepare_adapters(a, b, scaling)
    base = base_product(x, w, s, None)
    got = i8gemm.dynamic_scaled_mm_lora(x, packed, adapters, ids, out_dtype=dtype)
    check(got, base, x, a, b, scaling, ids)
    assert torch.equal(got[ids < 0], base[ids < 0].to(dtype))


def test_layouts_ids_and_ranks(cuda_device):
    """Ids of both integer types and out of range, rows in three dimensions, a strided x and strided ids, adapters of unequal ranks, one scaling for all."""
    from fused_cpp_b200 import i8gemm, lora

    x, w, s, a, b, scaling, ids, bias = make(60, 264, 200, 4, 24)
    packed, adapters = i8gemm.prepare(w, s), lora.prepare_adapters(a, b, scaling)
    want = i8gemm.dynamic_scaled_mm_lora(x, packed, adapters, ids, bias=bias)
    assert torch.equal(i8gemm.dynamic_scaled_mm_lora(x, packed, adapters, ids.int(), bias=bias), want)
    for outside in (4, 2 ** 31 - 1, -(2 ** 31)):
        far = torch.where(ids < 0, torch.full_like(ids, outside), ids)
        assert torch.equal(i8gemm.dynamic_scaled_mm_lora(x, packed, adapters, far, bias=bias), want)
        assert torch.equal(i8gemm.dynamic_scaled_mm_lora(x, packed, adapters, far.int(), bias=bias), want)
    assert torch.equal(i8gemm.dynamic_scaled_mm_lora(x, packed, adapters, torch.where(ids < 0, ids + 2 ** 40, ids), bias=bias), want)
    cube = i8gemm.dynamic_scaled_mm_lora(x.view(3, 20, 264), packed, adapters, ids.view(3, 20), bias=bias)
    assert cube.shape == (3, 20, 200) and torch.equal(cube.view(60, 200), want)
    wide = torch.zeros(60, 300, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:267] = x
    strided = torch.stack((ids, ids), 1)[:, 0]
    assert torch.equal(i8gemm.dynamic_scaled_mm_lora(wide[:, 3:267], packed, adapters, strided, bias=bias), want)
    empty = i8gemm.dynamic_scaled_mm_lora(x[:0], packed, adapters, ids[:0])
    assert empty.shape == (0, 200) and empty.dtype == torch.bfloat16
    # Unequal ranks, padded with zeros: the same as whole adapters whose other ranks are zero.
    ranks = (24, 3, 17, 1)
    cut = [(a[i, :r], b[i, :, :r]) for i, r in enumerate(ranks)]
    whole_a, whole_b = a.clone(), b.clone()
    for i, r in enumerate(ranks):
        whole_a[i, r:] = 0
        whole_b[i, :, r:] = 0
    unequal = lora.prepare_adapters([p[0] for p in cut], [p[1].cpu() for p in cut], 0.5)
    assert unequal.rank == 24 and unequal.scaling.tolist() == [0.5] * 4
    equal = lora.prepare_adapters(whole_a, whole_b, [0.5] * 4)
    assert torch.equal(i8gemm.dynamic_scaled_mm_lora(x, packed, unequal, ids), i8gemm.dynamic_scaled_mm_lora(x, packed, equal, ids))


def test_a_slot_is_exchanged_in_place(cuda_device):
    from fused_cpp_b200 import i8gemm, lora

    x, w, s, a, b, scaling, ids, _ = make(40, 256, 136, 3, 16)
    packed, adapters = i8gemm.prepare(w, s), lora.prepare_adapters(a, b, scaling)
    before = i8gemm.dynamic_scaled_mm_lora(x, packed, adapters, ids)
    new_a, new_b = a[1, :9].flip(1).contiguous(), b[1, :, :9].flip(0).contiguous()
    lora.set_adapter(adapters, 1, new_a, new_b, 0.75)
    after = i8gemm.dynamic_scaled_mm_lora(x, packed, adapters, ids)
    assert torch.equal(after[ids != 1], before[ids != 1])
    a, b, scaling = a.clone(), b.clone(), scaling.clone()
    a[1], b[1] = 0, 0
    a[1, :9], b[1, :, :9], scaling[1] = new_a, new_b, 0.75
    check(after, base_product(x, w, s, None), x, a, b, scaling, ids)


@pytest.mark.parametrize("rows", [40, 200, 1000])
def test_a_row_depends_on_itself_alone(cuda_device, rows):
    """Neighbours, their adapters, NaN and infinities among them, and the row's place change no bit of it, as long as the same kernel serves the batch."""
    from fused_cpp_b200 import i8gemm, lora

    x, w, s, a, b, scaling, ids, bias = make(rows, 512, 5000, 6, 16)
    packed, adapters = i8gemm.prepare(w, s), lora.prepare_adapters(a, b, scaling)
    want = i8gemm.dynamic_scaled_mm_lora(x, packed, adapters, ids, bias=bias)
    order = torch.randperm(rows, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    assert torch.equal(i8gemm.dynamic_scaled_mm_lora(x[order], packed, adapters, ids[order], bias=bias), want[order])
    broken, other = x.clone(), ids.clone()
    broken[::3, 7] = float("nan")
    broken[1::3, 9] = float("inf")
    other[::3] = (other[::3] + 1) % 6
    got = i8gemm.dynamic_scaled_mm_lora(broken, packed, adapters, other, bias=bias)
    assert torch.equal(got[2::3], want[2::3])


@pytest.mark.parametrize("a_value, b_value", [(float("inf"), 1.0), (1.0, float("nan"))])
def test_adapters_that_are_not_finite_are_refused(cuda_device, a_value, b_value):
    from fused_cpp_b200 import lora

    a, b = torch.ones(2, 4, 16).bfloat16(), torch.ones(2, 24, 4).bfloat16()
    a[1, 2, 3], b[1, 2, 3] = a_value, b_value
    with pytest.raises(ValueError, match="finite"):
        lora.prepare_adapters(a, b)
    with pytest.raises(ValueError, match="finite"):
        lora.prepare_adapters(a[:1], b[:1], float("inf"))


def test_refusals_on_the_gpu(cuda_device):
    from fused_cpp_b200 import i8gemm, lora

    x, w, s, a, b, scaling, ids, bias = make(10, 64, 48, 2, 8)
    packed, adapters = i8gemm.prepare(w, s), lora.prepare_adapters(a, b, scaling)
    mm = i8gemm.dynamic_scaled_mm_lora
    for call, error, text in (
            (lambda: mm(x.float(), packed, adapters, ids), TypeError, "CUDA bfloat16"),
            (lambda: mm(x[:, :32], packed, adapters, ids), ValueError, "K=64"),
            (lambda: mm(x, packed, lora.prepare_adapters(a[:, :, :32], b), ids), ValueError, "beside a weight"),
            (lambda: mm(x, packed, adapters, ids[:4]), ValueError, "one per row"),
            (lambda: mm(x, packed, adapters, ids.float()), TypeError, "int32 or int64"),
            (lambda: mm(x, packed, adapters, ids.cpu()), ValueError, "input's device"),
            (lambda: mm(x, packed, adapters, ids, bias=bias[:4]), ValueError, "bias must be"),
            (lambda: mm(x, packed, adapters, ids, out_dtype=torch.float16), ValueError, "out_dtype"),
            (lambda: mm(x, packed, adapters, ids, nthreads=-1), ValueError, "non-negative")):
        with pytest.raises(error, match=text):
            call()


def test_streams_and_graphs(cuda_device):
    """Calls on two streams at once, and two captured graphs replayed in turn on new rows and ids, each with a workspace of its own."""
    from fused_cpp_b200 import i8gemm, lora

    x, w, s, a, b, scaling, ids, bias = make(700, 512, 5000, 6, 16)
    packed, adapters = i8gemm.prepare(w, s), lora.prepare_adapters(a, b, scaling)
    parts = [(x[:30], ids[:30]), (x[30:], ids[30:])]
    want = [i8gemm.dynamic_scaled_mm_lora(*p[:1], packed, adapters, p[1], bias=bias) for p in parts]
    streams = [torch.cuda.Stream() for _ in parts]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for stream, p in zip(streams, parts):
            with torch.cuda.stream(stream):
                got.append(i8gemm.dynamic_scaled_mm_lora(p[0], packed, adapters, p[1], bias=bias))
        torch.cuda.synchronize()
        assert all(torch.equal(g, e) for g, e in zip(got, want))
    graphs = []
    for p in parts:
        inputs = (p[0].clone(), p[1].clone())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = i8gemm.dynamic_scaled_mm_lora(inputs[0], packed, adapters, inputs[1], bias=bias)
        graphs.append((graph, inputs, out))
    for round_ in range(3):
        for graph, inputs, _ in graphs:
            inputs[0].copy_(inputs[0].flip(0))
            inputs[1].copy_((inputs[1] + 1 + round_) % 7 - 1)
            graph.replay()
        torch.cuda.synchronize()
        for _, inputs, out in graphs:
            assert torch.equal(out, i8gemm.dynamic_scaled_mm_lora(inputs[0], packed, adapters, inputs[1], bias=bias))


def test_attention_output_then_feed_forward(cuda_device):
    """The two operators one after the other, as a layer has them: the attention's output projection with the requests' adapters, then the gated block, and the
    block's weights learning from what comes out."""
    from fused_cpp_b200 import deepseek_v4_w8a8, i8gemm, lora, moe

    x, w, s, a, b, scaling, ids, _ = make(50, 512, 256, 4, 16)
    packed, adapters = i8gemm.prepare(w, s), lora.prepare_adapters(a, b, scaling)
    g = torch.Generator(device="cuda").manual_seed(5)
    w13 = (torch.randn(256, 256, generator=g, device="cuda") / 16).bfloat16().requires_grad_(True)
    w2 = (torch.randn(256, 128, generator=g, device="cuda") / 12).bfloat16().requires_grad_(True)
    weight = deepseek_v4_w8a8.prepare_deepseek_v4_w8a8_linear_quantized_weight(w, s)
    projected = deepseek_v4_w8a8.deepseek_v4_wo_b_w8a8(x, weight, adapters=adapters, adapter_ids=ids)
    check(projected, base_product(x, w, s, None), x, a, b, scaling, ids)
    assert torch.equal(projected, i8gemm.dynamic_scaled_mm_lora(x, packed, adapters, ids))
    out = torch.empty_like(projected)
    assert deepseek_v4_w8a8.deepseek_v4_w8a8_linear(x, weight, out=out, adapters=adapters, adapter_ids=ids) is out and torch.equal(out, projected)
    with pytest.raises(ValueError, match="given together"):
        deepseek_v4_w8a8.deepseek_v4_w8a8_linear(x, weight, adapters=adapters)
    y = moe.gated_mlp(projected, w13, w2, swiglu_limit=10.0)
    with torch.no_grad():
        assert torch.equal(y, moe.gated_mlp(projected, w13, w2, swiglu_limit=10.0))
    y.float().square().mean().backward()
    assert w13.grad.isfinite().all() and w13.grad.any() and w2.grad.any()


@pytest.mark.parametrize("rows, k, n, count, rank", [
    (65, 8192, 200, 65, 64), (200, 4100, 300, 40, 64), (256, 8192, 136, 16, 70), (130, 3001, 520, 130, 33), (64, 8192, 200, 65, 64), (300, 8, 40, 5, 3),
    (270, 64, 64, 270, 17), (1500, 120, 72, 60, 130), (40, 130, 8200, 40, 7), (127, 2048, 128, 20, 200)])
@pytest.mark.parametrize("none", [0.0, 0.6])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sizes_about_the_rules(cuda_device, rows, k, n, count, rank, none, dtype):
    """Between the forms of the coefficients' kernel, many adapters in a tile, K ranges of one block, and row tiles of every size; x on no boundary too."""
    from fused_cpp_b200 import i8gemm, lora

    x, w, s, a, b, scaling, ids, bias = make(rows, k, n, count, rank, seed=rows, none=none)
    packed, adapters = i8gemm.prepare(w, s), lora.prepare_adapters(a, b, scaling)
    base = base_product(x, w, s, bias)
    got = i8gemm.dynamic_scaled_mm_lora(x, packed, adapters, ids, bias=bias, out_dtype=dtype)
    check(got, base, x, a, b, scaling, ids)
    assert torch.equal(got[ids < 0], base[ids < 0].to(dtype))
    shifted = torch.empty(rows * k + 1, dtype=x.dtype, device="cuda")[1:].view(rows, k).copy_(x)
    assert torch.equal(i8gemm.dynamic_scaled_mm_lora(shifted, packed, adapters, ids, bias=bias, out_dtype=dtype), got)


def test_adapters_in_training(cuda_device):
    """Adapters that are leaves of a graph are copied without it, and serve under and without recorded gradients."""
    from fused_cpp_b200 import i8gemm, lora

    x, w, s, a, b, scaling, ids, _ = make(20, 64, 40, 3, 8)
    packed = i8gemm.prepare(w, s)
    want = i8gemm.dynamic_scaled_mm_lora(x, packed, lora.prepare_adapters(a, b, scaling), ids)
    for first, second in ((a.clone().requires_grad_(True), b.clone().requires_grad_(True)), ([t.clone().requires_grad_(True) for t in a], list(b))):
        adapters = lora.prepare_adapters(first, second, scaling.clone().requires_grad_(True))
        assert not (adapters.a.requires_grad or adapters.b.requires_grad or adapters.scaling.requires_grad)
        assert torch.equal(i8gemm.dynamic_scaled_mm_lora(x, packed, adapters, ids), want)


def test_streams_at_once(cuda_device):
    """Calls of all forms on four streams at the same time, with the gated block's, give what they give alone."""
    from fused_cpp_b200 import i8gemm, lora, moe

    jobs = []
    for rows, k, n, count, rank in ((300, 1000, 520, 9, 40), (200, 4104, 304, 40, 64), (40, 512, 2000, 5, 16), (2000, 400, 3200, 30, 24)):
        x, w, s, a, b, scaling, ids, _ = make(rows, k, n, count, rank, seed=rows)
        packed, adapters = i8gemm.prepare(w, s), lora.prepare_adapters(a, b, scaling)
        w13, w2 = (torch.randn(shape, device="cuda").bfloat16() / 16 for shape in ((512, 256), (256, 256)))
        rows_in = torch.randn(rows, 256, device="cuda").bfloat16()

        def job(x=x, packed=packed, adapters=adapters, ids=ids, w13=w13, w2=w2, rows_in=rows_in):
            y, kept = moe.gated_mlp_forward(rows_in, w13, w2)
            return (i8gemm.dynamic_scaled_mm_lora(x, packed, adapters, ids), y, *moe.gated_mlp_backward(rows_in, rows_in, w13, w2, kept))
        jobs.append((job, job(), torch.cuda.Stream()))
    torch.cuda.synchronize()
    results = []
    for _ in range(20):
        for job, want, stream in jobs:
            with torch.cuda.stream(stream):
                results.append((job(), want))
    torch.cuda.synchronize()
    for got, want in results:
        assert all(torch.equal(g, v) for g, v in zip(got, want))
