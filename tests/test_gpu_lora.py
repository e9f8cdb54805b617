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
