"""Arguments of the adapter operators that are refused before anything reaches the GPU."""
import pytest
import torch

from fused_cpp_b200 import i8gemm, lora


def _bf16(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("a, b, scaling, error, text", [
    ([], [], 1.0, ValueError, "at least one"),
    ([_bf16(4, 16)], [], 1.0, ValueError, "as many a as b"),
    (torch.zeros(1, 4, 16), _bf16(1, 24, 4), 1.0, TypeError, "a must be torch.bfloat16"),
    (_bf16(1, 4, 16), torch.zeros(1, 24, 4), 1.0, TypeError, "b must be torch.bfloat16"),
    ([[1.0]], [_bf16(24, 4)], 1.0, TypeError, "must be a torch.Tensor"),
    ([_bf16(4)], [_bf16(24, 4)], 1.0, ValueError, "an adapter is a"),
    (_bf16(1, 4, 16), _bf16(1, 24, 5), 1.0, ValueError, "share R"),
    ([_bf16(4, 16), _bf16(4, 8)], [_bf16(24, 4), _bf16(24, 4)], 1.0, ValueError, "share K and N"),
    (_bf16(1, 513, 16), _bf16(1, 24, 513), 1.0, ValueError, "ranks must lie"),
    ([_bf16(0, 16)], [_bf16(24, 0)], 1.0, ValueError, "ranks must lie"),
    (_bf16(2, 4, 16), _bf16(2, 24, 4), [1.0, 2.0, 3.0], ValueError, "one per adapter"),
])
def test_prepare_refusals(a, b, scaling, error, text):
    with pytest.raises(error, match=text):
        lora.prepare_adapters(a, b, scaling)


def _holder(**changes):
    fields = {"a": _bf16(2, 4, 16), "b": _bf16(2, 24, 8), "scaling": torch.ones(2), "count": 2, "rank": 4, "k": 16, "n": 24}
    fields.update(changes)
    return lora.PreparedAdapters(**fields)


def test_set_adapter():
    """The holder's tensors may lie anywhere: a slot is exchanged in place, padding included."""
    holder = _holder(a=torch.ones(2, 4, 16).bfloat16(), b=torch.ones(2, 24, 8).bfloat16())
    lora.set_adapter(holder, 1, torch.full((3, 16), 2.0).bfloat16(), torch.full((24, 3), 3.0).bfloat16(), 0.5)
    assert holder.scaling.tolist() == [1.0, 0.5]
    assert (holder.a[0] == 1).all() and (holder.b[0] == 1).all()
    assert (holder.a[1, :3] == 2).all() and (holder.a[1, 3:] == 0).all()
    assert (holder.b[1, :, :3] == 3).all() and (holder.b[1, :, 3:] == 0).all()


@pytest.mark.parametrize("index, a, b, scaling, error, text", [
    (2, _bf16(4, 16), _bf16(24, 4), 1.0, ValueError, "index must lie"),
    (-1, _bf16(4, 16), _bf16(24, 4), 1.0, ValueError, "index must lie"),
    (0, _bf16(5, 16), _bf16(24, 5), 1.0, ValueError, "expected a"),
    (0, _bf16(4, 8), _bf16(24, 4), 1.0, ValueError, "expected a"),
    (0, _bf16(4, 16), torch.full((24, 4), float("inf")).bfloat16(), 1.0, ValueError, "finite"),
    (0, torch.full((4, 16), float("nan")).bfloat16(), _bf16(24, 4), 1.0, ValueError, "finite"),
    (0, _bf16(4, 16), _bf16(24, 4), float("inf"), ValueError, "finite"),
])
def test_set_adapter_refusals(index, a, b, scaling, error, text):
    with pytest.raises(error, match=text):
        lora.set_adapter(_holder(), index, a, b, scaling)


def test_projection_refusals():
    packed = i8gemm.PreparedI8GEMMWeight(torch.zeros(24, 16, dtype=torch.int8), torch.ones(24), 16, 24, 16, 24, "x")
    ids = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(TypeError, match="CUDA bfloat16"):
        i8gemm.dynamic_scaled_mm_lora(_bf16(3, 16), packed, _holder(), ids)
    with pytest.raises(TypeError, match="prepare_adapters"):
        i8gemm.dynamic_scaled_mm_lora(_bf16(3, 16), packed, None, ids)
    with pytest.raises(TypeError, match="i8gemm.prepare"):
        i8gemm.dynamic_scaled_mm_lora(_bf16(3, 16), None, _holder(), ids)
