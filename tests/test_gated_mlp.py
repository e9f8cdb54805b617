"""Arguments of the gated feed-forward block that are refused before anything reaches the GPU."""
import pytest
import torch

from fused_cpp_b200 import _lib, moe
from fused_cpp_b200.moe import gated


def _call(**changes):
    arguments = {"input": torch.zeros(3, 16, dtype=torch.bfloat16), "w13": torch.zeros(48, 16, dtype=torch.bfloat16),
                 "w2": torch.zeros(16, 24, dtype=torch.bfloat16)}
    options = {name: changes.pop(name) for name in list(changes) if name not in arguments}
    arguments.update(changes)
    return moe.gated_mlp(arguments["input"], arguments["w13"], arguments["w2"], **options)


@pytest.mark.parametrize("changes, error, text", [
    ({"input": torch.zeros(3, 16)}, TypeError, "input must be torch.bfloat16"),
    ({"w13": torch.zeros(48, 16)}, TypeError, "w13 must be torch.bfloat16"),
    ({"w2": torch.zeros(16, 24)}, TypeError, "w2 must be torch.bfloat16"),
    ({"input": [1.0]}, TypeError, "must be a torch.Tensor"),
    ({"input": torch.zeros(3, 24, dtype=torch.bfloat16)}, ValueError, "H=16"),
    ({"w13": torch.zeros(40, 16, dtype=torch.bfloat16)}, ValueError, "w13 must be"),
    ({"w2": torch.zeros(1, 16, 24, dtype=torch.bfloat16)}, ValueError, "weights must be"),
    ({"w13": torch.zeros(24, 16, dtype=torch.bfloat16), "w2": torch.zeros(16, 12, dtype=torch.bfloat16)}, ValueError, "multiples of 8"),
    ({"activation": "relu"}, ValueError, "activation must be"),
    ({"swiglu_limit": 7.0}, ValueError, "swiglu_limit=10.0"),
    ({"swiglu_limit": 10.0, "activation": "gelu"}, ValueError, "only valid with activation='silu'"),
    ({}, ValueError, "CUDA"),
])
def test_refusals(changes, error, text):
    with pytest.raises(error, match=text):
        _call(**changes)


@pytest.mark.parametrize("rows, inter", [(0, 8), (1, 8), (32, 32), (33, 40), (1333, 1024)])
def test_kept_derivatives_have_the_size_the_library_wants(rows, inter):
    assert gated._derivative_bytes(rows, inter) == 4 * _lib.load().fmoe_gated_mlp_derivative_count(rows, inter)
    assert gated._kept_bytes(rows, inter) == gated._derivative_bytes(rows, inter) + 2 * rows * inter


def test_backward_refusals():
    x, w13, w2 = (torch.zeros(*shape, dtype=torch.bfloat16) for shape in ((3, 16), (48, 16), (16, 24)))
    kept = torch.zeros(gated._kept_bytes(3, 24), dtype=torch.uint8)
    with pytest.raises(ValueError, match="input's shape"):
        moe.gated_mlp_backward(x[:2], x, w13, w2, kept)
    for wrong in (kept[:-1], kept.to(torch.int8), None):
        with pytest.raises(ValueError, match="what gated_mlp_forward returned"):
            moe.gated_mlp_backward(x, x, w13, w2, wrong)
    with pytest.raises(TypeError, match="dy must be torch.bfloat16"):
        moe.gated_mlp_backward(x.float(), x, w13, w2, kept)
    with pytest.raises(ValueError, match="needs"):
        moe.gated_mlp_backward(x, x, w13, w2, kept, needs=(True,))
    with pytest.raises(ValueError, match="CUDA"):
        moe.gated_mlp_backward(x, x, w13, w2, kept)
