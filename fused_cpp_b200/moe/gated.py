"""The gated feed-forward block with its gradients: y = (act(x Wg^T, x Wu^T)) W2^T on bf16 tensors.

    y = gated_mlp(x, w13, w2)                              # serving, or inside a differentiated program
    dx, dw13, dw2 = torch.autograd.grad(y, (x, w13, w2), dy)

The trainable companion of `shared_mlp_bf16_tiled`: the same weights ([2F, H] gate rows then up rows, and [H, F]) and the same
activations, as plain tensors that an optimiser updates.  Both projections, the activation and the product are one kernel, the down projection a
second; the backward pass is three launches.  Sums are fp32; h = act(..) is rounded to bf16 for the down projection, as in the fused MoE
operators.  `gated_mlp_forward` and `gated_mlp_backward` are the two passes for programs that keep their own tape.

What a forward pass keeps for the backward pass besides its inputs, in one buffer: the partial derivatives of h by gate and by up (fp32, in an
order of the library's own) and h [T, F].
"""
from __future__ import annotations

from typing import Any

import torch

from .. import _lib
from .bf16_tiled import _native_activation_name

_BF16 = torch.bfloat16
_ACTIVATIONS = {"silu": (_lib.ACTIVATION_SILU, 0.0), "silu_clamp10": (_lib.ACTIVATION_SILU, 10.0), "gelu": (_lib.ACTIVATION_GELU, 0.0),
                "swigluoai": (_lib.ACTIVATION_SWIGLUOAI, 0.0)}


def _activation(activation: Any, swiglu_limit: float | None) -> tuple[int, float]:
    name = _native_activation_name(activation, None, swiglu_limit)
    if name not in _ACTIVATIONS:
        raise ValueError(f"gated_mlp activation must be 'silu', 'gelu' or 'swigluoai', got {name!r}")
    return _ACTIVATIONS[name]


def _check_tensor(name: str, tensor: Any, index: int | None) -> None:
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if tensor.dtype is not _BF16:
        raise TypeError(f"{name} must be torch.bfloat16, got {tensor.dtype}")
    if index is not None and tensor.get_device() != index:
        raise ValueError(f"{name} must lie on the input's device")


def _check(input, w13, w2) -> tuple[int, int, int]:
    """(H, F, the CUDA device's index or -1) of tensors that go together."""
    _check_tensor("input", input, None)
    index = input.get_device()
    _check_tensor("w13", w13, index)
    _check_tensor("w2", w2, index)
    if w13.dim() != 2 or w2.dim() != 2:
        raise ValueError("gated_mlp weights must be [2F, H] and [H, F]")
    hidden, inter = w2.shape
    if w13.shape != (2 * inter, hidden):
        raise ValueError(f"w13 must be [2F, H] = [{2 * inter}, {hidden}] beside w2 [H, F], got {tuple(w13.shape)}")
    if input.dim() < 1 or input.shape[-1] != hidden:
        raise ValueError(f"input must be [..., H={hidden}], got {tuple(input.shape)}")
    if hidden % 8 or inter % 8 or not hidden or not inter:
        raise ValueError(f"H and F must be positive multiples of 8 (H={hidden}, F={inter})")
    return hidden, inter, index


def _require_cuda(index: int) -> None:
    if index < 0:
        raise ValueError("gated_mlp takes CUDA tensors (this build has no CPU path)")


def _rows(tensor: torch.Tensor, columns: int) -> torch.Tensor:
    """[..., columns] as rows that the kernels can read where they are: unit column stride, every row on a 16-byte boundary."""
    if tensor.dim() == 2 and tensor.is_contiguous() and tensor.data_ptr() % 16 == 0:
        return tensor
    rows = tensor.reshape(-1, columns)
    if rows.stride(1) == 1 and rows.data_ptr() % 16 == 0 and (rows.shape[0] == 1 or (rows.stride(0) % 8 == 0 and rows.stride(0) >= columns)):
        return rows
    rows = rows.contiguous()
    return rows if rows.data_ptr() % 16 == 0 else rows.clone()


def _like(input: torch.Tensor) -> torch.Tensor:
    """A contiguous result of the input's shape."""
    return torch.empty_like(input) if input.is_contiguous() else input.new_empty(input.shape)


def _stride(rows: torch.Tensor) -> int:
    """Elements from a row to the next; a single row may carry any stride."""
    return rows.stride(0) if rows.shape[0] > 1 else rows.shape[1]


def _whole(tensor: torch.Tensor) -> torch.Tensor:
    """A weight as contiguous rows on a 16-byte boundary."""
    tensor = tensor if tensor.is_contiguous() else tensor.contiguous()
    return tensor if tensor.data_ptr() % 16 == 0 else tensor.clone()


def _derivative_bytes(rows: int, inter: int) -> int:
    """4 * fmoe_gated_mlp_derivative_count: whole blocks of 32 rows x 32 channels x 2."""
    return -(-rows // 32) * -(-inter // 32) * 8192


def _kept_bytes(rows: int, inter: int) -> int:
    """The derivatives, then h."""
    return _derivative_bytes(rows, inter) + 2 * rows * inter


def _forward(index: int, rows, w13, w2, code: int, limit: float, keep: bool, y):
    """y, and what the backward pass needs (keep) or h alone, in one buffer (the caller's, so that it outlives the kernels on this stream)."""
    count, hidden = rows.shape
    inter = w2.shape[1]
    front = _derivative_bytes(count, inter) if keep else 0
    kept = rows.new_empty(front + 2 * count * inter, dtype=torch.uint8)
    address = kept.data_ptr()
    _lib.check(_lib.load().fmoe_gated_mlp_forward(rows.data_ptr(), _stride(rows), w13.data_ptr(), w2.data_ptr(), count, hidden, inter, code, limit,
                                                  address + front, address if keep else None, y.data_ptr(), _lib._stream_of(index)))
    return kept


def _backward(index: int, dy, rows, w13, w2, kept, need_x: bool, need_w13: bool, need_w2: bool):
    count, hidden = rows.shape
    inter = w2.shape[1]
    if count == 0:
        return (rows.new_zeros((0, hidden)) if need_x else None, w13.new_zeros(w13.shape) if need_w13 else None,
                w2.new_zeros(w2.shape) if need_w2 else None)
    dx = _like(rows) if need_x else None
    dw13 = torch.empty_like(w13) if need_w13 else None
    dw2 = torch.empty_like(w2) if need_w2 else None
    scratch = rows.new_empty((count, 2 * inter)) if need_x or need_w13 else None
    pointer = _lib._ptr
    address = kept.data_ptr()
    _lib.check(_lib.load().fmoe_gated_mlp_backward(dy.data_ptr(), _stride(dy), rows.data_ptr(), _stride(rows), w13.data_ptr(), w2.data_ptr(),
                                                   address + _derivative_bytes(count, inter), address, count, hidden, inter, pointer(scratch),
                                                   pointer(dx), pointer(dw13), pointer(dw2), _lib._stream_of(index)))
    return dx, dw13, dw2


class _GatedMLP(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, w13, w2, code, limit, index):
        return _lib.on_device(index, _GatedMLP._forward, ctx, input, w13, w2, code, limit, index)

    @staticmethod
    def _forward(ctx, input, w13, w2, code, limit, index):
        rows = _rows(input, w2.shape[0])
        y = _like(input)
        ctx.save_for_backward(input, w13, w2, _forward(index, rows, _whole(w13), _whole(w2), code, limit, True, y))
        ctx.index = index
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("gated_mlp is differentiable once: its backward pass has no gradient (create_graph)")
        return _lib.on_device(ctx.index, _GatedMLP._backward, ctx, dy)

    @staticmethod
    def _backward(ctx, dy):
        input, w13, w2, kept = ctx.saved_tensors
        hidden = w2.shape[0]
        dx, dw13, dw2 = _backward(ctx.index, _rows(dy, hidden), _rows(input, hidden), _whole(w13), _whole(w2), kept, *ctx.needs_input_grad[:3])
        return dx if dx is None or input.dim() == 2 else dx.view(input.shape), dw13, dw2, None, None, None


def gated_mlp(input, w13, w2, *, activation: Any = "silu", swiglu_limit: float | None = None, out=None):
    """bf16 [..., H] x w13 [2F, H], w2 [H, F] -> bf16 [..., H]; differentiable by input, w13 and w2 (once).

    activation: "silu", "gelu" or "swigluoai"; swiglu_limit: None, 0 or 10.0 (with "silu").  H and F are multiples of 8.  With `out`
    (contiguous, no gradients asked for) the result is written there and `out` returned.

    Both passes can be captured into a CUDA graph.  As with any function of torch, the engine refuses to capture a backward pass while an eager
    graph of the same leaves lives; `gated_mlp_forward` and `gated_mlp_backward` have no such condition."""
    _, _, index = _check(input, w13, w2)
    code, limit = _activation(activation, swiglu_limit)
    _require_cuda(index)
    if (input.requires_grad or w13.requires_grad or w2.requires_grad) and torch.is_grad_enabled():
        if out is not None:
            raise ValueError("out cannot be given where gradients are asked for")
        return _GatedMLP.apply(input, w13, w2, code, limit, index)
    return _lib.on_device(index, _serve, index, input, w13, w2, code, limit, out)


def _serve(index: int, input, w13, w2, code: int, limit: float, out):
    rows = _rows(input, w2.shape[0])
    if out is None:
        y = out = _like(input)
    else:
        _check_tensor("out", out, index)
        if out.shape != input.shape or not out.is_contiguous():
            raise ValueError("out must be contiguous and match the input shape")
        y = out if out.data_ptr() % 16 == 0 else rows.new_empty(input.shape)
    _forward(index, rows, _whole(w13), _whole(w2), code, limit, False, y)
    return out if y is out else out.copy_(y)


def gated_mlp_forward(input, w13, w2, *, activation: Any = "silu", swiglu_limit: float | None = None):
    """The forward pass without a tape: (y, kept), the second for `gated_mlp_backward`."""
    hidden, _, index = _check(input, w13, w2)
    code, limit = _activation(activation, swiglu_limit)
    _require_cuda(index)

    def call():
        rows = _rows(input.detach(), hidden)
        y = _like(rows).view(input.shape)
        return y, _forward(index, rows, _whole(w13.detach()), _whole(w2.detach()), code, limit, True, y)

    return _lib.on_device(index, call)


def gated_mlp_backward(dy, input, w13, w2, kept, *, needs: tuple = (True, True, True)):
    """(dx, dw13, dw2) from dy [..., H] and what `gated_mlp_forward` kept; None where `needs` says so."""
    hidden, inter, index = _check(input, w13, w2)
    _check_tensor("dy", dy, index)
    if dy.shape != input.shape:
        raise ValueError(f"dy must have the input's shape {tuple(input.shape)}, got {tuple(dy.shape)}")
    if not isinstance(kept, torch.Tensor) or kept.dtype is not torch.uint8 or kept.get_device() != index or not kept.is_contiguous() \
            or kept.shape != (_kept_bytes(input.numel() // hidden, inter),):
        raise ValueError("kept must be what gated_mlp_forward returned for this input")
    if len(needs) != 3:
        raise ValueError("needs must say for dx, dw13 and dw2 whether they are wanted")
    _require_cuda(index)

    def call():
        dx, dw13, dw2 = _backward(index, _rows(dy.detach(), hidden), _rows(input.detach(), hidden), _whole(w13.detach()), _whole(w2.detach()), kept,
                                  *(bool(need) for need in needs))
        return None if dx is None else dx.view(input.shape), dw13, dw2

    return _lib.on_device(index, call)
