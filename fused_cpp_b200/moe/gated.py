"""The gated feed-forward block with its gradients: y = (act(x Wg^T, x Wu^T)) W2^T on bf16 tensors.

    y = gated_mlp(x, w13, w2)                              # serving, or inside a differentiated program
    dx, dw13, dw2 = torch.autograd.grad(y, (x, w13, w2), dy)

The trainable companion of `shared_mlp_bf16_tiled`: the same weights ([2F, H] gate rows then up rows, and [H, F]) and the same
activations, as plain tensors that an optimiser updates.  Both projections, the activation and the product are one kernel, the down projection a
second; the backward pass is three launches.  Sums are fp32; h = act(..) is rounded to bf16 for the down projection, as in the fused MoE
operators.  `gated_mlp_forward` and `gated_mlp_backward` are the two passes for programs that keep their own tape.

What a forward pass keeps for the backward pass besides its inputs: h [T, F] and the partial derivatives of h by gate and by up, fp32 [T, 2F].
"""
from __future__ import annotations

from typing import Any

import torch

from .. import _lib
from .bf16_tiled import _native_activation_name

_ACTIVATIONS = {"silu": (_lib.ACTIVATION_SILU, 0.0), "silu_clamp10": (_lib.ACTIVATION_SILU, 10.0), "gelu": (_lib.ACTIVATION_GELU, 0.0),
                "swigluoai": (_lib.ACTIVATION_SWIGLUOAI, 0.0)}


def _activation(activation: Any, swiglu_limit: float | None) -> tuple[int, float]:
    name = _native_activation_name(activation, None, swiglu_limit)
    if name not in _ACTIVATIONS:
        raise ValueError(f"gated_mlp activation must be 'silu', 'gelu' or 'swigluoai', got {name!r}")
    return _ACTIVATIONS[name]


def _check_tensor(name: str, tensor: Any, device: torch.device | None) -> None:
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if tensor.dtype is not torch.bfloat16:
        raise TypeError(f"{name} must be torch.bfloat16, got {tensor.dtype}")
    if device is not None and tensor.device != device:
        raise ValueError(f"{name} must lie on the input's device")


def _check(input, w13, w2) -> tuple[int, int]:
    _check_tensor("input", input, None)
    _check_tensor("w13", w13, input.device)
    _check_tensor("w2", w2, input.device)
    if w13.dim() != 2 or w2.dim() != 2:
        raise ValueError("gated_mlp weights must be [2F, H] and [H, F]")
    hidden, inter = int(w2.shape[0]), int(w2.shape[1])
    if tuple(w13.shape) != (2 * inter, hidden):
        raise ValueError(f"w13 must be [2F, H] = [{2 * inter}, {hidden}] beside w2 [H, F], got {tuple(w13.shape)}")
    if input.dim() < 1 or input.shape[-1] != hidden:
        raise ValueError(f"input must be [..., H={hidden}], got {tuple(input.shape)}")
    if hidden % 8 or inter % 8 or not hidden or not inter:
        raise ValueError(f"H and F must be positive multiples of 8 (H={hidden}, F={inter})")
    return hidden, inter


def _require_cuda(tensor: torch.Tensor) -> None:
    if not tensor.is_cuda:
        raise ValueError("gated_mlp takes CUDA tensors (this build has no CPU path)")


def _rows(tensor: torch.Tensor, columns: int) -> torch.Tensor:
    """[..., columns] as rows that the kernels can read where they are: unit column stride, every row on a 16-byte boundary."""
    rows = tensor.reshape(-1, columns)
    if rows.stride(1) == 1 and rows.data_ptr() % 16 == 0 and (rows.shape[0] == 1 or (rows.stride(0) % 8 == 0 and rows.stride(0) >= columns)):
        return rows
    rows = rows.contiguous()
    return rows if rows.data_ptr() % 16 == 0 else rows.clone()


def _stride(rows: torch.Tensor) -> int:
    """Elements from a row to the next; a single row may carry any stride."""
    return rows.stride(0) if rows.shape[0] > 1 else rows.shape[1]


def _whole(tensor: torch.Tensor) -> torch.Tensor:
    """A weight as contiguous rows on a 16-byte boundary."""
    tensor = tensor if tensor.is_contiguous() else tensor.contiguous()
    return tensor if tensor.data_ptr() % 16 == 0 else tensor.clone()


def _forward(rows, w13, w2, code: int, limit: float, keep: bool, y):
    count, hidden = rows.shape
    inter = w2.shape[1]
    h = torch.empty((count, inter), dtype=torch.bfloat16, device=rows.device)
    derivatives = torch.empty((count, 2 * inter), dtype=torch.float32, device=rows.device) if keep else None
    _lib.check(_lib.load().fmoe_gated_mlp_forward(rows.data_ptr(), _stride(rows), w13.data_ptr(), w2.data_ptr(), count, hidden, inter, code, limit,
                                                  h.data_ptr(), _lib._ptr(derivatives), y.data_ptr(), _lib._stream()))
    return h, derivatives


def _backward(dy, rows, w13, w2, h, derivatives, needs):
    count, hidden = rows.shape
    inter = w2.shape[1]
    if count == 0:
        return tuple(torch.zeros_like(t, memory_format=torch.contiguous_format) if need else None for need, t in zip(needs, (rows, w13, w2)))
    dx = torch.empty((count, hidden), dtype=torch.bfloat16, device=rows.device) if needs[0] else None
    dw13 = torch.empty((2 * inter, hidden), dtype=torch.bfloat16, device=rows.device) if needs[1] else None
    dw2 = torch.empty((hidden, inter), dtype=torch.bfloat16, device=rows.device) if needs[2] else None
    d_gate_up = torch.empty((count, 2 * inter), dtype=torch.bfloat16, device=rows.device) if needs[0] or needs[1] else None
    _lib.check(_lib.load().fmoe_gated_mlp_backward(dy.data_ptr(), _stride(dy), rows.data_ptr(), _stride(rows), w13.data_ptr(), w2.data_ptr(), h.data_ptr(),
                                                   _lib._ptr(derivatives), count, hidden, inter, _lib._ptr(d_gate_up), _lib._ptr(dx), _lib._ptr(dw13),
                                                   _lib._ptr(dw2), _lib._stream()))
    return dx, dw13, dw2


class _GatedMLP(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, w13, w2, code, limit):
        with _lib.on_device_of(input):
            rows, w13_rows, w2_rows = _rows(input, w2.shape[0]), _whole(w13), _whole(w2)
            y = torch.empty(input.shape, dtype=torch.bfloat16, device=input.device)
            # dW2 needs h alone, dx and dW13 the derivatives.
            h, derivatives = _forward(rows, w13_rows, w2_rows, code, limit, ctx.needs_input_grad[0] or ctx.needs_input_grad[1], y)
        ctx.save_for_backward(input, w13, w2, h, derivatives)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        input, w13, w2, h, derivatives = ctx.saved_tensors
        with _lib.on_device_of(input):
            hidden = w2.shape[0]
            dx, dw13, dw2 = _backward(_rows(dy, hidden), _rows(input, hidden), _whole(w13), _whole(w2), h,
                                      derivatives, ctx.needs_input_grad[:3])
        return None if dx is None else dx.view(input.shape), dw13, dw2, None, None


def gated_mlp(input, w13, w2, *, activation: Any = "silu", swiglu_limit: float | None = None, out=None):
    """bf16 [..., H] x w13 [2F, H], w2 [H, F] -> bf16 [..., H]; differentiable by input, w13 and w2 (once).

    activation: "silu", "gelu" or "swigluoai"; swiglu_limit: None, 0 or 10.0 (with "silu").  H and F are multiples of 8.  With `out`
    (contiguous, no gradients asked for) the result is written there and `out` returned."""
    _check(input, w13, w2)
    code, limit = _activation(activation, swiglu_limit)
    _require_cuda(input)
    if torch.is_grad_enabled() and (input.requires_grad or w13.requires_grad or w2.requires_grad):
        if out is not None:
            raise ValueError("out cannot be given where gradients are asked for")
        return _GatedMLP.apply(input, w13, w2, code, limit)
    if out is None:
        out = torch.empty(input.shape, dtype=torch.bfloat16, device=input.device)
        y = out
    else:
        _check_tensor("out", out, input.device)
        if out.shape != input.shape or not out.is_contiguous():
            raise ValueError("out must be contiguous and match the input shape")
        y = out if out.data_ptr() % 16 == 0 else torch.empty(out.shape, dtype=out.dtype, device=out.device)
    with _lib.on_device_of(input):
        _forward(_rows(input, w2.shape[0]), _whole(w13), _whole(w2), code, limit, False, y)
    return out if y is out else out.copy_(y)


def gated_mlp_forward(input, w13, w2, *, activation: Any = "silu", swiglu_limit: float | None = None):
    """The forward pass without a tape: (y, h, derivatives), the last two for `gated_mlp_backward`."""
    _check(input, w13, w2)
    code, limit = _activation(activation, swiglu_limit)
    _require_cuda(input)
    with torch.no_grad(), _lib.on_device_of(input):
        y = torch.empty(input.shape, dtype=torch.bfloat16, device=input.device)
        h, derivatives = _forward(_rows(input, w2.shape[0]), _whole(w13), _whole(w2), code, limit, True, y)
    return y, h, derivatives


def gated_mlp_backward(dy, input, w13, w2, h, derivatives, *, needs: tuple = (True, True, True)):
    """(dx, dw13, dw2) from dy [..., H] and what `gated_mlp_forward` returned; None where `needs` says so."""
    hidden, inter = _check(input, w13, w2)
    _check_tensor("dy", dy, input.device)
    _check_tensor("h", h, input.device)
    if not isinstance(derivatives, torch.Tensor) or derivatives.dtype is not torch.float32 or derivatives.device != input.device:
        raise TypeError("derivatives must be the float32 tensor that gated_mlp_forward returned")
    if dy.shape != input.shape:
        raise ValueError(f"dy must have the input's shape {tuple(input.shape)}, got {tuple(dy.shape)}")
    rows = input.numel() // hidden
    if tuple(h.shape) != (rows, inter) or tuple(derivatives.shape) != (rows, 2 * inter) or not h.is_contiguous() or not derivatives.is_contiguous():
        raise ValueError("h and derivatives must be what gated_mlp_forward returned for this input")
    if len(needs) != 3:
        raise ValueError("needs must say for dx, dw13 and dw2 whether they are wanted")
    _require_cuda(input)
    with torch.no_grad(), _lib.on_device_of(input):
        dx, dw13, dw2 = _backward(_rows(dy, hidden), _rows(input, hidden), _whole(w13), _whole(w2), _whole(h), _whole(derivatives), tuple(bool(n) for n in needs))
    return None if dx is None else dx.view(input.shape), dw13, dw2
