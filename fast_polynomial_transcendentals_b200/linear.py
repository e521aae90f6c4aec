"""A linear layer with its bias, its activation and the residual connection in one kernel: `act(x @ weight.T + bias) + residual`.

Beside `gate_up` (the SwiGLU projection of the gated feed-forward) this is the projection of everything else in a block:
queries, keys and values with a bias, the attention's output onto the residual stream, a GELU feed-forward's two layers.
The activation and the residual are applied to the fp32 sums in registers and rounded once; nothing between the product and
the result is stored.  Any number of rows: one token streams the weight at the memory's rate, many rows run on the tensor
cores' pair form.

Differentiable for x, weight, bias and residual.  A training step keeps the slope of the activation in fp16 (times 2^15, so
that small slopes keep their precision) beside x and the weight (nothing where there is no activation); the gradients of x and
of the weight are products of the same kernels.
A second derivative and forward-mode differentiation are refused (RuntimeError).
Usable under `torch.compile` (`torch.ops.fpt_b200.linear_act`) and in captured graphs (what `qk_rope` says of captured backward
passes holds here too).
"""
from __future__ import annotations

import torch

from . import _lib
from .qk_rope import _choice, _ext

_FUNCTIONS = {"none": -1, "sigmoid": _lib.FN_SIGMOID, "tanh": _lib.FN_TANH, "silu": _lib.FN_SWISH, "swish": _lib.FN_SWISH,
              "gelu": _lib.FN_GELU}
_SOURCES = {"current": 0, "sollya": 1}


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, residual: torch.Tensor | None = None, *,
               activation: str = "none", degree: int = 0, coeff_source: str = "current") -> torch.Tensor:
    """x `[..., dim]`, weight `[out, dim]`, bias `[out]`, residual `[..., out]` -> `[..., out]`; float16 or bfloat16 (the bias
    float32 too), dim a multiple of 8, any out.

    activation: "none", "sigmoid", "tanh", "silu" ("swish") or "gelu" (the erf form).  degree 0 evaluates it in fp32;
    degree 3 .. 6 runs the packed polynomial program of `spline_ops` on the product rounded to the dtype, bit for bit what
    `spline_ops.<activation>_fwd_variant` gives on the stored product, and its gradient the derivative program of that
    degree.  x and weight whose rows are not contiguous or do not start on 16-byte boundaries are copied first."""
    function, source = _choice(_FUNCTIONS, activation, "activation"), _choice(_SOURCES, coeff_source, "coeff_source")
    if torch.compiler.is_compiling():
        return torch.ops.fpt_b200.linear_act(x, weight, bias, residual, function, int(degree), source)
    return _ext.linear_act(x, weight, bias, residual, function, int(degree), source)


def check_linear_status(device=None) -> None:
    """Wait for the work on `device` (default: the current one) and raise RuntimeError if a `linear_act` on it reported a
    device-side wait that ran out.  Without this call the same error surfaces, without blocking, at the next `linear_act` on
    that device, from whichever thread, and is cleared there."""
    torch.cuda.synchronize(device)
    index = None if device is None else torch.device(device).index
    _ext.poll_linear_status(torch.cuda.current_device() if index is None else index)


@torch.library.register_fake("fpt_b200::linear_act")
def _(x, weight, bias, residual, function, degree, source):
    return x.new_empty((*x.shape[:-1], weight.shape[0]))


@torch.library.register_fake("fpt_b200::linear_act_slope")
def _(x, weight, bias, residual, function, degree, source):
    rows = x.numel() // x.shape[-1]
    return (x.new_empty((*x.shape[:-1], weight.shape[0])),
            x.new_empty((rows if function != -1 else 0, (weight.shape[0] + 7) // 8 * 8), dtype=torch.float16))


@torch.library.register_fake("fpt_b200::linear_act_bwd")
def _(dy, slope, x, weight, x_shape, out, bias_dtype, want_x, want_weight, want_bias):
    return (dy.new_empty(x_shape if want_x else (0,)), dy.new_empty((out if want_weight else 0, x_shape[-1])),
            dy.new_empty((out if want_bias else 0,), dtype=(torch.float16, torch.bfloat16, torch.float32)[bias_dtype]))


__all__ = ["check_linear_status", "linear_act"]
