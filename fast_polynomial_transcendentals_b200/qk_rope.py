"""Queries and keys on their way into the attention: the norm of every head and the position rotation in one pass.

`qk_norm_rope` is the step that models with normalised queries and keys take between the projection and the attention, and
`rope_axes` the rotation of models whose tokens have a position on several axes (time, height and width of a video).  Both
take `[batch, sequence, heads, head_dim]` as the attention does (`sfu_repro.fa4`), by strides, so the views of one fused
projection need no copy, and return contiguous tensors of the same shape.  Both are differentiable, run without a
gradient at the cost of one launch, and are usable under `torch.compile` (`torch.ops.fpt_b200.qk_rope`).

They stand beside the reference's fused RoPE (`spline_ops.rope_apply_*`, positions 0 .. S - 1, fp16 arithmetic, no
gradient) and take the same parameter, `sfu_repro.rope.rope_phase_increments`: 32-bit fixed-point turns per position.  The
phase `position * increment` wraps as the angle does, so it is exact at every 32- or 64-bit position.  All arithmetic here
is fp32 with one rounding at the end, whatever the dtype (float16, bfloat16 or float32).

Forward and backward pass can be captured into CUDA graphs; drop every eager graph of the same leaves before a backward pass is
captured, as for PyTorch's own operators (a leaf's gradient accumulation stays on the stream of the graph that made it).

A second derivative through the norm is refused (RuntimeError; the rotation alone is linear and has every derivative), and so are
forward-mode differentiation and a call whose shapes, dtypes or devices do not fit.  `torch.func.grad`, `vjp` and `jacrev` and both
forms of activation checkpointing can be used.
"""
from __future__ import annotations

from typing import Sequence

import torch

from . import _lib

_lib.load()
try:
    from . import _fpt_torch as _ext
except ImportError as error:
    raise ImportError("the compiled PyTorch binding is missing: build it with "
                      "`python -m fast_polynomial_transcendentals_b200.build`") from error

_PAIRINGS = {"adjacent": 0, "halves": 1}
_ORDERS = {"blocked": 0, "cyclic": 1}


def _choice(table: dict[str, int], value: str, name: str) -> int:
    try:
        return table[value]
    except (KeyError, TypeError):
        raise ValueError(f"unknown {name} {value!r}, expected one of: {', '.join(table)}") from None


def _call(q, k, q_weight, k_weight, phase_increments, positions, sections, order: int, pairing: int, norm: bool, eps: float):
    if torch.compiler.is_compiling():
        return torch.ops.fpt_b200.qk_rope(q, k, q_weight, k_weight, phase_increments, positions, sections, order, pairing, norm, eps, False)
    return _ext.qk_rope(q, k, q_weight, k_weight, phase_increments, positions, sections, order, pairing, norm, eps)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                 phase_increments: torch.Tensor, *, positions: torch.Tensor | None = None,
                 sections: Sequence[int] | None = None, section_order: str = "blocked", pairing: str = "adjacent",
                 eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """`rotate(weight * x / sqrt(mean(x^2) + eps))` for every head of q `[B, S, Hq, D]` and k `[B, S, Hk, D]`.

    q_weight, k_weight: `[D]` (float16, bfloat16 or float32, the same for both) or None for ones.  phase_increments: int32,
    one entry per rotated pair (a multiple of four, at most D / 2; dimensions behind the pairs are normalised and pass
    through).  pairing: "adjacent" rotates (2i, 2i + 1), "halves" (i, i + pairs).  positions: int32 or int64, `[S]` or
    `[B, S]` (or `[1, S]`), any sign; None counts 0 .. S - 1.  sections, section_order: positions on several axes, as in
    `rope_axes`.  D is a multiple of eight, at most 256.  Gradients: q, k and the weights."""
    return _call(q, k, q_weight, k_weight, phase_increments, positions, [] if sections is None else list(sections),
                 _choice(_ORDERS, section_order, "section_order"), _choice(_PAIRINGS, pairing, "pairing"), True, float(eps))


def rope_axes(q: torch.Tensor, k: torch.Tensor, phase_increments: torch.Tensor, positions: torch.Tensor,
              sections: Sequence[int], *, section_order: str = "blocked",
              pairing: str = "adjacent") -> tuple[torch.Tensor, torch.Tensor]:
    """The rotation alone, each pair by the position on its own axis.

    positions: int32 or int64, `[axes, S]` or `[axes, B, S]` (or `[axes, 1, S]`), one to four axes.  sections: how many
    pairs each axis has; they add up to the entries of phase_increments, which hold one increment per pair whatever its
    axis (`sfu_repro.rope.rope_axis_phase_increments` starts the frequencies anew in every section).  section_order:
    "blocked" gives the first `sections[0]` pairs to axis 0 and so on.  "cyclic" deals the pairs out in turn until an axis has
    its share, and goes on among the others: [2, 3, 3] is 0 1 2 0 1 2 1 2.  A model that interleaves its axes and leaves every
    pair that is over to axis 0 means the same only where the other sections are equal and the first is not smaller.  pairing as in `qk_norm_rope`.  Gradients: q and k."""
    if sections is None or len(sections) == 0 or positions is None:
        raise RuntimeError("rope_axes needs sections and positions")
    return _call(q, k, None, None, phase_increments, positions, list(sections), _choice(_ORDERS, section_order, "section_order"),
                 _choice(_PAIRINGS, pairing, "pairing"), False, 0.0)


@torch.library.register_fake("fpt_b200::qk_rope")
def _(q, k, *_args):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.register_fake("fpt_b200::qk_norm_rope_bwd")
def _(dq_out, dk_out, q, k, q_weight, k_weight, phase_increments, positions, sections, order, pairing, eps, want_q, want_k):
    like = q_weight if q_weight is not None else k_weight if k_weight is not None else q
    return (q.new_empty(q.shape), k.new_empty(k.shape), like.new_empty(q.shape[-1] if want_q else 0),
            like.new_empty(q.shape[-1] if want_k else 0))


__all__ = ["qk_norm_rope", "rope_axes"]
