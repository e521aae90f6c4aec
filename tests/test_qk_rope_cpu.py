"""CPU: the per-head norm with rotation and the rotation with several axes refuse what does not fit before anything is
launched, through the Python surface and through the C ABI, and the phase increments per axis are what they say."""
import ctypes
import math

import pytest
import torch

from fast_polynomial_transcendentals_b200 import qk_rope
from fast_polynomial_transcendentals_b200.sfu_repro.rope import rope_axis_phase_increments, rope_phase_increments

INC = rope_phase_increments(64)


def heads(batch=2, seq=3, heads=4, dim=64, dtype=torch.bfloat16):
    return torch.zeros(batch, seq, heads, dim, dtype=dtype)


@pytest.mark.parametrize("change, message", [
    (dict(q=heads().flatten(2)), "shape"),
    (dict(q=heads(dtype=torch.float64)), "float16, bfloat16 or float32"),
    (dict(k=heads(dtype=torch.float16)), "same dtype"),
    (dict(k=heads(batch=1)), "batch"),
    (dict(k=heads(seq=4)), "sequence"),
    (dict(k=heads(dim=72)), "head dimensions"),
    (dict(k=heads(heads=0)), "at least one head"),
    (dict(q=heads(dim=60), k=heads(dim=60)), "multiple of eight"),
    (dict(q=heads(dim=264), k=heads(dim=264)), "multiple of eight"),
    (dict(phase_increments=INC.long()), "int32"),
    (dict(phase_increments=INC[::2]), "contiguous"),
    (dict(phase_increments=INC[:30].contiguous()), "multiple of four"),
    (dict(phase_increments=rope_phase_increments(128)), "head_dim / 2"),
    (dict(phase_increments=INC[:0]), "multiple of four"),
    (dict(q_weight=torch.ones(32)), "head_dim entries"),
    (dict(q_weight=torch.ones(64), k_weight=torch.ones(64, dtype=torch.bfloat16)), "same dtype"),
    (dict(q_weight=torch.ones(64, dtype=torch.float64)), "head_dim entries"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=math.nan), "eps"),
    (dict(eps=math.inf), "eps"),
    (dict(positions=torch.zeros(3)), "int32 or int64"),
    (dict(positions=torch.zeros(4, dtype=torch.int32)), "sequence length"),
    (dict(positions=torch.zeros(3, 3, dtype=torch.int32)), "batch size"),
    (dict(positions=torch.zeros(1, 2, 3, dtype=torch.int32)), "shape"),
    (dict(sections=[16, 16]), "positions"),
    (dict(sections=[16, 15], positions=torch.zeros(2, 3, dtype=torch.int32)), "add up"),
    (dict(sections=[33, -1], positions=torch.zeros(2, 3, dtype=torch.int32)), "between 0"),
    (dict(sections=[16, 16], positions=torch.zeros(3, 3, dtype=torch.int32)), "one row per section"),
    (dict(sections=[8, 8, 8, 4, 4], positions=torch.zeros(5, 3, dtype=torch.int32)), "at most 4"),
    (dict(), "must be a CUDA tensor"),
])
def test_norm_rotation_refusals(change, message):
    args = dict(q=heads(), k=heads(), q_weight=None, k_weight=None, phase_increments=INC)
    args.update(change)
    with pytest.raises(RuntimeError, match=message):
        qk_rope.qk_norm_rope(args.pop("q"), args.pop("k"), args.pop("q_weight"), args.pop("k_weight"),
                             args.pop("phase_increments"), **args)


def test_names_are_checked():
    with pytest.raises(ValueError, match="pairing"):
        qk_rope.qk_norm_rope(heads(), heads(), None, None, INC, pairing="odd")
    with pytest.raises(ValueError, match="section_order"):
        qk_rope.rope_axes(heads(), heads(), INC, torch.zeros(1, 3, dtype=torch.int32), [32], section_order="random")
    with pytest.raises(RuntimeError, match="sections and positions"):
        qk_rope.rope_axes(heads(), heads(), INC, torch.zeros(1, 3, dtype=torch.int32), [])
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        qk_rope.rope_axes(heads(), heads(), INC, torch.zeros(1, 3, dtype=torch.int32), [32])


def test_c_abi_checks_before_launch(fpt):
    lib = fpt.load()
    p, three = 256, (ctypes.c_int64 * 3)(0, 0, 0)

    def call(q_out=p, k_out=p, q=p, k=p, qw=None, kw=None, inc=p, pos=None, bits=0, pos_strides=None, axes=None, batch=1, seq=1,
             hq=1, hk=1, dim=64, pairs=32, qs=three, ks=three, pairing=0, norm=1, eps=1e-6, inverse=0, dtype=1, wdtype=2):
        return lib.fpt_qk_rope(q_out, k_out, q, k, qw, kw, inc, pos, bits, pos_strides, axes, batch, seq, hq, hk, dim, pairs, qs, ks,
                               pairing, norm, eps, inverse, dtype, wdtype, None)

    assert call(batch=-1) == -2 and call(seq=-1) == -2 and call(hq=-1) == -2
    assert call(batch=1 << 20, seq=1 << 20) == -2 and call(hq=65536) == -2
    assert call(dim=60) == -6 and call(dim=0) == -6 and call(dim=264) == -6
    assert call(pairs=0) == -6 and call(pairs=6) == -6 and call(pairs=36) == -6
    assert call(pairing=2) == -5 and call(dtype=3) == -5 and call(wdtype=-1) == -5
    assert call(pos=p, bits=16, pos_strides=three) == -5
    assert call(norm=1, inverse=1) == -5
    assert call(axes=bytes([4] * 32)) == -5
    assert call(eps=-1.0) == -2 and call(eps=math.nan) == -2
    assert call(q=None) == -1 and call(k_out=None) == -1 and call(inc=None) == -1 and call(qs=None) == -1
    assert call(pos=p, bits=32) == -1
    assert call(q_out=p + 2) == -3 and call(q=p + 1) == -3 and call(inc=p + 2) == -3 and call(kw=p + 2) == -3
    assert call(pos=p + 4, bits=64, pos_strides=three) == -3
    assert call(batch=0, q=None) == 0                                   # nothing to do

    def back(dq=p, dqw=None, g=p, gs=three, workspace=None, nbytes=0, eps=1e-6, batch=1):
        return lib.fpt_qk_norm_rope_bwd(dq, p, dqw, None, g, p, p, p, None, None, p, None, 0, None, None, workspace, nbytes, batch, 1, 1, 1,
                                        64, 32, three, three, gs, three, 0, eps, 1, 2, None)

    assert back(dq=None) == -1 and back(g=None) == -1 and back(gs=None) == -1
    assert back(g=p + 1) == -3 and back(dqw=p, workspace=p + 2) == -3
    assert back(eps=-1.0) == -2 and back(batch=-1) == -2


def test_increments_start_anew_in_every_section():
    inc = rope_axis_phase_increments([4, 8, 0, 2], theta=100.0)
    assert inc.dtype == torch.int32 and inc.numel() == 14
    assert torch.equal(inc[4:12], rope_phase_increments(16, theta=100.0))
    assert inc[0] == inc[4] == inc[12] == round(2 ** 32 / (2 * math.pi))


def test_eps_beyond_fp32_is_refused():
    with pytest.raises(RuntimeError, match="finite"):
        qk_rope.qk_norm_rope(heads(), heads(), None, None, INC, eps=1e39)
