"""GPU: the per-head norm with rotation, the rotation with several axes and their gradients against a plain
implementation in 64 bits.

Tolerances (u = 2^-24, the half step of fp32; all kernels work in fp32 and round once, by at most eps / 2 of the value,
plus half the smallest step in fp16):
  rotation     each output is two products and a sum (3 u of |a| + |b|) with a sine and a cosine that are off by the
               rounding of the phase to fp32 (pi 2^-25 < 2 u) and by sincospif itself (2 ulp = 4 u): < 9 u (|a| + |b|)
  norm         r carries the error of a sum of squares (at most 8 + 5 roundings), of 1 / D and of rsqrtf (2 ulp = 4 u) halved:
               < 13 u; two products follow: < 15 u.  Together < 24 u (|a| + |b|) <= 48 u max|v|; tested with 64 u max|v|.
  gradient     dx = r (h - u m): h carries the rotation and a product (< 12 u max|h| sqrt 2), m a dot product over the head
               (< 13 + 18 roundings of mean|h u| <= max|h|) and r: < 64 u r max|h| (1 + max|u|); tested with 96.
  weights      every term g u carries < 40 u of its size, a thread adds at most as many terms as it meets heads (n below),
               and 16 + 5 + 5 more additions join them: (66 + n) u sum|g u|; tested with (96 + n).
"""
import math

import pytest
import torch

from fast_polynomial_transcendentals_b200 import qk_rope
from fast_polynomial_transcendentals_b200.sfu_repro.rope import rope_axis_phase_increments, rope_phase_increments

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def half_step(dtype):
    """(relative, absolute) size of half a rounding step."""
    return torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0


def axis_of_pair(sections, order):
    if order == "blocked":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


def turns(increments, positions, batch, seq, sections=None, order="blocked"):
    """[batch, seq, 1, pairs] in turns, 64 bits: the phases are whole numbers of 2^-32 turns."""
    inc = increments.long().cpu()
    if positions is None:
        p = torch.arange(seq).view(1, seq, 1)
    elif sections is not None:
        pos = positions.long().cpu()
        pos = pos[:, None] if pos.dim() == 2 else pos
        p = torch.stack([pos[a] for a in axis_of_pair(sections, order)], dim=-1)
    else:
        pos = positions.long().cpu()
        p = (pos[None] if pos.dim() == 1 else pos)[..., None]
    # modulo 2^32 before the product: positions far out would pass 64 bits
    phase = torch.remainder(torch.remainder(p, 2 ** 32) * torch.remainder(inc, 2 ** 31) + torch.where(inc < 0, torch.remainder(p, 2) * 2 ** 31, 0), 2 ** 32)
    return (phase.double() / 2.0 ** 32).expand(batch, seq, -1)[:, :, None]


def rotate(x, turn, pairing, sign=1):
    c, s = torch.cos(2 * math.pi * turn), sign * torch.sin(2 * math.pi * turn)
    n = turn.shape[-1]
    y = x.clone()
    if pairing == "adjacent":
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        y[..., :n], y[..., n:2 * n] = a * c - b * s, b * c + a * s
    return y


def plain_norm(x, w, turn, pairing, eps):
    x = x.detach().double().cpu()
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    v = x * r * (1.0 if w is None else w.detach().double().cpu())
    return rotate(v, turn, pairing), v


def plain_norm_back(g, x, w, turn, pairing, eps):
    x, g = x.detach().double().cpu(), rotate(g.detach().double().cpu(), turn, pairing, -1)
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    u = x * r
    h = g if w is None else g * w.detach().double().cpu()
    dx = r * (h - u * (h * u).mean(-1, keepdim=True))
    scale = r * h.abs().amax(-1, keepdim=True) * (1 + u.abs().amax(-1, keepdim=True))
    return dx, scale, (g * u).sum((0, 1, 2)), (g * u).abs().sum((0, 1, 2))


def close(got, want, slack, what):
    rel, least = half_step(got.dtype)
    got = got.detach().double().cpu()
    assert got.shape == want.shape, what
    bound = rel * (want.abs() + slack) + least + slack
    worst = ((got - want).abs() - bound).max().item() if got.numel() else -1
    assert worst <= 0, f"{what}: {worst} above the tolerance"
    assert torch.isfinite(got).all(), what


def make(batch, seq, hq, hk, dim, dtype, device, seed=0, layout="plain"):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device=device, generator=g).to(dtype)
    if layout == "fused":                          # views of the rows of one projection
        rows = rand(batch, seq, (hq + 2 * hk) * dim)
        return rows[..., :hq * dim].unflatten(-1, (hq, dim)), rows[..., hq * dim:(hq + hk) * dim].unflatten(-1, (hk, dim))
    if layout == "heads first":
        return rand(batch, hq, seq, dim).transpose(1, 2), rand(batch, hk, seq, dim).transpose(1, 2)
    if layout == "odd start":                      # no row starts on a 16-byte boundary
        return tuple(rand(batch * seq * (h * dim + 3) + 1)[1:].view(batch, seq, h * dim + 3)[..., :h * dim].unflatten(-1, (h, dim))
                     for h in (hq, hk))
    if layout == "broadcast":
        return rand(1, seq, hq, dim).expand(batch, -1, -1, -1), rand(batch, 1, hk, dim).expand(-1, seq, -1, -1)
    if layout == "strided":                        # the head dimension itself is not contiguous
        return rand(batch, seq, hq, 2 * dim)[..., ::2], rand(batch, seq, hk, 2 * dim)[..., ::2]
    return rand(batch, seq, hq, dim), rand(batch, seq, hk, dim)


def check_norm(q, k, qw, kw, inc, pairing, positions=None, sections=None, order="blocked", eps=1e-6, grad=True, seed=1):
    batch, seq = q.shape[:2]
    turn = turns(inc, positions, batch, seq, sections, order)
    leaves = [t if t is None else t.detach().requires_grad_(grad) for t in (q, k, qw, kw)]
    out = qk_rope.qk_norm_rope(*leaves, inc, positions=positions, sections=sections, section_order=order, pairing=pairing, eps=eps)
    for name, y, x, w in zip("qk", out, (q, k), (qw, kw)):
        want, v = plain_norm(x, w, turn, pairing, eps)
        assert y.is_contiguous() and y.dtype == x.dtype
        close(y, want, 64 * U * v.abs().amax(-1, keepdim=True), f"{name} output")
    if not grad:
        return out
    g = torch.Generator(device=q.device)
    g.manual_seed(seed)
    grads = [torch.randn(t.shape, device=q.device, generator=g).to(t.dtype) for t in out]
    inputs = [t for t in leaves if t is not None]
    back = dict(zip([n for n, t in zip(("q", "k", "qw", "kw"), leaves) if t is not None], torch.autograd.grad(out, inputs, grads)))
    for name, x, w, go in (("q", q, qw, grads[0]), ("k", k, kw, grads[1])):
        dx, scale, dw, total = plain_norm_back(go, x, w, turn, pairing, eps)
        close(back[name], dx, 96 * U * scale, f"d{name}")
        if w is not None:
            n = 32 + batch * seq * x.shape[2] // 64      # at least 64 groups share the rows, tiles of up to 32 rows a group
            assert back[name + "w"].dtype == w.dtype
            close(back[name + "w"], dw, (96 + n) * U * total, f"d{name}_weight")
    return out


SHAPES = [  # batch, seq, q heads, k heads, head_dim, pairs
    (1, 1, 1, 1, 8, 4), (2, 7, 3, 1, 64, 32), (1, 33, 5, 2, 80, 40), (3, 17, 4, 4, 96, 24), (2, 130, 8, 2, 128, 64),
    (1, 9, 2, 2, 256, 128), (5, 1, 4, 1, 136, 4), (1, 1201, 16, 1, 64, 32), (1, 100, 130, 2, 128, 64), (33, 1, 32, 8, 128, 64)]


@pytest.mark.parametrize("pairing", ["adjacent", "halves"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_norm_rotation_and_gradients(cuda, shape, dtype, pairing):
    batch, seq, hq, hk, dim, pairs = shape
    q, k = make(batch, seq, hq, hk, dim, DTYPES[dtype], cuda, seed=sum(shape))
    wdtype = torch.float32 if seq % 2 else DTYPES[dtype]
    qw, kw = ((1 + 0.2 * torch.randn(dim, device=cuda)).to(wdtype) for _ in range(2))
    check_norm(q, k, qw, kw, rope_phase_increments(2 * pairs, 10000.0, cuda), pairing)


@pytest.mark.parametrize("layout", ["fused", "heads first", "odd start", "broadcast", "strided"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_layouts(cuda, layout, dtype):
    q, k = make(2, 19, 6, 2, 72, DTYPES[dtype], cuda, layout=layout)
    qw, kw = torch.rand(72, device=cuda) + 0.5, torch.rand(72, device=cuda) + 0.5
    check_norm(q, k, qw, kw, rope_phase_increments(64, device=cuda), "halves" if layout == "fused" else "adjacent")


@pytest.mark.parametrize("qw, kw", [(True, False), (False, True), (False, False)])
def test_one_weight_or_none(cuda, qw, kw):
    q, k = make(2, 5, 3, 2, 64, torch.bfloat16, cuda)
    check_norm(q, k, torch.rand(64, device=cuda) if qw else None, torch.rand(64, device=cuda) if kw else None,
               rope_phase_increments(64, device=cuda), "halves")


POSITIONS = {
    "row": lambda b, s, d: torch.arange(s, device=d, dtype=torch.int32) * 7,
    "batch": lambda b, s, d: torch.randint(0, 1 << 17, (b, s), device=d),
    "shared": lambda b, s, d: torch.randint(0, 1 << 17, (1, s), device=d),
    "far": lambda b, s, d: torch.randint(1 << 31, 1 << 45, (b, s), device=d),
    "negative": lambda b, s, d: -torch.arange(s, device=d, dtype=torch.int32).expand(b, s),
    "strided": lambda b, s, d: torch.randint(0, 1 << 20, (s, 2 * b), device=d).t()[::2],
}


@pytest.mark.parametrize("kind", list(POSITIONS))
@pytest.mark.parametrize("pairing", ["adjacent", "halves"])
def test_positions(cuda, kind, pairing):
    q, k = make(3, 21, 4, 2, 128, torch.float32, cuda)
    check_norm(q, k, None, None, rope_phase_increments(128, 500000.0, cuda), pairing, positions=POSITIONS[kind](3, 21, cuda))


def test_increments_of_either_sign(cuda):
    """A negative increment turns the other way; the phase is the product modulo 2^32."""
    q, k = make(1, 40, 2, 1, 64, torch.float32, cuda)
    inc = torch.randint(-(1 << 31), (1 << 31) - 1, (32,), device=cuda, dtype=torch.int32)
    check_norm(q, k, None, None, inc, "halves", positions=torch.randint(-1000, 1000, (40,), device=cuda))


@pytest.mark.parametrize("order", ["blocked", "cyclic"])
@pytest.mark.parametrize("sections, dim", [([16, 24, 24], 128), ([20, 20], 80), ([32], 64), ([5, 0, 3, 4], 32), ([1, 30, 1], 96)])
@pytest.mark.parametrize("dtype, pairing", [("bf16", "halves"), ("fp16", "adjacent"), ("fp32", "halves")])
def test_axes_and_gradients(cuda, sections, dim, order, dtype, pairing):
    batch, seq = 2, 23
    q, k = make(batch, seq, 4, 2, dim, DTYPES[dtype], cuda, layout="fused")
    inc = rope_axis_phase_increments(sections, device=cuda) if order == "blocked" else rope_phase_increments(2 * sum(sections), device=cuda)
    for positions in (torch.randint(0, 5000, (len(sections), batch, seq), device=cuda), torch.randint(0, 99, (len(sections), seq), device=cuda, dtype=torch.int32),
                      torch.randint(0, 99, (len(sections), 1, seq), device=cuda)):
        turn = turns(inc, positions, batch, seq, sections, order)
        leaves = [t.detach().requires_grad_() for t in (q, k)]
        out = qk_rope.rope_axes(*leaves, inc, positions, sections, section_order=order, pairing=pairing)
        grads = [torch.randn_like(t) for t in out]
        back = torch.autograd.grad(out, leaves, grads)
        for name, y, x, sign in (("q", out[0], q, 1), ("k", out[1], k, 1), ("dq", back[0], grads[0], -1), ("dk", back[1], grads[1], -1)):
            x = x.double().cpu()
            close(y, rotate(x, turn, pairing, sign), 24 * U * x.abs().amax(-1, keepdim=True), name)


def test_norm_with_axes(cuda):
    q, k = make(2, 11, 4, 2, 96, torch.bfloat16, cuda)
    w = torch.rand(96, device=cuda)
    for order in ("blocked", "cyclic"):
        check_norm(q, k, w, w, rope_phase_increments(80, device=cuda), "halves", positions=torch.randint(0, 300, (3, 2, 11), device=cuda),
                   sections=[10, 20, 10], order=order)


def test_one_axis_equals_the_plain_positions(cuda):
    q, k = make(2, 15, 4, 2, 64, torch.bfloat16, cuda)
    inc, pos = rope_phase_increments(64, device=cuda), torch.randint(0, 9999, (2, 15), device=cuda)
    a = qk_rope.rope_axes(q, k, inc, pos[None].expand(2, -1, -1), [12, 20])
    b = qk_rope.rope_axes(q, k, inc, pos[None], [32], section_order="cyclic")
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_rotation_agrees_with_the_fused_rope(cuda):
    """The framework's fp16 RoPE (adjacent pairs, positions 0 .. S - 1, [B, H, S, D] out) is the same rotation: its sines
    and cosines are fp16 polynomials (2^-9 is far above their error) and its products fp16 roundings."""
    from fast_polynomial_transcendentals_b200 import spline_ops
    q, k = make(2, 50, 4, 2, 128, torch.float16, cuda)
    inc = rope_phase_increments(128, device=cuda)
    ours = qk_rope.rope_axes(q, k, inc, torch.arange(50, device=cuda)[None], [64])
    theirs = spline_ops.rope_apply_fixed_half_turn_d5_d6_fp16(q, k, inc)
    for a, b in zip(ours, theirs):
        assert (a.float() - b.transpose(1, 2).float()).abs().max() <= 2.0 ** -9 * 2 * float(q.abs().max())


def test_zero_rows_and_rows_that_are_not_numbers(cuda):
    """A head of zeros gives zeros (eps keeps 1 / 0 away) and finite gradients; NaN and infinities stay in their head."""
    q, k = make(1, 6, 4, 2, 64, torch.bfloat16, cuda)
    q, k = q.clone(), k.clone()
    q[0, 1, 2] = 0
    check_norm(q, k, None, None, rope_phase_increments(64, device=cuda), "halves")
    inc = rope_phase_increments(64, device=cuda)
    clean = qk_rope.qk_norm_rope(q, k, None, None, inc)
    q[0, 3, 1, 5] = math.nan
    k[0, 2, 0, 9] = math.inf
    got = qk_rope.qk_norm_rope(q, k, None, None, inc)
    assert got[0][0, 3, 1].isnan().all() and got[1][0, 2, 0].isnan().any()
    for a, b, (s, h) in zip(got, clean, ((3, 1), (2, 0))):
        keep = torch.ones(a.shape[:3], dtype=torch.bool, device=cuda)
        keep[0, s, h] = False
        assert torch.equal(a[keep], b[keep])


@pytest.mark.parametrize("dim, pairs", [(64, 16), (40, 4), (128, 32)])
@pytest.mark.parametrize("pairing", ["adjacent", "halves"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_dimensions_behind_the_pairs_are_not_mixed(cuda, dtype, pairing, dim, pairs):
    """The rotation alone passes them through, infinities and -0 bit for bit and NaN as NaN (the conversion to 16 bits gives it
    one payload), and so does its gradient; under the norm one that is not finite makes NaN of itself only."""
    bits = torch.int32 if dtype == "fp32" else torch.int16
    inc, pos = rope_phase_increments(2 * pairs, device=cuda), torch.arange(6, device=cuda)[None]

    def spoiled(seed):
        out = make(1, 6, 4, 2, dim, DTYPES[dtype], cuda, seed=seed)
        for t in out:
            t[0, 1, 1, 2 * pairs + 1] = math.inf
            t[0, 2, 0, 2 * pairs + 4] = math.nan
            t[0, 3, 1, dim - 1] = -math.inf
            t[0, 4, :, 2 * pairs:] = -0.0
        return out
    x, dy = [t.requires_grad_() for t in spoiled(3)], spoiled(4)
    y = qk_rope.rope_axes(*x, inc, pos, [pairs], pairing=pairing)
    for got, want in (*zip(y, x), *zip(torch.autograd.grad(y, x, dy), dy)):
        a, b = (t.detach()[..., 2 * pairs:].contiguous() for t in (got, want))
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.view(bits)[~a.isnan()], b.view(bits)[~a.isnan()])
        assert torch.isfinite(got[..., :2 * pairs]).all()
    turn = turns(inc, None, 1, 6)
    with torch.no_grad():
        for got, t in zip(qk_rope.qk_norm_rope(*x, None, None, inc, pairing=pairing), x):
            want, _ = plain_norm(t, None, turn, pairing, 1e-6)
            assert torch.equal(got.isnan().cpu(), want.isnan())


@pytest.mark.parametrize("batch, seq", [(0, 5), (3, 0)])
def test_nothing_to_do(cuda, batch, seq):
    q, k = (torch.empty(batch, seq, h, 64, device=cuda, dtype=torch.bfloat16, requires_grad=True) for h in (4, 2))
    w = torch.ones(64, device=cuda, requires_grad=True)
    out = qk_rope.qk_norm_rope(q, k, w, w, rope_phase_increments(64, device=cuda))
    assert [tuple(t.shape) for t in out] == [(batch, seq, 4, 64), (batch, seq, 2, 64)]
    grads = torch.autograd.grad(out, [q, k, w], [torch.ones_like(t) for t in out])
    assert grads[0].shape == q.shape and torch.equal(grads[2], torch.zeros_like(w))


def test_gradient_against_differences(cuda):
    """<grad, direction> against a central difference of the 64-bit definition (step 2^-13: its own error is below 1e-7 of
    the sum of the terms; the kernel's gradients are fp32, off by less than 96 u of their scale)."""
    q, k = make(1, 9, 3, 2, 64, torch.float32, cuda)
    qw, kw = torch.rand(64, device=cuda) + 0.5, torch.rand(64, device=cuda) + 0.5
    inc = rope_phase_increments(48, device=cuda)
    turn, grads = turns(inc, None, 1, 9), [torch.randn_like(q), torch.randn_like(k)]
    leaves = [t.detach().requires_grad_() for t in (q, k, qw, kw)]
    back = torch.autograd.grad(qk_rope.qk_norm_rope(*leaves, inc, pairing="halves"), leaves, grads)

    def value(a, b, c, d):
        return sum((plain_norm(x, w, turn, "halves", 1e-6)[0] * g.double().cpu()).sum() for x, w, g in ((a, c, grads[0]), (b, d, grads[1])))

    for i, (leaf, d) in enumerate(zip(leaves, back)):
        direction = torch.randn(leaf.shape, dtype=torch.float64)
        args = [t.detach().double().cpu() for t in leaves]
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + 2.0 ** -13 * direction, args[i] - 2.0 ** -13 * direction
        want = (value(*up) - value(*down)) / 2.0 ** -12
        terms = d.double().cpu() * direction
        assert abs(terms.sum() - want) <= 2e-5 * terms.abs().sum(), i


def test_unused_output_and_shared_weight(cuda):
    """Only the queries' result is used: the keys' gradient is zero; one weight for both sides adds up."""
    q, k = (t.detach().requires_grad_() for t in make(2, 9, 3, 2, 64, torch.float32, cuda))
    w = (torch.rand(64, device=cuda) + 0.5).requires_grad_()
    inc = rope_phase_increments(64, device=cuda)
    out = qk_rope.qk_norm_rope(q, k, w, w, inc)
    dq, dk, dw = torch.autograd.grad(out[0].sum(), [q, k, w])
    assert torch.equal(dk, torch.zeros_like(k))
    a, b = w.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    g = [torch.randn_like(t) for t in out]
    both = torch.autograd.grad(qk_rope.qk_norm_rope(q, k, a, b, inc), [a, b], g)
    one = torch.autograd.grad(qk_rope.qk_norm_rope(q, k, w, w, inc), [w], g)[0]
    assert torch.equal(one, both[0] + both[1])


def test_no_second_gradient(cuda):
    q, k = (t.detach().requires_grad_() for t in make(1, 4, 2, 1, 64, torch.float32, cuda))
    out = qk_rope.qk_norm_rope(q, k, None, None, rope_phase_increments(64, device=cuda))
    with pytest.raises(RuntimeError, match="no second gradient"):
        torch.autograd.grad(out[0].sum(), [q], create_graph=True)


def test_results_do_not_change_from_run_to_run(cuda):
    q, k = make(2, 777, 8, 2, 128, torch.bfloat16, cuda)
    w = torch.rand(128, device=cuda).requires_grad_()
    inc = rope_phase_increments(128, device=cuda)
    runs = []
    for _ in range(3):
        out = qk_rope.qk_norm_rope(q, k, w, w, inc, pairing="halves")
        runs.append(torch.autograd.grad(out, [w], [torch.ones_like(t) for t in out])[0])
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_another_stream_and_captured_graphs(cuda):
    """Forward and backward captured twice on a stream of their own, replayed out of order with new inputs: each gives what
    an eager call gives (the workspace belongs to the call)."""
    inc = rope_phase_increments(128, device=cuda)
    stream, made = torch.cuda.Stream(cuda), []
    for seed, seq in ((1, 40), (2, 300)):
        q, k = (t.detach().requires_grad_() for t in make(2, seq, 8, 2, 128, torch.bfloat16, cuda, seed=seed))
        w = (torch.rand(128, device=cuda) + 0.5).requires_grad_()
        grads = [torch.randn_like(t) for t in (q, k)]

        def step(q=q, k=k, w=w, grads=grads):
            out = qk_rope.qk_norm_rope(q, k, w, w, inc, pairing="halves")
            return [*out, *torch.autograd.grad(out, [q, k, w], grads)]

        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
        made.append((graph, step, out, q, grads))
    for index in (1, 0, 1):
        graph, step, out, q, grads = made[index]
        with torch.no_grad():
            q.copy_(torch.randn_like(q))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))
    made[0][0].replay()
    made[1][0].replay()
    torch.cuda.synchronize()
    for _, step, out, *_ in made:
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_under_torch_compile(cuda):
    q, k = (t.detach().requires_grad_() for t in make(2, 12, 4, 2, 64, torch.bfloat16, cuda))
    w = (torch.rand(64, device=cuda) + 0.5).requires_grad_()
    inc = rope_phase_increments(64, device=cuda)

    def f(q, k, w):
        a, b = qk_rope.qk_norm_rope(q, k, w, w, inc, pairing="halves")
        return (a.float() * 2).sum() + b.float().sum()

    want = torch.autograd.grad(f(q, k, w), [q, k, w])
    got = torch.autograd.grad(torch.compile(f, backend="aot_eager", fullgraph=True)(q, k, w), [q, k, w])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
