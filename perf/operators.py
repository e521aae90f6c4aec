"""Three operators around the attention of a transformer block: the cases they are measured at, their plain forms and
their definitions in 64 bits.

  qk_norm_rope   y = rotate(w * x / sqrt(mean(x^2) + eps)) for every head of the queries and of the keys
  rope_axes      y = rotate(x) with the position of each pair taken from one of several axes (time, height, width)
  linear_act     y = act(x W^T + b) + r

Rotation of pair i by the angle 2 pi ((position * increment_i) mod 2^32) / 2^32, the increments being 32-bit fixed-point
turns per position.  The pairs are (2i, 2i + 1) ("adjacent") or (i, i + n) with n pairs in all ("halves"); dimensions
behind the last pair pass through.
"""
import math
from types import SimpleNamespace

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ITEM = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


# ---- cases ------------------------------------------------------------------------------------------------------------

def _qk(name, batch, seq, q_heads, k_heads, dim, rotary, dtype, pairing, positions, train):
    return {"name": name, "op": "qk_norm_rope", "batch": batch, "seq": seq, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
            "rotary": rotary, "dtype": dtype, "pairing": pairing, "positions": positions, "train": train}


def _axes(name, batch, grid, q_heads, k_heads, dim, sections, order, dtype, pairing, train):
    return {"name": name, "op": "rope_axes", "batch": batch, "grid": grid, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
            "sections": sections, "order": order, "dtype": dtype, "pairing": pairing, "train": train}


def _linear(name, rows, dim, out, activation, bias, residual, dtype, train):
    return {"name": name, "op": "linear_act", "rows": rows, "dim": dim, "out": out, "activation": activation, "bias": bias,
            "residual": residual, "dtype": dtype, "train": train}


def listed():
    return [
        # one new token of 32 sequences far into their contexts: the pass between the projection and the cached attention
        _qk("qk_norm_rope decode 32 x 1", 32, 1, 32, 8, 128, 128, "bf16", "halves", "far", False),
        # a prompt of the attention's own benchmark shape
        _qk("qk_norm_rope prefill 2 x 4096", 2, 4096, 32, 8, 128, 128, "bf16", "adjacent", "none", False),
        # a training step at that shape, several documents packed into each row (positions start anew)
        _qk("qk_norm_rope train 2 x 4096", 2, 4096, 32, 8, 128, 128, "bf16", "halves", "packed", True),
        # a small model in half precision: ragged length, three quarters of each head rotated
        _qk("qk_norm_rope train fp16 3 x 1021", 3, 1021, 12, 4, 64, 48, "fp16", "adjacent", "packed", True),
        # a clip of 8 frames of 45 x 44 patches in front of a language model's attention
        _axes("rope_axes video 8 x 45 x 44", 1, "8,45,44", 32, 8, 128, "16,24,24", "blocked", "bf16", "halves", False),
        # an image encoder's training step: rows and columns of 61 x 67 patches, heads of 80
        _axes("rope_axes image train 61 x 67", 2, "61,67", 16, 16, 80, "20,20", "cyclic", "fp16", "halves", True),
        # answering about an image: one new token of 8 sequences
        _axes("rope_axes decode 8 x 1", 8, "1,1,1", 32, 8, 128, "16,24,24", "cyclic", "bf16", "halves", False),
        # one token through the first feed-forward projection: the weight is all there is to read
        _linear("linear_act decode 1 row", 1, 4096, 14336, "gelu", True, False, "bf16", False),
        # a serving batch through the projection back, added to the residual stream
        _linear("linear_act decode 48 rows", 48, 14336, 4096, "none", False, True, "bf16", False),
        # a ragged prompt in half precision at the routed experts' sizes
        _linear("linear_act ragged fp16 1999 rows", 1999, 1408, 2048, "silu", True, True, "fp16", False),
        # a prompt through the first feed-forward projection
        _linear("linear_act prefill 4096 rows", 4096, 4096, 14336, "gelu", True, False, "bf16", False),
        # a training step of that layer, with the residual in the epilogue
        _linear("linear_act train 4096 rows", 4096, 4096, 4096, "gelu", True, True, "bf16", True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("qk_norm_rope", "rope_axes", "linear_act", "linear_act"))
    if op == "linear_act":
        while True:
            rows, dim, out = _log(rng, 1, 4096), 8 * _log(rng, 32, 1792), _log(rng, 256, 14336)
            train = rng.random() < 0.35
            if rows * dim * out * (3 if train else 1) <= 3 * 4096 ** 3:
                break
        return _linear("", rows, dim, out, rng.choice(("none", "gelu", "silu", "sigmoid", "tanh")), rng.random() < 0.6,
                       rng.random() < 0.5, rng.choice(("bf16", "bf16", "fp16")), train)
    while True:
        tokens = _log(rng, 1, 16384)
        batch = min(tokens, _log(rng, 1, 64))
        seq = max(1, tokens // batch)
        k_heads = rng.choice((1, 2, 4, 8, 16))
        q_heads = k_heads * rng.choice((1, 2, 3, 4, 8))
        dim = rng.choice((64, 80, 96, 128, 256))
        if q_heads <= 64 and batch * seq * (q_heads + k_heads) * dim <= 8192 * 40 * 128:
            break
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    pairing, train = rng.choice(("adjacent", "halves")), rng.random() < 0.4
    if op == "qk_norm_rope":
        rotary = rng.choice((dim, dim, dim // 2 // 8 * 8))
        return _qk("", batch, seq, q_heads, k_heads, dim, rotary, dtype, pairing, rng.choice(("none", "far", "packed")), train)
    axes = rng.choice((2, 3))
    pairs, sections = dim // 2, []
    for left in range(axes, 1, -1):
        sections.append(rng.randint(pairs // (2 * left), pairs // left))
        pairs -= sections[-1]
    sections.append(pairs)
    height = max(1, int(round(math.sqrt(seq / (4 if axes == 3 else 1)))))
    width = max(1, seq // (height * (4 if axes == 3 else 1)))
    grid = (4, height, width) if axes == 3 and seq >= 4 else (1,) * (axes - 2) + (height, width)
    while math.prod(grid) * batch * (q_heads + k_heads) * dim > 8192 * 40 * 128:
        batch = max(1, batch // 2)
    return _axes("", batch, ",".join(map(str, grid)), q_heads, k_heads, dim, ",".join(map(str, sections)),
                 rng.choice(("blocked", "cyclic")), dtype, pairing, train)


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _numbers(text):
    return [int(n) for n in text.split(",")]


def _increments(pairs, theta, device):
    """round(theta^(-i / pairs) 2^32 / 2 pi): turns per position in 32-bit fixed point."""
    i = torch.arange(pairs, dtype=torch.float64, device=device)
    return torch.round(theta ** (-i / pairs) * (2.0 ** 32 / (2 * math.pi))).to(torch.int32)


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = SimpleNamespace(case=case)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device=device, generator=g) * scale).to(dtype)

    if case["op"] == "linear_act":
        rows, dim, out = case["rows"], case["dim"], case["out"]
        s.x, s.weight = normal(rows, dim), normal(out, dim, scale=dim ** -0.5)
        s.bias = normal(out, scale=0.2) if case["bias"] else None
        s.residual = normal(rows, out) if case["residual"] else None
        s.grad = normal(rows, out) if case["train"] else None
        return s

    grid = _numbers(case["grid"]) if case["op"] == "rope_axes" else None
    batch, seq = case["batch"], math.prod(grid) if grid else case["seq"]
    hq, hk, dim = case["q_heads"], case["k_heads"], case["dim"]
    # queries, keys and values as one projection writes them; q and k are views of its rows
    fused = normal(batch, seq, (hq + 2 * hk) * dim)
    s.q = fused[..., :hq * dim].view(batch, seq, hq, dim)
    s.k = fused[..., hq * dim:(hq + hk) * dim].view(batch, seq, hk, dim)
    s.grads = (normal(batch, seq, hq, dim), normal(batch, seq, hk, dim)) if case["train"] else None
    if case["op"] == "qk_norm_rope":
        s.q_weight = (1 + 0.1 * torch.randn(dim, device=device, generator=g)).to(dtype)
        s.k_weight = (1 + 0.1 * torch.randn(dim, device=device, generator=g)).to(dtype)
        s.increments = _increments(case["rotary"] // 2, 500000.0, device)
        s.sections = s.order = None
        if case["positions"] == "none":
            s.positions = None
        elif case["positions"] == "far":
            first = torch.randint(0, 131072 - seq, (batch, 1), device=device, generator=g)
            s.positions = first + torch.arange(seq, device=device)
        else:
            # documents of random length after one another in every row, each counted from zero
            start = torch.rand(batch, seq, device=device, generator=g) < 4.0 / seq
            index = torch.arange(seq, device=device).expand(batch, seq)
            s.positions = (index - torch.where(start, index, 0).cummax(dim=1).values).to(torch.int32)
        return s
    s.sections, s.order = _numbers(case["sections"]), case["order"]
    s.increments = _increments(sum(s.sections), 10000.0, device)
    # a grid of patches behind `first` tokens of text, which every axis counts alike
    first = torch.randint(0, 4096, (batch, 1), device=device, generator=g)
    mesh = torch.meshgrid(*(torch.arange(n, device=device) for n in grid), indexing="ij")
    s.positions = torch.stack([first + m.reshape(1, -1) for m in mesh]).to(torch.int32)
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------

def _pair_axis(sections, order):
    """The axis of every pair: the sections after one another, or dealt out in turn until an axis has its share."""
    if order == "blocked":
        return [axis for axis, n in enumerate(sections) for _ in range(n)]
    left, found = list(sections), []
    while sum(left):
        for axis, n in enumerate(left):
            if n:
                left[axis] -= 1
                found.append(axis)
    return found


def _phase(s):
    """[batch or 1, seq, 1, pairs]: the 32-bit phase of every pair, in 64 bits."""
    if s.sections is not None:
        axis = torch.tensor(_pair_axis(s.sections, s.order), device=s.q.device)
        position = s.positions[axis].permute(1, 2, 0)
    elif s.positions is None:
        position = torch.arange(s.q.shape[1], device=s.q.device)[None, :, None]
    else:
        position = s.positions[:, :, None]
    return (position.long() * s.increments.long() & 0xFFFFFFFF)[:, :, None, :]


def _rotate(x, cos, sin, pairing):
    n = cos.shape[-1]
    turned, rest = x[..., :2 * n], x[..., 2 * n:]
    if pairing == "adjacent":
        a, b = turned[..., 0::2], turned[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = turned[..., :n], turned[..., n:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((y, rest), dim=-1) if rest.shape[-1] else y


def _norm_rotate(x, weight, cos, sin, pairing):
    x = x.float()
    unit = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return _rotate(unit * weight.float(), cos, sin, pairing)


def _norm_rotate_back(grad, x, weight, cos, sin, pairing):
    x, g = x.float(), _rotate(grad.float(), cos, -sin, pairing)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    unit = x * r
    dunit = g * weight.float()
    dx = r * (dunit - unit * (dunit * unit).mean(-1, keepdim=True))
    return dx, (g * unit).sum((0, 1, 2))


def _run_heads_plain(s):
    angle = _phase(s).double() * (2 * math.pi / 2.0 ** 32)
    cos, sin = angle.cos().float(), angle.sin().float()
    pairing = s.case["pairing"]
    if s.case["op"] == "qk_norm_rope":
        out = [_norm_rotate(s.q, s.q_weight, cos, sin, pairing).to(s.q.dtype), _norm_rotate(s.k, s.k_weight, cos, sin, pairing).to(s.k.dtype)]
        if s.grads is None:
            return out
        dq, dqw = _norm_rotate_back(s.grads[0], s.q, s.q_weight, cos, sin, pairing)
        dk, dkw = _norm_rotate_back(s.grads[1], s.k, s.k_weight, cos, sin, pairing)
        return out + [dq.to(s.q.dtype), dk.to(s.k.dtype), dqw.to(s.q_weight.dtype), dkw.to(s.k_weight.dtype)]
    out = [_rotate(x.float(), cos, sin, pairing).to(x.dtype) for x in (s.q, s.k)]
    if s.grads is None:
        return out
    return out + [_rotate(g.float(), cos, -sin, pairing).to(g.dtype) for g in s.grads]


def _run_heads_own(s):
    from fast_polynomial_transcendentals_b200 import qk_rope
    if s.case["op"] == "qk_norm_rope":
        if s.grads is None:
            return list(qk_rope.qk_norm_rope(s.q, s.k, s.q_weight, s.k_weight, s.increments, positions=s.positions,
                                             pairing=s.case["pairing"], eps=EPS))
        leaves = [t.detach().requires_grad_() for t in (s.q, s.k, s.q_weight, s.k_weight)]
        out = qk_rope.qk_norm_rope(*leaves, s.increments, positions=s.positions, pairing=s.case["pairing"], eps=EPS)
    else:
        if s.grads is None:
            return list(qk_rope.rope_axes(s.q, s.k, s.increments, s.positions, s.sections, section_order=s.order,
                                          pairing=s.case["pairing"]))
        leaves = [t.detach().requires_grad_() for t in (s.q, s.k)]
        out = qk_rope.rope_axes(*leaves, s.increments, s.positions, s.sections, section_order=s.order, pairing=s.case["pairing"])
    return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, s.grads))


def _activate(z, name):
    """act(z) and act'(z)."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "tanh":
        y = torch.tanh(z)
        return y, 1 - y * y
    if name == "gelu":
        phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    p = 1 / (1 + torch.exp(-z))
    if name == "sigmoid":
        return p, p * (1 - p)
    return z * p, p * (1 + z * (1 - p))


def _run_linear_plain(s):
    x, w, dtype = s.x.float(), s.weight.float(), s.x.dtype
    z = x @ w.T
    if s.bias is not None:
        z = z + s.bias.float()
    y, slope = _activate(z, s.case["activation"])
    if s.residual is not None:
        y = y + s.residual.float()
    if s.grad is None:
        return [y.to(dtype)]
    dz = s.grad.float() * slope
    out = [y.to(dtype), (dz @ w).to(dtype), (dz.T @ x).to(dtype)]
    if s.bias is not None:
        out.append(dz.sum(0).to(dtype))
    if s.residual is not None:
        out.append(s.grad)
    return out


def _run_linear_own(s):
    from fast_polynomial_transcendentals_b200.linear import linear_act
    if s.grad is None:
        return [linear_act(s.x, s.weight, s.bias, s.residual, activation=s.case["activation"])]
    x, w, b, r = (None if t is None else t.detach().requires_grad_() for t in (s.x, s.weight, s.bias, s.residual))
    y = linear_act(x, w, b, r, activation=s.case["activation"])
    return [y.detach(), *torch.autograd.grad(y, [t for t in (x, w, b, r) if t is not None], s.grad)]


def run(state):
    if own:
        return _run_linear_own(state) if state.case["op"] == "linear_act" else _run_heads_own(state)
    return _run_linear_plain(state) if state.case["op"] == "linear_act" else _run_heads_plain(state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(case):
    item = ITEM[case["dtype"]]
    if case["op"] == "linear_act":
        rows, dim, out = case["rows"], case["dim"], case["out"]
        acts, weights = rows * dim, out * dim
        read = acts + weights + (out if case["bias"] else 0) + (rows * out if case["residual"] else 0)
        write = rows * out
        flops = 2 * rows * dim * out
        if case["train"]:       # the gradient of the output (r's own too) comes in; those of x, W and b go out; two more products
            read += rows * out
            write += acts + weights + (out if case["bias"] else 0)
            flops *= 3
        return {"bytes": item * (read + write), "flops": flops}
    tokens = case["batch"] * (math.prod(_numbers(case["grid"])) if case["op"] == "rope_axes" else case["seq"])
    values = tokens * (case["q_heads"] + case["k_heads"]) * case["dim"]
    norm = case["op"] == "qk_norm_rope"
    moved = values * item * (4 if case["train"] else 2)             # x in, y out; gradient of y in, of x out
    flops = values * (7 if norm else 3) * (1 if not case["train"] else 3 if norm else 2)
    if norm:
        position = {"none": 0, "far": 8, "packed": 4}[case["positions"]] * tokens
        moved += position + 4 * case["dim"] * item
        moved += case["rotary"] * 2
    else:
        moved += 4 * tokens * len(_numbers(case["sections"])) + 2 * case["dim"]
    return {"bytes": moved, "flops": flops}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------

def _turned(x, turns, pairing):
    """Each pair as a complex number, times exp(2 pi i turns)."""
    n = turns.shape[-1]
    if pairing == "adjacent":
        z = torch.view_as_complex(x[..., :2 * n].unflatten(-1, (n, 2)).contiguous())
    else:
        z = torch.complex(x[..., :n].contiguous(), x[..., n:2 * n].contiguous())
    z = z * torch.polar(torch.ones_like(turns), 2 * math.pi * turns)
    y = torch.view_as_real(z).flatten(-2) if pairing == "adjacent" else torch.cat((z.real, z.imag), dim=-1)
    return torch.cat((y, x[..., 2 * n:]), dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear_act":
        names = [n for n in ("x", "weight", "bias", "residual") if getattr(s, n) is not None]
        leaves = {n: getattr(s, n).double().requires_grad_(case["train"]) for n in names}
        z = torch.einsum("rd,od->ro", leaves["x"], leaves["weight"])
        if "bias" in leaves:
            z = z + leaves["bias"]
        y = {"none": lambda: z, "gelu": lambda: z * torch.special.ndtr(z), "silu": lambda: z * torch.sigmoid(z),
             "sigmoid": lambda: torch.sigmoid(z), "tanh": lambda: torch.tanh(z)}[case["activation"]]()
        if "residual" in leaves:
            y = y + leaves["residual"]
        if not case["train"]:
            return [y]
        return [y.detach(), *torch.autograd.grad(y, list(leaves.values()), s.grad.double())]

    if s.sections is not None:
        position = torch.stack([s.positions[a] for a in _pair_axis(s.sections, s.order)], dim=-1).long()
    elif s.positions is None:
        position = torch.arange(case["seq"], device=s.q.device).view(1, -1, 1)
    else:
        position = s.positions.unsqueeze(-1).long()
    turns = torch.remainder(position * s.increments.long(), 2 ** 32).double().div(2.0 ** 32).unsqueeze(2)
    norm = case["op"] == "qk_norm_rope"
    leaves = [t.double().requires_grad_(case["train"]) for t in (s.q, s.k)]
    weights = [t.double().requires_grad_(case["train"]) for t in (s.q_weight, s.k_weight)] if norm else []
    out = []
    for i, x in enumerate(leaves):
        if norm:
            x = weights[i] * x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
        out.append(_turned(x, turns, case["pairing"]))
    if not case["train"]:
        return out
    grads = torch.autograd.grad(out, leaves + weights, [g.double() for g in s.grads])
    return [t.detach() for t in out] + list(grads)
