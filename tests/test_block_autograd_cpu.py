"""CPU: what the operators around the attention answer to PyTorch's automatic differentiation, on meta tensors (shapes and
graphs without values)."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from fast_polynomial_transcendentals_b200 import linear, qk_rope  # noqa: F401  (registers torch.ops.fpt_b200)

GELU = 4


def meta(*shape, grad=False):
    return torch.empty(*shape, dtype=torch.bfloat16, device="meta", requires_grad=grad)


def layer(x, weight, bias=None, residual=None):
    return torch.ops.fpt_b200.linear_act(x, weight, bias, residual, GELU, 0, 0)


def heads(q, k, q_weight=None, k_weight=None, norm=True):
    inc = torch.empty(32, dtype=torch.int32, device="meta")
    return torch.ops.fpt_b200.qk_rope(q, k, q_weight, k_weight, inc, None, [], 0, 0, norm, 1e-6, False)


LAYER = (4, 16), (8, 16), (8,), (4, 8)
HEADS = (2, 3, 4, 64), (2, 3, 2, 64), (64,), (64,)


@pytest.mark.parametrize("call, shapes", [(layer, LAYER), (heads, HEADS)])
@pytest.mark.parametrize("which", range(4))
def test_forward_mode_is_refused(call, shapes, which):
    """No tangent is dropped without a word, whichever input carries it."""
    args = [meta(*s) for s in shapes]
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.empty_like(args[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(*args)


def test_jvp_of_the_rotation_alone_is_refused():
    q, k = meta(2, 3, 4, 64), meta(2, 3, 2, 64)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda q: heads(q, k, norm=False)[0], (q,), (torch.empty_like(q),))


def checkpointed_layer(x, w, b, r):
    return layer(x, w, b, r)


def checkpointed_norm_of_the_layer(x, w, b, r):
    return heads(layer(x, w, b, r).view(1, 4, 2, 64), layer(x, w).view(1, 4, 2, 64))[0].reshape(4, 128)


def checkpointed_rotation(x, w, b, r):
    return heads(layer(x, w, b, r).view(1, 4, 2, 64), x.view(1, 4, 2, 64), norm=False)[0].reshape(4, 128)


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("region", [checkpointed_layer, checkpointed_norm_of_the_layer, checkpointed_rotation])
def test_checkpointed_regions(region, reentrant):
    """A region that ends in one of the operators: its node is the first to need its saved tensors, and the region runs again
    inside the node's unpacking."""
    from torch.utils.checkpoint import checkpoint
    args = [meta(4, 128, grad=True), meta(128, 128, grad=True), meta(128, grad=True), meta(4, 128, grad=True)]
    for call in (lambda *a: checkpoint(region, *a, use_reentrant=reentrant),
                 lambda *a: a[0] + checkpoint(region, *(2 * t for t in a), use_reentrant=reentrant)):
        for t in args:
            t.grad = None
        call(*args).sum().backward()
        assert all(t.grad is not None and t.grad.shape == t.shape for t in args)


@pytest.fixture
def cpu_kernels():
    """Plain forms of the kernels behind the dispatcher's CPU key (GELU and the norm with adjacent pairs and no angle), for what
    autograd and the compiler do above them."""
    def z_of(x, weight, bias):
        z = x.double() @ weight.double().T
        return z if bias is None else z + bias.double()

    def forward(x, weight, bias, residual, function, degree, source):
        y = torch.nn.functional.gelu(z_of(x, weight, bias))
        return (y if residual is None else y + residual.double()).to(x.dtype)

    def with_slope(x, weight, bias, residual, function, degree, source):
        z = z_of(x, weight, bias).reshape(-1, weight.shape[0])
        slope = torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
        kept = torch.zeros(z.shape[0], (z.shape[1] + 7) // 8 * 8, dtype=torch.float16)
        kept[:, :z.shape[1]] = slope
        return forward(x, weight, bias, residual, function, degree, source), kept

    def backward(dy, slope, x, weight, x_shape, out, bias_dtype, want_x, want_weight, want_bias):
        dz = dy.reshape(-1, out).double() * slope[:, :out].double()
        none = dy.new_empty(0)
        return ((dz @ weight.double()).to(dy.dtype).reshape(x_shape) if want_x else none,
                (dz.T @ x.double().reshape(-1, x_shape[-1])).to(dy.dtype) if want_weight else none,
                dz.sum(0).to((torch.float16, torch.bfloat16, torch.float32)[bias_dtype]) if want_bias else none)

    def norm(t, w):
        u = t.double() * torch.rsqrt(t.double().square().mean(-1, keepdim=True) + 1e-6)
        return (u if w is None else u * w.double()).to(t.dtype)

    def rope(q, k, q_weight, k_weight, inc, positions, sections, order, pairing, with_norm, eps, inverse):
        return (norm(q, q_weight), norm(k, k_weight)) if with_norm else (q.clone(), k.clone())

    def rope_backward(dq, dk, q, k, q_weight, k_weight, inc, positions, sections, order, pairing, eps, want_q, want_k):
        out = []
        for g, t, w, want in ((dq, q, q_weight, want_q), (dk, k, k_weight, want_k)):
            t, g = t.double(), g.double()
            r = torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6)
            u, h = t * r, g if w is None else g * w.double()
            out.append(((r * (h - u * (h * u).mean(-1, keepdim=True))).to(dq.dtype), (g * u).sum((0, 1, 2)).to(w.dtype) if want else q.new_empty(0)))
        return out[0][0], out[1][0], out[0][1], out[1][1]

    library = torch.library.Library("fpt_b200", "IMPL")
    for name, kernel in (("linear_act", forward), ("linear_act_slope", with_slope), ("linear_act_bwd", backward), ("qk_rope", rope),
                         ("qk_norm_rope_bwd", rope_backward)):
        library.impl(name, kernel, "CPU")
    yield
    library._destroy()


def values(*shape, seed=0, grad=True):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).requires_grad_(grad)


def layer_args(rows):
    return [values(rows, 16, seed=1), values(24, 16, seed=2), values(24, seed=3), values(rows, 24, seed=4)]


def heads_args(rows):
    return [values(2, rows, 4, 64, seed=1), values(2, rows, 2, 64, seed=2), values(64, seed=3), values(64, seed=4)]


def cpu_heads(q, k, q_weight, k_weight):
    return torch.cat(torch.ops.fpt_b200.qk_rope(q, k, q_weight, k_weight, torch.zeros(32, dtype=torch.int32), None, [], 0, 0, True, 1e-6, False), dim=2)


@pytest.mark.parametrize("call, make, row_axis", [(layer, layer_args, 0), (cpu_heads, heads_args, 1)], ids=["layer", "heads"])
@pytest.mark.parametrize("marked", [True, False])
def test_compiled_training_step_with_any_number_of_rows(cpu_kernels, call, make, row_axis, marked):
    """One graph for all row counts: none is written into the operators' gradients."""
    torch._dynamo.reset()
    compiled = torch.compile(call, backend="aot_eager", fullgraph=True, dynamic=None if marked else True)
    with torch._dynamo.config.patch(recompile_limit=2, error_on_recompile=False):
        for rows in (50, 3, 7, 11, 200):
            args = make(rows)
            if marked:
                for t in args:
                    if t.dim() > row_axis and t.shape[row_axis] == rows and t.dim() > 1:
                        torch._dynamo.mark_dynamic(t, row_axis)
            want = torch.autograd.grad(call(*args).float().sum(), args)
            got = torch.autograd.grad(compiled(*args).float().sum(), args)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), rows
    torch._dynamo.reset()


def cpu_rotation(q, k):
    return torch.cat(torch.ops.fpt_b200.qk_rope(q, k, None, None, torch.zeros(32, dtype=torch.int32), None, [], 0, 0, False, 0.0, False), dim=2)


CALLS = {"layer": (layer, layer_args), "heads": (cpu_heads, heads_args), "rotation": (cpu_rotation, lambda rows: heads_args(rows)[:2])}


@pytest.mark.parametrize("name", list(CALLS))
def test_function_transforms_give_the_gradients_of_autograd(cpu_kernels, name):
    call, make = CALLS[name]
    args = make(5)
    every = tuple(range(len(args)))
    cotangent = values(*call(*args).shape, seed=9, grad=False)
    want = torch.autograd.grad(call(*args), args, cotangent)
    plain = [t.detach() for t in args]
    loss = lambda *a: (call(*a) * cotangent).sum()
    assert all(torch.equal(a, b) for a, b in zip(torch.func.grad(loss, argnums=every)(*plain), want))
    y, pull = torch.func.vjp(call, *plain)
    assert torch.equal(y, call(*plain)) and all(torch.equal(a, b) for a, b in zip(pull(cotangent), want))
    rows = torch.func.jacrev(lambda t: call(t, *plain[1:]).flatten()[:3])(plain[0])
    for i in range(3):
        one = torch.zeros_like(cotangent)
        one.view(-1)[i] = 1
        assert torch.equal(rows[i], torch.autograd.grad(call(*args), args[0], one)[0])


@pytest.mark.parametrize("name", list(CALLS))
def test_a_transform_in_a_transform(cpu_kernels, name):
    """The outer transform sees the inner one's value as it sees a plain call, and no second derivative that is not there."""
    call, make = CALLS[name]
    plain = [t.detach() for t in make(5)]
    loss = lambda a, b: call(a, b, *plain[2:]).float().square().sum()
    inner = lambda a, b: torch.func.grad_and_value(loss)(a, b)
    want = torch.func.grad(loss, argnums=1)(*plain[:2])
    assert torch.equal(torch.func.grad(lambda b: inner(plain[0], b)[1])(plain[1]), want)
    if name != "rotation":
        with pytest.raises(RuntimeError, match="no second gradient"):
            torch.func.grad(lambda b: inner(plain[0], b)[0].float().sum())(plain[1])
        with pytest.raises(RuntimeError, match="no second gradient"):
            torch.func.grad(lambda a: inner(a, plain[1])[0].float().sum())(plain[0])
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.hessian(loss)(*plain[:2])


def test_the_rotation_alone_has_every_derivative(cpu_kernels):
    """It is linear: its gradient is the rotation backwards, which has a gradient.  The second derivative of a sum of squares."""
    q, k = heads_args(3)[:2]
    loss = lambda q: cpu_rotation(q, k.detach()).double().square().sum()
    second = torch.func.grad(lambda q: torch.func.grad(loss)(q).double().sum())(q.detach())
    assert torch.equal(second, torch.full_like(q, 2))
    first, = torch.autograd.grad(loss(q), q, create_graph=True)
    assert torch.equal(torch.autograd.grad(first.double().sum(), q)[0], torch.full_like(q, 2))


@pytest.mark.parametrize("activation", [GELU, -1])
@pytest.mark.parametrize("which", range(4))
def test_vjp_of_one_argument(activation, which):
    """Shapes only: the plain form above knows GELU alone."""
    args = [meta(*s) for s in LAYER]

    def call(t):
        return torch.ops.fpt_b200.linear_act(*args[:which], t, *args[which + 1:], activation, 0, 0)
    y, pull = torch.func.vjp(call, args[which])
    assert pull(torch.empty_like(y))[0].shape == args[which].shape


@pytest.mark.parametrize("name", ["layer", "heads"])
def test_create_graph_is_refused(cpu_kernels, name):
    call, make = CALLS[name]
    args = make(5)
    with pytest.raises(RuntimeError, match="no second gradient"):
        torch.autograd.grad(call(*args).float().sum(), args[:1], create_graph=True)


def test_the_parts_of_a_training_step_are_recorded(cpu_kernels):
    """Called by themselves: the result has the layer's gradient, the slope and the gradients refuse theirs."""
    x, w, b, r = layer_args(4)
    y, slope = torch.ops.fpt_b200.linear_act_slope(x, w, b, r, GELU, 0, 0)
    dy = torch.ones_like(y)
    assert all(torch.equal(s, t) for s, t in zip(torch.autograd.grad(y, (x, w, b, r), dy), torch.autograd.grad(layer(x, w, b, r), (x, w, b, r), dy)))
    with pytest.raises(RuntimeError, match="no second gradient"):
        torch.autograd.grad(slope.float().sum(), x)
    dx, *_ = torch.ops.fpt_b200.linear_act_bwd(dy, slope.detach(), x, w, x.shape, 24, 1, True, True, True)
    with pytest.raises(RuntimeError, match="no second gradient"):
        torch.autograd.grad(dx.float().sum(), w)
    q, k, qw, kw = heads_args(3)
    dq, *_ = torch.ops.fpt_b200.qk_norm_rope_bwd(q.detach(), k.detach(), q, k, qw, kw, torch.zeros(32, dtype=torch.int32), None, [], 0, 0, 1e-6, True, True)
    with pytest.raises(RuntimeError, match="no second gradient"):
        torch.autograd.grad(dq.float().sum(), q)
