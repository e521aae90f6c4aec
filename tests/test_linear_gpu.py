"""GPU: act(x W^T + b) + r and its gradients against a plain implementation in 64 bits.

Tolerances.  h = half a rounding step of the data type (eps / 2 of the value, and 2^-25 for fp16), u = 2^-23 (the tensor
cores may truncate, so a whole step of fp32 is counted), S = sum |x w| + |b|.
  z            products of 16-bit values are exact in fp32; 16 of them join the accumulator in one step, counted as two
               roundings of at most S, and up to 8 partial sums follow: dz <= (dim / 8 + 10) u S
  act          |act'| <= 1.13; ex2, rcp, erff and tanhf are good to 2 ulp and their arguments to one, logistic(z) to 4 u, so
               act(z) to 4 u (1 + |z|): |y - y_exact| <= h |y| + 1.13 dz + 4 u (1 + |z| + |r|)
  slope        |act''| <= 1: dz + 8 u (1 + |z|), then half a step of fp16 (2^-11 of it, 2^-25)
  dz           |dy| times the slope's error, then h
  dx, dW       the errors of dz times |W| or |x| summed up, the accumulation as for z (out / 8 or rows / 8 steps), then h
  db           the slope's part of the errors of dz (it is summed unrounded) and (rows / 8 + 64) u sum |dz|, then its h
"""
import math

import pytest
import torch

from fast_polynomial_transcendentals_b200 import spline_ops
from fast_polynomial_transcendentals_b200.linear import check_linear_status, linear_act

pytestmark = pytest.mark.gpu
U = 2.0 ** -23
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ACTIVATIONS = ["none", "sigmoid", "tanh", "silu", "gelu"]


@pytest.fixture
def tuning(fpt):
    lib = fpt.load()

    def set_form(tokens=-1, split=0, columns=0):
        for key, value in ((b"linear_tokens", tokens), (b"linear_split", split), (b"linear_columns", columns)):
            assert lib.fpt_set_tuning(key, value) == 0
    yield set_form
    set_form()


def half(dtype):
    return torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0


def act_and_slope(z, name):
    if name == "none":
        return z, torch.ones_like(z)
    if name == "tanh":
        return torch.tanh(z), 1 / torch.cosh(z) ** 2
    if name == "gelu":
        phi = torch.special.ndtr(z)
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    p = torch.sigmoid(z)
    return (p, p * (1 - p)) if name == "sigmoid" else (z * p, p * (1 + z * (1 - p)))


def near(got, want, slack, what):
    rel, least = half(got.dtype) if got.dtype != torch.float32 else (2.0 ** -24, 0.0)
    assert got.shape == want.shape, what
    over = ((got.double() - want).abs() - (rel * (want.abs() + slack) + least + slack))
    worst = over.max().item() if got.numel() else -1.0
    assert worst <= 0 and torch.isfinite(got).all(), f"{what}: {worst} above the tolerance"


def inputs(rows, dim, out, dtype, device, bias=True, residual=True, seed=0, bias_dtype=None):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device=device, generator=g)
    x, w = rand(rows, dim).to(dtype), (rand(out, dim) / math.sqrt(dim)).to(dtype)
    return x, w, rand(out).to(bias_dtype or dtype) if bias else None, rand(rows, out).to(dtype) if residual else None, rand(rows, out).to(dtype)


def check(x, w, b, r, dy, activation, grad=True, what=""):
    rows, dim, out = x.numel() // x.shape[-1], x.shape[-1], w.shape[0]
    leaves = [None if t is None else t.detach().requires_grad_(grad) for t in (x, w, b, r)]
    y = linear_act(*leaves, activation=activation)
    xd, wd = x.double().reshape(rows, dim), w.double()
    z, size = xd @ wd.T, xd.abs() @ wd.abs().T
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    value, slope = act_and_slope(z, activation)
    z_err = (dim / 8 + 10) * U * size
    want, slack = value, 1.13 * z_err + 4 * U * (1 + z.abs())
    if r is not None:
        want, slack = want + r.double().reshape(rows, out), slack + 4 * U * r.double().abs().reshape(rows, out)
    near(y.detach().reshape(rows, out), want, slack, f"{what} y")
    assert y.shape == (*x.shape[:-1], out) and y.is_contiguous()
    if not grad:
        return y
    names = [n for n, t in zip(("dx", "dw", "db", "dr"), leaves) if t is not None]
    got = dict(zip(names, torch.autograd.grad(y, [t for t in leaves if t is not None], dy)))
    d = dy.double().reshape(rows, out)
    dz = d * slope
    slope_err = 0 * z if activation == "none" else (2.0 ** -11 * slope.abs() + 2.0 ** -25 + 1.001 * (z_err + 8 * U * (1 + z.abs())))
    sum_err = d.abs() * slope_err
    rel, least = half(x.dtype)
    dz_err = sum_err + (0 if activation == "none" else rel * (dz.abs() + sum_err) + least)
    near(got["dx"].reshape(rows, dim), dz @ wd, dz_err @ wd.abs() + (out / 8 + 10) * U * ((dz.abs() + dz_err) @ wd.abs()), f"{what} dx")
    near(got["dw"], dz.T @ xd, dz_err.T @ xd.abs() + (rows / 8 + 10) * U * ((dz.abs() + dz_err).T @ xd.abs()), f"{what} dw")
    if b is not None:
        near(got["db"], dz.sum(0), sum_err.sum(0) + (rows / 8 + 64) * U * (dz.abs() + sum_err).sum(0), f"{what} db")
    if r is not None:
        assert torch.equal(got["dr"], dy)
    return y


SHAPES = [(1, 8, 1), (1, 64, 8), (2, 72, 3), (15, 200, 100), (16, 520, 127), (17, 128, 128), (33, 64, 129), (64, 1000, 200), (65, 192, 256),
          (100, 256, 257), (129, 72, 600), (257, 328, 264), (300, 136, 1003), (513, 64, 40)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_layer_and_gradients(cuda, shape, dtype):
    activation = ACTIVATIONS[sum(shape) % 5]
    check(*inputs(*shape, DTYPES[dtype], cuda, seed=sum(shape)), activation)
    check_linear_status()


@pytest.mark.parametrize("rows", [3, 40, 300])
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bias, residual", [(False, False), (True, False), (False, True)])
def test_every_activation_and_epilogue(cuda, rows, activation, dtype, bias, residual):
    check(*inputs(rows, 192, 144, DTYPES[dtype], cuda, bias, residual, seed=rows), activation)


@pytest.mark.parametrize("tokens", [0, 16, 32, 64, 128])
@pytest.mark.parametrize("shape", [(1, 640, 130), (50, 1032, 264), (200, 584, 384)], ids=str)
def test_every_form(cuda, tuning, tokens, shape):
    """Each tile form at every split, forward and backward, on the same inputs."""
    args = inputs(*shape, torch.bfloat16, cuda)
    for split in ([1, 2, 3, 5, 8] if tokens else [0]):
        tuning(tokens, split)
        check(*args, "gelu", what=f"tokens {tokens} split {split}")
    check_linear_status()


@pytest.mark.parametrize("columns", range(64, 257, 32))
def test_every_tile_width(cuda, tuning, columns):
    for shape in ((300, 200, 520), (70, 136, 1003)):
        tuning(0, 0, columns)
        check(*inputs(*shape, torch.bfloat16, cuda), "gelu", what=f"columns {columns}")
    check_linear_status()


@pytest.mark.parametrize("split, columns", [(2, 64), (2, 128), (2, 256), (4, 128), (4, 256)])
def test_pairs_that_share_a_tile(cuda, tuning, split, columns):
    """The K blocks of a tile over the pairs of a cluster, whole and ragged runs of them (the weight's gradient contracts over the
    rows: fewer K blocks than pairs fall back to one)."""
    for shape, dtype in (((300, 520, 264), "bf16"), ((70, 1288, 1003), "bf16"), ((513, 640, 40), "fp16"), ((1100, 1024, 512), "fp16")):
        tuning(0, split, columns)
        args = inputs(*shape, DTYPES[dtype], cuda)
        y = check(*args, "gelu", what=f"{shape}")
        assert torch.equal(y, linear_act(*args[:4], activation="gelu"))
    check_linear_status()


def test_several_tiles_per_block(cuda, tuning):
    """More output tiles than pairs of SMs: the persistent form goes round and alternates its accumulators."""
    tuning(0)
    check(*inputs(256 * 11 + 3, 72, 256 * 21 + 8, torch.bfloat16, cuda), "silu")


def test_long_contraction(cuda):
    for rows in (1, 20, 130, 400):
        check(*inputs(rows, 14336, 264, torch.bfloat16, cuda), "none")


@pytest.mark.parametrize("bias_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [5, 280])
def test_bias_types(cuda, bias_dtype, rows):
    check(*inputs(rows, 64, 136, torch.bfloat16, cuda, bias_dtype=bias_dtype), "gelu")


def odd_start(t):
    """The same values with rows that start on no 16-byte boundary."""
    wide = torch.zeros(t.shape[0], t.shape[1] + 3, dtype=t.dtype, device=t.device)
    wide[:, 1:-2] = t
    return wide[:, 1:-2]


@pytest.mark.parametrize("rows", [6, 290])
@pytest.mark.parametrize("layout", ["odd start", "wide rows", "transposed", "broadcast", "three dimensions"])
def test_layouts(cuda, rows, layout):
    x, w, b, r, dy = inputs(rows, 96, 152, torch.bfloat16, cuda)
    if layout == "odd start":
        x, w, r, dy = (odd_start(t) for t in (x, w, r, dy))
        b = torch.cat([b, b])[1:1 + b.numel()]
    elif layout == "wide rows":
        x, w, r, dy = (torch.cat([t, t], dim=1)[:, :t.shape[1]] for t in (x, w, r, dy))
        b = torch.stack([b, b], dim=1)[:, 0]
    elif layout == "transposed":
        x, w, r, dy = (t.t().contiguous().t() for t in (x, w, r, dy))
    elif layout == "broadcast":
        x, r, dy = x[:1].expand(rows, -1), r[:, :1].expand(-1, 152), dy[:1, :1].expand(rows, 152)
    else:
        x, r, dy = (t.view(2, rows // 2, -1) for t in (x, r, dy))
    check(x, w, b, r, dy, "silu")


def test_one_row_without_a_row_dimension(cuda):
    x, w, b, _, _ = inputs(1, 64, 24, torch.float16, cuda)
    assert torch.equal(linear_act(x[0], w, b, activation="tanh"), linear_act(x, w, b, activation="tanh")[0])


@pytest.mark.parametrize("dtype, source", [("fp16", "current"), ("bf16", "current"), ("bf16", "sollya")])
@pytest.mark.parametrize("activation", ["sigmoid", "tanh", "silu", "gelu"])
def test_polynomial_programs_bit_for_bit(cuda, activation, dtype, source):
    """degree 3 .. 6: the stored product through spline_ops, and the derivative program of that degree in the gradient."""
    name = "swish" if activation == "silu" else activation
    for rows, degree in ((7, 3), (300, 4), (7, 5), (300, 6)):
        x, w, b, r, dy = inputs(rows, 128, 200, DTYPES[dtype], cuda, seed=degree)
        x = x * 2
        z = linear_act(x, w, b)
        want = spline_ops._unary(z, name, 0, degree, int(source == "sollya"))
        got = linear_act(x, w, b, activation=activation, degree=degree, coeff_source=source)
        assert torch.equal(got, want), (degree, rows)
        with_residual = linear_act(x, w, b, r, activation=activation, degree=degree, coeff_source=source)
        assert torch.equal(with_residual, (want.float() + r.float()).to(want.dtype))
        one = torch.ones_like(z)
        slope = spline_ops._binary(one, z, name, degree, int(source == "sollya"))     # 1 * F'(z)
        bias = b.detach().float().requires_grad_()
        # b's cast to fp32 changes nothing (its values are 16-bit), and its gradient comes back in fp32
        y = linear_act(x, w, bias, activation=activation, degree=degree, coeff_source=source)
        db, = torch.autograd.grad(y, [bias], dy)
        terms = dy.double() * slope.double()
        assert ((db.double() - terms.sum(0)).abs() <= (2.0 ** -25 * dy.double().abs()).sum(0) + (rows / 8 + 64) * U * terms.abs().sum(0)).all()


def test_missing_program_is_refused(cuda):
    x, w, b, _, _ = inputs(4, 64, 24, torch.bfloat16, cuda)
    with pytest.raises(RuntimeError, match="degree"):
        linear_act(x, w, b, activation="gelu", degree=2)


@pytest.mark.parametrize("need", ["x", "weight", "bias", "residual"])
@pytest.mark.parametrize("activation", ["none", "gelu"])
def test_one_gradient_alone(cuda, need, activation):
    x, w, b, r, dy = inputs(20, 64, 40, torch.bfloat16, cuda)
    args = dict(x=x, weight=w, bias=b, residual=r)
    every = {k: v.detach().requires_grad_() for k, v in args.items()}
    want = dict(zip(every, torch.autograd.grad(linear_act(**every, activation=activation), list(every.values()), dy)))
    args[need] = args[need].detach().requires_grad_()
    got, = torch.autograd.grad(linear_act(**args, activation=activation), [args[need]], dy)
    assert torch.equal(got, want[need])


@pytest.mark.parametrize("activation", ["none", "gelu"])
def test_no_rows(cuda, activation):
    x, w, b, r, dy = inputs(0, 64, 41, torch.bfloat16, cuda)
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
    y = linear_act(*leaves, activation=activation)
    assert y.shape == (0, 41)
    dx, dw, db, dr = torch.autograd.grad(y, leaves, dy)
    assert dx.shape == (0, 64) and dr.shape == (0, 41) and torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros_like(b))


def test_gradient_against_differences(cuda):
    """<gradient, direction> against a central difference of the 64-bit definition.  With step 2^-12 the difference is off by
    (2^-24 / 6) |third derivative| < 1e-7 of the terms; the gradients carry roundings to bf16 (slope 2^-12, dz and the
    result 2^-9 each, independent from term to term): below 3 * 2^-9 of the sum of |terms|."""
    x, w, b, r, dy = inputs(40, 64, 72, torch.bfloat16, cuda)
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
    grads = torch.autograd.grad(linear_act(*leaves, activation="gelu"), leaves, dy)
    args = [t.double() for t in (x, w, b, r)]
    value = lambda x, w, b, r: ((act_and_slope(x @ w.T + b, "gelu")[0] + r) * dy.double()).sum()
    for i, g in enumerate(grads):
        direction = torch.randn_like(args[i])
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + 2.0 ** -12 * direction, args[i] - 2.0 ** -12 * direction
        terms = g.double() * direction
        assert abs(terms.sum() - (value(*up) - value(*down)) * 2.0 ** 11) <= 3 * 2.0 ** -9 * terms.abs().sum(), i


def test_no_second_gradient(cuda):
    x, w, *_ = inputs(4, 64, 24, torch.bfloat16, cuda)
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="no second gradient"):
        torch.autograd.grad(linear_act(x, w, activation="gelu").float().sum(), [x], create_graph=True)


def test_tail_of_gelu(cuda):
    """Relative to the result, where GELU(z) is small: z = x exactly (identity weight), so what is left is half a step of the
    dtype (fp16: at least 2^-25), the fit of the tail (1e-6) and its exponential, whose argument of at most 15 is rounded by
    2^-21 and twice 2^-24 of it (3e-6 together): (1 + 2^-10) h + 4e-6."""
    weight = torch.eye(64, device=cuda)
    for dtype in DTYPES.values():
        z = (-torch.arange(64 * 64, device=cuda).double() / (64 * 64) * 5.4).reshape(64, 64).to(dtype)
        want = z.double() * torch.special.ndtr(z.double())
        rel, least = half(dtype)
        for x in (z, z[:3]):
            got = linear_act(x, weight.to(dtype), activation="gelu").double()
            assert ((got - want[:len(x)]).abs() <= ((1 + 2.0 ** -10) * rel + 4e-6) * want[:len(x)].abs() + least).all()


def test_values_that_are_not_finite_stay_in_their_row(cuda):
    for rows in (9, 300):
        x, w, b, r, _ = inputs(rows, 64, 136, torch.bfloat16, cuda)
        clean = linear_act(x, w, b, r, activation="gelu")
        x[4, 7] = math.nan
        got = linear_act(x, w, b, r, activation="gelu")
        keep = torch.arange(rows, device=cuda) != 4
        assert got[4].isnan().all() and torch.equal(got[keep], clean[keep])


def test_results_do_not_change_from_run_to_run(cuda):
    for rows in (30, 200, 700):
        x, w, b, r, dy = inputs(rows, 2048, 1408, torch.bfloat16, cuda)
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        runs = []
        for _ in range(3):
            y = linear_act(*leaves, activation="gelu")
            runs.append([y, *torch.autograd.grad(y, leaves, dy)])
        assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(runs[0], run))


@pytest.mark.parametrize("rows", [5, 100, 300])
def test_output_rows_wider_than_the_result(cuda, fpt, rows):
    """Through the C ABI: what lies behind the last column and the last row stays as it was."""
    x, w, b, _, _ = inputs(rows, 64, 43, torch.bfloat16, cuda)
    wide = torch.full((rows + 2, 50), 7.0, dtype=torch.bfloat16, device=cuda)
    stream = torch.cuda.current_stream().cuda_stream
    fpt.call("fpt_linear", wide.data_ptr(), None, x.data_ptr(), w.data_ptr(), b.data_ptr(), None, rows, 64, 43, 64, 64, 50, 0, 0, 1, 1, 4, 0, 0, None, stream)
    assert torch.equal(wide[:rows, :43], linear_act(x, w, b, activation="gelu"))
    assert (wide[:rows, 43:] == 7).all() and (wide[rows:] == 7).all()


def test_another_stream_and_captured_graphs(cuda):
    stream, made = torch.cuda.Stream(cuda), []
    for rows in (10, 150, 600):
        x, w, b, r, dy = inputs(rows, 256, 264, torch.bfloat16, cuda, seed=rows)
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]

        def step(leaves=leaves, dy=dy):
            y = linear_act(*leaves, activation="gelu")
            return [y, *torch.autograd.grad(y, leaves, dy)]

        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
        made.append((graph, step, out, leaves[0]))
    for index in (2, 0, 1, 0):
        graph, step, out, x = made[index]
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))
    for graph, *_ in made:
        graph.replay()
    check_linear_status()
    for _, step, out, _ in made:
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_two_streams_at_once(cuda):
    args = [inputs(rows, 2048, 1024, torch.bfloat16, cuda, seed=rows) for rows in (24, 700)]
    want = [linear_act(x, w, b, r, activation="silu") for x, w, b, r, _ in args]
    streams = [torch.cuda.Stream(cuda) for _ in args]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for s, (x, w, b, r, _) in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(linear_act(x, w, b, r, activation="silu"))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_under_torch_compile(cuda):
    x, w, b, r, dy = inputs(12, 64, 40, torch.bfloat16, cuda)
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
    f = lambda x, w, b, r: linear_act(x, w, b, r, activation="gelu") * 2
    want = torch.autograd.grad(f(*leaves), leaves, dy)
    got = torch.autograd.grad(torch.compile(f, backend="aot_eager", fullgraph=True)(*leaves), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_random_shapes(cuda):
    """Random shapes over both forms and the rule that picks one."""
    g = torch.Generator().manual_seed(5)
    for i in range(24):
        rows, dim, out = (int(torch.randint(lo, hi, (1,), generator=g)) for lo, hi in ((1, 700), (1, 60), (1, 900)))
        check(*inputs(rows, 8 * dim, out, DTYPES["fp16" if i % 3 == 0 else "bf16"], cuda, seed=i), ACTIVATIONS[i % 5], what=str((rows, 8 * dim, out)))


def test_compiled_training_step_with_any_number_of_rows(cuda):
    """One compiled graph, row counts of every tile form: the bits of the eager call."""
    torch._dynamo.reset()
    f = lambda x, w, b, r: linear_act(x, w, b, r, activation="gelu") * 2
    compiled = torch.compile(f, backend="aot_eager", fullgraph=True)
    with torch._dynamo.config.patch(recompile_limit=2):
        for rows in (12, 2, 40, 300, 1025):
            x, w, b, r, dy = inputs(rows, 64, 40, torch.bfloat16, cuda, seed=rows)
            leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
            for t in (leaves[0], leaves[3]):
                torch._dynamo.mark_dynamic(t, 0)
            want = torch.autograd.grad(f(*leaves), leaves, dy)
            got = torch.autograd.grad(compiled(*leaves), leaves, dy)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), rows
    torch._dynamo.reset()


def test_a_thread_that_has_made_no_call_yet(cuda, fpt):
    """The first call of a new host thread is the layer's, through the C ABI and through the operator (its output comes from the
    allocator's cache): the thread has no context of its own before it."""
    import threading
    lib, (x, w, b, _, _) = fpt.load(), inputs(300, 64, 24, torch.bfloat16, cuda)
    want, out, got = linear_act(x, w, b, activation="gelu"), torch.empty(300, 24, dtype=torch.bfloat16, device=cuda), []
    spare = torch.empty_like(out)
    del spare
    stream = torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()
    calls = [lambda: lib.fpt_linear(out.data_ptr(), None, x.data_ptr(), w.data_ptr(), b.data_ptr(), None, 300, 64, 24, 64, 64, 24, 0, 0, 1, 1, 4,
                                    0, 0, None, stream),
             lambda: linear_act(x, w, b, activation="gelu")]
    for call in calls:
        thread = threading.Thread(target=lambda: got.append(call()))
        thread.start()
        thread.join()
    torch.cuda.synchronize()
    assert got[0] == 0 and len(got) == 2
    assert torch.equal(out, want) and torch.equal(got[1], want)


def test_threads_with_rings_of_two_sizes(cuda, fpt):
    """One kernel with a ring of 216 KB (a block alone on its SM) and of 108 KB, from threads that call at once (ctypes lets go of
    the interpreter's lock).  No launch fails on a limit that another thread set."""
    import threading
    lib, args = fpt.load(), [inputs(1, n, n, torch.bfloat16, cuda, residual=False)[:3] for n in (4096, 1024)]
    want = [linear_act(*a, activation="gelu") for a in args]
    made, failures, start = [], [], threading.Barrier(4)
    torch.cuda.synchronize()

    def run(i):
        x, w, b = args[i % 2]
        n, out, stream = x.shape[1], torch.zeros_like(x), torch.cuda.Stream(cuda)
        call = (out.data_ptr(), None, x.data_ptr(), w.data_ptr(), b.data_ptr(), None, 1, n, n, n, n, n, 0, 0, 1, 1, 4, 0, 0, None, stream.cuda_stream)
        made.append((i, out, stream))
        start.wait()
        for _ in range(5000):
            status = lib.fpt_linear(*call)
            if status:
                failures.append(status)
                return

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    torch.cuda.synchronize()
    assert not failures
    assert len(made) == 4 and all(torch.equal(out, want[i % 2]) for i, out, _ in made)


@pytest.mark.parametrize("rows", [3, 300])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("activation, low, high", [("sigmoid", -26, 26), ("tanh", -13, 13), ("silu", -26, -3), ("gelu", -7, -3)])
def test_small_slopes_keep_their_precision(cuda, activation, low, high, dtype, rows):
    """Relative to the gradient, where the slope is small.  With the identity for a weight z = x and dx = dz, so dx is dy times the
    slope with its roundings: h for the result, h of fp16 for the slope as it is kept (steps of 2^-10 from 1 on: 2^-11 of the value;
    below 2^-29, where 2^15 times the slope is subnormal, steps of 2^-24 2^-15: 2^-40), and what the exponential carries.  That is the rounding of its argument, at most 4 |z| u in sigmoid, SiLU and tanh and
    2 z^2 u in GELU, and 16 u for ex2, rcp and the products."""
    w = torch.eye(64, device=cuda).to(DTYPES[dtype])
    x = torch.linspace(low, high, rows * 64, device=cuda).reshape(rows, 64).to(DTYPES[dtype])
    dy = torch.randn(rows, 64, device=cuda).to(DTYPES[dtype])
    leaf = x.detach().requires_grad_()
    dx, = torch.autograd.grad(linear_act(leaf, w, activation=activation), leaf, dy)
    z, d = x.double(), dy.double()
    want = d * (torch.sigmoid(z) * torch.sigmoid(-z) if activation == "sigmoid" else act_and_slope(z, activation)[1])   # 1 - p would cancel
    rel, least = half(DTYPES[dtype])
    exponential = (2 * z * z if activation == "gelu" else 4 * z.abs()) + 16
    slack = (2.0 ** -11 + exponential * U) * want.abs() + 2.0 ** -40 * d.abs()
    assert ((dx.double() - want).abs() <= rel * (want.abs() + slack) + slack + least).all()


def test_column_sums_of_nearly_2_31_rows(cuda, fpt):
    """The last block's rows would end past 31 bits (740 chunks of 2902005 rows): they count all the same."""
    rows = 2 ** 31 - 300
    dy = torch.zeros(rows, 1, dtype=torch.bfloat16, device=cuda)
    dy[0], dy[rows // 2], dy[-1] = 1, 2, 4
    lib, db = fpt.load(), torch.empty(1, device=cuda)
    nbytes = lib.fpt_linear_grad_act_workspace_bytes(rows, 1)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=cuda)
    fpt.call("fpt_linear_grad_act", None, db.data_ptr(), dy.data_ptr(), None, workspace.data_ptr(), nbytes, rows, 1, 8, 1, 8, 1, 2,
             torch.cuda.current_stream().cuda_stream)
    assert db.item() == 7


def test_a_reported_wait_belongs_to_its_device(cuda):
    """A status word that the host writes as a kernel would: the next call on that device raises, once; another device's word is
    left for calls there."""
    import ctypes
    from fast_polynomial_transcendentals_b200 import _fpt_torch
    x, w, b, _, _ = inputs(4, 64, 24, torch.bfloat16, cuda)
    want = linear_act(x, w, b)
    check_linear_status()
    words = [ctypes.c_uint32.from_address(_fpt_torch.linear_status_address(i)) for i in (0, 1)]
    words[1].value = 0x80000052
    assert torch.equal(linear_act(x, w, b), want)
    check_linear_status(cuda)
    with pytest.raises(RuntimeError, match="cuda:1"):
        _fpt_torch.poll_linear_status(1)
    assert words[1].value == 0
    words[0].value = 0x80000052
    with pytest.raises(RuntimeError, match="cuda:0"):
        linear_act(x, w, b)
    assert words[0].value == 0 and torch.equal(linear_act(x, w, b), want)
    words[0].value = 0x80000053
    with pytest.raises(RuntimeError, match="cuda:0"):
        check_linear_status(0)
    check_linear_status("cuda")
