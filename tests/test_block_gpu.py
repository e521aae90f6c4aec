"""GPU: the operators around the attention in a run, as a transformer block uses them: projection with bias, norm of queries
and keys with the rotation (one axis, or three), the attention kernel, projection onto the residual stream, GELU
feed-forward onto the residual stream; forward, gradients, a captured step, and the feed-forward through the adapter."""
import math

import pytest
import torch
from torch import nn

from fast_polynomial_transcendentals_b200 import qk_rope
from fast_polynomial_transcendentals_b200.linear import check_linear_status, linear_act
from fast_polynomial_transcendentals_b200.sfu_repro import adapters, fa4
from fast_polynomial_transcendentals_b200.sfu_repro.rope import rope_phase_increments

pytestmark = pytest.mark.gpu
B, S, HQ, HK, D, HIDDEN = 2, 200, 4, 2, 128, 1000
DIM = HQ * D
BF = torch.bfloat16


def weights(device, seed=0):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    rand = lambda *s, scale=1.0: (torch.randn(*s, device=device, generator=g) * scale).to(BF)
    return dict(qkv=rand((HQ + 2 * HK) * D, DIM, scale=DIM ** -0.5), qkv_bias=rand((HQ + 2 * HK) * D, scale=0.1),
                q_norm=1 + rand(D, scale=0.1), k_norm=1 + rand(D, scale=0.1), out=rand(DIM, DIM, scale=DIM ** -0.5),
                up=rand(HIDDEN, DIM, scale=DIM ** -0.5), up_bias=rand(HIDDEN, scale=0.1), down=rand(DIM, HIDDEN, scale=HIDDEN ** -0.5),
                down_bias=rand(DIM, scale=0.1)), rand(B, S, DIM)


def attention(q, k, v):
    config = fa4.resolve_fa4_config(fa4.FA4Config(mode="softmax"), sequence_length=S)
    return fa4._fa4(q, k, v, softmax_scale=None, causal=True, config=config)


def split_heads(qkv):
    return (qkv[..., :HQ * D].unflatten(-1, (HQ, D)), qkv[..., HQ * D:(HQ + HK) * D].unflatten(-1, (HK, D)),
            qkv[..., (HQ + HK) * D:].unflatten(-1, (HK, D)))


def block(x, w, inc, positions, sections):
    q, k, v = split_heads(linear_act(x, w["qkv"], w["qkv_bias"]))
    if sections is None:
        q, k = qk_rope.qk_norm_rope(q, k, w["q_norm"], w["k_norm"], inc, positions=positions, pairing="halves")
    else:
        q, k = qk_rope.rope_axes(q, k, inc, positions, sections, pairing="halves")
    x = linear_act(attention(q, k, v.contiguous()).flatten(2), w["out"], None, x)
    return linear_act(linear_act(x, w["up"], w["up_bias"], activation="gelu"), w["down"], w["down_bias"], x)


class RoundGrad(torch.autograd.Function):
    """bf16 value, bf16 gradient: where an operator of the run hands on a tensor"""

    @staticmethod
    def forward(ctx, x):
        return x.to(BF).float()

    @staticmethod
    def backward(ctx, g):
        return g.to(BF).float()


def plain_block(x, w, inc, positions, sections):
    """The same in fp32 with roundings to bf16 at the operators' borders, around the same attention kernel."""
    f = {n: t.float() for n, t in w.items()}
    rnd = RoundGrad.apply
    xf = x.float()
    q, k, v = split_heads(rnd(xf @ f["qkv"].T + f["qkv_bias"]))
    if sections is None:
        position = positions[..., None].double()
        q, k = (t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * f[n] for t, n in ((q, "q_norm"), (k, "k_norm")))
    else:
        position = torch.stack([positions[a] for a, n in enumerate(sections) for _ in range(n)], dim=-1).double()
    angle = (position * inc.double() * (2 * math.pi / 2 ** 32))[:, :, None]
    c, s = angle.cos().float(), angle.sin().float()
    turn = lambda t: rnd(torch.cat((t[..., :D // 2] * c - t[..., D // 2:] * s, t[..., D // 2:] * c + t[..., :D // 2] * s), dim=-1))
    xf = rnd(attention(turn(q).to(BF), turn(k).to(BF), v.to(BF)).float().flatten(2) @ f["out"].T + xf)
    hidden = rnd(torch.nn.functional.gelu(xf @ f["up"].T + f["up_bias"]))
    return rnd(hidden @ f["down"].T + f["down_bias"] + xf)


def case(cuda, axes):
    w, x = weights(cuda)
    inc = rope_phase_increments(D, 10000.0, cuda)
    if axes:
        return w, x, inc, torch.randint(0, 60, (3, B, S), device=cuda), [16, 24, 24]
    return w, x, inc, torch.arange(S, device=cuda).expand(B, S) + torch.tensor([[0], [5000]], device=cuda), None


@pytest.mark.parametrize("axes", [False, True])
def test_a_block_and_its_gradients(cuda, axes):
    """Both runs round at the same places, so values differ where a rounding falls the other way (one step, 2^-8 of the value,
    carried on through up to six operators: root mean square below 2^-8); in the gradients the operators also round dz before
    its products (2^-8 at most, 2^-9.3 root mean square, at three layers): below 2^-7."""
    w, x, inc, positions, sections = case(cuda, axes)
    leaves = {n: t.detach().requires_grad_() for n, t in w.items() if not (axes and n.endswith("_norm"))}
    xs = x.detach().requires_grad_()
    names = ["x", *leaves]
    grad = torch.randn_like(x)
    results = []
    for f in (block, plain_block):
        y = f(xs, {**w, **leaves}, inc, positions, sections)
        results.append((y.detach().float(), torch.autograd.grad(y, [xs, *leaves.values()], grad.to(y.dtype))))
    relative = lambda a, b: ((a.float() - b.float()).norm() / b.float().norm()).item()
    assert relative(results[0][0], results[1][0]) < 2.0 ** -8
    for n, a, b in zip(names, results[0][1], results[1][1]):
        assert relative(a, b) < 2.0 ** -7, (n, relative(a, b))
    fa4.check_attention_status()
    check_linear_status()


def test_a_captured_step(cuda):
    """Forward and backward of the run in one graph, replayed with new inputs; the attention adds its dQ in no fixed order, so
    only what does not pass through it is compared bit for bit."""
    w, x, inc, positions, sections = case(cuda, False)
    leaves = {n: t.detach().requires_grad_() for n, t in w.items()}
    grad = torch.randn_like(x)

    def step():
        y = block(x, leaves, inc, positions, sections)
        return y, *torch.autograd.grad(y, [leaves["up"], leaves["down"], leaves["up_bias"]], grad)

    stream = torch.cuda.Stream(cuda)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    for _ in range(2):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))
    fa4.check_attention_status()
    check_linear_status()


def test_one_token_at_a_time_equals_the_prompt(cuda):
    """Serving: the projections, norms and rotations of single tokens at their positions give what the whole prompt gives, up
    to the order of the fp32 sums (another tile form), one step of bf16."""
    w, x, inc, positions, _ = case(cuda, False)
    whole = split_heads(linear_act(x, w["qkv"], w["qkv_bias"]))
    q, k = qk_rope.qk_norm_rope(*whole[:2], w["q_norm"], w["k_norm"], inc, positions=positions, pairing="halves")
    for t in (0, 1, 77, S - 1):
        one = split_heads(linear_act(x[:, t:t + 1], w["qkv"], w["qkv_bias"]))
        q1, k1 = qk_rope.qk_norm_rope(*one[:2], w["q_norm"], w["k_norm"], inc, positions=positions[:, t:t + 1], pairing="halves")
        for a, b in ((q1, q[:, t:t + 1]), (k1, k[:, t:t + 1])):
            # one step (2^-7 of the largest of a pair) of the projection, another of the result
            assert (a.float() - b.float()).abs().max() <= 2 * 2.0 ** -7 * float(b.float().abs().max())
            assert ((a.float() - b.float()).norm() / b.float().norm()).item() < 2.0 ** -9


class Mlp(nn.Module):
    def __init__(self, act):
        super().__init__()
        self.fc1, self.fc2, self.activation_fn = nn.Linear(256, 600), nn.Linear(600, 256), act

    def forward(self, x):
        return self.fc2(self.activation_fn(self.fc1(x)))


@pytest.mark.parametrize("act", [nn.GELU(), nn.SiLU()], ids=["gelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_adapter_runs_the_feed_forward(cuda, act, dtype):
    """Against the same module in fp32: the patched one rounds the hidden values, dz and the results (four roundings of at
    most eps / 2)."""
    torch.manual_seed(1)
    model = Mlp(act).to(cuda, dtype)
    x, grad = torch.randn(70, 256, device=cuda).to(dtype).requires_grad_(), torch.randn(70, 256, device=cuda).to(dtype)
    exact = Mlp(act).to(cuda)
    exact.load_state_dict({n: t.float() for n, t in model.state_dict().items()})
    xf = x.detach().float().requires_grad_()
    want_y = exact(xf)
    want = torch.autograd.grad(want_y, [xf, *exact.parameters()], grad.float())
    assert adapters.patch_mlp_epilogues(model) == 1
    y = model(x)
    got = torch.autograd.grad(y, [x, *model.parameters()], grad)
    for a, b in zip((y, *got), (want_y, *want)):
        assert ((a.float() - b).norm() / b.norm()).item() < 4 * torch.finfo(dtype).eps / 2
    poly = Mlp(act).to(cuda, dtype)
    poly.load_state_dict(model.state_dict())
    assert adapters.patch_mlp_epilogues(poly, variant="polynomial") == 1
    assert ((poly(x).float() - want_y).norm() / want_y.norm()).item() < 0.05         # the programs' own error
    assert adapters.restore(model) == 1
    torch.testing.assert_close(model(x).float(), y.float(), rtol=0, atol=8 * torch.finfo(dtype).eps)
    check_linear_status()


def test_adapter_leaves_hooked_projections_alone(cuda):
    model = Mlp(nn.GELU()).to(cuda, BF)
    x = torch.randn(5, model.fc1.in_features, device=cuda).to(BF)
    model.fc1.register_forward_hook(lambda module, args, out: 2 * out)
    with torch.no_grad():
        want = model(x)
        assert adapters.patch_mlp_epilogues(model) == 1
        assert torch.equal(model(x), want)


def test_calls_from_two_threads_at_once(cuda):
    """Two threads, each on a stream of its own, few and many rows, forward and gradients: the same bits as one after another."""
    import threading
    inc = rope_phase_increments(D, device=cuda)

    def step(seed):
        g = torch.Generator(device=cuda)
        g.manual_seed(seed)
        out = []
        for rows in (3, 256, 700):
            x = torch.randn(rows, 2048, device=cuda, generator=g).to(BF).requires_grad_()
            w = (torch.randn(6 * D, 2048, device=cuda, generator=g) / 45).to(BF).requires_grad_()
            y = linear_act(x, w, activation="gelu")
            q, k = qk_rope.qk_norm_rope(*y.view(1, rows, 6, D).split([4, 2], dim=2), None, None, inc)
            out += [y, q, k, *torch.autograd.grad((q, k), [x, w], [torch.ones_like(q), torch.ones_like(k)])]
        return out

    want = [step(seed) for seed in (1, 2)]
    torch.cuda.synchronize()
    got = [[], []]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i].append(step(i + 1))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    for i in range(2):
        assert len(got[i]) == 10
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
    check_linear_status()


def test_offsets_past_31_bits(cuda):
    """Results of more than 2^31 elements, rows checked at both ends and in between.  One rounding to bf16 (eps / 2 = 2^-8 of
    the value: eight significant bits) and fp32 sums of 64 terms of size 64 / 8 in all (18 u S, S < 100: below 3e-4)."""
    rows, out = 66000, 33000
    x, w = torch.randn(rows, 64, device=cuda).to(BF), torch.randn(out, 64, device=cuda).to(BF)
    y = linear_act(x, w, activation="silu")
    for i in (0, 1, 32767, 65535, 65536, rows - 1):
        z = x[i].double() @ w.double().T
        want = z * torch.sigmoid(z)
        assert ((y[i].double() - want).abs() <= 2.0 ** -8 * want.abs() + 3e-4).all(), i
    del y
    seq = 270000                                       # 2 x 270000 x 32 x 128 > 2^31, and a batch entry beyond 4 GB of rows
    wide = torch.empty(2, seq, 34 * 128 * 2, dtype=BF, device=cuda)
    q = wide[..., :32 * 128].unflatten(-1, (32, 128))
    k = wide[..., 32 * 128:34 * 128].unflatten(-1, (2, 128))
    picks = [(0, 0), (0, 1), (0, 246723), (0, seq - 1), (1, 0), (1, 123456), (1, seq - 1)]
    for b, s in picks:
        wide[b, s] = torch.randn(wide.shape[-1], device=cuda).to(BF)
    inc = rope_phase_increments(128, device=cuda)
    got = qk_rope.rope_axes(q, k, inc, torch.arange(seq, device=cuda)[None], [64], pairing="halves")
    for b, s in picks:
        one = qk_rope.rope_axes(q[b:b + 1, s:s + 1].contiguous(), k[b:b + 1, s:s + 1].contiguous(), inc,
                                torch.tensor([[s]], device=cuda), [64], pairing="halves")
        assert torch.equal(got[0][b, s], one[0][0, 0]) and torch.equal(got[1][b, s], one[1][0, 0]), (b, s)


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_checkpointed_block(cuda, reentrant):
    """Activation checkpointing of the run, which ends in a layer with a residual: the same values, and gradients whose bits are the
    same where they do not pass through the attention (it adds its dQ in no fixed order: root mean square below 2^-8)."""
    from torch.utils.checkpoint import checkpoint
    w, x, inc, positions, sections = case(cuda, False)
    leaves = {n: t.detach().requires_grad_() for n, t in w.items()}
    xs, grad = x.detach().requires_grad_(), torch.randn_like(x)
    runs = []
    for call in (block, lambda *args: checkpoint(block, *args, use_reentrant=reentrant)):
        for t in (xs, *leaves.values()):
            t.grad = None
        y = call(xs, leaves, inc, positions, sections)
        y.backward(grad)
        runs.append((y.detach(), {"x": xs.grad, **{n: t.grad for n, t in leaves.items()}}))
    assert torch.equal(runs[0][0], runs[1][0])
    for n, want in runs[0][1].items():
        got = runs[1][1][n]
        if n in ("up", "up_bias", "down", "down_bias"):
            assert torch.equal(got, want), n
        else:
            assert ((got.float() - want.float()).norm() / want.float().norm()).item() < 2.0 ** -8, n
    fa4.check_attention_status()
    check_linear_status()


def test_a_checkpointed_patched_feed_forward(cuda):
    from torch.utils.checkpoint import checkpoint
    model = Mlp(nn.GELU()).to(cuda, BF)
    assert adapters.patch_mlp_epilogues(model) == 1
    x = torch.randn(40, 256, device=cuda).to(BF).requires_grad_()
    want = torch.autograd.grad(x + model(x), [x, *model.parameters()], torch.ones_like(x))
    y = x + checkpoint(model, x, use_reentrant=False)
    got = torch.autograd.grad(y, [x, *model.parameters()], torch.ones_like(x))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_function_transforms(cuda):
    """torch.func gives the bits of autograd; the rotation alone, which is linear, has a second derivative too (of half the sum of
    squares: the rotation there and back, three roundings to fp32 of values below 6: 2^-18)."""
    w, x, inc, positions, _ = case(cuda, False)
    names = ("up", "up_bias", "q_norm")

    def loss(x, up, up_bias, q_norm):
        hidden = linear_act(x, up, up_bias, activation="gelu")[..., :768].unflatten(-1, (6, D))
        q, k = qk_rope.qk_norm_rope(hidden[..., :4, :], hidden[..., 4:, :], q_norm, None, inc, positions=positions, pairing="halves")
        return q.float().square().sum() + k.float().sum()

    args = [t.detach() for t in (x, *(w[n] for n in names))]
    leaves = [t.detach().requires_grad_() for t in args]
    want = torch.autograd.grad(loss(*leaves), leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.func.grad(loss, argnums=(0, 1, 2, 3))(*args), want))
    value, pull = torch.func.vjp(loss, *args)
    assert all(torch.equal(a, b) for a, b in zip(pull(torch.ones_like(value)), want))
    with pytest.raises(RuntimeError, match="no second gradient"):
        torch.func.grad(lambda x: torch.func.grad(loss)(x, *args[1:]).float().sum())(args[0])
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda x: loss(x, *args[1:]), (args[0],), (args[0],))
    q, k = torch.randn(1, 9, 2, D, device=cuda, requires_grad=True), torch.randn(1, 9, 1, D, device=cuda)
    half = lambda q: 0.5 * qk_rope.rope_axes(q, k, inc, torch.arange(9, device=cuda)[None], [D // 2])[0].square().sum()
    first, = torch.autograd.grad(half(q), q, create_graph=True)
    second, = torch.autograd.grad(first, q, torch.ones_like(q))
    assert (second - 1).abs().max() <= 2.0 ** -18 and (first - q).abs().max() <= 2.0 ** -18


def test_results_read_on_a_second_stream(cuda):
    """Launches that begin while the kernel before them drains, back to back, with inputs that the kernel before has just written
    (positions too) and results that another stream copies behind an event: the bits of calls with a wait after each."""
    w, x0, inc, _, _ = case(cuda, False)

    def run(settle, read):
        x, pos, out = x0.clone(), torch.zeros(B, S, dtype=torch.int32, device=cuda), []
        for _ in range(40):
            pos.add_(997)
            settle()
            q, k, v = split_heads(linear_act(x, w["qkv"], w["qkv_bias"]))
            settle()
            q, k = qk_rope.qk_norm_rope(q, k, w["q_norm"], w["k_norm"], inc, positions=pos, pairing="halves")
            settle()
            out += read(q, k)
            x = linear_act(q.flatten(2), w["out"], None, x0)
            settle()
            out += read(x)
        torch.cuda.synchronize()
        return out

    side = torch.cuda.Stream(cuda)

    def aside(*tensors):
        side.wait_event(torch.cuda.current_stream().record_event())
        with torch.cuda.stream(side):
            for t in tensors:
                t.record_stream(side)
            return [t.clone() for t in tensors]

    want = run(torch.cuda.synchronize, lambda *tensors: [t.clone() for t in tensors])
    got = run(lambda: None, aside)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    check_linear_status()
