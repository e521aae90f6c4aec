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
