"""CPU: which feed-forward modules the epilogue adapter takes, and that what it takes behaves as before off the GPU."""
import pytest
import torch
from torch import nn

from fast_polynomial_transcendentals_b200.sfu_repro import adapters


class Mlp(nn.Module):
    def __init__(self, act=None, dropout=None, names=("fc1", "fc2")):
        super().__init__()
        setattr(self, names[0], nn.Linear(16, 32))
        setattr(self, names[1], nn.Linear(32, 16))
        self.names = names
        self.activation_fn = act if act is not None else nn.GELU()
        if dropout is not None:
            self.dropout = nn.Dropout(dropout)

    def forward(self, x):
        return getattr(self, self.names[1])(self.activation_fn(getattr(self, self.names[0])(x)))


class Gated(nn.Module):
    def __init__(self):
        super().__init__()
        self.gate_proj, self.up_proj, self.down_proj = nn.Linear(16, 32), nn.Linear(16, 32), nn.Linear(32, 16)
        self.act_fn = nn.SiLU()


def test_takes_what_it_should_and_reports_the_rest():
    model = nn.ModuleDict({"gelu": Mlp(), "silu": Mlp(nn.SiLU()), "function": Mlp(torch.nn.functional.gelu), "named": Mlp(names=("c_fc", "c_proj")),
                           "no_dropout": Mlp(dropout=0.0), "dropout": Mlp(dropout=0.1), "tanh": Mlp(nn.GELU(approximate="tanh")),
                           "relu": Mlp(nn.ReLU()), "gated": Gated()})
    skipped = []
    assert adapters.patch_mlp_epilogues(model, skipped=skipped) == 5
    assert sorted(n for n, _ in skipped) == ["dropout", "relu", "tanh"]
    assert "forward" not in model["gated"].__dict__ and "forward" in model["gelu"].__dict__


def test_own_forward_off_the_gpu_and_restore():
    model = Mlp()
    x = torch.randn(3, 16)
    want = model(x)
    assert adapters.patch_mlp_epilogues(model) == 1 and adapters.patch_mlp_epilogues(model) == 1       # twice is once
    assert torch.equal(model(x), want)
    assert adapters.restore(model) == 1 and "forward" not in model.__dict__ and torch.equal(model(x), want)


def test_own_parameters_keep_a_module_as_it_is():
    model = Mlp()
    model.scale = nn.Parameter(torch.ones(16))
    skipped = []
    assert adapters.patch_mlp_epilogues(model, skipped=skipped) == 0
    assert skipped == [("", "also holds scale")]


def test_hooks_and_forwards_of_the_projections_are_seen():
    class Scaled(nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    plain, hooked, scaled, bound = Mlp(), Mlp(), Mlp(), Mlp()
    hooked.fc1.register_forward_hook(lambda module, args, out: 2 * out)
    scaled.fc2 = Scaled(32, 16)
    bound.fc1.forward = lambda x: x
    assert adapters._as_it_comes(plain.fc1, plain.fc2, plain.activation_fn)
    for model in (hooked, scaled, bound):
        assert not adapters._as_it_comes(model.fc1, model.fc2, model.activation_fn)


@pytest.fixture
def as_on_the_gpu(monkeypatch):
    """The adapter's own path on the CPU: it takes every input, and the layer is its plain form."""
    def plain(x, weight, bias=None, *, activation="none", degree=0, coeff_source="current"):
        return {"none": lambda z: z, "gelu": nn.functional.gelu, "silu": nn.functional.silu}[activation](nn.functional.linear(x, weight, bias))
    monkeypatch.setattr(adapters, "_epilogue_input", lambda x: True)
    monkeypatch.setattr(adapters, "linear_act", plain)


def test_further_arguments_are_not_dropped(as_on_the_gpu):
    class Optional(Mlp):
        def forward(self, x, residual=None):
            y = super().forward(x)
            return y if residual is None else y + residual

    model, x, r = Optional(), torch.randn(3, 16), torch.randn(3, 16)
    want = model(x), model(x, r), model(x, residual=r)
    assert adapters.patch_mlp_epilogues(model) == 1
    assert all(torch.equal(a, b) for a, b in zip(want, (model(x), model(x, r), model(x, residual=r))))


class WithResidual(Mlp):
    def forward(self, x, residual):
        return super().forward(x) + residual


class AddsItsInput(Mlp):
    def forward(self, x):
        y = super().forward(x)
        y += x
        return y


class ActivatesTwice(Mlp):
    def forward(self, x):
        return self.activation_fn(super().forward(x))


class DropsBetween(Mlp):
    def __init__(self, p=0.1):
        super().__init__()
        self.p = p

    def forward(self, x):
        hidden = nn.functional.dropout(self.activation_fn(self.fc1(x)), p=self.p, training=self.training)
        return self.fc2(hidden)


class DropsInPlace(DropsBetween):
    def forward(self, x):
        y = self.fc2(self.activation_fn(self.fc1(x)))
        return nn.functional.dropout(y, p=self.p, training=self.training, inplace=True)


class GatedInside(Mlp):
    def __init__(self):
        super().__init__()
        self.fc1 = nn.Linear(16, 64)

    def forward(self, x):
        hidden, gate = self.fc1(x).chunk(2, dim=-1)
        return self.fc2(self.activation_fn(gate) * hidden)


class GatedByItself(Mlp):
    def forward(self, x):
        hidden = self.fc1(x)
        return self.fc2(self.activation_fn(hidden) * hidden)


class SkipsItsActivation(Mlp):
    def forward(self, x):
        return self.fc2(self.fc1(x))


class WithABias(Mlp):
    def forward(self, x):
        return super().forward(x), self.fc2.bias


class ByItsWeights(Mlp):
    def forward(self, x):
        return self.fc2(self.activation_fn(nn.functional.linear(x, 2 * self.fc1.weight, self.fc1.bias)))


@pytest.mark.parametrize("kind", [WithResidual, AddsItsInput, ActivatesTwice, DropsBetween, DropsInPlace, GatedInside, GatedByItself,
                                  SkipsItsActivation, WithABias, ByItsWeights])
def test_forwards_that_do_more_are_left_alone(kind):
    model, skipped = kind(), []
    state = torch.random.get_rng_state()
    assert adapters.patch_mlp_epilogues(model, skipped=skipped) == 0 and [n for n, _ in skipped] == [""]
    assert "forward" not in model.__dict__ and model.training and isinstance(model.fc1, nn.Linear)
    assert torch.equal(state, torch.random.get_rng_state())


def test_a_forward_set_on_the_module_is_left_alone():
    model, skipped = Mlp(), []
    model.forward = lambda x: 2 * x
    assert adapters.patch_mlp_epilogues(model, skipped=skipped) == 0 and skipped == [("", "a forward of its own")]


def test_a_dropout_that_begins_to_drop_is_not_lost(as_on_the_gpu):
    for model, change in ((DropsBetween(0.0), lambda m: setattr(m, "p", 0.9)), (Mlp(dropout=0.0), lambda m: setattr(m.dropout, "p", 0.9))):
        calls = []
        assert adapters.patch_mlp_epilogues(model) == 1
        original = model.__dict__[adapters._ORIGINAL]
        model.__dict__[adapters._ORIGINAL] = lambda x: calls.append(1) or original(x)
        model(torch.randn(3, 16))
        assert not calls                        # the fused path
        change(model)
        model(torch.randn(3, 16))
        assert calls == [1]


def test_a_module_that_cannot_be_copied_is_left_alone():
    class Alone(Mlp):
        def __copy__(self):
            raise TypeError("there is one of it")

    model, skipped = Alone(), []
    assert adapters.patch_mlp_epilogues(model, skipped=skipped) == 0 and "there is one of it" in skipped[0][1]
