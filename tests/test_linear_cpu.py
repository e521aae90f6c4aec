"""CPU: the linear layer with its epilogue refuses what does not fit before anything is launched, through the Python surface
and through the C ABI."""
import pytest
import torch

from fast_polynomial_transcendentals_b200.linear import linear_act

BF = torch.bfloat16


def zeros(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("args, kwargs, error, message", [
    ((zeros(4, 16, dtype=torch.float32), zeros(8, 16)), {}, RuntimeError, "float16 or bfloat16"),
    ((zeros(4, 16), zeros(8, 16, dtype=torch.float16)), {}, RuntimeError, "same dtype"),
    ((zeros(4, 16), zeros(8, 24)), {}, RuntimeError, "16 columns, the weight wants 24"),
    ((zeros(4, 16), zeros(2, 8, 16)), {}, RuntimeError, r"\[out, dim\]"),
    ((torch.zeros((), dtype=BF), zeros(8, 16)), {}, RuntimeError, r"\[out, dim\]"),
    ((zeros(4, 12), zeros(8, 12)), {}, RuntimeError, "multiple of 8"),
    ((zeros(4, 0), zeros(8, 0)), {}, RuntimeError, "multiple of 8"),
    ((zeros(4, 16), zeros(0, 16)), {}, RuntimeError, "at least one row"),
    ((zeros(4, 16), zeros(8, 16), zeros(9)), {}, RuntimeError, "8 entries"),
    ((zeros(4, 16), zeros(8, 16), torch.zeros(8, dtype=torch.float64)), {}, RuntimeError, "8 entries"),
    ((zeros(4, 16), zeros(8, 16), None, zeros(1, 8)), {}, RuntimeError, "shape of the result"),
    ((zeros(4, 16), zeros(8, 16), None, zeros(4, 8, dtype=torch.float16)), {}, RuntimeError, "same dtype"),
    ((zeros(4, 16), zeros(8, 16)), dict(activation="relu6"), ValueError, "activation"),
    ((zeros(4, 16), zeros(8, 16)), dict(coeff_source="other"), ValueError, "coeff_source"),
    ((zeros(4, 16), zeros(8, 16)), dict(degree=3), RuntimeError, "degree"),
    ((zeros(4, 16), zeros(8, 16)), dict(activation="gelu", degree=7), RuntimeError, "degree"),
    ((zeros(4, 16, dtype=torch.float16), zeros(8, 16, dtype=torch.float16)), dict(activation="gelu", degree=5, coeff_source="sollya"),
     RuntimeError, "coeff_source=current"),
    ((zeros(4, 16), zeros(8, 16)), {}, RuntimeError, "must be a CUDA tensor"),
])
def test_refusals(args, kwargs, error, message):
    with pytest.raises(error, match=message):
        linear_act(*args, **kwargs)


def test_c_abi_checks_before_launch(fpt):
    lib, p = fpt.load(), 256

    def call(out=p, slope=None, x=p, w=p, b=None, r=None, rows=1, dim=16, n=8, x_ld=16, w_ld=16, out_ld=8, res_ld=8, slope_ld=8, dtype=1,
             bias_dtype=2, function=-1, degree=0, source=0):
        return lib.fpt_linear(out, slope, x, w, b, r, rows, dim, n, x_ld, w_ld, out_ld, res_ld, slope_ld, dtype, bias_dtype, function, degree,
                              source, None, None)

    assert call(rows=-1) == -2 and call(dim=0) == -2 and call(n=0) == -2 and call(rows=1 << 31) == -2
    assert call(dim=12) == -6 and call(dtype=2) == -5 and call(b=p, bias_dtype=3) == -5
    assert call(function=3) == -5 and call(function=5) == -5 and call(source=2) == -5
    assert call(degree=3) == -4 and call(function=4, degree=9) == -4 and call(dtype=0, function=4, degree=5, source=1) == -4
    assert call(x=None) == -1 and call(out=None) == -1
    assert call(x_ld=8) == -2 and call(w_ld=8) == -2 and call(out_ld=7) == -2 and call(r=p, res_ld=7) == -2 and call(slope=p, slope_ld=7, function=4) == -2 and call(slope=p) == -4
    assert call(x=p + 8) == -3 and call(w_ld=20) == -3 and call(out=p + 1) == -3 and call(b=p + 2) == -3
    assert call(rows=0, x=None, out=None) == 0

    def dx(d=p, z=p, w=p, rows=1, dim=16, n=8, dx_ld=16, dz_ld=8, w_ld=16):
        return lib.fpt_linear_grad_input(d, z, w, rows, dim, n, dx_ld, dz_ld, w_ld, 1, None, None)

    assert dx(d=None) == -1 and dx(dx_ld=8) == -2 and dx(dz_ld=4) == -2 and dx(z=p + 2) == -3 and dx(n=9, dz_ld=9) == -3 and dx(rows=0, z=None) == 0

    def dw(d=p, z=p, x=p, rows=1, dim=16, n=8, dw_ld=16, dz_ld=8, x_ld=16):
        return lib.fpt_linear_grad_weight(d, z, x, rows, dim, n, dw_ld, dz_ld, x_ld, 1, None, None)

    assert dw(d=None) == -1 and dw(z=None) == -1 and dw(dw_ld=8) == -2 and dw(x_ld=8) == -2 and dw(x=p + 2) == -3

    def act(dz=p, db=None, dy=p, slope=None, work=None, nbytes=0, rows=1, n=8, dz_ld=8, dy_ld=8, slope_ld=8):
        return lib.fpt_linear_grad_act(dz, db, dy, slope, work, nbytes, rows, n, dz_ld, dy_ld, slope_ld, 1, 2, None)

    assert act(dy=None) == -1 and act(n=9, dy_ld=9, dz_ld=9) == -2 and act(dz=p + 2) == -3 and act(slope=p, slope_ld=12) == -3
    assert act(db=p) == -1 and act(db=p, work=p, nbytes=31) == -9 and act(db=p + 2, work=p, nbytes=32) == -3
    assert lib.fpt_linear_grad_act_workspace_bytes(1, 8) == 32 and lib.fpt_linear_grad_act_workspace_bytes(0, 8) == 0


def test_tuning_keys(fpt):
    lib = fpt.load()
    for key, good, bad in ((b"linear_tokens", (0, 16, 32, 64, 128, -1), (8, 256, -2)), (b"linear_split", (1, 8, 0), (9, -1)),
                           (b"linear_columns", (64, 96, 256, 0), (32, 100, 288, -1))):
        assert all(lib.fpt_set_tuning(key, v) == -2 for v in bad)
        assert all(lib.fpt_set_tuning(key, v) == 0 for v in good)         # the last one is the default
