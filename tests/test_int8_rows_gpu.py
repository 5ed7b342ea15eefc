"""Rows in 8-bit integers: what their first tests leave out."""
import pytest
import torch

from test_int8_gpu import DEV, EPS, holds, ops, plain_rows, rand  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


def test_more_rows_than_a_launch_has_threads_for(ops):
    """A workgroup of 64 threads a row: 2^26 rows are 2^32 threads, which a launch takes modulo 2^32."""
    rows = 2 ** 26 + 64
    x = rand(rows, 1, seed=1)
    picked = torch.tensor([0, 1, 63, 64, 65, 2 ** 25, 2 ** 26 - 1, 2 ** 26, 2 ** 26 + 63], device=DEV)
    values, scales = plain_rows(x[picked])
    for operator in ("quantize", "norm", "norm, chosen"):
        out = ops.int8_rows(rows, 1, DEV)
        out.values[picked], out.scales[picked] = 55, -1.0
        if operator == "quantize":
            ops.quantize_int8(x, out)
            assert torch.equal(out.scales[picked], scales)
            back = torch.empty(rows, 1, device=DEV)
            back[picked] = -1.0
            ops.dequantize_int8(out, back)
            assert torch.equal(back[picked], values * scales[:, None])
        elif operator == "norm":
            added = x.clone()
            ops.rmsnorm_int8(added, torch.ones(1, device=DEV), EPS, out, delta=x)
            assert torch.equal(added, x + x)
            assert bool((out.scales[picked] > 0).all())
        else:
            index = torch.arange(rows - 1, -1, -1, dtype=torch.int32, device=DEV)
            ops.rmsnorm_int8(x, torch.ones(1, device=DEV), EPS, out, rows=index)
            values = values.flip(0)                             # (the picked rows are those from the other end then, in the other order)
            values, _ = plain_rows(x[rows - 1 - picked])
            assert bool((out.scales[picked] > 0).all())
        assert torch.equal(out.values[picked, :1].float(), values) and not out.values[picked, 1:].any()
        del out


# rows whose squares overflow float32 (whole rows, a single element, sums only) and, without an eps to speak of, vanish in it; one row in two is an ordinary one
@pytest.mark.parametrize("k", [1, 3, 520, 4096, 16390, 33003])
@pytest.mark.parametrize("eps", [EPS, 0.0, 1e-36])
def test_norm_of_rows_whose_squares_do_not_fit_float32(ops, k, eps):
    x, weight = rand(16, k, seed=1).clamp(-4.0, 4.0), rand(k, seed=2, scale=0.2) + 1.0
    x[:, 0] = 1.0
    x[0] *= 1e18
    x[2] *= 1e19
    x[4] *= 8e37
    x[6, 0] = 3.4e38
    x[8] = 3.4028234e38
    if eps < 1e-30:
        x[10] *= 1e-18
        x[12] *= 1e-30
        x[14] *= 1e-41                                          # denormal
    y = x.double() / torch.sqrt((x.double() ** 2).mean(1, keepdim=True) + eps) * weight.double()
    out, alone = ops.int8_rows(16, k, DEV), ops.int8_rows(1, k, DEV)
    before = x.clone()
    ops.rmsnorm_int8(x, weight, eps, out)
    assert torch.equal(x, before)
    holds(out, y, 16, k)
    added = torch.zeros(1, k, device=DEV)
    ops.rmsnorm_int8(added, weight, eps, alone, delta=before[4:5].contiguous())
    assert torch.equal(alone.values, out.values[4:5]) and torch.equal(alone.scales, out.scales[4:5]) and torch.equal(added, before[4:5])


def test_norm_of_huge_rows_that_hold_an_infinity_or_a_nan(ops):
    x = rand(4, 300, seed=1).abs() * 1e30 + 1e30
    x[1, 5], x[2, 6] = float("inf"), float("nan")
    x[3] = 0.0
    for eps in (EPS, 0.0):
        out = ops.int8_rows(4, 300, DEV)
        ops.rmsnorm_int8(x, torch.ones(300, device=DEV), eps, out)
        assert bool(torch.isnan(out.scales[1:3]).all()) and not out.values[1:].any() and bool(out.scales[0] > 0)
        assert bool(out.scales[3] == 0) if eps > 0 else bool(torch.isnan(out.scales[3]))      # (without an eps: zero by zero)


def test_norm_of_rows_chosen_of_none(ops):
    x, out = rand(0, 300), ops.int8_rows(3, 300, DEV)
    out.values.fill_(55)
    ops.rmsnorm_int8(x, torch.ones(300, device=DEV), EPS, out, rows=torch.tensor([0, -1, 7], dtype=torch.int32, device=DEV))
    assert bool(torch.isnan(out.scales).all()) and not out.values.any()
