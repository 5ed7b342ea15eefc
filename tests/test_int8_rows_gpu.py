"""Rows in 8-bit integers: what their first tests leave out."""
import pytest
import torch

from test_int8_gpu import DEV, EPS, ops, plain_rows, rand  # noqa: F401  (ops: the fixture)

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
