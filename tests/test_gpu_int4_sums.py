"""GPU: the sums of Int4MatMulLayer for rows whose mean is not 0, where a sum of codes and its zero
points' part cancel.

Bound, in the 2-norm of the result's error over n outputs of a row.  Products of codes and 16-bit
values are exact.  A sum runs group by group: a group's codes and its zero points' part, then the
next group, so that no partial sum is larger than the result so far (its square grows evenly to
R^2, or R as a whole at the start) and one group's two parts, at most G = max over groups of
sum |a| max(c, z) s.  Matrix instructions 16 deep round k / 16 + groups times, by at most half a
step, 2^-24 of that; from group to group a sum is brought to the next one's scale, in two factors,
2^-23 of it each.  Of either sign: 2^-24 sqrt(k / 16 + 9 groups) (R + G).  With all of k between the two
parts G would be `groups` times as large.

The result is seen through its residual, the negative of its own rounding: what is left has half
a step of its own size, eps / 2 (and of f16's subnormal numbers 2^-25)."""
import math

import pytest
import torch

from onnxsharp_amd.lm_layers import Int4MatMulLayer
from test_gpu_int4_matmul import make, weight

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# a token, few rows, large and small tiles, with k that ends inside a group
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, False), (128, True), (256, True)])
@pytest.mark.parametrize("m,n,k", [(1, 400, 8192), (40, 300, 4096), (70, 16384, 8192), (300, 4200, 4096), (2100, 2049, 4100)])
@pytest.mark.parametrize("rows", ["positive", "silu"])
def test_rows_that_do_not_average_zero(cuda, m, n, k, group, zeros, dtype, rows):
    print(f"int4 sums {m} x {n} x {k} groups of {group} {dtype} {rows}", flush=True)
    dt = TYPES[dtype]
    t = make(cuda, m, n, k, group, zeros, dt)
    t["x"] = (torch.rand_like(t["x"].float()) if rows == "positive" else torch.nn.functional.silu(t["x"].float())).to(dt)
    # codes about their zero point
    t["scales"] = (0.5 + torch.rand_like(t["scales"].float())).to(dt)
    at = torch.arange(k, device=cuda) // group
    z = t["zeros"][:, at] if zeros else torch.full_like(t["codes"], 8)
    step = torch.randint(-7, 8, z.shape, device=cuda)
    t["codes"] = (z.int() + step).clamp(0, 15).to(torch.uint8)
    s = t["scales"].double()[:, at]
    c, z, x = t["codes"].double(), z.double(), t["x"].double()
    want = x @ ((c - z) * s).T
    groups = -(-k // group)
    each = torch.maximum(c, z) * s
    most = torch.zeros_like(want)
    for e in range(groups):
        a, b = e * group, min(k, (e + 1) * group)
        most = torch.maximum(most, x[:, a:b].abs() @ each[:, a:b].T.contiguous())
    res = (-want).to(dt)
    got = Int4MatMulLayer().forward(t["x"], weight(t), None, res).double()
    left = want + res.double()
    norm = lambda v: float(v.pow(2).mean().sqrt())  # noqa: E731
    bound = 2.0 ** -24 * math.sqrt(k / 16 + 9 * groups) * (norm(want) + norm(most))
    bound += torch.finfo(dt).eps / 2 * (norm(left) + bound) + (2.0 ** -25 if dt == torch.float16 else 0.0)
    err = norm(got - left)
    print(f"   {err:.3e} of {bound:.3e}, result {norm(want):.3e}", flush=True)
    assert err <= bound
