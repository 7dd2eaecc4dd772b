"""GPU: QuantMatMulLayer's activations over their arguments, against 64 bits.

The product is 0 and the bias the argument, so that it is exact.  u = 2^-24.
GELU into float32: z = x / sqrt 2 is 2 u off, which moves erfc(z) by (2 z^2 + 1) 2 u of
itself; erfcf is within 16 steps, 32 u, and two products add 2: (2 x^2 + 36) u.
SiLU: x log2 e is 2 u off, moving the exponential by 2 |x| u; exponential, sum, quotient
or reciprocal and product add 2 u each at most: (2 |x| + 8) u.
GELU into 16 bits: its fit is within 5e-4 of its value down to -8 and 2.5e-3 below.
Outputs add half a step of their type; below the normal numbers it is half a step of
those there, and |x| times the smallest normal one where a factor was subnormal."""
import pytest
import torch

from onnxsharp_amd.lm_layers import QuantMatMulLayer

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _run(cuda, act, dtype, x, m):
    n = len(x)
    a, w = torch.zeros(m, 16, dtype=torch.int8, device=cuda), torch.zeros(n, 16, dtype=torch.int8, device=cuda)
    y = QuantMatMulLayer(act, dtype).forward(a, torch.ones(m, device=cuda), w, torch.ones(n, device=cuda), x)
    assert torch.equal(y.nan_to_num(nan=7.0), y[:1].expand(m, n).nan_to_num(nan=7.0))
    return y[0]


# rows of the few-row kernel, tiles of 64 and of 128 fed both ways
@pytest.mark.parametrize("m", [1, 100, 2100])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ["Gelu", "Silu"])
def test_activation_over_its_arguments(cuda, act, dtype, m):
    x = torch.linspace(-13.0, 13.0, 2040, device=cuda)
    x = torch.cat([x, torch.tensor([0.0, -0.0, 1e-30, -1e-30, -40.0, 40.0, -80.0, 80.0], device=cuda)])
    y, d = _run(cuda, act, dtype, x, m).double(), x.double()
    fi = torch.finfo(dtype)
    if act == "Gelu":
        want = d * 0.5 * torch.erfc(-d * 0.5 ** 0.5)
        rel = (2 * d * d + 36) * U if dtype == torch.float32 else torch.where(d > -8, 5e-4, 2.5e-3)
    else:
        want = d * torch.sigmoid(d)
        rel = (2 * d.abs() + 8) * U
    bound = (fi.eps / 2 + rel) * want.abs() + fi.smallest_normal * fi.eps / 2 + d.abs().clamp(max=1e3) * 2.0 ** -126
    err = (y - want).abs()
    assert (err <= bound).all(), (float(x[(err - bound).argmax()]), float((err - bound).max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ["Gelu", "Silu", "Relu"])
def test_activation_at_large_arguments(cuda, act, dtype):
    inf = float("inf")
    x = torch.tensor([3e38, 6e4, -6e4, -3e38, inf, float("nan"), -inf, 1.0], device=cuda)
    for m in (3, 100):
        y = _run(cuda, act, dtype, x, m)
        assert torch.equal(y[:2], x[:2].to(dtype)) and (y[2:4] == 0).all() and y[4] == inf and y[5].isnan()
        if act != "Silu":  # x sigmoid(x) has no value at -infinity
            assert y[6] == 0
        assert torch.isfinite(y[7])
