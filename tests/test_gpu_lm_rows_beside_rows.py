"""GPU: outputs whose rows lie beside an operand's rows in one buffer, as the halves of a wider
tensor do, give what separate tensors give."""
import pytest
import torch

from onnxsharp_amd import native as N
from onnxsharp_amd.lm_layers import QuantMatMulLayer, RmsNormQuantLayer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [5, 200, 4096])
def test_norm_beside_its_rows(cuda, cols):
    wide = torch.randn(9, 3 * cols, device=cuda).bfloat16()
    x, r, out = (wide[:, i * cols:(i + 1) * cols] for i in range(3))
    gamma = torch.randn(cols, device=cuda).bfloat16()
    want = RmsNormQuantLayer().forward(x.clone(), gamma, r.clone())
    keep = wide[:, :2 * cols].clone()
    got = RmsNormQuantLayer().forward(x, gamma, r, out_h=out)
    assert got[0] is out and all(torch.equal(a.float(), b.float()) for a, b in zip(got, want))
    assert torch.equal(wide[:, :2 * cols], keep)
    with pytest.raises(N.OshError, match="overlaps x"):
        RmsNormQuantLayer().forward(x, gamma, r, out_h=wide[:, 1:cols + 1])


@pytest.mark.parametrize("m", [3, 100, 700])
def test_matmul_beside_its_residual(cuda, m):
    n, k = 264, 144
    a, w = (torch.randint(-127, 128, (r, k), device=cuda).to(torch.int8) for r in (m, n))
    sa, sw = torch.rand(m, device=cuda), torch.rand(n, device=cuda)
    wide = torch.randn(m, 2 * n, device=cuda).half()
    out, r = wide[:, :n], wide[:, n:]
    want = QuantMatMulLayer("Relu", torch.float16).forward(a, sa, w, sw, residual=r.clone())
    keep = r.clone()
    got = QuantMatMulLayer("Relu", torch.float16).forward(a, sa, w, sw, residual=r, out=out)
    assert torch.equal(got, want) and torch.equal(wide[:, n:], keep)
    with pytest.raises(N.OshError, match="overlaps"):
        QuantMatMulLayer("Relu", torch.float16).forward(a, sa, w, sw, residual=r, out=wide[:, 1:n + 1])
