"""GPU: the sums of QuantMatMulLayer for operands quantized from normals, into float32.

Bound, in the 2-norm of the result against 64 bits.  Products of 8-bit values are exact
in FP32; a sum of k of them by MFMAs 32 deep rounds k / 32 times, each by at most half a
step, 2^-24, of a partial sum whose square grows evenly to the result's.  Roundings of
either sign: 2^-24 sqrt(k / 64) of the result, 6.7e-7 at k = 8192, and three roundings of
the scaled sum, 2^-24 sqrt(3): below 1e-6 for every k here."""
import pytest
import torch

from onnxsharp_amd.lm_layers import QuantMatMulLayer

pytestmark = pytest.mark.gpu
Q = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def _quantize(v, q):
    t, top = Q[q]
    s = v.abs().amax(1) / top
    v = (v / s[:, None]).clamp(-top, top)
    return (v.round() if q == "int8" else v).to(t), s


# few rows, tiles of both sizes, operands on and off 16 bytes, several tiles a workgroup,
# outputs on and off 16 bytes, k that cuts a k-block
@pytest.mark.parametrize("q", Q)
@pytest.mark.parametrize("m,n,k", [(1, 768, 64), (5, 300, 512), (16, 512, 8192), (24, 8200, 1040), (40, 200, 2048),
                                   (64, 8192, 128), (100, 200, 1283), (300, 500, 8192), (2100, 2048, 512),
                                   (2100, 2050, 528), (2048, 3000, 65), (4100, 4104, 1024), (4099, 4101, 4096)])
def test_matmul_sums_into_float32(cuda, m, n, k, q):
    g = torch.Generator(device=cuda).manual_seed(m + n + k)
    a, sa = _quantize(torch.randn(m, k, generator=g, device=cuda), q)
    w, sw = _quantize(torch.randn(n, k, generator=g, device=cuda) / k ** 0.5, q)
    print(f"matmul sums {m} x {n} x {k} {q}", flush=True)
    y = QuantMatMulLayer(None, torch.float32).forward(a, sa, w, sw)
    want = (a.double() * sa.double()[:, None]) @ (w.double() * sw.double()[:, None]).t().contiguous()
    err = float((y.double() - want).norm() / want.norm())
    assert err < 1e-6, err


def test_matmul_every_e4m3_value(cuda):
    # every code times one, NaN too, through each kernel
    codes = torch.arange(256, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
    one = lambda r: torch.ones(r, device=cuda)  # noqa: E731
    for m, n in ((3, 256), (100, 256), (2100, 2048)):
        a = torch.zeros(m, 144, device=cuda)
        a[:, 77] = 1.0
        w = torch.zeros(n, 144, device=cuda).to(torch.float8_e4m3fn)
        w[:, 77] = codes.repeat(n // 256)
        y = QuantMatMulLayer(None, torch.float32).forward(a.to(torch.float8_e4m3fn), one(m), w, one(n))
        want = codes.float().repeat(n // 256).expand(m, n)
        assert torch.equal(y.nan_to_num(nan=1000.0), want.nan_to_num(nan=1000.0))
