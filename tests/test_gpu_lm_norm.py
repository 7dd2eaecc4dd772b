"""GPU: RmsNormQuantLayer against its formula in 64 bits.

Bounds.  u = 2^-24.  A row's sum of squares is one rounding per value of a lane
(32 at most) and one per join of lanes and waves (6 + 15), and its square root
halves the error: 27 u; mean, eps, root, reciprocal, two products and the division
by the top add 8: the scale is within 40 u.  What rounds to 8 bits is y / scale
with 5 more roundings, 127 or 448 at most: int8 within half a step (1 + 1e-4), e4m3
within 2^-4 of its value or half its smallest step, 2^-10, (1 + 1e-4)."""
import pytest
import torch

from onnxsharp_amd.lm_layers import RmsNormQuantLayer

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _make(cuda, rows, cols, dtype, seed):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device=cuda).to(dtype)
    r = (4 * torch.randn(rows, cols, generator=g, device=cuda)).to(dtype)
    return x, r, (1 + 0.2 * torch.randn(cols, generator=g, device=cuda)).to(dtype)


def _check(x, r, gamma, h, q, scale, q_type, eps=1e-5):
    want = x if r is None else (x.float() + r.float()).to(x.dtype)
    assert torch.equal(h, want)
    f = want.double()
    y = f / (f.pow(2).mean(1, keepdim=True) + eps).sqrt() * gamma.double()
    top = 127.0 if q_type == "int8" else 448.0
    s = y.abs().amax(1) / top
    assert ((scale.double() - s).abs() <= 40 * 2.0 ** -24 * s).all()
    v = torch.where(s[:, None] > 0, y / s[:, None], 0.0)
    d = (q.double() - v).abs()
    bound = torch.full_like(v, 0.5) if q_type == "int8" else (v.abs() * 2.0 ** -4).clamp(min=2.0 ** -10)
    assert (d <= bound * (1 + 1e-4)).all(), float((d - bound).max())


@pytest.mark.parametrize("q_type", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (300, 5), (3, 8), (5, 9), (7, 64), (1, 511), (9, 513), (2, 1283), (1, 4096),
                                       (33, 2047), (3, 4100), (17, 8192), (2, 16384), (1, 32768), (2, 30001)])
def test_norm(cuda, rows, cols, dtype, q_type):
    x, r, gamma = _make(cuda, rows, cols, TYPES[dtype], rows * 7 + cols)
    layer = RmsNormQuantLayer(q_type=q_type)
    print(f"norm {rows} x {cols} {dtype} {q_type}", flush=True)
    _check(x, r, gamma, *layer.forward(x, gamma, r), q_type)
    h, q, scale = layer.forward(x, gamma)
    assert h is x
    _check(x, None, gamma, h, q, scale, q_type)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_many_rows(cuda, dtype):
    x, r, gamma = _make(cuda, 70001, 72, TYPES[dtype], 5)
    _check(x, r, gamma, *RmsNormQuantLayer(q_type="int8").forward(x, gamma, r), "int8")


@pytest.mark.parametrize("cols", [40, 1283, 4096])
def test_norm_strided_rows_and_in_place(cuda, cols):
    # rows and gamma inside wider tensors at odd offsets
    wide, r, g = _make(cuda, 6, 2 * cols + 3, torch.bfloat16, 3)
    x, res, gamma = wide[:, 1:cols + 1], r[::2].repeat(2, 1)[:, cols:2 * cols], g[2:cols + 2]
    _check(x, res, gamma, *RmsNormQuantLayer().forward(x, gamma, res), "e4m3")
    before = wide.clone()
    h, q, scale = RmsNormQuantLayer().forward(x, gamma, res, out_h=x)
    assert h is x
    _check(before[:, 1:cols + 1], res, gamma, h, q, scale, "e4m3")
    assert torch.equal(wide[:, 0], before[:, 0]) and torch.equal(wide[:, cols + 1:], before[:, cols + 1:])
    res2 = res.contiguous()
    keep = res2.clone()
    h, q, scale = RmsNormQuantLayer().forward(before[:, 1:cols + 1], gamma, res2, out_h=res2)
    _check(before[:, 1:cols + 1], keep, gamma, res2, q, scale, "e4m3")


@pytest.mark.parametrize("cols", [6, 200, 2000, 9000])
@pytest.mark.parametrize("q_type", ["int8", "e4m3"])
def test_norm_zero_and_nonfinite_rows(cuda, cols, q_type):
    x, r, gamma = _make(cuda, 6, cols, torch.bfloat16, 9)
    x[1], r[1] = 0, 0
    x[2, cols // 2] = float("nan")
    x[3, 0] = float("inf")
    r[4, cols - 1] = -float("inf")
    h, q, scale = RmsNormQuantLayer(q_type=q_type).forward(x, gamma, r)
    assert scale[1] == 0 and (q[1].float() == 0).all()
    assert scale[2:5].isnan().all() and scale[[0, 5]].isfinite().all()
    ok = [0, 5]
    _check(x[ok], r[ok], gamma, h[ok], q[ok], scale[ok], q_type)
    gamma[cols // 3] = float("nan")
    assert RmsNormQuantLayer(q_type=q_type).forward(x, gamma, r)[2][[0, 5]].isnan().all()


def test_norm_no_rows(cuda):
    h, q, scale = RmsNormQuantLayer().forward(torch.empty(0, 64, device=cuda), torch.ones(64, device=cuda))
    assert q.shape == (0, 64) and scale.shape == (0,)


def test_norm_on_a_stream_and_in_a_graph(cuda):
    x, r, gamma = _make(cuda, 5, 1283, torch.float16, 4)
    layer = RmsNormQuantLayer()
    want = layer.forward(x, gamma, r)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        layer.forward(x, gamma, r)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = layer.forward(x, gamma, r)
    torch.cuda.current_stream().wait_stream(st)
    for i in range(3):
        x.mul_(1.25)
        want = layer.forward(x, gamma, r)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a.float(), b.float())
