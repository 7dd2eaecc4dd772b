"""GPU: Int4Weight and Int4MatMulLayer against their formula in 64 bits.

Bounds.  u = 2^-24.  Codes, zero points and the pieces of the rows are exact in the matrix
instructions' operands, so what is off are FP32 sums of a (c - z) s, computed as sum a c -
z sum a.  A value passes through the sum of its group (at most 128 of it at a time, a
rounding each at worst, in both sums), the product with z, the scaling, one addition a
group of a wave and one a wave: at most 2 * 128 + 4 k / 32 / 8 + 16 roundings of what adds up
to no more than S = sum |a| (c + z) s.  For k up to 8192 that is 400 u S.  Bias, residual
and activation (1.13 is the largest slope of GELU, 1.1 of SiLU) add 4 u of their sizes; for
16-bit outputs GELU is 8e-8 off.  The result is rounded once."""
import math

import pytest
import torch

from onnxsharp_amd import native as N
from onnxsharp_amd.lm_layers import Int4MatMulLayer, Int4Weight

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def _two(c):
    c = torch.nn.functional.pad(c, (0, c.shape[1] % 2))
    return (c[:, 0::2] | c[:, 1::2] << 4).contiguous()


def make(cuda, m, n, k, group, zeros, dtype, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed + m + 3 * n + 7 * k + group)
    groups = -(-k // group)
    t = dict(k=k, group=group)
    t["x"] = torch.randn(m, k, generator=g, device=cuda).to(dtype)
    t["codes"] = torch.randint(0, 16, (n, k), generator=g, device=cuda, dtype=torch.uint8)
    t["scales"] = ((0.5 + torch.rand(n, groups, generator=g, device=cuda)) / math.sqrt(20 * k)).to(dtype)
    t["zeros"] = torch.randint(0, 16, (n, groups), generator=g, device=cuda, dtype=torch.uint8) if zeros else None
    t["bias"] = torch.randn(n, generator=g, device=cuda)
    t["res"] = torch.randn(m, n, generator=g, device=cuda).to(dtype)
    return t


def weight(t):
    return Int4Weight(_two(t["codes"]), t["scales"], None if t["zeros"] is None else _two(t["zeros"]), k=t["k"],
                      group=t["group"])


def check(t, y, act=None, bias=None, res=None):
    at = torch.arange(t["k"], device=y.device) // t["group"]
    z = t["zeros"].double()[:, at] if t["zeros"] is not None else 8.0
    s, c, x = t["scales"].double()[:, at], t["codes"].double(), t["x"].double()
    want = x @ ((c - z) * s).T
    size = 400 * U * (x.abs() @ ((c + z) * s.abs()).T)
    if bias is not None:
        want, size = want + bias.double(), size + 4 * U * bias.abs().double()
    if act == "Relu":
        want = want.clamp(min=0)
    elif act == "Silu":
        want = want * torch.sigmoid(want)
    elif act == "Gelu":
        want = want * 0.5 * torch.erfc(-want / math.sqrt(2.0))
    size = 1.13 * size + 4 * U * want.abs() + (8e-8 if act == "Gelu" else 0.0)
    if res is not None:
        want = want + res.double()
    half = torch.finfo(y.dtype).eps / 2
    bound = size + half * want.abs() * (1 + 1e-6) + (2.0 ** -25 if y.dtype == torch.float16 else 0.0)
    d = (y.double() - want).abs()
    assert (d <= bound).all(), (float((d - bound).max()), int((d > bound).sum()))


SIZES = [(1, 1, 1), (1, 16, 32), (1, 15, 33), (2, 17, 127), (3, 70, 129), (16, 48, 256), (17, 33, 300), (32, 64, 640),
         (33, 100, 257), (64, 96, 1024), (65, 130, 384), (130, 257, 513), (300, 200, 1283)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_int4_matmul(cuda, m, n, k, group, dtype):
    print(f"int4 {m} x {n} x {k} groups of {group} {dtype}", flush=True)
    for zeros in (False, True):
        t = make(cuda, m, n, k, group, zeros, TYPES[dtype])
        check(t, Int4MatMulLayer().forward(t["x"], weight(t)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("m,n,k", [(4101, 2055, 300), (2050, 4200, 264)])
def test_many_rows(cuda, m, n, k, group, dtype):
    print(f"int4 {m} x {n} x {k} groups of {group} {dtype}", flush=True)
    for zeros in (False, True):
        t = make(cuda, m, n, k, group, zeros, TYPES[dtype])
        check(t, Int4MatMulLayer("Silu").forward(t["x"], weight(t), t["bias"], t["res"]), "Silu", t["bias"], t["res"])


@pytest.mark.parametrize("act", [None, "Relu", "Silu", "Gelu"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 768, 768), (24, 500, 4096), (200, 512, 1024), (129, 131, 200)])
def test_epilogue(cuda, m, n, k, dtype, act):
    t = make(cuda, m, n, k, 64, True, TYPES[dtype])
    w, layer = weight(t), Int4MatMulLayer(act)
    print(f"int4 {m} x {n} x {k} {dtype} {act}", flush=True)
    check(t, layer.forward(t["x"], w, t["bias"], t["res"]), act, t["bias"], t["res"])
    check(t, layer.forward(t["x"], w, t["bias"]), act, t["bias"])
    out = t["res"].clone()
    y = layer.forward(t["x"], w, None, out, out=out)
    assert y is out
    check(t, y, act, None, t["res"])


@pytest.mark.parametrize("m", [1, 40, 150])
@pytest.mark.parametrize("dtype", TYPES)
def test_strides(cuda, m, dtype):
    # rows, residual and output inside wider tensors at odd offsets
    dt = TYPES[dtype]
    t = make(cuda, m, 77, 300, 32, True, dt)
    wide = torch.randn(m, 303, device=cuda).to(dt)
    wide[:, 1:301] = t["x"]
    out, res = torch.full((m, 81), 7.0, device=cuda, dtype=dt), torch.randn(m, 99, device=cuda).to(dt)
    y = Int4MatMulLayer().forward(wide[:, 1:301], weight(t), None, res[:, 5:82], out=out[:, 3:80])
    check(t, y, None, None, res[:, 5:82])
    assert (out[:, :3] == 7).all() and (out[:, 80:] == 7).all()


def test_weights_inside_wider_tensors(cuda):
    t = make(cuda, 5, 40, 200, 64, True, torch.bfloat16)
    codes, scales, zeros = _two(t["codes"]), t["scales"], _two(t["zeros"])
    pad = lambda a: torch.cat((a, a[:, :3], a), 1)[:, a.shape[1] + min(3, a.shape[1]):]  # noqa: E731
    w = Int4Weight(pad(codes), pad(scales), pad(zeros), k=200, group=64)
    check(t, Int4MatMulLayer().forward(t["x"], w))


@pytest.mark.parametrize("m", [1, 70])
def test_rows_of_float32_keep_their_24_bits(cuda, m):
    # values of very different size in one row, whose differences small codes pick out
    t = make(cuda, m, 64, 256, 128, False, torch.float32)
    t["x"] *= 10.0 ** (torch.arange(256, device=cuda) % 7 - 3)
    check(t, Int4MatMulLayer().forward(t["x"], weight(t)))
    # one code apart: y is x[5] itself, all 24 bits of it
    t["codes"][:] = 8
    t["codes"][:, 5] = 9
    t["scales"][:] = 1
    y = Int4MatMulLayer().forward(t["x"], weight(t)).double()
    assert ((y - t["x"][:, 5:6].double()).abs() <= 400 * U * 17 * t["x"].double().abs().sum(1, keepdim=True)).all()
    t["x"][:] = 0
    t["x"][:, 5] = 1 + 2.0 ** -23
    assert (Int4MatMulLayer().forward(t["x"], weight(t)) == 1 + 2.0 ** -23).all()


@pytest.mark.parametrize("m", [3, 70, 300])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_scales_of_any_size(cuda, m, group, dtype):
    # zeros, the type's smallest numbers, signs, and neighbours many powers of two apart
    dt = TYPES[dtype]
    t = make(cuda, m, 200, 1280, group, True, dt)
    torch.manual_seed(m + group)
    lo, hi = (-24, 3) if dtype == "f16" else (-100, 30)
    e = torch.randint(lo, hi, t["scales"].shape, device=cuda).float()
    t["scales"] = (torch.exp2(e) * (1 + torch.rand_like(e)) * torch.where(torch.rand_like(e) < 0.3, -1.0, 1.0)).to(dt)
    t["scales"][torch.rand_like(e) < 0.2] = 0
    t["scales"][:20] = 0
    t["scales"][20:40, 1:] = 0
    t["x"] *= 0.01
    y = Int4MatMulLayer().forward(t["x"], weight(t))
    check(t, y)
    assert (y[:, :20] == 0).all()


@pytest.mark.parametrize("m", [3, 70])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_are_not_finite(cuda, m, dtype):
    t = make(cuda, m, 40, 130, 32, False, TYPES[dtype])
    good = Int4MatMulLayer().forward(t["x"], weight(t))
    t["x"][1, 3], t["x"][2, 129] = float("nan"), float("inf")
    y = Int4MatMulLayer().forward(t["x"], weight(t))
    assert not y[1:3].isfinite().any()
    rest = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(y[rest], good[rest])


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 128])
def test_quantize(cuda, group, zeros):
    g = torch.Generator(device=cuda).manual_seed(1)
    wf = torch.randn(50, 300, generator=g, device=cuda)
    wf[3, :group] = 0
    w = Int4Weight.quantize(wf, group, zeros, torch.float32)
    got = Int4MatMulLayer().forward(torch.eye(300, device=cuda), w).T
    full = torch.nn.functional.pad(wf, (0, -300 % group)).reshape(50, -1, group)
    step = ((full.amax(2).clamp(min=0) - full.amin(2).clamp(max=0)) / 15 if zeros else full.abs().amax(2) / 7)
    # a zero point is rounded too: at the ends of a group another half step
    bound = (1.0 if zeros else 0.5) * step.repeat_interleave(group, 1)[:, :300] * (1 + 1e-5) + 1e-6
    assert ((got - wf).abs() <= bound).all()
    assert (got[3, :group] == 0).all()


def test_empty(cuda):
    t = make(cuda, 4, 8, 64, 32, False, torch.bfloat16)
    assert Int4MatMulLayer().forward(t["x"][:0], weight(t)).shape == (0, 8)
    w = Int4Weight(torch.zeros(0, 32, dtype=torch.uint8, device=cuda), torch.zeros(0, 2, device=cuda), k=64, group=32)
    assert Int4MatMulLayer().forward(torch.zeros(3, 64, device=cuda), w).shape == (3, 0)


@pytest.mark.parametrize("m,dtype", [(1, "bf16"), (100, "f32"), (200, "f16")])
def test_captured_and_other_streams(cuda, m, dtype):
    t = make(cuda, m, 256, 512, 64, True, TYPES[dtype])
    w, layer = weight(t), Int4MatMulLayer("Silu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = layer.forward(t["x"], w, t["bias"])
    s.synchronize()
    check(t, y, "Silu", t["bias"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer.forward(t["x"], w, t["bias"])
    for _ in range(3):
        t["x"].normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, layer.forward(t["x"], w, t["bias"]))
