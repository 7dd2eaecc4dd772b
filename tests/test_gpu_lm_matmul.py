"""GPU: QuantMatMulLayer against its formula in 64 bits.

Operands are whole numbers in both types (e4m3 holds those up to 16), so every sum is
exact in FP32 and in int32 and the epilogue alone rounds.  Bounds, u = 2^-24: the
scaled sum takes 3 roundings, bias, residual 1 each, an activation's exponential or
erf at most 16 u of its result where its argument stays below 16 (|x| u for the
product with log2 e, 4 u for the functions): 2^-19 of |scaled sum| + |bias| + |res|.
The output adds half a step of its type.  One test takes arbitrary e4m3 values: each
of the k additions then rounds by at most 2 u of the sum of magnitudes."""
import pytest
import torch

from onnxsharp_amd.lm_layers import QuantMatMulLayer

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
Q = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _make(cuda, m, n, k, q, dtype, seed, bias=True, res=True):
    g = torch.Generator(device=cuda).manual_seed(seed)
    top = 127 if q == "int8" else 16
    whole = lambda r: torch.randint(-top, top + 1, (r, k), generator=g, device=cuda).float().to(Q[q])  # noqa: E731
    t = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    scale = 3.0 / (top * k ** 0.5)
    return dict(a=whole(m), a_scale=scale * (0.5 + t(m).abs()), w=whole(n), w_scale=(0.5 + t(n).abs()) / top,
                bias=t(n) if bias else None, residual=t(m, n).to(TYPES[dtype]) if res else None)


def _ref(s, act):
    y = (s["a"].double() @ s["w"].double().t().contiguous()) * s["a_scale"].double()[:, None] * s["w_scale"].double()
    size = y.abs()
    if s["bias"] is not None:
        y = y + s["bias"].double()
        size = size + s["bias"].double().abs()
    if act == "Relu":
        y = y.clamp(min=0)
    elif act == "Silu":
        y = y * torch.sigmoid(y)
    elif act == "Gelu":
        y = y * 0.5 * torch.erfc(-y * 0.5 ** 0.5)
    if s["residual"] is not None:
        y = y + s["residual"].double()
        size = size + s["residual"].double().abs()
    return y, size


def _check(out, s, act, dtype, extra=0.0):
    y, size = _ref(s, act)
    t = TYPES[dtype]
    assert out.dtype == t and out.shape == y.shape
    # the smallest normal's step bounds the rounding near zero
    bound = torch.finfo(t).eps / 2 * y.abs() + (2.0 ** -19 + extra) * size + torch.finfo(t).smallest_normal
    d = (out.double() - y).abs()
    assert (d <= bound).all(), float((d - bound).max())


# rows at the borders of the few-row kernels and the tiles; k inside, at and past a
# 128-byte block; odd pitches
SIZES = [(1, 1, 1), (1, 768, 768), (2, 17, 127), (16, 33, 128), (17, 64, 129), (24, 130, 1000), (32, 48, 256), (33, 65, 64),
         (64, 64, 640), (65, 300, 383), (100, 129, 16), (129, 257, 144), (200, 96, 1283), (257, 511, 384), (700, 900, 272)]


@pytest.mark.parametrize("q", Q)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul(cuda, m, n, k, dtype, q):
    print(f"matmul {m} x {n} x {k} {q} {dtype}", flush=True)
    acts = [None, "Relu", "Silu", "Gelu"]
    for i, (bias, res) in enumerate([(True, True), (False, True), (True, False), (False, False)]):
        act = acts[(i + m + n + k) % 4]
        s = _make(cuda, m, n, k, q, dtype, m + 3 * n + 5 * k, bias, res)
        _check(QuantMatMulLayer(act, TYPES[dtype]).forward(**s), s, act, dtype)


@pytest.mark.parametrize("q", Q)
@pytest.mark.parametrize("m,n,k", [(2100, 2048, 512), (4000, 1100, 400), (5, 9001, 2048), (48, 5000, 4096), (300, 4096, 1027),
                                   (2048, 3000, 65)])
def test_matmul_large(cuda, m, n, k, q):
    s = _make(cuda, m, n, k, q, "bf16", 11)
    _check(QuantMatMulLayer("Gelu", torch.bfloat16).forward(**s), s, "Gelu", "bf16")


@pytest.mark.parametrize("q", Q)
@pytest.mark.parametrize("m,n,k,dtype", [(4100, 4104, 272, "bf16"), (4099, 4101, 384, "f16"), (4100, 4112, 256, "f32"),
                                         (2100, 2056, 144, "f32"), (1500, 3333, 1040, "bf16")])
def test_matmul_several_tiles_a_workgroup(cuda, m, n, k, dtype, q):
    # more tiles than a launch holds at once, cut rows, columns and k-blocks
    for act, bias, res in ((None, False, True), ("Gelu", True, False)):
        s = _make(cuda, m, n, k, q, dtype, m + n, bias, res)
        _check(QuantMatMulLayer(act, TYPES[dtype]).forward(**s), s, act, dtype)


@pytest.mark.parametrize("m,n,k", [(3, 70, 8192), (40, 200, 2000), (300, 500, 700)])
def test_matmul_arbitrary_e4m3(cuda, m, n, k):
    s = _make(cuda, m, n, k, "e4m3", "f32", 2, bias=False, res=False)
    g = torch.Generator(device=cuda).manual_seed(3)
    for f in ("a", "w"):
        s[f] = (100 * torch.randn(s[f].shape, generator=g, device=cuda)).clamp(-448, 448).to(torch.float8_e4m3fn)
    out = QuantMatMulLayer(None, torch.float32).forward(**s)
    size = (s["a"].double().abs() @ s["w"].double().abs().t().contiguous()) * s["a_scale"].double()[:, None] * s["w_scale"].double()
    y, _ = _ref(s, None)
    assert ((out.double() - y).abs() <= (2 * k + 4) * 2.0 ** -24 * size).all()


def test_matmul_int8_extremes(cuda):
    # -128 everywhere: the largest sum that int32 has to hold
    for m, n, k in ((3, 20, 131071), (70, 80, 131071)):
        a, w = (torch.full((r, k), -128, dtype=torch.int8, device=cuda) for r in (m, n))
        one = lambda r: torch.ones(r, device=cuda)  # noqa: E731
        out = QuantMatMulLayer(None, torch.float32).forward(a, one(m), w, one(n))
        assert (out == float(16384 * 131071)).all()


def test_matmul_e4m3_nan_stays_in_its_row_and_column(cuda):
    for m in (5, 100):
        s = _make(cuda, m, 150, 200, "e4m3", "f32", 6)
        s["a"][2, 199] = float("nan")
        s["w"][140, 3] = float("nan")
        out = QuantMatMulLayer(None, torch.float32).forward(**s)
        want = torch.zeros(m, 150, dtype=torch.bool, device=cuda)
        want[2], want[:, 140] = True, True
        assert torch.equal(out.isnan(), want)
        # Relu keeps a NaN
        assert torch.equal(QuantMatMulLayer("Relu", torch.float32).forward(**s).isnan(), want)


@pytest.mark.parametrize("act,lo,hi", [("Silu", -0.0, float("inf")), ("Gelu", -0.0, float("inf")), ("Relu", 0.0, float("inf"))])
def test_matmul_activations_at_large_arguments(cuda, act, lo, hi):
    a = torch.ones(2, 16, dtype=torch.int8, device=cuda)
    w = torch.ones(4, 16, dtype=torch.int8, device=cuda)
    bias = torch.tensor([-3e38, 3e38, -200.0, 200.0], device=cuda)
    out = QuantMatMulLayer(act, torch.float32).forward(a, torch.full((2,), 1e-3, device=cuda), w,
                                                       torch.ones(4, device=cuda), bias)
    assert (out[:, 0] == lo).all() and (out[:, 2].abs() < 1e-30).all()
    assert torch.allclose(out[:, 1], bias[1]) and torch.allclose(out[:, 3], bias[3] + 0.016)


@pytest.mark.parametrize("m", [7, 90, 600])
def test_matmul_strided_and_in_place(cuda, m):
    n, k = 333, 260
    s = _make(cuda, m, n, k + 7, "int8", "f16", 8)
    s["a"], s["w"] = s["a"][:, 3:k + 3], s["w"][:, 5:k + 5]  # odd pitches and addresses
    wide = torch.randn(m, 2 * n, device=cuda).half()
    s["residual"] = wide[:, 1:n + 1]
    before = wide.clone()
    out = QuantMatMulLayer("Silu", torch.float16).forward(**s, out=s["residual"])
    assert out.data_ptr() == wide.data_ptr() + 2
    s["residual"] = before[:, 1:n + 1]
    _check(out, s, "Silu", "f16")
    assert torch.equal(wide[:, 0], before[:, 0]) and torch.equal(wide[:, n + 1:], before[:, n + 1:])
    # one row of scales spread out, w an expanded row
    s["a_scale"] = torch.rand(m, 2, device=cuda)[:, 1]
    s["w"] = s["w"][:1].expand(n, k)
    _check(QuantMatMulLayer("Silu", torch.float16).forward(**s), s, "Silu", "f16")


def test_matmul_empty(cuda):
    z = lambda *s: torch.zeros(*s, dtype=torch.int8, device=cuda)  # noqa: E731
    o = lambda r: torch.ones(r, device=cuda)  # noqa: E731
    assert QuantMatMulLayer().forward(z(0, 8), o(0), z(4, 8), o(4)).shape == (0, 4)
    assert QuantMatMulLayer().forward(z(3, 8), o(3), z(0, 8), o(0)).shape == (3, 0)


@pytest.mark.parametrize("m", [1, 64, 300])
def test_matmul_on_a_stream_and_in_a_graph(cuda, m):
    s = _make(cuda, m, 200, 512, "e4m3", "bf16", 12)
    layer = QuantMatMulLayer("Gelu")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        layer.forward(**s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = layer.forward(**s)
    torch.cuda.current_stream().wait_stream(st)
    for i in range(3):
        s["a_scale"].mul_(1.1)
        want = layer.forward(**s)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
