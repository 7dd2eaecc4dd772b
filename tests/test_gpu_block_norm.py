"""GPU: BlockNormLayer against its formula in 64 bits.

Bounds.  u = 2^-24.  A norm's sum of squares is one rounding per value of a lane (32 at
most) and one per join of lanes and waves (6 + 15), its square root halves the error: 27 u;
mean, eps, root, reciprocal and products add 8: 36 u.  A sigmoid adds 16 u for gates below 8
(the argument's rounding times its size, exp2, sum, reciprocal).  So before its own rounding h
is within 60 u of the sizes of its two terms, and y, the norm of the h that is stored, within
40 u; each is then rounded once, by half a step of its type or half of its smallest
subnormal number."""
import pytest
import torch

from onnxsharp_amd.lm_layers import BlockNormLayer

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}


def _make(cuda, rows, cols, dtype, seed):
    g = torch.Generator(device=cuda).manual_seed(seed)
    t = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    return dict(x=(3 * t(rows, cols)).to(dtype), branch=t(rows, cols).to(dtype), gamma=(1 + 0.2 * t(cols)).to(dtype),
                post=(1 + 0.2 * t(cols)).to(dtype), gate_cols=t(cols).to(dtype), gate_rows=t(rows, cols).to(dtype))


def _rms(f, eps):
    return (f.pow(2).mean(1, keepdim=True) + eps).sqrt()


def _close(got, want, size, dtype):
    half = torch.finfo(dtype).eps / 2
    d = (got.double() - want).abs()
    bound = half * want.abs() * (1 + 1e-6) + 60 * U * size + TINY[dtype]
    assert (d <= bound).all(), float((d - bound).max())


def check(layer, x, gamma, branch, post, gate, h, y, eps=1e-5):
    dtype = x.dtype
    if branch is None:
        assert h is x
    else:
        n = branch.double()
        if post is not None:
            n = n / _rms(n, eps) * post.double()
        if gate is not None:
            n = n * (torch.sigmoid(gate.double()) if layer.gate_activation else gate.double())
        a, b = layer.residual_scale * x.double(), layer.branch_scale * n
        _close(h, a + b, a.abs() + b.abs(), dtype)
    if gamma is None:
        assert y is None
    else:
        want = h.double() / _rms(h.double(), eps) * gamma.double()
        _close(y, want, want.abs(), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (300, 5), (3, 8), (5, 9), (7, 64), (1, 511), (9, 513), (2, 1283), (1, 4096),
                                       (33, 2047), (3, 4100), (17, 8192), (2, 16384), (1, 32768), (2, 30001)])
def test_block_norm(cuda, rows, cols, dtype):
    t = _make(cuda, rows, cols, TYPES[dtype], rows * 7 + cols)
    print(f"block norm {rows} x {cols} {dtype}", flush=True)
    for act, gate, post, gamma in ((None, None, t["post"], t["gamma"]), ("Sigmoid", t["gate_rows"], t["post"], t["gamma"]),
                                   (None, t["gate_cols"], None, t["gamma"]), ("Sigmoid", t["gate_cols"], t["post"], None),
                                   (None, t["gate_rows"], None, None)):
        layer = BlockNormLayer(residual_scale=0.5, branch_scale=1.25, gate_activation=act)
        h, y = layer.forward(t["x"], gamma, t["branch"], post, gate)
        check(layer, t["x"], gamma, t["branch"], post, gate, h, y)
    layer = BlockNormLayer()
    check(layer, t["x"], t["gamma"], None, None, None, *layer.forward(t["x"], t["gamma"]))


@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows(cuda, dtype):
    t = _make(cuda, 70001, 72, TYPES[dtype], 5)
    layer = BlockNormLayer(branch_scale=-2.0)
    check(layer, t["x"], t["gamma"], t["branch"], t["post"], None, *layer.forward(t["x"], t["gamma"], t["branch"], t["post"]))


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("cols", [6, 40, 1283, 4096, 9001, 17000])
def test_strided_rows_and_in_place(cuda, cols, post):
    # operands inside wider tensors at odd offsets; h over x and over the branch
    t = _make(cuda, 6, 2 * cols + 3, torch.bfloat16, 3)
    part = lambda name: t[name][..., 1:cols + 1]  # noqa: E731
    gamma, gate, pg = part("gamma"), part("gate_rows"), part("post") if post else None
    layer = BlockNormLayer(gate_activation="Sigmoid")
    for target in ("x", "branch"):
        for g in (gamma, None):
            wide = {n: t[n].clone() for n in ("x", "branch")}
            x, br = wide["x"][:, 1:cols + 1], wide["branch"][:, 1:cols + 1]
            keep_x, keep_b = x.clone(), br.clone()
            h, y = layer.forward(x, g, br, pg, gate, out_h={"x": x, "branch": br}[target])
            check(layer, keep_x, g, keep_b, pg, gate, h, y)
            assert torch.equal(wide[target][:, 0], t[target][:, 0])
            assert torch.equal(wide[target][:, cols + 1:], t[target][:, cols + 1:])
            other = "branch" if target == "x" else "x"
            assert torch.equal(wide[other], t[other])


@pytest.mark.parametrize("cols", [5, 200, 2000, 9000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_beyond_the_squares_range(cuda, cols, dtype):
    # rows whose squares overflow, vanish or are zero, beside ordinary ones
    dt = TYPES[dtype]
    t = _make(cuda, 6, cols, dt, 11)
    sizes = torch.tensor([1.0, 1e25, 1e-30, 1.0, 0.0, 1e30], device=cuda)[:, None]
    x, br = (t["x"].float() * sizes).to(dt), (t["branch"].float() * sizes.flip(0)).to(dt)
    for eps in (0.0, 1e-5):
        layer = BlockNormLayer(eps=eps)
        h, y = layer.forward(x, t["gamma"])
        f = x.double()
        r = _rms(f, eps)
        _close(y, torch.where(r > 0, f / r, 0.0) * t["gamma"].double(), (f / r).nan_to_num(0.0).abs() * 2, dt)
        h, y = layer.forward(torch.zeros_like(x), None, br, t["post"])
        f = br.double()
        r = _rms(f, eps)
        want = torch.where(r > 0, f / r, 0.0) * t["post"].double()
        _close(h, want, want.abs(), dt)


@pytest.mark.parametrize("cols", [6, 200, 2000, 9000])
def test_rows_that_are_not_finite(cuda, cols):
    t = _make(cuda, 5, cols, torch.bfloat16, 9)
    t["branch"][1, cols // 2] = float("nan")
    t["branch"][3, 0] = float("inf")
    h, y = BlockNormLayer().forward(t["x"], t["gamma"], t["branch"], t["post"])
    bad = torch.tensor([False, True, False, True, False], device=cuda)
    assert torch.equal(h.isnan().all(1), bad) and torch.equal(y.isnan().all(1), bad)
    assert h[~bad].isfinite().all() and y[~bad].isfinite().all()


def test_empty_and_other_streams(cuda):
    t = _make(cuda, 4, 640, torch.float16, 2)
    h, y = BlockNormLayer().forward(t["x"][:0], t["gamma"], t["branch"][:0])
    assert h.shape == y.shape == (0, 640)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    layer = BlockNormLayer()
    with torch.cuda.stream(s):
        h, y = layer.forward(t["x"], t["gamma"], t["branch"], t["post"])
    s.synchronize()
    check(layer, t["x"], t["gamma"], t["branch"], t["post"], None, h, y)


def test_captured(cuda):
    t = _make(cuda, 9, 1283, torch.float16, 4)
    layer = BlockNormLayer()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, y = layer.forward(t["x"], t["gamma"], t["branch"], t["post"], t["gate_cols"])
    for seed in range(3):
        other = _make(cuda, 9, 1283, torch.float16, 40 + seed)
        for n in ("x", "branch", "post"):
            t[n].copy_(other[n])
        graph.replay()
        torch.cuda.synchronize()
        eh, ey = layer.forward(t["x"], t["gamma"], t["branch"], t["post"], t["gate_cols"])
        assert torch.equal(h, eh) and torch.equal(y, ey)
