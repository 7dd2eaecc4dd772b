"""GPU: Int4MatMulLayer's kernel for few rows of large weights, whose sums over parts of k meet in
the scratch.  Which shapes take it is seen from the scratch: parts of k times rows times outputs
(up to a multiple of 128) in FP32, or nothing where one part holds all of k."""
import ctypes as C

import pytest
import torch

from onnxsharp_amd import native as N
from onnxsharp_amd.lm_layers import Int4MatMulLayer
from test_gpu_int4_matmul import check, make, weight

pytestmark = pytest.mark.gpu
TYPES = {"f32": (torch.float32, N.T_F32), "f16": (torch.float16, N.T_F16), "bf16": (torch.bfloat16, N.T_BF16)}


def parts(m, n, k, group, code):
    size = C.c_size_t()
    N.call("osh_int4_matmul_scratch_bytes", m, n, k, group, code, C.byref(size))
    row = m * -(-n // 128) * 128 * 4
    assert size.value % row == 0, "not sums of parts"
    return size.value // row


def blocks(k):
    return -(-k // 128)


# 16 rows, 32 and 64 (32 and 32 in FP32) a workgroup, and more than one workgroup's; one block of
# 128 k a part and several; parts that end short; k and n that end inside a group, a block, a tile
HALF = [(1, 36000, 5000), (2, 33000, 4100), (8, 16390, 8190), (16, 16385, 3200), (17, 8200, 8190), (24, 4099, 8190),
        (32, 12000, 5500), (33, 12100, 4100), (64, 4100, 4200), (64, 16000, 3333), (100, 4096, 2176), (200, 5000, 2500)]
FULL = [(1, 4099, 4200), (1, 16390, 4100), (3, 8200, 8190), (16, 8200, 4100), (17, 8200, 4100), (33, 4099, 1100),
        (100, 4096, 2176), (70, 7000, 1000)]
CASES = [(d, *s) for d in ("f16", "bf16") for s in HALF] + [("f32", *s) for s in FULL]


@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype,m,n,k", CASES)
def test_few_rows(cuda, dtype, m, n, k, group):
    dt, code = TYPES[dtype]
    cut = parts(m, n, k, group, code)
    print(f"int4 {m} x {n} x {k} groups of {group} {dtype}: {blocks(k)} blocks of k in {cut} parts", flush=True)
    assert cut > 1
    for zeros in (False, True):
        t = make(cuda, m, n, k, group, zeros, dt)
        check(t, Int4MatMulLayer().forward(t["x"], weight(t)))
    act = {32: "Silu", 64: "Gelu", 128: "Relu", 256: None}[group]
    y = Int4MatMulLayer(act).forward(t["x"], weight(t), t["bias"], t["res"])
    check(t, y, act, t["bias"], t["res"])


def test_the_cases_reach_every_form():
    # blocks of k a part by the shapes above: one and several, whole and cut short
    seen = set()
    for dtype, m, n, k in CASES:
        cut, all_k = parts(m, n, k, 128, TYPES[dtype][1]), blocks(k)
        rows = 16 if m <= 16 else 32 if m <= 32 or dtype == "f32" else 64
        per = -(-all_k // cut)
        seen.add((dtype, rows, per > 1, all_k % per != 0))
    for dtype, rows in (("f16", 16), ("f16", 32), ("f16", 64), ("bf16", 16), ("bf16", 32), ("bf16", 64), ("f32", 16),
                        ("f32", 32)):
        assert (dtype, rows, True, True) in seen, (dtype, rows, sorted(seen))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(5, 16390, 8190), (24, 8200, 8192), (60, 8200, 4104)])
def test_few_rows_strides(cuda, m, n, k, dtype):
    # rows, residual and output inside wider tensors at odd offsets; the output over the residual
    dt, code = TYPES[dtype]
    assert parts(m, n, k, 64, code) > 1
    t = make(cuda, m, n, k, 64, True, dt)
    wide = torch.randn(m, k + 3, device=cuda).to(dt)
    wide[:, 1:k + 1] = t["x"]
    out, res = torch.full((m, n + 5), 7.0, device=cuda, dtype=dt), torch.randn(m, n + 9, device=cuda).to(dt)
    w = weight(t)
    y = Int4MatMulLayer().forward(wide[:, 1:k + 1], w, None, res[:, 5:n + 5], out=out[:, 3:n + 3])
    check(t, y, None, None, res[:, 5:n + 5])
    assert (out[:, :3] == 7).all() and (out[:, n + 3:] == 7).all()
    keep = t["res"].clone()
    y = Int4MatMulLayer().forward(t["x"], w, None, t["res"], out=t["res"])
    check(t, y, None, None, keep)


@pytest.mark.parametrize("m", [8, 24, 64])
@pytest.mark.parametrize("dtype", TYPES)
def test_few_rows_that_are_not_finite(cuda, m, dtype):
    dt, code = TYPES[dtype]
    assert parts(m, 16400, 4100, 32, code) > 1
    t = make(cuda, m, 16400, 4100, 32, False, dt)
    w = weight(t)
    good = Int4MatMulLayer().forward(t["x"], w)
    t["x"][1, 3], t["x"][2, 4099] = float("nan"), float("inf")
    y = Int4MatMulLayer().forward(t["x"], w)
    assert not y[1:3].isfinite().any()
    rest = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(y[rest], good[rest])


@pytest.mark.parametrize("m,dtype", [(1, "f32"), (24, "bf16"), (64, "f16")])
def test_few_rows_captured_and_other_streams(cuda, m, dtype):
    dt, code = TYPES[dtype]
    assert parts(m, 16400, 4100, 64, code) > 1
    t = make(cuda, m, 16400, 4100, 64, True, dt)
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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(150, 77, 296), (300, 520, 1024), (2100, 1100, 264)])
def test_tiles_of_rows_at_odd_addresses(cuda, m, n, k, dtype):
    # k of whole chunks, whose rows the tiles read where they lie
    dt = TYPES[dtype][0]
    t = make(cuda, m, n, k, 32, True, dt)
    for pitch in (k + 3, k + 8):
        wide = torch.randn(m, pitch, device=cuda).to(dt)
        wide[:, 1:k + 1] = t["x"]
        out, res = torch.full((m, n + 4), 7.0, device=cuda, dtype=dt), torch.randn(m, n + 9, device=cuda).to(dt)
        y = Int4MatMulLayer().forward(wide[:, 1:k + 1], weight(t), None, res[:, 5:n + 5], out=out[:, 3:n + 3])
        check(t, y, None, None, res[:, 5:n + 5])
        assert (out[:, :3] == 7).all() and (out[:, n + 3:] == 7).all()
