"""GPU: Int4MatMulLayer with groups that are longer than k, a scale a row: whatever their length says,
the work is that of k.  (A loop over a group's length would pass 2^30 / 128 times for nothing, a
tenth of a second; the product itself takes microseconds.)"""
import pytest
import torch

from onnxsharp_amd.lm_layers import Int4MatMulLayer
from test_gpu_int4_matmul import check, make, weight

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [1 << 20, 1 << 30, 2 ** 31 - 128])
@pytest.mark.parametrize("m,n,k", [(1, 70, 300), (40, 4100, 4200), (200, 256, 512), (300, 130, 515)])
def test_one_group_for_all_of_k(cuda, m, n, k, group, dtype):
    print(f"int4 {m} x {n} x {k} groups of {group} {dtype}", flush=True)
    for zeros in (False, True):
        t = make(cuda, m, n, k, group, zeros, TYPES[dtype])
        w, layer = weight(t), Int4MatMulLayer()
        check(t, layer.forward(t["x"], w))
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        layer.forward(t["x"], w)
        b.record()
        b.synchronize()
        assert a.elapsed_time(b) < 5.0
