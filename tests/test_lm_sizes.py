"""Sizes beyond the C ABI's 32 bits are refused: cut down to those they would name another, smaller
product, whose result would stand in the first part of the output.  Meta tensors: nothing is allocated."""
import pytest
import torch

from onnxsharp_amd import native as N
from onnxsharp_amd.lm_layers import BlockNormLayer, Int4MatMulLayer, Int4Weight, QuantMatMulLayer, RmsNormQuantLayer

BIG = 2 ** 32 + 64  # 64 in 32 bits


def t(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def refused():
    return pytest.raises(N.OshUnsupported, match=str(BIG))


def test_int4_weight():
    with refused():
        Int4Weight(t(1, BIG // 2, dtype=torch.uint8), t(1, BIG // 32), k=BIG, group=32)
    with refused():
        Int4Weight(t(BIG, 16, dtype=torch.uint8), t(BIG, 1), k=32, group=32)
    with refused():
        Int4Weight(t(8, 16, dtype=torch.uint8), t(8, 1), k=32, group=BIG)


def test_int4_matmul():
    w = Int4Weight.__new__(Int4Weight)
    w.n, w.k, w.group, w.dtype, w.has_zeros, w.packed = 4, 32, 32, torch.bfloat16, False, t(4096, dtype=torch.uint8)
    with refused():
        Int4MatMulLayer().forward(t(BIG, 32), w)


def test_norms():
    with refused():
        BlockNormLayer().forward(t(2, BIG), t(BIG))
    with refused():
        RmsNormQuantLayer().forward(t(2, BIG), t(BIG))


@pytest.mark.parametrize("m,n,k", [(BIG, 4, 32), (4, BIG, 32), (4, 4, BIG)])
def test_quant_matmul(m, n, k):
    with refused():
        QuantMatMulLayer().forward(t(m, k, dtype=torch.int8), t(m, dtype=torch.float32), t(n, k, dtype=torch.int8),
                                   t(n, dtype=torch.float32))
