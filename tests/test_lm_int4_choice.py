"""Which kernel Int4MatMul takes for few rows, as the scratch shows: none where one launch does it,
sums of parts of k where the weights' own reading pays for a second launch.  Both sides were measured
with weights that come from memory, as a model's do, not from a cache that holds one of them."""
import ctypes as C

import pytest

from onnxsharp_amd import native as N

# rows, outputs, k of bf16 products in groups of 128, and whether two launches were the faster
MEASURED = [(1, 768, 768, False), (1, 4096, 4096, False), (1, 8192, 8192, False), (4, 8192, 8192, False),
            (1, 16384, 8192, True), (2, 16384, 8192, True), (1, 32768, 8192, True), (1, 151936, 4096, True),
            (8, 12288, 4096, False), (8, 16384, 8192, True), (16, 4096, 4096, False), (16, 12288, 4096, True),
            (32, 4096, 4096, False), (32, 12288, 4096, True), (32, 8192, 8192, True)]


@pytest.mark.parametrize("m,n,k,two", MEASURED)
def test_few_rows_take_the_faster_kernel(m, n, k, two):
    size = C.c_size_t()
    N.call("osh_int4_matmul_scratch_bytes", m, n, k, 128, N.T_BF16, C.byref(size))
    assert (size.value > 0) == two
