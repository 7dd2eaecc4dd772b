"""GPU: attention over 4-bit pages at the ends of FP32's range, on both sides of the 512 rows of a
key head from which bf16 calls take f16 pages.

Where all scores are 0 in FP32 the weights are 1 each, exact in every type: o is the mean of the
visible values.  A value or its weight is rounded by at most half a step of bf16, 2^-9 of the
largest value seen V, the output by as much again; sums in FP32 and values in f16 stay far
below: 2^-8 V in all."""
import pytest
import torch

from test_gpu_kv4_attention import make, ref, run

pytestmark = pytest.mark.gpu
F32_TINY = 2.0 ** -126


def check_mean(s, window, sinks, scale):
    o, _, (_, vc, _, vs), _ = ref(s, window, sinks, scale)
    out = run(s, window, sinks, scale).double()
    v = vs.double().nan_to_num(0.0)
    top = (v[..., 1].abs() + 15 * v[..., 0].abs()).amax()
    assert out.isfinite().all()
    assert ((out - o).abs() <= 2.0 ** -8 * top).all(), float(((out - o).abs() / top).max())


@pytest.mark.parametrize("new", [3, 40, 130, 300])
@pytest.mark.parametrize("q_size,k_size,scale", [(1e-25, 1e-25, None), (1e-30, 1e-30, 0.1), (1e-4, 1e-4, F32_TINY),
                                                 (1.0, 1e-37, F32_TINY), (1e-37, 1.0, F32_TINY)])
def test_scores_below_the_range(cuda, q_size, k_size, scale, new):
    s = make(cuda, 4, 1, 64, 32, 16, [(new, 400), (1, 90)], "bf16", new)
    s["q"] = (s["q"].float() * q_size).bfloat16()
    s["k"] = (s["k"].float() * k_size).bfloat16()
    s["cache"].k_scales.copy_((s["cache"].k_scales.float() * k_size).bfloat16())
    check_mean(s, 100, 4, scale)


@pytest.mark.parametrize("new", [3, 40, 130, 300])
@pytest.mark.parametrize("size", [1.0, 1e15, 1e19, 1e30])
def test_products_of_zero_between_large_operands(cuda, size, new):
    # queries in one half of a head, keys in the other
    s = make(cuda, 4, 1, 64, 32, 16, [(new, 400), (1, 90)], "bf16", new)
    s["q"] = (s["q"].float() * size).bfloat16()
    s["k"] = (s["k"].float() * size).bfloat16()
    s["q"][..., 32:] = 0
    s["k"][..., :32] = 0
    s["cache"].k_scales.copy_((s["cache"].k_scales.float() * size).bfloat16())
    s["cache"].k_scales[..., 0, :].mul_(0)
    check_mean(s, 100, 4, None)
