"""GPU: how far attention over 4-bit pages is from its formula beside what the rounding of its output
costs by itself.

Bound, in the 2-norm of a head's error.  With r the norm of the error that rounding the result in 64
bits to the type leaves: products of codes are exact, and what is kept of a weight in the product with
them has 16 bits and more, 2^-17 of its size at most, times codes up to 15 and scales: 2^-17 *
15 scale, next to which r is 2^-10 (f16 2^-13) of o's size or more.  Sums in FP32 add as
little.  Both together stay below a tenth of r for keys and values of one size: 1.1 r."""
import pytest
import torch

from test_gpu_kv4_attention import check, make, ref, run

pytestmark = pytest.mark.gpu


def ratio(s, window, sinks, heads=slice(None), values=slice(None)):
    o = ref(s, window, sinks)[0][:, heads, values]
    out = run(s, window, sinks)[:, heads, values].double()
    return float((out - o).norm() / (o.to(s["q"].dtype).double() - o).norm())


# one, two and four heads a key head, drafts, 16 rows and row blocks, each group size
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d,group,lens", [
    (12, 4, 64, 32, [(1, 600)]), (8, 2, 128, 128, [(1, 3000), (1, 700)]), (8, 2, 128, 32, [(1, 3000), (1, 700)]),
    (4, 4, 64, 64, [(1, 900)]), (8, 1, 128, 64, [(1, 2000)]), (8, 2, 128, 128, [(2, 900), (1, 300)]),
    (16, 1, 64, 64, [(1, 900)]), (16, 1, 128, 128, [(1, 2000), (1, 40)]), (8, 2, 128, 64, [(40, 500)]),
    (4, 2, 256, 32, [(1, 900)]), (8, 2, 256, 128, [(3, 900)]), (4, 1, 128, 64, [(200, 500)])])
def test_error_is_that_of_the_output(cuda, hq, hkv, d, group, lens, dtype):
    s = make(cuda, hq, hkv, d, group, 16, lens, dtype, 5)
    r = ratio(s, None, 0)
    print(hq, hkv, d, group, lens, dtype, r, flush=True)
    assert r <= 1.1


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new,hq", [(1, 4), (4, 8), (50, 4)])
@pytest.mark.parametrize("power", [4, 8, 12])
def test_groups_of_one_head_apart(cuda, power, new, hq, dtype):
    # one group's values 2^power times the others': each group has the error of its own size
    s = make(cuda, hq, 2, 128, 32, 16, [(new, 700)], dtype, 6)
    s["v"][..., 32:64] *= 2.0 ** (power - 6)
    s["v"][..., :32] *= 2.0 ** -6
    s["v"][..., 64:] *= 2.0 ** -6
    s["cache"].v_scales[..., :, :] *= 2.0 ** -6
    s["cache"].v_scales[..., 1, :] *= 2.0 ** power
    for g in range(4):
        r = ratio(s, None, 0, values=slice(32 * g, 32 * g + 32))
        print(power, new, hq, dtype, g, r, flush=True)
        assert r <= 1.1


@pytest.mark.parametrize("dtype,power", [("f16", 10), ("bf16", 10), ("bf16", 60)])
@pytest.mark.parametrize("where", [150, 690])
def test_a_large_key_that_other_queries_see(cuda, where, dtype, power):
    # the first query alone sees a key whose values are 2^power times the others'
    s = make(cuda, 4, 2, 128, 64, 16, [(3, 700)], dtype, 7)
    window = 700 - 3 + 1 - where
    pg = s["table"][0, where // 16].long()
    s["cache"].v_scales[pg, where % 16] *= 2.0 ** power
    o, out = ref(s, window, 0)[0], run(s, window, 0).double()
    rounded = o.to(s["q"].dtype).double()
    for i in range(3):
        r = float((out[i] - o[i]).norm() / (rounded[i] - o[i]).norm())
        print(where, dtype, power, i, r, flush=True)
        assert r <= 1.1


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,new,group", [(4, 1, 64), (8, 3, 32), (4, 60, 128), (8, 130, 64)])
def test_scales_below_zero(cuda, hq, new, group, dtype):
    # pages that another program filled from the largest value down: lo + scale code all the same
    s = make(cuda, hq, 2, 128, group, 16, [(new, 700)], dtype, 9)
    for codes, pairs in ((s["cache"].k_codes, s["cache"].k_scales), (s["cache"].v_codes, s["cache"].v_scales)):
        codes.copy_(255 - codes)
        pairs[..., 1] += 15 * pairs[..., 0]
        pairs[..., 0].neg_()
    check(s, None, 0)
