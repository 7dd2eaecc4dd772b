"""GPU: the new tokens of an attention call over 4-bit pages are quantized once each, or by a few row
blocks, but not by all.

A prompt of n tokens under a short window with sinks has work that grows as n: n / 16 row blocks,
each over the window's keys.  Were a block to quantize every new token among its keys' positions, the
sinks the first of them, the work would grow as n^2.  From 2048 to 16384 tokens n grows 8 times and n^2
64 times; a call has a cost of its own, so a time that grows less than 20 times is no n^2."""
import pytest
import torch

from test_gpu_kv4_attention import make, run

pytestmark = pytest.mark.gpu


def best(fn):
    fn()
    times = []
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        fn()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b))
    return min(times)


def test_time_grows_with_the_tokens(cuda):
    took = {}
    for n in (2048, 16384):
        s = make(cuda, 8, 2, 128, 64, 64, [(n, n)], "f16", 3)
        took[n] = best(lambda: run(s, 64, 4))
    print({n: f"{1e3 * t:.0f} us" for n, t in took.items()}, flush=True)
    assert took[16384] <= 20 * took[2048]
