"""GPU: WindowAttentionLayer's sequences of a batch apart from one another, and what a
captured call writes.

A sequence's bits depend on its own tokens and keys, the call's bounds and the number of
workgroups its keys are split over, which few and long sequences raise: alone and in a
batch they are the same where that number is, else within twice the bound against 64 bits
that test_gpu_lm_attention derives."""
import pytest
import torch

from onnxsharp_amd.lm_layers import PagedKvCache, WindowAttentionLayer
from test_gpu_lm_attention import _make, _ref, _run, _same

pytestmark = pytest.mark.gpu


def _alone(s, i, window, sinks):
    """Sequence i of s as a batch of one, under the batch's bounds."""
    cu = s["cu"].tolist()
    rows = slice(cu[i], cu[i + 1])
    cache = PagedKvCache(s["kp"].clone(), s["vp"].clone(), s["table"][i:i + 1])
    new = torch.tensor([0, cu[i + 1] - cu[i]], dtype=torch.int32, device=s["kl"].device)
    out = WindowAttentionLayer(window, sinks).forward(
        s["q"][rows], s["k"][rows], s["v"][rows], cache, new, s["kl"][i:i + 1], max(q for q, _ in s["lens"]),
        max(k for _, k in s["lens"]))
    return out, rows, cache


# single tokens, drafted tokens, pieces of prompts and whole ones; spans of one split
@pytest.mark.parametrize("hq,hkv,d,lens,window", [
    (8, 2, 128, [(1, 500), (1, 77), (1, 1)], 100), (4, 4, 64, [(1, 300), (1, 400), (1, 20)], 300),
    (8, 2, 80, [(3, 200), (5, 90), (1, 1)], 100), (4, 1, 128, [(150, 400), (1, 90), (40, 40)], 64),
    (2, 2, 256, [(1, 200), (30, 300)], 100)])
def test_attention_alone_and_in_a_batch(cuda, hq, hkv, d, lens, window):
    s = _make(cuda, hq, hkv, d, 16, lens, "bf16", 31)
    alone = [_alone(s, i, window, 4) for i in range(len(lens))]
    before = s["kp"].clone()
    out = _run(s, window, 4)
    for i, (one, rows, cache) in enumerate(alone):
        assert _same(out[rows], one)
        pages = s["table"][i][:(lens[i][1] + 15) // 16].long()
        assert _same(s["kp"][pages], cache.k_pages[pages]) and _same(s["vp"][pages], cache.v_pages[pages])
    # other data and lengths of the others change nothing
    s["kp"].copy_(before)
    first = slice(0, lens[0][0])
    for f in ("q", "k", "v"):
        s[f][lens[0][0]:] *= -3.0
    s["kl"][1:] -= 1
    s["kl"][1:].clamp_(min=0)
    again = _run(s, window, 4)
    assert _same(again[first], out[first])


@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_alone_and_in_a_batch_of_long_ones(cuda, d):
    lens = [(1, 5000), (1, 3000), (1, 700), (1, 4999)]
    s = _make(cuda, 4, 1, d, 64, lens, "f16", 32)
    o, big, _, _ = _ref(s, 4500, 4, None, s["kp"], s["vp"])
    alone = [_alone(s, i, 4500, 4) for i in range(len(lens))]
    out = _run(s, 4500, 4)
    bound = 2.0 ** -11 * (o.abs() + big) + 2.0 ** -12 * big + 2.0 ** -14
    for one, rows, _ in alone:
        assert ((one.double() - out[rows].double()).abs() <= 2 * bound[rows]).all()


@pytest.mark.parametrize("lens", [[(1, 700), (1, 30)], [(1, 6000)], [(150, 400), (1, 90)]])
def test_attention_in_a_graph_writes_the_cache(cuda, lens):
    # every replay runs over slots that hold something else
    s = _make(cuda, 8, 1, 128, 16, lens, "bf16", 33)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        _run(s, 4000, 4)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = _run(s, 4000, 4)
    torch.cuda.current_stream().wait_stream(st)
    at = [(int(s["table"][i, j // 16]), j % 16) for i, (ql, kl) in enumerate(lens) for j in range(kl - ql, kl)]
    pages, slots = (torch.tensor(t, device=cuda) for t in zip(*at))
    for _ in range(3):
        for f in ("q", "k", "v"):
            s[f].mul_(0.9)
        want = _run(s, 4000, 4)
        kp, vp = s["kp"].clone(), s["vp"].clone()
        assert _same(kp[pages, slots], s["k"]) and _same(vp[pages, slots], s["v"])
        s["kp"][pages, slots] = 5.0
        s["vp"][pages, slots] = -5.0
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        assert _same(out, want) and _same(s["kp"], kp) and _same(s["vp"], vp)
