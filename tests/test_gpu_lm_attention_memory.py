"""GPU: WindowAttentionLayer where its operands lie in one another's memory: views that
interleave give what separate tensors give, views that share bytes are refused."""
import pytest
import torch

from onnxsharp_amd import native as N
from onnxsharp_amd.lm_layers import PagedKvCache, WindowAttentionLayer
from test_gpu_lm_attention import _make, _run, _same

pytestmark = pytest.mark.gpu
LENS = [(20, 90), (1, 40)]


def test_attention_into_the_buffer_that_holds_q(cuda):
    s = _make(cuda, 8, 2, 64, 16, LENS, "bf16", 21)
    want = _run(s, 32, 4)
    wide = torch.zeros(21, 16, 64, dtype=torch.bfloat16, device=cuda)
    wide[:, :8] = s["q"]
    s["q"] = wide[:, :8]
    out = _run(s, 32, 4, out=wide[:, 8:])
    assert _same(out, want)
    heads = torch.zeros(21, 8, 2, 64, dtype=torch.bfloat16, device=cuda)  # every other head
    heads[:, :, 1] = s["q"]
    s["q"] = heads[:, :, 1]
    assert _same(_run(s, 32, 4, out=heads[:, :, 0]), want)


def test_attention_refuses_shared_views(cuda):
    s = _make(cuda, 8, 2, 64, 16, LENS, "bf16", 22)
    layer = WindowAttentionLayer(32, 4)

    def run(k_pages, v_pages, **kw):
        layer.forward(s["q"], s["k"], s["v"], PagedKvCache(k_pages, v_pages, s["table"]), s["cu"], s["kl"], 20, 90, **kw)

    kp, vp = s["kp"], s["vp"]
    with pytest.raises(N.OshError, match="share memory"):
        run(kp, kp)
    with pytest.raises(N.OshError, match="share memory"):
        run(kp, vp[:1].expand(vp.shape))
    with pytest.raises(N.OshError, match="share memory"):
        run(torch.cat([kp, vp])[:len(kp)], torch.empty_like(vp), out=s["q"][:1].clone().expand(s["q"].shape))
    with pytest.raises(N.OshError, match="overlaps the cache"):
        run(kp, vp, out=vp.view(-1, 8, 64)[:21])
    with pytest.raises(N.OshError, match="overlaps an operand"):
        run(kp, vp, out=s["q"])


@pytest.mark.parametrize("max_q", [1, 3, 40, 200])
def test_attention_more_new_tokens_than_the_bound(cuda, max_q):
    # every row of a sequence above max_q is NaN, the others keep their bits, and nothing of
    # it goes to the pages
    lens = [(max_q, 300), (max_q + 157, 400), (1, 20)]
    s = _make(cuda, 4, 2, 64, 16, lens, "bf16", 23)
    kp, vp = s["kp"].clone(), s["vp"].clone()

    def run():
        cache = PagedKvCache(s["kp"], s["vp"], s["table"])
        return WindowAttentionLayer(32, 2).forward(s["q"], s["k"], s["v"], cache, s["cu"], s["kl"], max_q, 400,
                                                   out=torch.full_like(s["q"], 7.0))

    out = run()
    first, last = lens[0][0], lens[0][0] + lens[1][0]
    assert out[first:last].isnan().all() and out[:first].isfinite().all() and out[last:].isfinite().all()
    for i in range(lens[1][1]):
        slot = int(s["table"][1, i // 16]), i % 16
        assert _same(s["kp"][slot], kp[slot]) and _same(s["vp"][slot], vp[slot])
    s["kl"][1] = -1  # refused for another reason
    assert _same(run().nan_to_num(nan=5.0), out.nan_to_num(nan=5.0))


def test_attention_rows_of_no_sequence_stay(cuda):
    s = _make(cuda, 4, 2, 64, 16, [(3, 50), (2, 40), (4, 30)], "f16", 24)
    s["cu"].copy_(torch.tensor([2, 5, 7, 7]))
    s["kl"][2] = 26
    out = _run(s, 32, 2, out=torch.full_like(s["q"], 7.0))
    assert (out[:2] == 7.0).all() and (out[7:] == 7.0).all() and (out[2:7] != 7.0).any(-1).all()
