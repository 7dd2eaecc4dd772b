"""GPU: WindowAttentionLayer against its formula in 64 bits.

Bounds.  A weight is rounded to the type before its product with v, half a step h =
eps / 2 of its size, and the output rounds once more: h (|o| + W) with W = sum of the
weights times |v|.  Scores are FP32 sums of d exact products, scaled to base 2 (at
most d / 8 + 4 roundings of 2^-24 of sum |q k| scale), sums and joins of weights and
values take at most one rounding per key of a lane and one per join; scores here
stay below 32 in size: 2^-12 W covers them for these lengths."""
import pytest
import torch

from onnxsharp_amd.lm_layers import PagedKvCache, WindowAttentionLayer

pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _make(cuda, hq, hkv, d, page, lens, dtype, seed, spare=3, stale=float("nan")):
    """lens: (new, whole) of each sequence.  Slots that hold no token are `stale`."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    t = TYPES[dtype]
    rnd = lambda *s: torch.randn(*s, generator=g, device=cuda).to(t)  # noqa: E731
    b = len(lens)
    width = max((kl + page - 1) // page for _, kl in lens) + 1
    pages = sum((kl + page - 1) // page for _, kl in lens) + spare
    s = dict(hq=hq, hkv=hkv, d=d, page=page, lens=lens)
    kp = torch.full((pages, page, hkv, d), stale, dtype=t, device=cuda)
    vp = kp.clone()
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((b, width), -1, dtype=torch.int32)
    for i, (ql, kl) in enumerate(lens):
        for j in range((kl + page - 1) // page):
            pg = order.pop()
            table[i, j] = pg
            n = max(0, min(page, kl - ql - j * page))
            kp[pg, :n], vp[pg, :n] = rnd(n, hkv, d), rnd(n, hkv, d)
    tokens = sum(ql for ql, _ in lens)
    s["q"], s["k"], s["v"] = rnd(tokens, hq, d), rnd(tokens, hkv, d), rnd(tokens, hkv, d)
    s["kp"], s["vp"], s["table"] = kp, vp, table.to(cuda)
    cu = [0]
    for ql, _ in lens:
        cu.append(cu[-1] + ql)
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device=cuda)
    s["kl"] = torch.tensor([kl for _, kl in lens], dtype=torch.int32, device=cuda)
    return s


def _run(s, window, sinks, scale=None, slack=0, **kw):
    layer = WindowAttentionLayer(window=window, sinks=sinks, scale=scale)
    cache = PagedKvCache(s["kp"], s["vp"], s["table"])
    max_q = max(ql for ql, _ in s["lens"]) + slack
    max_kv = max(max(kl for _, kl in s["lens"]), 1) + slack
    return layer.forward(s["q"], s["k"], s["v"], cache, s["cu"], s["kl"], max_q, max_kv, **kw)


def _ref(s, window, sinks, scale, kp, vp):
    """o, its bound's W, and the cache afterwards (from the cache before)."""
    kp, vp = kp.clone(), vp.clone()
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    big = torch.zeros_like(o)
    page, table, group = s["page"], s["table"].cpu(), s["hq"] // s["hkv"]
    scale = s["d"] ** -0.5 if scale is None else scale
    c = 0
    for i, (ql, kl) in enumerate(s["lens"]):
        at = torch.arange(kl)
        pg, sl = table[i, at // page].long().to(kp.device), (at % page).to(kp.device)
        kp[pg[kl - ql:], sl[kl - ql:]] = s["k"][c:c + ql]
        vp[pg[kl - ql:], sl[kl - ql:]] = s["v"][c:c + ql]
        for t in range(ql):
            p = kl - ql + t
            lo = 0 if window is None else max(0, p - window + 1)
            js = list(range(min(sinks, lo))) + list(range(lo, p + 1))
            js = torch.tensor(js, device=kp.device)
            k, v = kp[pg[js], sl[js]].double(), vp[pg[js], sl[js]].double()
            k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
            e = (s["q"][c + t].double() * k).sum(-1) * scale
            w = torch.softmax(e, 0)[..., None]
            o[c + t], big[c + t] = (w * v).sum(0), (w * v.abs()).sum(0)
        c += ql
    return o, big, kp, vp


def _same(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


def _check(s, window, sinks, scale=None, **kw):
    kp, vp = s["kp"].clone(), s["vp"].clone()
    out = _run(s, window, sinks, scale, **kw)
    o, big, kp, vp = _ref(s, window, sinks, scale, kp, vp)
    half = torch.finfo(out.dtype).eps / 2
    d = (out.double() - o).abs()
    bound = half * (o.abs() + big) + 2.0 ** -12 * big + torch.finfo(out.dtype).smallest_normal
    assert out.shape == o.shape and (d <= bound).all(), float((d - bound).max())
    assert _same(s["kp"], kp) and _same(s["vp"], vp)
    return out


# hq, hkv, d, page, (new, whole), window, sinks
CASES = [
    (1, 1, 8, 1, [(1, 1)], 1, 0),
    (4, 4, 32, 16, [(1, 1), (1, 2), (1, 17), (1, 33)], 16, 0),
    (12, 4, 64, 16, [(1, 600)], 512, 4),
    (8, 1, 128, 64, [(1, 1000), (1, 3), (0, 70), (1, 129), (0, 0)], 300, 4),
    (16, 2, 80, 16, [(1, 77), (1, 400)], 64, 16),
    (6, 2, 24, 7, [(1, 50), (1, 8)], 20, 3),
    (4, 2, 256, 32, [(1, 300), (1, 31)], 1000, 0),
    (3, 3, 136, 16, [(1, 90)], 33, 1),
    (40, 2, 64, 16, [(1, 100), (2, 40)], 50, 2),
    (8, 2, 96, 16, [(3, 100), (5, 5), (1, 64), (8, 200)], 32, 4),
    (4, 1, 64, 16, [(70, 70), (33, 100), (1, 90), (130, 131)], 40, 4),
    (4, 2, 128, 32, [(200, 500), (64, 64)], 128, 130),
    (2, 2, 40, 5, [(90, 95)], 1, 0),
    (2, 1, 64, 16, [(100, 300)], 1, 7),
    (5, 5, 72, 16, [(40, 40)], None, 0),
    (8, 8, 32, 128, [(150, 700), (1, 650), (17, 17)], None, 0),
    (6, 1, 128, 16, [(300, 300), (257, 900)], 100, 1000),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(cuda, case, dtype):
    hq, hkv, d, page, lens, window, sinks = CASES[case]
    print(f"attention {CASES[case]} {dtype}", flush=True)
    _check(_make(cuda, hq, hkv, d, page, lens, dtype, case), window, sinks)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_long_splits(cuda, d):
    # few sequences with long histories: the keys are split and joined
    _check(_make(cuda, 4, 1, d, 64, [(1, 6000), (1, 100)], "bf16", 1), 5000, 4)
    _check(_make(cuda, 4, 1, d, 64, [(3, 5000)], "f16", 2), None, 0)
    _check(_make(cuda, 2, 1, d, 16, [(24, 3001)], "bf16", 3), 2500, 16)


def test_attention_long_prompt(cuda):
    _check(_make(cuda, 8, 2, 128, 64, [(1100, 1100), (300, 1500)], "bf16", 4), 256, 4)
    _check(_make(cuda, 4, 4, 64, 16, [(600, 600)], "f16", 5), None, 0)


def test_attention_bounds_above_the_lengths(cuda):
    # the host's bounds may be loose: same outputs
    lens = [(3, 50), (1, 200), (0, 9)]
    s = _make(cuda, 4, 2, 64, 16, lens, "bf16", 6)
    s["table"] = torch.cat([s["table"], torch.full((3, 400), -1, dtype=torch.int32, device=cuda)], 1)
    _check(s, 100, 2, slack=1000)


def test_attention_scale_and_large_scores(cuda):
    s = _make(cuda, 4, 2, 64, 16, [(40, 100), (1, 300)], "f16", 7)
    _check(s, 64, 4, scale=0.4)
    # one key far above the others: its value comes back, from any place
    s = _make(cuda, 2, 2, 64, 16, [(1, 900)], "bf16", 8)
    s["q"].fill_(8.0)
    s["kp"][s["table"][0, 20].long(), 3] = 8.0
    out = _run(s, None, 0)
    assert _same(out[0], s["vp"][s["table"][0, 20].long(), 3])


def test_attention_strided_inputs_and_pages(cuda):
    hq, hkv, d, page = 8, 2, 64, 16
    lens = [(20, 90), (1, 40)]
    s = _make(cuda, hq, hkv, d, page, lens, "bf16", 9)
    # q, k, v as parts of one projection's rows; pages with heads outside slots
    qkv = torch.cat([s[f].reshape(21, -1) for f in "qkv"], 1)
    s["q"] = qkv[:, :hq * d].view(21, hq, d)
    s["k"] = qkv[:, hq * d:(hq + hkv) * d].view(21, hkv, d)
    s["v"] = qkv[:, (hq + hkv) * d:].view(21, hkv, d)
    both = torch.stack([s["kp"], s["vp"]], 1).transpose(2, 3).contiguous().transpose(2, 3)
    s["kp"], s["vp"] = both[:, 0], both[:, 1]
    assert not s["kp"].is_contiguous()
    wide = torch.zeros(21, hq, d + 3, dtype=torch.bfloat16, device=cuda)
    out = _check(s, 32, 4, out=wide[..., 2:d + 2])
    assert out.data_ptr() == wide.data_ptr() + 4
    assert not wide[..., :2].any() and not wide[..., d + 2:].any()
    # pages at odd addresses
    flat = torch.zeros(s["kp"].numel() + 1, dtype=torch.bfloat16, device=cuda)
    kp = flat[1:].view(s["kp"].shape)
    kp.copy_(s["kp"])
    s["kp"], s["q"], s["k"] = kp, s["q"].contiguous(), s["k"].transpose(0, 1).contiguous().transpose(0, 1)
    _check(s, 32, 4)


def test_attention_pages_before_the_window_are_not_read(cuda):
    # entries and slots that no query sees: ids outside the cache, NaN, infinities
    s = _make(cuda, 4, 2, 64, 16, [(1, 400), (30, 300)], "bf16", 10)
    want = _check(s, 64, 4)
    for i, (ql, kl) in enumerate(s["lens"]):
        first = kl - ql - 64 + 1
        for j in range(1, first // 16):
            pg = int(s["table"][i, j])
            s["kp"][pg], s["vp"][pg] = float("inf"), float("nan")
            s["table"][i, j] = [-1, 1 << 30, -2 ** 31, 999][j % 4]
        pg = int(s["table"][i, first // 16])
        s["kp"][pg, :first % 16], s["vp"][pg, :first % 16] = float("nan"), float("-inf")
        pg = int(s["table"][i, 0])
        s["kp"][pg, 4:], s["vp"][pg, 4:] = float("nan"), float("nan")
    assert _same(_run(s, 64, 4), want)


def test_attention_bad_page_is_nan_where_it_is_seen(cuda):
    lens = [(1, 100), (1, 100), (40, 100)]
    s = _make(cuda, 4, 2, 64, 16, lens, "f16", 11)
    good = _run(s, 32, 0)
    kp, vp = s["kp"].clone(), s["vp"].clone()
    s["table"][0, 5] = s["kp"].shape[0]  # positions 80..95, seen by sequence 0's query at 99
    s["table"][1, 0] = -5                # position 0..15, outside sequence 1's window
    s["table"][2, 6] = -1                # positions 96..99: seen by its last four queries, which are new there
    out = _run(s, 32, 0)
    assert out[0].isnan().all() and _same(out[1], good[1])
    # new tokens come from k and v, so their page only misses their copy
    assert _same(out[2:], good[2:])
    assert _same(s["kp"], kp) and _same(s["vp"], vp)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,ql,kl", [(64, 3, 40), (128, 90, 130), (256, 60, 90)])
def test_attention_nonfinite_keys_reach_only_who_sees_them(cuda, d, ql, kl, dtype):
    # a new token's key and an old key are not finite: the queries that see neither keep
    # the bits that finite ones give
    s, window = _make(cuda, 4, 2, d, 16, [(ql, kl)], dtype, d + ql), 24
    past = kl - ql
    old, tk = past - 10, ql - 2  # the old one leaves the window of later tokens
    good = _run(s, window, 2)
    s["k"][tk, 0, 1] = float("nan")
    s["kp"][int(s["table"][0, old // 16]), old % 16, 0, 7] = float("nan")
    out = _run(s, window, 2)
    pos = past + torch.arange(ql, device=cuda)
    want = torch.zeros(out.shape, dtype=torch.bool, device=cuda)
    for j in (past + tk, old):
        want[(j <= pos) & (j > pos - window), :2] = True
    assert torch.equal(out.isnan(), want)
    assert torch.equal(out[~want], good[~want])


def test_attention_lengths_that_contradict(cuda):
    s = _make(cuda, 4, 2, 64, 16, [(2, 50), (3, 60), (1, 20)], "bf16", 12)
    good = _run(s, 32, 2)
    kp = s["kp"].clone()
    for kl in (2, 10 ** 6, -1):  # below its new tokens, past its table, negative
        s["kl"][1] = kl
        out = _run(s, 32, 2)
        assert out[2:5].isnan().all() and _same(out[:2], good[:2]) and _same(out[5:], good[5:])
        assert _same(s["kp"], kp)


def test_attention_does_not_depend_on_other_sequences(cuda):
    # a batch gives each sequence the bits that it gets alone under the same bounds
    lens = [(1, 500), (1, 77), (1, 1)]
    s = _make(cuda, 8, 2, 128, 16, lens, "bf16", 13)
    all_ = _run(s, 100, 4)
    again = _run(s, 100, 4)
    assert _same(all_, again)


def test_attention_empty(cuda):
    s = _make(cuda, 4, 2, 64, 16, [(0, 40), (0, 0)], "f16", 14)
    kp = s["kp"].clone()
    assert _run(s, 32, 2).shape == (0, 4, 64) and _same(s["kp"], kp)


@pytest.mark.parametrize("lens", [[(1, 700), (1, 30)], [(1, 6000)], [(150, 400), (1, 90)]])
def test_attention_on_a_stream_and_in_a_graph(cuda, lens):
    s = _make(cuda, 8, 1, 128, 16, lens, "bf16", 15)
    _run(s, 4000, 4)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        _run(s, 4000, 4)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = _run(s, 4000, 4)
    torch.cuda.current_stream().wait_stream(st)
    for i in range(3):
        s["q"].mul_(1.1)
        s["k"].mul_(0.9)
        want = _run(s, 4000, 4)
        kp = s["kp"].clone()
        s["kp"][int(s["table"][0, (lens[0][1] - 1) // 16])].zero_()
        s["kp"].copy_(kp)
        g.replay()
        torch.cuda.synchronize()
        assert _same(out, want) and _same(s["kp"], kp)


def test_attention_offsets_past_32_bits(cuda):
    # 2^31 elements of K in front of the pages that are used
    hkv, d, page = 8, 128, 16
    pages = 2 ** 31 // (page * hkv * d) + 40
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 12 GiB")
    s = _make(cuda, 8, hkv, d, page, [(1, 300), (40, 60)], "f16", 16)
    n = s["kp"].shape[0]
    kp, vp = (torch.empty(pages, page, hkv, d, dtype=torch.float16, device=cuda) for _ in "kv")
    kp[pages - n:], vp[pages - n:] = s["kp"], s["vp"]
    o, big, _, _ = _ref(s, 100, 4, None, s["kp"], s["vp"])
    s["table"] = torch.where(s["table"] >= 0, s["table"] + (pages - n), s["table"])
    s["kp"], s["vp"] = kp, vp
    out = _run(s, 100, 4)
    assert ((out.double() - o).abs() <= 2.0 ** -11 * (o.abs() + big) + 2.0 ** -12 * big + 2.0 ** -14).all()
