"""Performance cases of the operators of a served language model's block: the
RMS norm that adds the residual and leaves 8-bit rows with scales, the 8-bit
product with bias, activation and residual in its epilogue, and attention over
a paged cache with a sliding window and first tokens that stay visible.

`run` computes them in their plain form from torch's elementary operations, or
through the framework's layers where `own` is true.  The listed cases stand
for ranges that `draw` samples.

Inputs: activations N(0, 1) with a few large channels, as residual streams
have them; 8-bit operands quantized from normals, a scale per row of the
activations and per output of the weights; queries, keys and values N(0, 1);
pages handed out in no order.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_Q8 = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
_EPS = 1e-5

_MM_OPS = 2.0 * 8192 * 4096 * 8192
_NORM_VALUES = 16384 * 4096
_ATTN_SCORES = 32.0 * 8192 * 8192       # scores the plain form holds at once
_ATTN_CACHE = 64.0 * 8192 * 8 * 128     # values of K in the cache


def listed():
    return [
        # one token's residual stream in an answer being written: latency
        dict(name="norm_token", kind="norm", rows=1, cols=4096, dtype="bf16", q="e4m3", res=True),
        # a ragged sequence at an odd width (rows without alignment), into int8
        dict(name="norm_ragged", kind="norm", rows=1028, cols=1283, dtype="f16", q="int8", res=True),
        # a batch of prompts: memory-bound
        dict(name="norm_large", kind="norm", rows=16384, cols=4096, dtype="bf16", q="e4m3", res=True),
        # one token through a small projection: latency
        dict(name="mm_token", kind="mm", m=1, k=768, n=768, q="int8", dtype="f32", act="None", bias=True, res=False),
        # a step of 24 sequences through a feed-forward layer: reads the weights
        dict(name="mm_decode", kind="mm", m=24, k=4096, n=8192, q="e4m3", dtype="bf16", act="Silu", bias=True,
             res=False),
        # a ragged sequence through an encoder's feed-forward layer
        dict(name="mm_ragged", kind="mm", m=1028, k=1280, n=5120, q="int8", dtype="f16", act="Gelu", bias=True,
             res=False),
        # a batch of prompts back into the residual stream: the throughput end
        dict(name="mm_large", kind="mm", m=8192, k=4096, n=8192, q="e4m3", dtype="bf16", act="None", bias=False,
             res=True),
        # one token of one sequence: latency
        dict(name="attn_token", kind="attn", b=1, hq=12, hkv=4, d=64, q_max=1, kv_max=600, window=512, sinks=4,
             page=16, dtype="f16", ragged=False),
        # a step of 64 sequences of different lengths: reads the cache
        dict(name="attn_decode", kind="attn", b=64, hq=32, hkv=8, d=128, q_max=1, kv_max=8192, window=4096, sinks=4,
             page=64, dtype="bf16", ragged=True),
        # few sequences with long histories: one sequence has to fill the card
        dict(name="attn_decode_long", kind="attn", b=3, hq=32, hkv=8, d=128, q_max=1, kv_max=65536, window=32768,
             sinks=16, page=64, dtype="bf16", ragged=False),
        # pieces of prompts behind histories of odd lengths, heads of 80
        dict(name="attn_chunks", kind="attn", b=5, hq=16, hkv=4, d=80, q_max=701, kv_max=3001, window=1024, sinks=4,
             page=16, dtype="f16", ragged=True),
        # a whole long prompt
        dict(name="attn_prompt", kind="attn", b=1, hq=32, hkv=8, d=128, q_max=8192, kv_max=8192, window=2048, sinks=4,
             page=64, dtype="bf16", ragged=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "mm", "mm", "attn", "attn"])
    while True:
        if kind == "norm":
            dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
            # rounding to int8 is compared at 16 bits, so FP32 rows go into e4m3
            q = "e4m3" if dtype == "f32" else rng.choice(["int8", "e4m3"])
            c = dict(kind="norm", rows=_log_int(rng, 1, 16384), cols=_log_int(rng, 64, 16384), dtype=dtype, q=q,
                     res=rng.random() < 0.7)
            if rng.random() < 0.6:  # the round widths of real models
                c["cols"] = (c["cols"] + 63) // 64 * 64
            if c["rows"] * c["cols"] <= _NORM_VALUES // (2 if dtype == "f32" else 1):
                return c
        elif kind == "mm":
            c = dict(kind="mm", m=_log_int(rng, 1, 8192), k=_log_int(rng, 64, 8192), n=_log_int(rng, 64, 8192),
                     q=rng.choice(["int8", "e4m3"]), dtype=rng.choice(["f32", "f16", "bf16", "bf16"]),
                     act=rng.choice(["None", "Relu", "Silu", "Gelu"]), bias=rng.random() < 0.5,
                     res=rng.random() < 0.5)
            if rng.random() < 0.7:
                c["k"], c["n"] = (c["k"] + 63) // 64 * 64, (c["n"] + 63) // 64 * 64
            if 2.0 * c["m"] * c["k"] * c["n"] <= _MM_OPS:
                return c
        else:
            hkv = rng.choice([1, 2, 4, 8])
            q_max = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 4096)])
            c = dict(kind="attn", b=_log_int(rng, 1, 64), hq=hkv * rng.choice([1, 2, 3, 4, 8]), hkv=hkv,
                     d=rng.choice([32, 64, 80, 96, 128, 128, 256]), q_max=q_max,
                     kv_max=q_max + _log_int(rng, 1, 16384) - 1, window=_log_int(rng, 16, 8192),
                     sinks=rng.choice([0, 1, 4, 4, 16, 130]), page=rng.choice([16, 32, 64, 128]),
                     dtype=rng.choice(["f16", "bf16"]), ragged=rng.random() < 0.6)
            if (1.0 * c["b"] * c["hq"] * c["q_max"] * c["kv_max"] <= _ATTN_SCORES / 4
                    and 1.0 * c["b"] * c["kv_max"] * c["hkv"] * c["d"] <= _ATTN_CACHE / 4):
                return c


# ------------------------------------------------------------------- inputs

def _quantize(v, q):
    """Rows of v in 8 bits, and the rows' scales."""
    t, top = _Q8[q]
    s = v.abs().amax(1) / top
    v = (v / s[:, None]).clamp(-top, top)
    return (v.round() if q == "int8" else v).to(t), s


def _lens(case, seed):
    """The sequences' new and whole lengths, as the host of a server knows them: the
    case's own lengths, with the histories dealt out by the seed."""
    b, q_max, past = case["b"], case["q_max"], case["kv_max"] - case["q_max"]
    if not case["ragged"]:
        return [q_max] * b, [q_max + past] * b
    g = torch.Generator().manual_seed(b * 1000003 + q_max * 1009 + past)
    ql = torch.randint((q_max + 3) // 4, q_max + 1, (b,), generator=g)
    old = torch.randint(past // 4, past + 1, (b,), generator=g)
    ql[0], old[-1] = q_max, past
    old = old[torch.randperm(b, generator=g.manual_seed(seed))]
    return ql.tolist(), (ql + old).tolist()


def prepare(case, seed):
    seed = int(seed) % (1 << 62)
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    s = dict(case)
    if case["kind"] == "norm":
        t = _DT[case["dtype"]]
        loud = 1.0 + 20.0 * (torch.rand(case["cols"], generator=g, device="cuda") < 0.01).float()
        s["x"] = normal(case["rows"], case["cols"]).to(t)
        s["r"] = (normal(case["rows"], case["cols"]) * loud).to(t) if case["res"] else None
        s["gamma"] = (1.0 + 0.2 * normal(case["cols"])).to(t)
    elif case["kind"] == "mm":
        m, n, k, t = case["m"], case["n"], case["k"], _DT[case["dtype"]]
        s["a"], s["sa"] = _quantize(normal(m, k), case["q"])
        s["w"], s["sw"] = _quantize(normal(n, k) / math.sqrt(k), case["q"])
        s["b"] = 0.1 * normal(n) if case["bias"] else None
        s["r"] = normal(m, n).to(t) if case["res"] else None
    else:
        t, b, page = _DT[case["dtype"]], case["b"], case["page"]
        ql, kl = _lens(case, seed)
        width = (case["kv_max"] + page - 1) // page
        shape = (b * width, page, case["hkv"], case["d"])
        s["kp"], s["vp"] = normal(*shape).to(t), normal(*shape).to(t)
        s["table"] = torch.randperm(b * width, generator=g, device="cuda").reshape(b, width).to(torch.int32)
        starts = [sum(ql[:i]) for i in range(b + 1)]
        s["cu"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        s["kl"] = torch.tensor(kl, dtype=torch.int32, device="cuda")
        s["x"] = normal(starts[-1], case["hq"], case["d"]).to(t)
        s["k"] = normal(starts[-1], case["hkv"], case["d"]).to(t)
        s["v"] = normal(starts[-1], case["hkv"], case["d"]).to(t)
    return s


# -------------------------------------------------------------- plain forms

def _activate(y, act):
    if act == "Relu":
        return torch.where(y > 0, y, torch.zeros_like(y))
    if act == "Silu":
        return y / (1.0 + torch.exp(-y))
    if act == "Gelu":
        return 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    return y


def _plain_norm(s):
    t, top = _Q8[s["q"]]
    h = s["x"] if s["r"] is None else (s["x"].float() + s["r"].float()).to(s["x"].dtype)
    f = h.float()
    y = f * (1.0 / torch.sqrt((f * f).mean(1, keepdim=True) + _EPS)) * s["gamma"].float()
    scale = y.abs().amax(1) / top
    v = (y / scale[:, None]).clamp(-top, top)
    return h, (v.round() if s["q"] == "int8" else v).to(t), scale


def _plain_mm(s):
    y = (s["a"].float() @ s["w"].float().t().contiguous()) * s["sa"][:, None] * s["sw"]
    if s["b"] is not None:
        y = y + s["b"]
    y = _activate(y, s["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    return y.to(_DT[s["dtype"]])


def _plain_attn(s):
    b, hq, hkv, d, page, q_max = s["b"], s["hq"], s["hkv"], s["d"], s["page"], s["q_max"]
    x, table, cu, kl = s["x"], s["table"].long(), s["cu"].long(), s["kl"].long()
    # the new tokens' sequences and positions, and their places in the cache
    tok = torch.arange(x.shape[0], device=x.device)
    seq = torch.searchsorted(cu, tok, right=True) - 1
    pos = kl[seq] - (cu[seq + 1] - tok)
    place = (table[seq, pos // page], pos % page)
    s["kp"][place] = s["k"]
    s["vp"][place] = s["v"]
    # every sequence's keys and values in order, queries padded to the longest
    keys = s["kp"][table].reshape(b, -1, hkv, d).float().permute(0, 2, 3, 1).contiguous()
    vals = s["vp"][table].reshape(b, -1, hkv, d).float().transpose(1, 2).contiguous()
    row = tok - cu[seq]
    q = torch.zeros((b, q_max, hq, d), device=x.device)
    q[seq, row] = x.float()
    q = q.reshape(b, q_max, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    p = torch.zeros((b, q_max), dtype=torch.long, device=x.device)
    p[seq, row] = pos
    j = torch.arange(keys.shape[3], device=x.device)
    seen = (j <= p[..., None]) & ((j > p[..., None] - s["window"]) | (j < s["sinks"]))
    e = torch.matmul(q, keys).mul_(1.0 / math.sqrt(d)).reshape(b, hkv, hq // hkv, q_max, -1)
    e = e.masked_fill_(~seen[:, None, None], -math.inf)
    e = e.sub_(e.amax(-1, keepdim=True)).exp_()
    e = e.div_(e.sum(-1, keepdim=True)).reshape(b, hkv, -1, keys.shape[3])
    o = torch.matmul(e, vals).reshape(b, hq, q_max, d).transpose(1, 2)
    return o[seq, row].to(x.dtype), s["kp"], s["vp"]


# -------------------------------------------------------------------- calls

def _own_norm(s):
    from onnxsharp_amd.lm_layers import RmsNormQuantLayer
    return RmsNormQuantLayer(eps=_EPS, q_type=s["q"]).forward(s["x"], s["gamma"], s["r"])


def _own_mm(s):
    from onnxsharp_amd.lm_layers import QuantMatMulLayer
    layer = QuantMatMulLayer(activation=None if s["act"] == "None" else s["act"], out_dtype=_DT[s["dtype"]])
    return layer.forward(s["a"], s["sa"], s["w"], s["sw"], s["b"], s["r"])


def _own_attn(s):
    from onnxsharp_amd.lm_layers import PagedKvCache, WindowAttentionLayer
    cache = PagedKvCache(s["kp"], s["vp"], s["table"])
    layer = WindowAttentionLayer(window=s["window"], sinks=s["sinks"])
    o = layer.forward(s["x"], s["k"], s["v"], cache, s["cu"], s["kl"], max_q=s["q_max"], max_kv=s["kv_max"])
    return o, s["kp"], s["vp"]


def run(state):
    kind = state["kind"]
    if kind == "norm":
        h, q, scale = _own_norm(state) if own else _plain_norm(state)
        if state["q"] == "int8":  # the values that the integers stand for
            q = torch.mul(q, scale[:, None], out=torch.empty_like(h))
        return h, q, scale
    if kind == "mm":
        return _own_mm(state) if own else _plain_mm(state)
    return _own_attn(state) if own else _plain_attn(state)


# --------------------------------------------------------------------- work

def _pairs(ql, kl, window, sinks):
    """Visible (query, key) pairs of one sequence, and the keys that any query sees."""
    start = kl - ql
    pairs = sum(min(p + 1, window) + min(sinks, max(0, p + 1 - window)) for p in range(start, kl))
    first = max(0, start - window + 1)
    return pairs, kl - first + min(sinks, first)


def work(case):
    if case["kind"] == "norm":
        n, e = case["rows"] * case["cols"], _DT[case["dtype"]].itemsize
        return dict(bytes=n * ((3 if case["res"] else 1) * e + 1) + case["cols"] * e + 4 * case["rows"],
                    flops=8.0 * n)
    if case["kind"] == "mm":
        m, n, k, e = case["m"], case["n"], case["k"], _DT[case["dtype"]].itemsize
        return dict(bytes=m * k + n * k + 4 * (m + n * (2 if case["bias"] else 1))
                    + m * n * e * (2 if case["res"] else 1), flops=2.0 * m * n * k)
    ql, kl = _lens(case, 0)
    both = [_pairs(x, y, case["window"], case["sinks"]) for x, y in zip(ql, kl)]
    e, d = _DT[case["dtype"]].itemsize, case["d"]
    return dict(bytes=2 * e * d * (case["hkv"] * (sum(k for _, k in both) + 2 * sum(ql)) + case["hq"] * sum(ql)),
                flops=4.0 * d * case["hq"] * sum(p for p, _ in both))


# ------------------------------------------------------- results in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        t, top = _Q8[case["q"]]
        h = s["x"].double()
        if s["r"] is not None:
            h = (h + s["r"].double()).to(s["x"].dtype).double()
        y = h / (h.pow(2).sum(1, keepdim=True) / case["cols"] + _EPS).sqrt() * s["gamma"].double()
        scale = y.abs().max(1, keepdim=True).values / top
        if case["q"] == "int8":
            return h, (y / scale).round() * scale, scale[:, 0]
        return h, (y / scale).to(t).double(), scale[:, 0]
    if case["kind"] == "mm":
        y = (s["a"].double() * s["sa"].double()[:, None]) @ (s["w"].double() * s["sw"].double()[:, None]).T
        if s["b"] is not None:
            y += s["b"].double()
        if case["act"] == "Relu":
            y = y.clamp(min=0)
        elif case["act"] == "Silu":
            y = y * torch.sigmoid(y)
        elif case["act"] == "Gelu":
            y = y * 0.5 * torch.erfc(-y / math.sqrt(2.0))
        return y if s["r"] is None else y + s["r"].double()
    # one sequence and one head of keys at a time, over its own tokens
    out = torch.empty(s["x"].shape, dtype=torch.float64, device="cuda")
    ql, kl = _lens(case, int(seed) % (1 << 62))
    groups, page, start = case["hq"] // case["hkv"], case["page"], 0
    for i, (nq, nk) in enumerate(zip(ql, kl)):
        at = torch.arange(nk, device="cuda")
        pages, slots = s["table"][i, at // page].long(), at % page
        s["kp"][pages[nk - nq:], slots[nk - nq:]] = s["k"][start:start + nq]
        s["vp"][pages[nk - nq:], slots[nk - nq:]] = s["v"][start:start + nq]
        p = at[nk - nq:, None]
        hidden = (at > p) | ((at <= p - case["window"]) & (at >= case["sinks"]))
        for h in range(case["hkv"]):
            k, v = s["kp"][pages, slots, h].double(), s["vp"][pages, slots, h].double()
            for u in range(h * groups, (h + 1) * groups):
                logits = s["x"][start:start + nq, u].double() @ k.T / math.sqrt(case["d"])
                out[start:start + nq, u] = torch.softmax(logits.masked_fill(hidden, -math.inf), 1) @ v
        start += nq
    return out, s["kp"], s["vp"]
