"""GPU: a decoder block of BlockNormLayer, Int4MatMulLayer and WindowAttentionLayer over a
PagedKv4Cache against the same block in 64 bits, which rounds where the block rounds.

Bounds.  The weights are the packed codes' own values.  A key or value may take the neighbouring
code where its 16-bit rounding falls the other way: it stays within a step and the rounding of
what the formula gives, and the attention goes on from what the cache holds.  After that the
stream passes eight 16-bit roundings (q, o, branch, h, y, up, down, h) of at most 2^-8 of a value
each, and norms and residuals that do not enlarge them: 2^-5 of the stream's norm."""
import pytest
import torch

from onnxsharp_amd.decoder import Int4DecoderBlock, main, random_weights
from onnxsharp_amd.lm_layers import Int4MatMulLayer, PagedKv4Cache

pytestmark = pytest.mark.gpu
HQ, HKV, D, WIDTH, HIDDEN, PAGE = 8, 2, 64, 384, 640, 16


def _rms(x, gamma, eps=1e-5):
    return x / (x.pow(2).mean(1, keepdim=True) + eps).sqrt() * gamma.double()


def _cached(codes, pairs, group):
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double().unflatten(-1, (-1, group))
    p = pairs.double()
    return (p[..., 1:] + p[..., :1] * c).flatten(-2), p[..., 0].repeat_interleave(group, -1)


@pytest.mark.parametrize("group,zeros,dtype", [(64, True, torch.bfloat16), (32, False, torch.float16)])
def test_block_prompts_then_tokens(cuda, group, zeros, dtype):
    window, sinks = 48, 3
    block = Int4DecoderBlock(random_weights(WIDTH, HIDDEN, HQ, HKV, D, cuda, 5), HQ, HKV, D, window, sinks, group, zeros,
                             dtype=dtype)
    # what the packed weights stand for, through the product with the unit matrix (exact: one term)
    w = {n: Int4MatMulLayer().forward(torch.eye(p.k, device=cuda, dtype=dtype), p).double().T for n, p in block.w.items()}
    g, n = torch.Generator(device=cuda).manual_seed(6), 36  # 12 pages each: 192 positions for at most 187
    cache = PagedKv4Cache.empty(n, PAGE, HKV, D, torch.randperm(n, device=cuda).to(torch.int32).view(3, 12), 32, dtype)
    r = lambda t: t.to(dtype).double()  # noqa: E731
    lens = [0, 0, 0]
    # prompts, a piece of one beside single tokens, then single tokens alone
    for new in ([140, 33, 1], [41, 1, 1], [1, 1, 1], [1, 0, 1], [4, 100, 2]):
        lens = [a + b for a, b in zip(lens, new)]
        cu = [sum(new[:i]) for i in range(4)]
        x = torch.randn(cu[-1], WIDTH, generator=g, device=cuda).to(dtype)
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
        out = block.forward(x, cache, ints(cu), ints(lens), max(new), max(lens))
        for i in range(3):
            if not new[i]:
                continue
            xs = x[cu[i]:cu[i + 1]].double()
            qkv = r(r(_rms(xs, block.gamma["norm1"])) @ w["qkv"].T).view(-1, HQ + 2 * HKV, D)
            at = torch.arange(lens[i], device=cuda)
            pg, slot = cache.table[i, at // PAGE].long(), at % PAGE
            k, k_step = _cached(cache.k_codes[pg, slot], cache.k_scales[pg, slot], 32)
            v, v_step = _cached(cache.v_codes[pg, slot], cache.v_scales[pg, slot], 32)
            for got, step, want in ((k, k_step, qkv[:, HQ:HQ + HKV]), (v, v_step, qkv[:, HQ + HKV:])):
                got, step = got[-new[i]:], step[-new[i]:]
                # a group's ends may move with their roundings too
                top = want.abs().unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1)
                assert ((got - want).abs() <= step + 2.0 ** -6 * top).all()
            pos = torch.arange(lens[i] - new[i], lens[i], device=cuda)[:, None]
            seen = (at <= pos) & ((at > pos - window) | (at < sinks))
            o = torch.empty(new[i], HQ, D, dtype=torch.float64, device=cuda)
            for h in range(HQ):
                e = (qkv[:, h] @ k[:, h // (HQ // HKV)].T.contiguous()) * D ** -0.5
                o[:, h] = torch.softmax(e.masked_fill(~seen, float("-inf")), 1) @ v[:, h // (HQ // HKV)].contiguous()
            branch = r(r(o).reshape(new[i], -1) @ w["out"].T)
            hs = r(xs + torch.sigmoid(block.gamma["gate"].double()) * _rms(branch, block.gamma["post1"]))
            up = r(_rms(hs, block.gamma["norm3"])) @ w["up"].T
            down = r(r(up * torch.sigmoid(up)) @ w["down"].T)
            want = r(hs + _rms(down, block.gamma["post2"]))
            err = float((out[cu[i]:cu[i + 1]].double() - want).norm() / want.norm())
            print(group, zeros, dtype, new, i, err, flush=True)
            assert err <= 2.0 ** -5


def test_example_runs(cuda, capsys):
    main(tokens=40, steps=2, four=True)
    assert capsys.readouterr().out.count("rms") == 3
