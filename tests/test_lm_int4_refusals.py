"""Refusals of the operators of a decoder block in 4 bits, before anything touches a device: the
layers' checks on host tensors and the C entry points' on pointers that are never read."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

from onnxsharp_amd import native as N
from onnxsharp_amd.lm_layers import (BlockNormLayer, Int4MatMulLayer, Int4Weight, PagedKv4Cache, PagedKvCache,
                                     WindowAttentionLayer)

INCLUDE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
E, U, OK = N.OSH_E_INVALID, N.OSH_E_UNSUPPORTED, N.OSH_OK


def _p(i, off=0):
    return C.c_void_p((i << 40) + off)  # distinct addresses, never dereferenced


# ------------------------------------------------------------------- layers

def test_block_norm_layer_refusals():
    with pytest.raises(ValueError, match="eps"):
        BlockNormLayer(eps=-1.0)
    with pytest.raises(ValueError, match="gate activation"):
        BlockNormLayer(gate_activation="Relu")
    f, x, g = BlockNormLayer().forward, torch.zeros(3, 16), torch.zeros(16)
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        f(x.double(), g)
    with pytest.raises(N.OshError, match="rows, cols"):
        f(x[0], g)
    with pytest.raises(N.OshError, match="neither"):
        f(x)
    for kw in (dict(post_gamma=g), dict(gate=g), dict(out_h=x)):
        with pytest.raises(N.OshError, match="without a branch"):
            f(x, g, **kw)
    with pytest.raises(N.OshError, match="branch must"):
        f(x, g, x[:2])
    with pytest.raises(TypeError, match="post_gamma"):
        f(x, g, x, g.half())
    with pytest.raises(N.OshError, match="gate"):
        f(x, g, x, None, x[:, :8])
    with pytest.raises(N.OshError, match="contiguous rows"):
        f(x, g, x, out_h=torch.zeros(16, 3).t())
    with pytest.raises(ValueError, match="device tensors"):
        f(x, g, x)


def test_int4_layer_refusals():
    codes, scales, zeros = torch.zeros(5, 50, dtype=torch.uint8), torch.zeros(5, 4), torch.zeros(5, 2, dtype=torch.uint8)
    for k, group, match in ((98, 32, "codes must"), (0, 32, "codes must"), (99, 0, "codes must"), (99, 64, "scales must")):
        with pytest.raises(N.OshError, match=match):
            Int4Weight(codes, scales, zeros, k=k, group=group)
    with pytest.raises(TypeError, match="codes"):
        Int4Weight(codes.char(), scales, zeros, k=99, group=32)
    with pytest.raises(TypeError, match="scales"):
        Int4Weight(codes, scales.double(), zeros, k=99, group=32)
    with pytest.raises(N.OshError, match="zeros must"):
        Int4Weight(codes, scales, zeros[:, :1], k=99, group=32)
    with pytest.raises(ValueError, match="device tensors"):
        Int4Weight(codes, scales, zeros, k=99, group=32)
    with pytest.raises(ValueError, match="cannot be fused"):
        Int4MatMulLayer("Tanh")
    w = Int4Weight.__new__(Int4Weight)
    w.n, w.k, w.group, w.dtype, w.has_zeros, w.packed = 5, 99, 32, torch.float32, True, codes
    f, a = Int4MatMulLayer().forward, torch.zeros(3, 99)
    with pytest.raises(TypeError, match="scales"):
        f(a.half(), w)
    with pytest.raises(N.OshError, match="a must"):
        f(a[:, :98], w)
    with pytest.raises(TypeError, match="bias"):
        f(a, w, torch.zeros(5).half())
    with pytest.raises(N.OshError, match="residual"):
        f(a, w, None, torch.zeros(3, 4))
    with pytest.raises(N.OshError, match="contiguous rows"):
        f(a, w, out=torch.zeros(5, 3).t())
    with pytest.raises(ValueError, match="device tensors"):
        f(a, w)


def test_kv4_cache_refusals():
    codes = torch.zeros(4, 16, 2, 32, dtype=torch.uint8)
    scales, table = torch.zeros(4, 16, 2, 2, 2, dtype=torch.float16), torch.zeros(2, 2, dtype=torch.int32)
    make = lambda k=codes, v=codes, ks=scales, vs=scales, t=table: PagedKv4Cache(k, v, ks, vs, t)  # noqa: E731
    assert make().group == 32 and make().head_dim == 64
    with pytest.raises(N.OshError, match="codes must"):
        make(codes[0])
    with pytest.raises(TypeError, match="k_codes"):
        make(codes.char())
    with pytest.raises(N.OshError, match="v_codes"):
        make(v=codes[:3])
    with pytest.raises(N.OshError, match="scales must"):
        make(ks=scales[..., 0])
    with pytest.raises(TypeError, match="scales must"):
        make(ks=scales.float())
    with pytest.raises(TypeError, match="v_scales"):
        make(vs=scales.bfloat16())
    with pytest.raises(N.OshError, match="groups"):
        make(ks=torch.zeros(4, 16, 2, 3, 2).half(), vs=torch.zeros(4, 16, 2, 3, 2).half())
    with pytest.raises(N.OshError, match="codes must be contiguous"):
        make(codes.transpose(2, 3).contiguous().transpose(2, 3))
    with pytest.raises(N.OshError, match="scales must be contiguous"):
        make(ks=scales.transpose(3, 4).contiguous().transpose(3, 4))
    with pytest.raises(TypeError, match="table"):
        make(t=table.long())
    cache = make()
    q, k = torch.zeros(3, 4, 64, dtype=torch.float16), torch.zeros(3, 2, 64, dtype=torch.float16)
    cu, kl = torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    f = WindowAttentionLayer(window=8).forward
    with pytest.raises(TypeError, match="the cache"):
        f(q.bfloat16(), k, k, cache, cu, kl, 3, 3)
    with pytest.raises(N.OshError, match="stored"):
        f(q, k, k, cache, cu, kl, 3, 3, stored=(k, k[:2]))
    with pytest.raises(N.OshError, match="stored must"):
        f(q, k, k, cache, cu, kl, 3, 3, stored=(k, k.transpose(1, 2).contiguous().transpose(1, 2)))
    pages = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    with pytest.raises(N.OshError, match="not held in 4 bits"):
        f(q, k, k, PagedKvCache(pages, pages.clone(), table), cu, kl, 3, 3, stored=(k, k.clone()))
    with pytest.raises(ValueError, match="device tensors"):
        f(q, k, k, cache, cu, kl, 3, 3)


# ---------------------------------------------------------- C entry points

def _norm(rows=4, cols=16, dtype=N.T_BF16, x=_p(1), ldx=16, b=_p(2), ldb=16, post=_p(3), gate=_p(4), ldg=0,
          act=N.ACT_SIGMOID, gamma=_p(5), eps=1e-5, h=_p(6), ldh=16, y=_p(7), ldy=16):
    return N.lib().osh_block_norm(rows, cols, dtype, x, ldx, 1.0, b, ldb, 1.0, post, gate, ldg, act, gamma, eps, h, ldh, y,
                                  ldy, None)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(rows=-1), E, "negative"), (dict(cols=0), E, "without columns"), (dict(dtype=N.T_I8), E, "f32"),
    (dict(eps=float("nan")), E, "eps"), (dict(act=N.ACT_RELU), E, "sigmoid"), (dict(b=None), E, "not there"),
    (dict(b=None, post=None, gate=None, gamma=None), E, "neither"), (dict(x=None), E, "NULL"), (dict(h=None), E, "NULL"),
    (dict(y=None), E, "NULL"), (dict(ldx=15), E, "pitch"), (dict(ldh=15), E, "pitch"), (dict(ldg=15), E, "pitch"),
    (dict(cols=32769, ldx=40000, ldb=40000, ldh=40000, ldy=40000), U, "at most"),
    (dict(h=_p(1, 2)), E, "without being it"), (dict(h=_p(2), ldh=17), E, "without being it"),
    (dict(h=_p(5)), E, "overlaps another"), (dict(y=_p(1)), E, "overlaps another"), (dict(y=_p(6)), E, "overlaps another"),
    (dict(y=_p(4)), E, "overlaps another"), (dict(rows=0, x=None), OK, None),
])
def test_block_norm_entry_refusals(kw, status, msg):
    assert _norm(**kw) == status
    assert not msg or msg in N.last_error()


def _pack(n=8, k=64, group=32, dtype=N.T_F16, codes=_p(1), ldc=32, scales=_p(2), lds=2, zeros=_p(3), ldz=1, out=_p(4)):
    return N.lib().osh_int4_pack(n, k, group, dtype, codes, ldc, scales, lds, zeros, ldz, out, None)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(n=-1), E, "negative"), (dict(k=0), E, "k is 0"), (dict(dtype=N.T_I8), E, "f32"), (dict(group=0), E, "groups of 0"),
    (dict(group=48), U, "groups of 48"), (dict(group=192, lds=1), U, "groups of 192"), (dict(codes=None), E, "NULL"),
    (dict(ldc=31), E, "pitch"), (dict(lds=1), E, "pitch"), (dict(ldz=0), E, "pitch"), (dict(out=_p(4, 8)), E, "16-byte"),
    (dict(out=_p(1)), E, "overlap"), (dict(out=_p(3)), E, "overlap"), (dict(k=(1 << 28) + 1), U, "weights"),
    (dict(n=0, codes=None), OK, None),
])
def test_int4_pack_entry_refusals(kw, status, msg):
    assert _pack(**kw) == status
    assert not msg or msg in N.last_error()


def _mm(m=4, n=8, k=64, group=32, dtype=N.T_F16, a=_p(1), lda=64, w=_p(2), zeros=1, bias=_p(3), act=N.ACT_SILU, res=_p(4),
        ldr=8, y=_p(5), ldy=8, scratch=_p(6)):
    return N.lib().osh_int4_matmul(m, n, k, group, dtype, a, lda, w, zeros, bias, act, res, ldr, y, ldy, scratch, None)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(m=-1), E, "negative"), (dict(k=0), E, "k is 0"), (dict(dtype=N.T_I8), E, "f32"), (dict(group=96), U, "groups"),
    (dict(act=N.ACT_SIGMOID), E, "activation"), (dict(w=None), E, "NULL"), (dict(lda=63), E, "pitch"),
    (dict(ldy=7), E, "pitch"), (dict(ldr=7), E, "pitch"), (dict(w=_p(2, 8)), E, "16-byte"),
    (dict(m=1 << 20, n=1 << 20, ldy=1 << 20, ldr=1 << 20), U, "outputs"),
    (dict(m=4000, k=100, lda=100, scratch=None), E, "scratch"), (dict(m=4000, k=100, lda=100, scratch=_p(6, 4)), E, "scratch"),
    (dict(m=4000, k=100, lda=100, scratch=_p(1)), E, "scratch overlaps"),
    (dict(y=_p(1)), E, "overlaps"), (dict(y=_p(2)), E, "overlaps"), (dict(y=_p(3)), E, "overlaps"),
    (dict(y=_p(4), ldy=9), E, "overlaps"), (dict(m=0, a=None), OK, None), (dict(n=0), OK, None),
])
def test_int4_matmul_entry_refusals(kw, status, msg):
    assert _mm(**kw) == status
    assert not msg or msg in N.last_error()


def test_int4_sizes():
    n, lib = C.c_size_t(), N.lib()
    assert lib.osh_int4_packed_bytes(8, 64, 32, N.T_F16, 1, None) == E
    assert lib.osh_int4_packed_bytes(17, 129, 32, N.T_F16, 1, C.byref(n)) == OK
    assert n.value == 2 * 2 * (1024 + 2 * 4 * 16 * 2)  # 2 x 2 blocks of codes, scales and zero points
    assert lib.osh_int4_matmul_scratch_bytes(-1, 8, 64, 32, N.T_F16, C.byref(n)) == E
    assert lib.osh_int4_matmul_scratch_bytes(1, 768, 768, 32, N.T_F16, C.byref(n)) == OK and n.value == 0
    assert lib.osh_int4_matmul_scratch_bytes(0, 768, 768, 32, N.T_F16, C.byref(n)) == OK and n.value == 0


def _attn(group=64, **kw):
    w = N.WindowAttn(dtype=N.T_BF16, batch=2, q_heads=4, kv_heads=2, head_dim=64, window=32, sinks=4, max_q=2, max_kv=64,
                     pages=8, page=16, table_width=4, tokens=4, d_q=1 << 40, d_k_new=2 << 40, d_v_new=3 << 40,
                     d_o=4 << 40, d_k_pages=5 << 40, d_v_pages=6 << 40, d_table=7 << 40, d_cu=8 << 40, d_kl=9 << 40,
                     q_stride=(256, 64), k_new_stride=(128, 64), v_new_stride=(128, 64), o_stride=(256, 64),
                     k_stride=(1024, 32, 512), v_stride=(1024, 32, 512), table_stride=4)
    p = N.Kv4Attn(w=w, group=group, d_k_scales=10 << 40, d_v_scales=11 << 40, d_k_stored=12 << 40, d_v_stored=13 << 40,
                  k_scale_stride=(64, 2, 32), v_scale_stride=(64, 2, 32), k_stored_stride=(128, 64),
                  v_stored_stride=(128, 64))
    scratch = kw.pop("scratch", None)
    for f, v in kw.items():
        setattr(p if hasattr(p, f) else p.w, f, v)
    return N.lib().osh_kv4_attention(C.byref(p), scratch, None)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(dtype=N.T_F32), E, "f16 or bf16"), (dict(kv_heads=3), E, "over 3 key heads"), (dict(page=0), E, "bad sizes"),
    (dict(window=0), E, "window"), (dict(group=48), U, "groups of 48"), (dict(group=128), U, "heads of 64"),
    (dict(head_dim=96), U, "heads of 96"), (dict(batch=65536, max_q=1), U, "65536 sequences"),
    (dict(d_table=None), E, "NULL"), (dict(d_k_scales=None), E, "NULL"), (dict(d_v_stored=None), E, "NULL"),
    (dict(max_kv=6000, table_width=400, table_stride=400, window=6000), E, "NULL"),  # splits need scratch
    (dict(max_kv=6000, table_width=400, table_stride=400, window=6000, scratch=_p(20, 4)), E, "NULL"),
    (dict(o_stride=(-1, 64)), E, "negative stride"), (dict(k_scale_stride=(64, -2, 32)), E, "negative stride"),
    (dict(k_stride=(1 << 31, 32, 512)), U, "above 2"), (dict(k_stride=(1032, 32, 512)), U, "16-byte"),
    (dict(d_k_pages=(5 << 40) + 8), U, "16-byte"), (dict(v_scale_stride=(65, 2, 32)), U, "4-byte"),
    (dict(d_k_scales=(10 << 40) + 2), U, "4-byte"), (dict(table_stride=3), E, "table stride"),
    (dict(d_v_pages=5 << 40), E, "share memory"), (dict(k_stride=(0, 32, 512)), E, "share memory"),
    (dict(d_v_scales=10 << 40), E, "share memory"), (dict(d_k_stored=4 << 40), E, "share memory"),
    (dict(k_stored_stride=(64, 64)), E, "share memory"), (dict(d_o=1 << 40), E, "overlaps"),
    (dict(d_k_stored=2 << 40), E, "overlaps"), (dict(batch=0), OK, None), (dict(max_q=0), OK, None),
    (dict(tokens=0, d_q=None), OK, None),
])
def test_kv4_attention_entry_refusals(kw, status, msg):
    assert _attn(**kw) == status
    assert not msg or msg in N.last_error()


def test_kv4_attention_scratch():
    n, lib = C.c_size_t(), N.lib()
    assert lib.osh_kv4_attention_scratch_bytes(None, C.byref(n)) == E
    assert lib.osh_kv4_attention_scratch_bytes(C.byref(N.Kv4Attn()), None) == E
    assert lib.osh_kv4_attention(None, None, None) == E
    # many rows: f16 pages of what is visible, or none where they would pass 16 GiB
    w = N.WindowAttn(dtype=N.T_BF16, batch=1, q_heads=8, kv_heads=1, head_dim=128, window=1000, sinks=70, max_q=100,
                     max_kv=1 << 20, pages=1, page=16, table_width=1 << 16, tokens=100)
    p = N.Kv4Attn(w=w, group=64)
    assert lib.osh_kv4_attention_scratch_bytes(C.byref(p), C.byref(n)) == OK
    pages = (2 + 18 + 1) * 2 * 64 * 128 * 2
    assert pages < n.value < pages + (1 << 24)
    p.w.window, p.w.batch = 1 << 20, 64
    p.w.max_q = 64
    assert lib.osh_kv4_attention_scratch_bytes(C.byref(p), C.byref(n)) == OK and n.value < 1 << 30


def test_kv4_struct_has_the_c_layout(tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("no gcc")
    fields = [f for f, _ in N.Kv4Attn._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "osh_hip.h"\nint main(void) {\n'
                   + "".join(f'  printf("%zu\\n", offsetof(osh_kv4_attn, {f}));\n' for f in fields)
                   + '  printf("%zu\\n", sizeof(osh_kv4_attn));\n  return 0;\n}\n')
    subprocess.run(["gcc", "-I", INCLUDE, str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(N.Kv4Attn, f).offset for f in fields] + [C.sizeof(N.Kv4Attn)]


def test_kv4_packing_is_the_struct():
    from onnxsharp_amd.lm_layers import _KV4_ATTN, _WINDOW_ATTN
    assert _WINDOW_ATTN.size + _KV4_ATTN.size == C.sizeof(N.Kv4Attn)
    values = list(range(1, 17))
    p = N.Kv4Attn.from_buffer_copy(bytes(_WINDOW_ATTN.size) + _KV4_ATTN.pack(*values))
    got = []
    for f, t in N.Kv4Attn._fields_[1:]:
        got += list(getattr(p, f)) if issubclass(t, C.Array) else [getattr(p, f)]
    assert got == values
