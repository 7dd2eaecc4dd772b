"""Refusals of the language-model operators, before anything touches a device: the
layers' checks on host tensors and the C entry points' on pointers that are never
read.  And which keys and slots a call of osh_window_attention reaches: the kernel's
own rules (csrc/osh_window_addr.h, plain C++ on the host) against their definition."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

from onnxsharp_amd import native as N
from onnxsharp_amd.lm_layers import PagedKvCache, QuantMatMulLayer, RmsNormQuantLayer, WindowAttentionLayer

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "onnxsharp_amd", "csrc")


def _p(i):
    return C.c_void_p(i << 40)  # distinct addresses, never dereferenced


# ------------------------------------------------------------------- layers

def test_norm_layer_refusals():
    with pytest.raises(ValueError, match="q_type"):
        RmsNormQuantLayer(q_type="int4")
    with pytest.raises(ValueError, match="eps"):
        RmsNormQuantLayer(eps=-1.0)
    f = RmsNormQuantLayer().forward
    x, g = torch.zeros(3, 16), torch.zeros(16)
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        f(x.double(), g)
    with pytest.raises(TypeError, match="gamma"):
        f(x, g.half())
    with pytest.raises(N.OshError, match="gamma"):
        f(x, g[:8])
    with pytest.raises(N.OshError, match="rows, cols"):
        f(x[0], g)
    with pytest.raises(N.OshError, match="residual"):
        f(x, g, x[:2])
    with pytest.raises(N.OshError, match="without a residual"):
        f(x, g, out_h=x)
    with pytest.raises(ValueError, match="device tensors"):
        f(x, g, x)


def test_matmul_layer_refusals():
    with pytest.raises(ValueError, match="cannot be fused"):
        QuantMatMulLayer(activation="Tanh")
    with pytest.raises(ValueError, match="out_dtype"):
        QuantMatMulLayer(out_dtype=torch.int8)
    f = QuantMatMulLayer().forward
    a, w = torch.zeros(3, 8, dtype=torch.int8), torch.zeros(5, 8, dtype=torch.int8)
    sa, sw = torch.ones(3), torch.ones(5)
    with pytest.raises(TypeError, match="both be int8"):
        f(a, sa, w.to(torch.float8_e4m3fn), sw)
    with pytest.raises(TypeError, match="both be int8"):
        f(a.float(), sa, w, sw)
    with pytest.raises(N.OshError, match=r"\[m, k\] and \[n, k\]"):
        f(a, sa, w.t(), sw)
    with pytest.raises(N.OshError, match="w_scale"):
        f(a, sa, w, sw[:4])
    with pytest.raises(TypeError, match="a_scale"):
        f(a, sa.half(), w, sw)
    with pytest.raises(TypeError, match="residual"):
        f(a, sa, w, sw, residual=torch.zeros(3, 5))
    with pytest.raises(ValueError, match="device tensors"):
        f(a, sa, w, sw)


def test_attention_layer_refusals():
    for kw in (dict(window=0), dict(sinks=-1), dict(scale=0.0), dict(scale=float("nan"))):
        with pytest.raises(ValueError):
            WindowAttentionLayer(**kw)
    pages = torch.zeros(4, 16, 2, 32, dtype=torch.float16)
    table = torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(TypeError, match="table"):
        PagedKvCache(pages, pages, table.long())
    with pytest.raises(N.OshError, match="v_pages"):
        PagedKvCache(pages, pages[:3], table)
    with pytest.raises(TypeError, match="pages"):
        PagedKvCache(pages.float(), pages.float(), table)
    with pytest.raises(N.OshError, match="contiguous"):
        PagedKvCache(pages.transpose(2, 3), pages.transpose(2, 3), table)
    with pytest.raises(N.OshError, match="table"):
        PagedKvCache(pages, pages, table.t())
    cache = PagedKvCache(pages, pages.clone(), table)
    q, k = torch.zeros(3, 4, 32, dtype=torch.float16), torch.zeros(3, 2, 32, dtype=torch.float16)
    cu, kl = torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    f = WindowAttentionLayer(window=8).forward
    with pytest.raises(N.OshError, match="q must be"):
        f(q[..., :16], k, k, cache, cu, kl, 1, 1)
    with pytest.raises(TypeError, match="the cache"):
        f(q.bfloat16(), k, k, cache, cu, kl, 1, 1)
    with pytest.raises(N.OshError, match="v must"):
        f(q, k, k[:2], cache, cu, kl, 1, 1)
    with pytest.raises(TypeError, match="cu_seqlens"):
        f(q, k, k, cache, cu.long(), kl, 1, 1)
    with pytest.raises(N.OshError, match="kv_lens"):
        f(q, k, k, cache, cu, kl[:1], 1, 1)
    with pytest.raises(ValueError, match="device tensors"):
        f(q, k, k, cache, cu, kl, 1, 1)


# ---------------------------------------------------------- C entry points

def _norm(rows=4, cols=16, dtype=N.T_BF16, x=_p(1), ldx=16, res=_p(2), ldr=16, g=_p(3), eps=1e-5, h=_p(4), ldh=16,
          q_type=N.T_E4M3, q=_p(5), ldq=16, scale=_p(6)):
    return N.lib().osh_rms_norm_quant(rows, cols, dtype, x, ldx, res, ldr, g, eps, h, ldh, q_type, q, ldq, scale, None)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(rows=-1), N.OSH_E_INVALID, "negative"), (dict(cols=0), N.OSH_E_INVALID, "without columns"),
    (dict(dtype=N.T_I8), N.OSH_E_INVALID, "f32"), (dict(q_type=N.T_F16), N.OSH_E_INVALID, "int8 or e4m3"),
    (dict(eps=float("nan")), N.OSH_E_INVALID, "eps"), (dict(x=None), N.OSH_E_INVALID, "NULL"),
    (dict(h=None), N.OSH_E_INVALID, "NULL"), (dict(ldx=15), N.OSH_E_INVALID, "pitch"),
    (dict(ldh=15), N.OSH_E_INVALID, "pitch"),
    (dict(cols=32769, ldx=40000, ldr=40000, ldh=40000, ldq=40000), N.OSH_E_UNSUPPORTED, "at most"),
    (dict(h=C.c_void_p((1 << 40) + 2)), N.OSH_E_INVALID, "overlaps x"),
    (dict(h=_p(2), ldh=17), N.OSH_E_INVALID, "overlaps the residual"),
    (dict(q=_p(1)), N.OSH_E_INVALID, "overlaps another"), (dict(scale=_p(5)), N.OSH_E_INVALID, "overlaps another"),
    (dict(rows=0, x=None), N.OSH_OK, None),
])
def test_norm_entry_refusals(kw, status, msg):
    assert _norm(**kw) == status
    if msg:
        assert msg in N.last_error()


def _mm(m=4, n=8, k=16, q=N.T_I8, a=_p(1), lda=16, sa=_p(2), w=_p(3), ldw=16, sw=_p(4), bias=_p(5), act=N.ACT_SILU,
        dtype=N.T_F16, res=_p(6), ldr=8, y=_p(7), ldy=8):
    return N.lib().osh_quant_matmul(m, n, k, q, a, lda, sa, w, ldw, sw, bias, act, dtype, res, ldr, y, ldy, None)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(m=-1), N.OSH_E_INVALID, "negative"), (dict(k=0), N.OSH_E_INVALID, "k is 0"),
    (dict(q=N.T_F16), N.OSH_E_INVALID, "i8 or e4m3"), (dict(dtype=N.T_I8), N.OSH_E_INVALID, "f32"),
    (dict(act=N.ACT_SIGMOID), N.OSH_E_INVALID, "activation"), (dict(sw=None), N.OSH_E_INVALID, "NULL"),
    (dict(lda=15), N.OSH_E_INVALID, "pitch"), (dict(ldy=7), N.OSH_E_INVALID, "pitch"),
    (dict(ldr=7), N.OSH_E_INVALID, "pitch"),
    (dict(k=131072, lda=131072, ldw=131072), N.OSH_E_UNSUPPORTED, "131071"),
    (dict(m=1 << 20, n=1 << 20, ldy=1 << 20, ldr=1 << 20), N.OSH_E_UNSUPPORTED, "outputs"),
    (dict(y=_p(1)), N.OSH_E_INVALID, "overlaps"), (dict(y=_p(6), ldy=9), N.OSH_E_INVALID, "overlaps"),
    (dict(y=C.c_void_p((6 << 40) + 2)), N.OSH_E_INVALID, "overlaps"),
    (dict(m=0, a=None), N.OSH_OK, None), (dict(n=0), N.OSH_OK, None),
])
def test_matmul_entry_refusals(kw, status, msg):
    assert _mm(**kw) == status
    if msg:
        assert msg in N.last_error()


def _attn(**kw):
    p = N.WindowAttn(dtype=N.T_BF16, batch=2, q_heads=4, kv_heads=2, head_dim=64, window=32, sinks=4, max_q=2, max_kv=64,
                     pages=8, page=16, table_width=4, tokens=4, d_q=1 << 40, d_k_new=2 << 40, d_v_new=3 << 40,
                     d_o=4 << 40, d_k_pages=5 << 40, d_v_pages=6 << 40, d_table=7 << 40, d_cu=8 << 40, d_kl=9 << 40,
                     q_stride=(256, 64), k_new_stride=(128, 64), v_new_stride=(128, 64), o_stride=(256, 64),
                     k_stride=(2048, 128, 64), v_stride=(2048, 128, 64), table_stride=4)
    for f, v in kw.items():
        setattr(p, f, v)
    return N.lib().osh_window_attention(C.byref(p), None, None)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(dtype=N.T_F32), N.OSH_E_INVALID, "f16 or bf16"), (dict(kv_heads=3), N.OSH_E_INVALID, "over 3 key heads"),
    (dict(batch=-1), N.OSH_E_INVALID, "bad sizes"), (dict(page=0), N.OSH_E_INVALID, "bad sizes"),
    (dict(window=0), N.OSH_E_INVALID, "window"), (dict(sinks=-1), N.OSH_E_INVALID, "sinks"),
    (dict(scale=-1.0), N.OSH_E_INVALID, "scale"), (dict(scale=float("nan")), N.OSH_E_INVALID, "scale"),
    (dict(head_dim=60), N.OSH_E_UNSUPPORTED, "multiples of 8"), (dict(head_dim=264), N.OSH_E_UNSUPPORTED, "up to 256"),
    (dict(max_q=65), N.OSH_E_INVALID, "lengths"), (dict(max_kv=(1 << 30) + 1), N.OSH_E_UNSUPPORTED, "lengths"),
    (dict(d_table=None), N.OSH_E_INVALID, "NULL"), (dict(table_stride=3), N.OSH_E_INVALID, "table stride"),
    (dict(o_stride=(-1, 64)), N.OSH_E_INVALID, "negative stride"), (dict(d_o=1 << 40), N.OSH_E_INVALID, "overlaps"),
    (dict(batch=0), N.OSH_OK, None), (dict(max_q=0), N.OSH_OK, None), (dict(tokens=0, d_q=None), N.OSH_OK, None),
])
def test_attention_entry_refusals(kw, status, msg):
    assert _attn(**kw) == status
    if msg:
        assert msg in N.last_error()


def test_attention_scratch_refusals():
    n = C.c_size_t()
    assert N.lib().osh_window_attention_scratch_bytes(None, C.byref(n)) == N.OSH_E_INVALID
    assert N.lib().osh_window_attention_scratch_bytes(C.byref(N.WindowAttn()), None) == N.OSH_E_INVALID
    assert N.lib().osh_window_attention(None, None, None) == N.OSH_E_INVALID


def test_window_attn_struct_has_the_c_layout(tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("no gcc")
    fields = [f for f, _ in N.WindowAttn._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "osh_hip.h"\nint main(void) {\n'
                   + "".join(f'  printf("%zu\\n", offsetof(osh_window_attn, {f}));\n' for f in fields)
                   + '  printf("%zu\\n", sizeof(osh_window_attn));\n  return 0;\n}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(CSRC, "..", "..", "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(N.WindowAttn, f).offset for f in fields] + [C.sizeof(N.WindowAttn)]


def test_window_attn_packing_is_the_struct():
    from onnxsharp_amd.lm_layers import _WINDOW_ATTN
    assert _WINDOW_ATTN.size == C.sizeof(N.WindowAttn)
    values = list(range(1, 13)) + [0.5, 13] + list(range(14, 39))
    p, got = N.WindowAttn.from_buffer_copy(_WINDOW_ATTN.pack(*values)), []
    for f, t in N.WindowAttn._fields_:
        got += list(getattr(p, f)) if issubclass(t, C.Array) else [getattr(p, f)]
    assert got == values


# ------------------------------------------------- keys and slots of a call

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>
#include "osh_window_addr.h"
using namespace osh;

static void die(const char *what, int a, int b, int c) { printf("%s (%d, %d, %d)\n", what, a, b, c); exit(1); }

int main() {
    osh_window_attn p = {};
    // keys of every token range against the rule itself
    for (int window : {1, 2, 7, 32, 0x7fffffff})
        for (int sinks : {0, 1, 5, 40, 0x7fffffff})
            for (int past : {0, 1, 6, 31, 70})
                for (int ql : {1, 2, 9}) {
                    p.window = window, p.sinks = sinks;
                    WinSeq s{0, ql, past + ql, past, true};
                    for (int t0 = 0; t0 < ql; t0++)
                        for (int t1 = t0; t1 < ql; t1++) {
                            const WinKeys k = win_keys(p, s, t0, t1);
                            std::set<int> got;
                            int before = -1;
                            for (int v = 0; v < k.count; v++) {
                                if (k.at(v) <= before) die("keys out of order", window, sinks, v);
                                got.insert(before = k.at(v));
                            }
                            for (int j = 0; j < s.kl; j++) {
                                bool any = false;
                                for (int t = t0; t <= t1; t++) any |= j <= past + t && (j > (long long)past + t - window || j < sinks);
                                if (any != (got.count(j) > 0)) die("key set", window, sinks, j);
                                for (int t = t0; t <= t1; t++)
                                    if (win_sees(p, past + t, j) != (j <= past + t && (j > (long long)past + t - window || j < sinks)))
                                        die("win_sees", past + t, j, window);
                            }
                            if (!got.empty() && (*got.begin() < 0 || *got.rbegin() >= s.kl)) die("key range", t0, t1, ql);
                        }
                }
    // lengths that contradict each other stay inside the tensors
    const int32_t bad[] = {-2147483647 - 1, -1, 0, 1, 3, 5, 9, 2147483647};
    p.window = 4, p.sinks = 1, p.batch = 1, p.tokens = 5, p.max_q = 3, p.max_kv = 9, p.page = 4, p.table_width = 2;
    for (int32_t c0 : bad)
        for (int32_t c1 : bad)
            for (int32_t kl : bad) {
                const int32_t cu[2] = {c0, c1};
                p.d_cu = cu, p.d_kl = &kl;
                const WinSeq s = win_seq(p, 0);
                const bool fits = c0 >= 0 && c1 >= c0 && c1 <= 5 && (long long)c1 - c0 <= 3 && kl >= c1 - c0 && kl <= 8;
                if (s.ok != fits) die("ok", c0, c1, kl);
                if (s.c0 < 0 || s.ql < 0 || s.c0 + s.ql > 5 || s.ql > 3) die("rows", c0, c1, kl);
                if (s.ok && (s.c0 != c0 || s.ql != c1 - c0 || s.past != kl - s.ql)) die("lengths", c0, c1, kl);
            }
    // page ids outside the cache; offsets past 32 bits
    const int32_t table[] = {7, -1, 8, 0, 2147483647, 6};
    p.d_table = table, p.table_stride = 3, p.pages = 8, p.page = 5;
    const int64_t stride[3] = {1LL << 33, 1LL << 20, 128};
    for (int b = 0; b < 2; b++)
        for (int j = 0; j < 15; j++) {
            const int pg = table[3 * b + j / 5];
            const long long want = pg < 0 || pg >= 8 ? -1 : pg * stride[0] + j % 5 * stride[1] + 3 * stride[2];
            if (win_cache_at(p, b, j, stride, 3) != want) die("slot", b, j, pg);
        }
    printf("ok\n");
    return 0;
}
"""


def test_window_keys_and_slots(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    src, exe = tmp_path / "keys.cpp", tmp_path / "keys"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", CSRC, "-I",
                    os.path.join(CSRC, "..", "..", "include"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr
