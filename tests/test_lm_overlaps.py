"""Operands of the language-model operators that share memory: the rule itself
(csrc/osh_overlap.h, plain C++ on the host) against sets of bytes, and the C entry
points' refusals on pointers that are never read."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from onnxsharp_amd import native as N

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "onnxsharp_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include "osh_overlap.h"
using namespace osh;

static std::set<long long> bytes(const Strided &a, long long at, bool &twice) {
    std::set<long long> out;
    twice = false;
    const int n0 = a.dims > 0 ? (int)a.n[0] : 1, n1 = a.dims > 1 ? (int)a.n[1] : 1, n2 = a.dims > 2 ? (int)a.n[2] : 1;
    for (int i = 0; i < n0; i++)
        for (int j = 0; j < n1; j++)
            for (int k = 0; k < n2; k++)
                for (int e = 0; e < (int)a.len; e++) {
                    const long long o = at + e + (a.dims > 0 ? i * (long long)a.step[0] : 0) +
                                        (a.dims > 1 ? j * (long long)a.step[1] : 0) + (a.dims > 2 ? k * (long long)a.step[2] : 0);
                    twice |= !out.insert(o).second;
                }
    return out;
}

int main() {
    std::mt19937 rng(5);
    auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (unsigned)(hi - lo + 1)); };
    int exact = 0, apart = 0, kept = 0, shared = 0;
    for (int round = 0; round < 60000; round++) {
        // steps that enclose each other, or any
        const bool nested = round % 3 != 0, equal = round % 2;
        auto make = [&](long long at, const Strided *like) {
            Strided a(reinterpret_cast<const char *>(0x10000 + at), pick(1, 6));
            int inner = (int)a.len;
            for (int k = 0; k < 3; k++) {
                const int n = pick(0, 9) == 0 ? 1 : pick(1, 4);
                const int step = like && k < like->dims ? (int)like->step[k] : nested ? inner + pick(0, 12) : pick(0, 40);
                a.by(n, step);
                inner += (n - 1) * step;
            }
            return a;
        };
        const long long at = pick(0, 200) - 100;
        Strided a = make(0, nullptr), b = make(at, equal ? &a : nullptr);
        bool ta, tb;
        const std::set<long long> sa = bytes(a, 0, ta), sb = bytes(b, at, tb);
        if (ta && !shares_itself(a)) return printf("missed itself %d\n", round), 1;
        if (nested && !equal && (shares_itself(a) || shares_itself(b))) return printf("enclosed steps %d\n", round), 1;
        bool both = false;
        for (long long o : sb) both |= sa.count(o) > 0;
        const bool got = share_bytes(a, b);
        if (got != share_bytes(b, a)) return printf("not symmetric %d\n", round), 1;
        if (both && !got) return printf("missed %d\n", round), 1;
        shared += both;
        kept += got && !both;
        if (nested && equal && !shares_itself(b)) {
            exact++;
            apart += !both;
            if (got != both) return printf("refused %d\n", round), 1;
        }
    }
    // sizes past 64 bits
    Strided huge(reinterpret_cast<const char *>(64), 512);
    huge.by(1 << 30, (Strided::wide)(1LL << 62)).by(1 << 30, (Strided::wide)(1LL << 62));
    if (!shares_itself(huge) || share_bytes(Strided(reinterpret_cast<const char *>(8), 8), huge)) return printf("huge\n"), 1;
    if (share_bytes(Strided(nullptr, 8), huge) || share_bytes(huge, Strided(reinterpret_cast<const char *>(64), 0)))
        return printf("nothing\n"), 1;
    // keys and values in turn in one tensor: [pages][2][page][heads][values]
    for (int two = 0; two < 2; two++) {
        auto part = [&](long long off) {
            return Strided(reinterpret_cast<const char *>(4096 + off), 128).by(50, 8192 - 64 * two).by(16, 256).by(2, 128);
        };
        if (shares_itself(part(0)) || share_bytes(part(0), part(4096)) != (two == 1)) return printf("in turn %d\n", two), 1;
    }
    printf("ok %d\n", exact > 1000 && apart > 100 && shared > 1000);
    return 0;
}
"""


def test_share_rules(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    src, exe = tmp_path / "share.cpp", tmp_path / "share"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", CSRC, str(src),
                    "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok 1\n", r.stdout + r.stderr


def _attn(**kw):
    p = N.WindowAttn(dtype=N.T_BF16, batch=2, q_heads=4, kv_heads=2, head_dim=64, window=32, sinks=4, max_q=2, max_kv=64,
                     pages=8, page=16, table_width=4, tokens=4, d_q=1 << 40, d_k_new=2 << 40, d_v_new=3 << 40,
                     d_o=4 << 40, d_k_pages=5 << 40, d_v_pages=6 << 40, d_table=7 << 40, d_cu=8 << 40, d_kl=9 << 40,
                     q_stride=(256, 64), k_new_stride=(128, 64), v_new_stride=(128, 64), o_stride=(256, 64),
                     k_stride=(2048, 128, 64), v_stride=(2048, 128, 64), table_stride=4)
    for f, v in kw.items():
        setattr(p, f, v)
    return N.lib().osh_window_attention(C.byref(p), None, None)


# pages: 8 * 2048 * 2 bytes; o: 4 * 256 * 2 bytes
@pytest.mark.parametrize("kw,msg", [
    (dict(d_o=5 << 40), "o overlaps the cache"), (dict(d_o=(6 << 40) + 32766), "o overlaps the cache"),
    (dict(d_o=(5 << 40) - 2046), "o overlaps the cache"),
    (dict(o_stride=(0, 64)), "rows of o share"), (dict(o_stride=(256, 0)), "rows of o share"),
    (dict(o_stride=(192, 64)), "rows of o share"),
    (dict(d_v_pages=5 << 40), "slots of the cache share"), (dict(d_v_pages=(5 << 40) + 2), "slots of the cache share"),
    (dict(k_stride=(0, 128, 64)), "slots of the cache share"), (dict(v_stride=(2048, 0, 64)), "slots of the cache share"),
    (dict(v_stride=(2048, 128, 56)), "slots of the cache share"),
    (dict(d_q=5 << 40), "cache overlaps an operand"), (dict(d_k_new=(6 << 40) + 1024), "cache overlaps an operand"),
    (dict(d_table=(5 << 40) + 4), "cache overlaps an operand"), (dict(d_kl=6 << 40), "cache overlaps an operand"),
    (dict(d_cu=4 << 40), "o overlaps an operand"), (dict(d_table=(4 << 40) - 4), "o overlaps an operand"),
    (dict(d_k_new=4 << 40), "o overlaps an operand"),
])
def test_attention_refuses_shared_memory(kw, msg):
    assert _attn(**kw) == N.OSH_E_INVALID
    assert msg in N.last_error()


def _p(i, off=0):
    return C.c_void_p((i << 40) + off)


def _norm(rows=4, cols=16, x=_p(1), ldx=16, res=_p(2), ldr=16, g=_p(3), h=_p(4), ldh=16, q=_p(5), ldq=16, scale=_p(6)):
    return N.lib().osh_rms_norm_quant(rows, cols, N.T_BF16, x, ldx, res, ldr, g, 1e-5, h, ldh, N.T_I8, q, ldq, scale, None)


@pytest.mark.parametrize("kw", [
    dict(h=_p(1), ldx=40, ldh=41), dict(h=_p(1, 30), ldx=40, ldh=40), dict(h=_p(1, 50), ldx=40, ldh=40),
    dict(h=_p(3, 30)), dict(q=_p(4, 127)), dict(q=_p(2), ldr=20, ldq=40), dict(scale=_p(1, 124)), dict(scale=_p(5, 60)),
    dict(scale=_p(3, -12)), dict(res=None, h=None, q=_p(1, 1)), dict(res=None, h=None, scale=_p(5)),
])
def test_norm_refuses_shared_memory(kw):
    assert _norm(**kw) == N.OSH_E_INVALID and "overlaps" in N.last_error()


def _mm(m=4, n=8, k=16, a=_p(1), lda=16, w=_p(3), ldw=16, bias=_p(5), res=_p(6), ldr=8, y=_p(7), ldy=8):
    return N.lib().osh_quant_matmul(m, n, k, N.T_I8, a, lda, _p(2), w, ldw, _p(4), bias, N.ACT_NONE, N.T_F16, res, ldr, y,
                                    ldy, None)


@pytest.mark.parametrize("kw", [
    dict(y=_p(1), ldy=8), dict(y=_p(3, 127)), dict(y=_p(2, 15)), dict(y=_p(4, -60)), dict(y=_p(5, 31)),
    dict(y=_p(6, 14), ldr=16, ldy=16), dict(y=_p(6, 18), ldr=16, ldy=16), dict(y=_p(6), ldr=16, ldy=17),
])
def test_matmul_refuses_shared_memory(kw):
    assert _mm(**kw) == N.OSH_E_INVALID and "overlaps" in N.last_error()
