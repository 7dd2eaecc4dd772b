"""Bounds and scales that the language-model layers refuse before anything touches a
device, and the rows that a sequence of contradicting lengths holds."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

from onnxsharp_amd import native as N
from onnxsharp_amd.lm_layers import PagedKvCache, WindowAttentionLayer

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "onnxsharp_amd", "csrc")


def test_attention_bounds():
    pages = torch.zeros(4, 16, 2, 32, dtype=torch.float16)
    q, k = torch.zeros(3, 4, 32, dtype=torch.float16), torch.zeros(3, 2, 32, dtype=torch.float16)
    f = WindowAttentionLayer(window=8).forward

    def call(batch, max_q, max_kv):
        cache = PagedKvCache(pages, pages.clone(), torch.zeros(batch, 2, dtype=torch.int32))
        f(q, k, k, cache, torch.zeros(batch + 1, dtype=torch.int32), torch.zeros(batch, dtype=torch.int32), max_q, max_kv)

    with pytest.raises(N.OshError, match="3 tokens, but 2 sequences of at most 0"):
        call(2, 0, 5)
    with pytest.raises(N.OshError, match="3 tokens, but 0 sequences"):
        call(0, 3, 5)
    for max_q, max_kv in ((3, 2), (1, 2 ** 31), (2 ** 40, 2 ** 40)):
        with pytest.raises(N.OshError, match="max_q"):
            call(2, max_q, max_kv)
    with pytest.raises(ValueError, match="device tensors"):
        call(2, 3, 5)


@pytest.mark.parametrize("scale", [1e-50, 1e-46, 3e38, 1e39, -0.5])
def test_attention_scales_that_are_no_float(scale):
    # 1e-50 would be 0, which stands for 1 / sqrt(head_dim)
    with pytest.raises(ValueError, match="scale"):
        WindowAttentionLayer(scale=scale)
    assert WindowAttentionLayer(scale=1e-30).scale == 1e-30


def test_attention_entry_refuses_a_scale_without_room():
    p = N.WindowAttn(dtype=N.T_BF16, batch=1, q_heads=1, kv_heads=1, head_dim=64, window=1, max_q=1, max_kv=1, pages=1,
                     page=1, table_width=1, tokens=1, scale=2.9e38)
    n = C.c_size_t()
    assert N.lib().osh_window_attention_scratch_bytes(C.byref(p), C.byref(n)) == N.OSH_E_INVALID
    assert "scale" in N.last_error()


PROGRAM = r"""
#include <cstdio>
#include "osh_window_addr.h"
using namespace osh;

int main() {
    osh_window_attn p = {};
    const int32_t some[] = {-2147483647 - 1, -1, 0, 1, 3, 5, 9, 2147483647};
    p.window = 4, p.sinks = 1, p.batch = 1, p.tokens = 5, p.max_q = 2, p.max_kv = 9, p.page = 4, p.table_width = 2;
    for (int32_t c0 : some)
        for (int32_t c1 : some)
            for (int32_t kl : some) {
                const int32_t cu[2] = {c0, c1};
                p.d_cu = cu, p.d_kl = &kl;
                const WinSeq s = win_seq(p, 0);
                int held = 0, first = -1;
                for (int r = 0; r < 5; r++)
                    if (r >= c0 && r < c1) first = held++ ? first : r;
                if (s.held != held || (held && s.c0 != first) || (s.ok && s.ql != held) || s.ql > held || s.c0 + s.held > 5)
                    return printf("%d %d %d\n", c0, c1, kl), 1;
            }
    printf("ok\n");
    return 0;
}
"""


def test_rows_of_a_refused_sequence(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    src, exe = tmp_path / "held.cpp", tmp_path / "held"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", CSRC, "-I",
                    os.path.join(CSRC, "..", "..", "include"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr
