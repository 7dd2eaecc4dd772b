// osh_window_addr.h -- which keys and which cache slots a call of
// osh_window_attention reaches.  Plain C++ (no HIP header), so that the rules can
// also be compiled for the host and checked there.
#pragma once

#include <stdint.h>

#include "osh_hip.h"

#ifdef __HIPCC__
#define OSH_HD __host__ __device__ __forceinline__
#else
#define OSH_HD inline
#endif

namespace osh {

OSH_HD int win_min(int a, int b) { return a < b ? a : b; }
OSH_HD int win_max(int a, int b) { return a > b ? a : b; }

// A sequence's rows and lengths.  ok is false where they contradict each other,
// the host's bounds or the table; c0, ql and held, all of its rows, stay within the
// tensors even then, so that they can be filled with NaN.
struct WinSeq {
    int c0, ql, kl, past, held;
    bool ok;
};
OSH_HD WinSeq win_seq(const osh_window_attn &p, int b) {
    WinSeq s;
    const long long n = p.tokens;
    long long c0 = p.d_cu[b], c1 = p.d_cu[b + 1];
    s.kl = p.d_kl[b];
    s.ok = c0 >= 0 && c1 >= c0 && c1 <= n && c1 - c0 <= p.max_q && s.kl >= c1 - c0 && s.kl <= p.max_kv &&
           (long long)p.table_width * p.page >= s.kl;
    c0 = c0 < 0 ? 0 : c0 > n ? n : c0;
    c1 = c1 < c0 ? c0 : c1 > n ? n : c1;
    s.c0 = (int)c0;
    s.held = (int)(c1 - c0);
    s.ql = (int)(c1 - c0 < p.max_q ? c1 - c0 : p.max_q);
    s.past = s.kl - s.ql;
    return s;
}

// The keys that any of the tokens t0..t1 (of the new ones) of a sequence sees:
// the sinks below the first one's window, then one range up to the last one.
// Key number v in [0, count) is position at(v).
struct WinKeys {
    int sink_end, lo, count;
    OSH_HD int at(int v) const { return v < sink_end ? v : v - sink_end + lo; }
};
OSH_HD WinKeys win_keys(const osh_window_attn &p, const WinSeq &s, int t0, int t1) {
    WinKeys k;
    k.lo = win_max(0, s.past + t0 - p.window + 1);
    k.sink_end = win_min(p.sinks, k.lo);
    k.count = k.sink_end + s.past + t1 + 1 - k.lo;
    return k;
}

// Whether the query at position pos sees position j.
OSH_HD bool win_sees(const osh_window_attn &p, int pos, int j) {
    return j <= pos && (j > pos - p.window || j < p.sinks);
}

// Element offset of cache position j at key head h, or -1 for a page outside the
// cache.
OSH_HD long long win_cache_at(const osh_window_attn &p, int b, int j, const int64_t *stride, int h) {
    const int pg = p.d_table[b * p.table_stride + j / p.page];
    if ((unsigned)pg >= (unsigned)p.pages) return -1;
    return pg * (long long)stride[0] + (long long)(j % p.page) * stride[1] + (long long)h * stride[2];
}

}  // namespace osh
