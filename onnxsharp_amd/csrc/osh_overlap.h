// osh_overlap.h -- whether strided operands share memory.  Plain C++ (no HIP header), so
// that it can also be compiled for the host and checked there.
#pragma once

#include <stdint.h>

namespace osh {

// Bytes base + sum_k i_k step[k] + [0, len), 0 <= i_k < n[k], steps ascending.
struct Strided {
    typedef __int128 wide;  // offsets of any int and any int64 stride
    const char *base = nullptr;
    wide len = 0;
    int dims = 0;
    wide n[3], step[3];

    Strided(const void *p, wide bytes) : base(static_cast<const char *>(p)), len(bytes) {}
    Strided &by(wide count, wide step_bytes) {  // one more dimension, of at most three
        if (count <= 0) base = nullptr;
        if (count <= 1) return *this;
        int k = dims++;
        for (; k > 0 && step[k - 1] > step_bytes; k--) n[k] = n[k - 1], step[k] = step[k - 1];
        n[k] = count, step[k] = step_bytes;
        return *this;
    }
    bool none() const { return !base || len <= 0; }
    wide extent() const {
        wide e = len;
        for (int k = 0; k < dims; k++) e += (n[k] - 1) * step[k];
        return e;
    }
};

// Rows of `cols` bytes.
inline Strided strided_rows(const void *p, long long rows, long long pitch, long long cols) {
    return Strided(p, cols).by(rows, pitch);
}

// Whether two index tuples reach the same byte.  Steps that do not enclose each other count
// as sharing.
inline bool shares_itself(const Strided &a) {
    if (a.none()) return false;
    Strided::wide inner = a.len;
    for (int k = 0; k < a.dims; k++) {
        if (a.step[k] < inner) return true;
        inner += (a.n[k] - 1) * a.step[k];
    }
    return false;
}

// b's start lies `diff` bytes behind a's; the dimensions ka.. and kb.. down are still open.
inline bool share_from(const Strided &a, int ka, const Strided &b, int kb, Strided::wide diff, int &budget) {
    typedef Strided::wide wide;
    if (--budget < 0) return true;
    wide ea = a.len, eb = b.len;
    for (int k = 0; k < ka; k++) ea += (a.n[k] - 1) * a.step[k];
    for (int k = 0; k < kb; k++) eb += (b.n[k] - 1) * b.step[k];
    if (diff >= ea || -diff >= eb) return false;
    if (ka == 0 && kb == 0) return true;
    // the widest step, of both where they have it in common
    const bool in_a = ka && (!kb || a.step[ka - 1] >= b.step[kb - 1]), in_b = kb && (!ka || b.step[kb - 1] >= a.step[ka - 1]);
    const wide s = in_a ? a.step[ka - 1] : b.step[kb - 1];
    if (s <= 0) return true;
    const wide lo = in_a ? -(a.n[ka - 1] - 1) : 0, hi = in_b ? b.n[kb - 1] - 1 : 0;
    if (in_a) ea -= (a.n[ka - 1] - 1) * s;
    if (in_b) eb -= (b.n[kb - 1] - 1) * s;
    // offsets t s with -eb < diff + t s < ea
    const auto floor_div = [](wide x, wide y) { return x / y - (x % y < 0); };
    wide t0 = floor_div(-eb - diff, s) + 1, t1 = -floor_div(diff - ea, s) - 1;
    if (t0 < lo) t0 = lo;
    if (t1 > hi) t1 = hi;
    for (wide t = t0; t <= t1; t++)
        if (share_from(a, ka - in_a, b, kb - in_b, diff + t * s, budget)) return true;
    return false;
}

// Whether a and b share a byte.  Exact for layouts that a few dozen trials decide (equal
// strides, as views of one tensor have, take two a dimension), else true where the ranges meet.
inline bool share_bytes(const Strided &a, const Strided &b) {
    if (a.none() || b.none()) return false;
    int budget = 256;
    return share_from(a, a.dims, b, b.dims, (Strided::wide)((intptr_t)b.base - (intptr_t)a.base), budget);
}

}  // namespace osh
