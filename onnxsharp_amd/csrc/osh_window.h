// osh_window.h -- what the attention kernels over paged caches (osh_window_attn.hip,
// osh_kv4_attn.hip) have in common: the arguments, a sequence's rows, MFMA and LDS
// wrappers, and the join of splits.
#pragma once

#include <algorithm>

#include "osh_int4.h"
#include "osh_window_addr.h"

namespace osh {

struct WinArgs {
    osh_window_attn p;
    int group, tile_rows, tiles, splits;
    bool wide;       // few rows: eight waves a row block instead of four and splits
    int page_shift;  // of a page that is a power of two, else -1
    float scale_log2;
    float *part_o, *part_ml;  // of a split: [unit][split][tile_rows][head_dim], [unit][split][tile_rows][2]
    const float *expanded;    // [batch][kv_heads][2]: the powers of two that f16 pages of K and V were taken times
};

constexpr int WIN_MAX_SPLITS = 64;  // a lane a split in the join

// l plus the eight values of w, in FP32, two an instruction.
__device__ __forceinline__ float add8(f16x8 w, float l) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 one = {(_Float16)1, (_Float16)1};
#pragma unroll
    for (int i = 0; i < 8; i += 2) l = __builtin_amdgcn_fdot2(f16x2{w[i], w[i + 1]}, one, l, false);
    return l;
}
__device__ __forceinline__ float add8(bf16x8 w, float l) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
    for (int i = 0; i < 8; i += 2) l = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{w[i], w[i + 1]}, one, l, false);
    return l;
}

// What stands in for a row that is not read: zeros for a key past the last one and
// for the value of a page outside the cache, NaN (0x7fff in both types) for its key.
#define WIN_NAN4 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu
#define WIN_NAN32 WIN_NAN4, WIN_NAN4, WIN_NAN4, WIN_NAN4, WIN_NAN4, WIN_NAN4, WIN_NAN4, WIN_NAN4
static __device__ const unsigned win_zero_row[128] = {};
static __device__ const unsigned win_nan_row[128] = {WIN_NAN32, WIN_NAN32, WIN_NAN32, WIN_NAN32};
#undef WIN_NAN4
#undef WIN_NAN32

// All rows of a sequence whose lengths contradict each other or the bounds (it may hold
// more than the call's row blocks cover), at one key head's query heads.
template <typename T>
__device__ __forceinline__ void win_fill_nan(const osh_window_attn &p, const WinSeq &sq, int h, int G, int tid,
                                             int threads) {
    const int d = p.head_dim;
    for (long long e = tid; e < (long long)sq.held * G * d; e += threads) {
        const long long r = e / d;
        static_cast<T *>(p.d_o)[(sq.c0 + r / G) * p.o_stride[0] + (h * G + r % G) * p.o_stride[1] + e % d] =
            (T)__builtin_nanf("");
    }
}

// The tokens whose first row lies in rows r0 .. r0 + n go to their pages.
template <typename T>
__device__ __forceinline__ void win_append(const osh_window_attn &p, const WinSeq &sq, int b, int h, int G, int r0, int n,
                                           int tid, int threads) {
    const T *kn = static_cast<const T *>(p.d_k_new), *vn = static_cast<const T *>(p.d_v_new);
    T *kp = static_cast<T *>(p.d_k_pages), *vp = static_cast<T *>(p.d_v_pages);
    const int t0 = cdiv(r0, G), t1 = min(cdiv(r0 + n, G), sq.ql);
    const int chunks = p.head_dim / 8;
    for (int e = tid; e < (t1 - t0) * chunks; e += threads) {
        const int t = t0 + e / chunks, c = e % chunks * 8;
        const long long ko = win_cache_at(p, b, sq.past + t, p.k_stride, h);
        const long long vo = win_cache_at(p, b, sq.past + t, p.v_stride, h);
        if (ko < 0) continue;
        const long long row = sq.c0 + t;
        __builtin_memcpy(kp + ko + c, kn + row * p.k_new_stride[0] + h * p.k_new_stride[1] + c, 16);
        __builtin_memcpy(vp + vo + c, vn + row * p.v_new_stride[0] + h * p.v_new_stride[1] + c, 16);
    }
}

// Slot of a 16-byte chunk in an LDS row of C chunks: chunk ^ swizzle(row).
template <int C>
__device__ __forceinline__ int win_k_swizzle(int r) {
    return C >= 16 ? r & 15 : C == 8 ? r >> 1 & 7 : r >> 2 & 3;
}
template <int C>
__device__ __forceinline__ int win_v_swizzle(int r) {
    return C >= 16 ? (r & 3) << 2 | (r >> 2 & 3) : C == 8 ? (r >> 1 & 1) << 2 : 0;
}

// Where a key's rows of K and V are; its page is looked up one step ahead.  Selects
// in place of branches: the lanes of a wave mix new tokens, pages and keys past the
// end (branches cost 30 us of the 340 of an 8192-token prompt).  Strides fit 31 bits.
template <typename T>
struct WinRows {
    const T *k, *v;
};
template <typename T>
__device__ __forceinline__ const T *win_row(bool fresh, unsigned i0, unsigned i1, const void *fresh_base,
                                            const int64_t *fresh_stride, const void *base, const int64_t *stride, int h) {
    const T *f = static_cast<const T *>(fresh_base) + h * fresh_stride[1];
    const T *c = static_cast<const T *>(base) + h * stride[2];
    const unsigned s0 = fresh ? (unsigned)fresh_stride[0] : (unsigned)stride[0];
    return (fresh ? f : c) + ((unsigned long long)i0 * s0 + (unsigned long long)i1 * (unsigned)stride[1]);
}
template <typename T>
__device__ __forceinline__ WinRows<T> win_rows(const osh_window_attn &p, const WinSeq &sq, const WinKeys &keys, int v,
                                               int page_id, int page_shift, int h) {
    const int j = keys.at(v);
    const bool past_end = v >= keys.count, fresh = j >= sq.past;
    const bool bad = !fresh && (unsigned)page_id >= (unsigned)p.pages;
    const unsigned in = page_shift >= 0 ? j & (p.page - 1) : j % p.page;
    const unsigned i0 = fresh ? sq.c0 + j - sq.past : page_id, i1 = fresh ? 0 : in;
    WinRows<T> r;
    r.k = win_row<T>(fresh, i0, i1, p.d_k_new, p.k_new_stride, p.d_k_pages, p.k_stride, h);
    r.v = win_row<T>(fresh, i0, i1, p.d_v_new, p.v_new_stride, p.d_v_pages, p.v_stride, h);
    if (past_end || bad) {
        r.k = reinterpret_cast<const T *>(past_end ? win_zero_row : win_nan_row);
        r.v = reinterpret_cast<const T *>(win_zero_row);
    }
    return r;
}
__device__ __forceinline__ int win_page(const osh_window_attn &p, const WinSeq &sq, const WinKeys &keys, int b, int v,
                                        int page_shift) {
    if (sq.past == 0) return 0;
    const int j = win_min(keys.at(v), sq.past - 1);  // a key past the pages takes no page
    return p.d_table[b * p.table_stride + (page_shift >= 0 ? j >> page_shift : j / p.page)];
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// Of the 16 lanes of a group, lane 4 j + q reads values 4 q .. 4 q + 3 of row j; lane i
// gets value i of rows 0..3.
__device__ __forceinline__ s16x4 read_transposed(const unsigned char *at) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)at);
}

// Joins the splits of four rows, a wave a row: the splits' weights first, a lane a
// split, then the sums, eight splits' loads in flight.  Latency bounds it: 6 us for 21
// splits of 24 blocks.
template <typename T>
static __global__ __launch_bounds__(256) void window_attn_join_kernel(WinArgs a) {
    const osh_window_attn &p = a.p;
    const int quads = a.tile_rows / 4, d = p.head_dim, G = a.group;
    const int unit = blockIdx.x / quads, lane = threadIdx.x & 63;
    int id = unit;
    const int tile = a.tile_rows > 16 ? a.tiles - 1 - id % a.tiles : id % a.tiles;
    id /= a.tiles;
    const int h = id % p.kv_heads, b = id / p.kv_heads;
    const WinSeq sq = win_seq(p, b);
    const int r = blockIdx.x % quads * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = tile * a.tile_rows + r;
    if (!sq.ok || row >= sq.ql * G) return;
    const float *ml = a.part_ml + ((long long)unit * a.splits * a.tile_rows + r) * 2;
    const float *os = a.part_o + ((long long)unit * a.splits * a.tile_rows + r) * d;
    const long long next = a.tile_rows;
    const bool mine = lane < a.splits;  // at most WIN_MAX_SPLITS = 64
    const float m = mine ? ml[lane * next * 2] : -__builtin_inff(), l = mine ? ml[lane * next * 2 + 1] : 0.0f;
    float top = m;
#pragma unroll
    for (int o = 32; o; o >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o));
    const float w = __builtin_amdgcn_exp2f(m - (top == -__builtin_inff() ? 0.0f : top));
    float sum = w * l;
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    const float scale = w / sum;
    T *out = static_cast<T *>(p.d_o) + (long long)(sq.c0 + row / G) * p.o_stride[0] + (h * G + row % G) * p.o_stride[1];
    for (int c = lane * 2; c < d; c += 128) {
        float2 f = {0.0f, 0.0f};
        for (int s = 0; s < a.splits; s += 8) {
            float2 v[8];
#pragma unroll
            for (int e = 0; e < 8; e++)
                v[e] = *reinterpret_cast<const float2 *>(os + min(s + e, a.splits - 1) * next * d + c);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                // lanes past the head's values left the loop: read the weight by its lane
                const float we = s + e < a.splits ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(scale), s + e)) : 0.0f;
                f.x = s + e < a.splits ? __builtin_fmaf(we, v[e].x, f.x) : f.x;
                f.y = s + e < a.splits ? __builtin_fmaf(we, v[e].y, f.y) : f.y;
            }
        }
        out[c] = (T)f.x;
        out[c + 1] = (T)f.y;
    }
}

template <typename T>
static osh_status win_join(const WinArgs &a, unsigned units, hipStream_t st) {
    if (a.splits > 1) {
        OSH_LAUNCH(window_attn_join_kernel<T>, dim3(units * (a.tile_rows / 4)), dim3(256), 0, st, a);
        OSH_LAUNCH_CHECK("window_attn_join_kernel");
    }
    return OSH_OK;
}

// The attention over 16-bit pages of a planned and checked call (osh_window_attn.hip).
osh_status win_run(const WinArgs &a, unsigned units, hipStream_t st);
// The same of bf16 queries over pages of f16 that hold the new tokens too, taken times
// a.expanded; more than 16 rows a key head.
osh_status win_run_expanded(const WinArgs &a, unsigned units, hipStream_t st);

// Row blocks, splits and scratch of a call.
static osh_status win_plan(const osh_window_attn *p, WinArgs &a, size_t &scratch) {
    if (!p) return fail(OSH_E_INVALID, "WindowAttention: NULL parameters");
    if (p->dtype != OSH_T_F16 && p->dtype != OSH_T_BF16)
        return fail(OSH_E_INVALID, "WindowAttention: queries, keys and values are f16 or bf16");
    if (p->batch < 0 || p->q_heads <= 0 || p->kv_heads <= 0 || p->head_dim <= 0 || p->max_q < 0 || p->max_kv < 0 ||
        p->pages < 0 || p->page <= 0 || p->table_width < 0 || p->tokens < 0)
        return fail(OSH_E_INVALID, "WindowAttention: bad sizes");
    if (p->q_heads % p->kv_heads) return fail(OSH_E_INVALID, "WindowAttention: %d query heads over %d key heads",
                                              p->q_heads, p->kv_heads);
    if (p->window < 1 || p->sinks < 0) return fail(OSH_E_INVALID, "WindowAttention: window %d, sinks %d", p->window,
                                                   p->sinks);
    if (!(p->scale >= 0.0f) || p->scale > 2e38f)  // times log2(e) it stays finite
        return fail(OSH_E_INVALID, "WindowAttention: bad scale");
    if (p->head_dim % 8 || p->head_dim > 256)
        return fail(OSH_E_UNSUPPORTED, "WindowAttention: heads of %d values (multiples of 8 up to 256)", p->head_dim);
    if (p->max_kv > (1 << 30) || p->tokens > (1 << 30) || p->max_q > p->max_kv)
        return fail(p->max_q > p->max_kv ? OSH_E_INVALID : OSH_E_UNSUPPORTED,
                    "WindowAttention: lengths up to %d new, %d in all", p->max_q, p->max_kv);
    a.p = *p;
    a.group = p->q_heads / p->kv_heads;
    if ((long long)p->max_q * a.group > (1 << 30))
        return fail(OSH_E_UNSUPPORTED, "WindowAttention: %d new tokens of %d heads", p->max_q, p->q_heads);
    a.page_shift = (p->page & (p->page - 1)) == 0 ? __builtin_ctz(p->page) : -1;
    a.scale_log2 = (p->scale == 0.0f ? 1.0f / __builtin_sqrtf((float)p->head_dim) : p->scale) * 1.4426950408889634f;
    const int rows = p->max_q * a.group;
    const long long heads = (long long)p->batch * p->kv_heads;
    // More than one block of 16 rows would read the keys again for each: 32 rows of 8
    // sequences to 8192 take 35 us as two blocks and 31 in a tile of 128, 60 rows 56 and 32.
    a.tile_rows = rows > 16 ? 128 : 16;
    a.tiles = cdiv(rows, a.tile_rows);
    const long long units = heads * a.tiles;
    if (units >= (1LL << 22)) return fail(OSH_E_UNSUPPORTED, "WindowAttention: too many row blocks (%lld)", units);
    const long long span = std::min<long long>(p->max_kv, (long long)p->window + p->sinks + a.tile_rows / a.group);
    // Two workgroups a CU, all resident at once: three sequences of 65536 with window
    // 32768 take 87 us as 504 workgroups, 104 as 528 (16 of them in a second round), 90
    // as 1024; 64 ragged ones of 8192 191 us unsplit, 207 split in two.
    const long long want = units ? std::max(1LL, 2LL * device_cus() / units) : 1;
    a.splits = (int)std::max(1LL, std::min({want, span / 256, (long long)WIN_MAX_SPLITS}));
    // One launch of eight waves for short spans, else four waves, splits and a join.  Device
    // times, eight waves against four, over 64, 200, 400, 640, 800 and 1000 keys: one sequence
    // of 12 heads of 64 on 4: 6.3 (5.9), 7.0 (7.8), 8.6 (10.9), 10.2 (12.6), 11.8 (12.5), 13.0
    // (13.0) us; 4 of 32 heads of 128 on 8: 7.9 (7.3), 8.9 (9.7), 11.7 (14.0), 13.6 (15.2), 15.7
    // (15.3), 18.2 (15.6); 32 of them, a workgroup a CU: 8.2 (7.5), 9.7 (10.1), 16.9 (18.0),
    // 20.3 (26.1), 23.5 (29.6), 26.6 (32.2).  Few workgroups lose past 640 keys, many do not;
    // below 100 keys four waves are 0.7 us ahead.
    a.wide = a.tile_rows == 16 && span <= 640 && units <= device_cus() && p->head_dim <= 128;
    if (a.wide) a.splits = 1;
    const long long parts = a.splits > 1 ? units * a.splits : 0;
    scratch = (size_t)parts * a.tile_rows * (p->head_dim + 2) * 4;
    return OSH_OK;
}

}  // namespace osh
