// osh_kv4_attn.hip -- the attention of osh_window_attn.hip over a paged cache held in 4
// bits (osh_kv4_attention): a group of a head's values is lo + scale * code.
//
// Up to 512 rows of a key head, and f16 calls (kv4_rows_kernel): the products take the codes,
// which are exact in 16 bits; scales and minima stay in FP32:
//   q . k_j = sum over groups of scale_j (q . code_j) + lo_j (sum of q over the group),
//   sum_j p_j v_j = sum_j (p_j scale_j) code_j + sum_j p_j lo_j.
// The matrix instructions take p_j scale_j as two numbers of dtype, the second what rounding to
// the first leaves: 16 bits of a bf16 weight, 22 of an f16 one.  The first alone leaves the output
// a quarter more error than its own rounding (2.2e-3 of o for 1.7e-3 in bf16) and is 2 to 8% faster
// (64 sequences of 5000 keys, 32 heads of 128 on 8: 70.2 us for 72.2 in groups of 128, 104.5 for
// 108.5 of 32).
// More rows in bf16: the visible cache is expanded to f16 pages once, and the kernel of
// osh_window_attn.hip reads those.
#include <limits.h>

#include "osh_overlap.h"
#include "osh_window.h"

using namespace osh;

namespace osh {

struct Kv4Args {
    WinArgs w;
    const void *ks, *vs;  // scale pairs
    void *k_stored, *v_stored;
    long long ks_stride[3], vs_stride[3], k_stored_stride[2], v_stored_stride[2];
    unsigned page_mul, page_log;  // j / page = umulhi(4 j, page_mul) >> page_log for j < 2^30
    bool append;                  // row blocks quantize the new tokens themselves, else a launch in front
    // many bf16 rows: the visible cache in f16, and what the 16-bit kernel is told about it
    _Float16 *k_wide, *v_wide;    // [batch * wide_blocks][kv_heads][WIDE_PAGE][head_dim]
    float *wide_by;               // [batch][kv_heads][2]: what K and V are taken times
    float *wide_top;              // [batch][kv_heads][RANGE_PARTS][2]: the largest of each part of the keys
    int32_t *wide_table, *wide_kl;
    int wide_blocks, wide_width;  // pages of a sequence, entries of its table
};

constexpr int WIDE_PAGE = 64, RANGE_PARTS = 16;

// -------------------------------------------------------------- quantization

// Tokens t0 .. t1 of the sequence's new ones into the cache, at key heads h0 .. h1, dealt out to
// `threads` threads (whole waves).  Eight neighbouring values a lane, the GL lanes of a group
// next to each other.
template <typename T, int GL>
__device__ __forceinline__ void kv4_append(const Kv4Args &a, const WinSeq &sq, int b, int h0, int h1, int t0, int t1,
                                           long long tid, long long threads) {
    const osh_window_attn &p = a.w.p;
    const int chunks = p.head_dim / 8, heads = h1 - h0;
    const long long total = (long long)(t1 - t0) * heads * 2 * chunks;
    for (long long e0 = tid & ~63LL; e0 < total; e0 += threads) {
        const long long e = e0 + (tid & 63);
        const bool in = e < total;
        long long item = 0, t = 0;
        int c = 0, h = h0;
        if (total <= INT_MAX) {  // divisions of 32 bits
            const unsigned u = in ? (unsigned)e : 0u, i = u / (unsigned)chunks, at = i / 2 / (unsigned)heads;
            c = (int)(u - i * chunks), h += (int)(i / 2 - at * heads), item = i, t = t0 + (int)at;
        } else if (in) {
            item = e / chunks, c = (int)(e - item * chunks), h += (int)(item / 2 % heads), t = t0 + item / 2 / heads;
        }
        const bool is_v = item & 1;
        const long long row = sq.c0 + t;
        const T *src = static_cast<const T *>(is_v ? p.d_v_new : p.d_k_new);
        const int64_t *st = is_v ? p.v_new_stride : p.k_new_stride;
        f32x8 f = {};
        if (in) f = load8(src + row * st[0] + h * st[1] + 8 * c);
        // NaN and infinities are above and below everything, as integers of the floats' order
        float lo = f[0], hi = f[0];
        bool finite = true;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            lo = __builtin_fminf(lo, f[i]), hi = __builtin_fmaxf(hi, f[i]);
            finite &= (__float_as_uint(f[i]) & 0x7f800000u) != 0x7f800000u;
        }
        int bad = !finite;
#pragma unroll
        for (int o = 1; o < GL; o <<= 1) {
            lo = __builtin_fminf(lo, __shfl_xor(lo, o));
            hi = __builtin_fmaxf(hi, __shfl_xor(hi, o));
            bad |= __shfl_xor(bad, o);
        }
        T scale = (T)((hi - lo) / 15.0f), low = (T)lo;
        if (bad || !(hi - lo < __builtin_inff())) scale = low = (T)__builtin_nanf("");
        const float s = (float)scale, l = (float)low;
        unsigned word = 0;
        f32x8 kept;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float q = s > 0.0f ? __builtin_rintf((f[i] - l) / s) : 0.0f;
            q = __builtin_fminf(__builtin_fmaxf(q, 0.0f), 15.0f);
            word |= (unsigned)(int)q << (4 * i);
            kept[i] = __builtin_fmaf(s, q, l);
        }
        if (!in) continue;
        // where it is kept; a sequence of contradicting lengths is not
        long long at = -1;
        const int64_t *cst = is_v ? p.v_stride : p.k_stride;
        const long long *sst = is_v ? a.vs_stride : a.ks_stride;
        if (sq.ok) {
            const int j = sq.past + (int)t, pg = p.d_table[b * p.table_stride + j / p.page], slot = j % p.page;
            if ((unsigned)pg < (unsigned)p.pages) {
                at = pg * (long long)cst[0] + (long long)slot * cst[1] + (long long)h * cst[2];
                unsigned char *codes = static_cast<unsigned char *>(is_v ? p.d_v_pages : p.d_k_pages);
                *reinterpret_cast<unsigned *>(codes + at + 4 * c) = word;
                if (c % GL == 0) {
                    T pair[2] = {scale, low};
                    T *to = const_cast<T *>(static_cast<const T *>(is_v ? a.vs : a.ks)) + pg * sst[0] + slot * sst[1] +
                            h * sst[2] + c / GL * 2;
                    __builtin_memcpy(__builtin_assume_aligned(to, 4), pair, 4);
                }
            }
        }
        if (T *out = static_cast<T *>(is_v ? a.v_stored : a.k_stored)) {
            const long long *ost = is_v ? a.v_stored_stride : a.k_stored_stride;
            store8(out + row * ost[0] + h * ost[1] + 8 * c, at < 0 ? f32x8{} + __builtin_nanf("") : kept);
        }
    }
}

// All new tokens.  blockIdx.y is the sequence.
template <typename T, int GL>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4Args a) {
    const WinSeq sq = win_seq(a.w.p, blockIdx.y);
    kv4_append<T, GL>(a, sq, blockIdx.y, 0, a.w.p.kv_heads, 0, sq.held, blockIdx.x * 256LL + threadIdx.x, gridDim.x * 256LL);
}

// The keys that any of a sequence's queries sees, by their blocks of WIDE_PAGE: first those of
// the sinks, then those of the window.
struct WideBlocks {
    int sinks, first, count;
    __device__ int at(int i) const { return i < sinks ? i : first + i - sinks; }  // below count
};
__device__ __forceinline__ WideBlocks kv4_blocks(const osh_window_attn &p, const WinSeq &sq, const WinKeys &keys) {
    const int sinks = cdiv(min(p.sinks, p.max_kv), WIDE_PAGE);
    return {sinks, max(keys.lo / WIDE_PAGE, sinks), cdiv(sq.kl, WIDE_PAGE)};
}

// The power of two that keeps a head's largest visible key, and value, within 1.  f16's 11 bits
// are then 8 times as close as bf16's rounding of the output down to 2^-14 of it (bf16 keys and
// values add as much error as the output's own rounding twice over).  First the largest of each
// of RANGE_PARTS parts of the keys; kv4_expand_kernel joins them.  blockIdx: part and head, sequence.
template <typename T>
__global__ __launch_bounds__(256) void kv4_range_kernel(Kv4Args a, int groups) {
    const osh_window_attn &p = a.w.p;
    const int b = blockIdx.y, h = blockIdx.x / RANGE_PARTS, part = blockIdx.x % RANGE_PARTS;
    const WinSeq sq = win_seq(p, b);
    if (!sq.ok || sq.ql == 0) return;
    const WinKeys keys = win_keys(p, sq, 0, sq.ql - 1);
    __shared__ float s_top[2][4];
    float top[2] = {0.0f, 0.0f};
    for (int v = part * 256 + threadIdx.x; v < keys.count; v += RANGE_PARTS * 256) {
        const int j = keys.at(v), slot = j % p.page, id = p.d_table[b * p.table_stride + j / p.page];
        if ((unsigned)id >= (unsigned)p.pages) continue;
#pragma unroll
        for (int is_v = 0; is_v < 2; is_v++) {
            const long long *st = is_v ? a.vs_stride : a.ks_stride;
            const T *pair = static_cast<const T *>(is_v ? a.vs : a.ks) + id * st[0] + slot * st[1] + h * st[2];
            for (int e = 0; e < groups; e++) {
                const float s = (float)pair[2 * e], lo = (float)pair[2 * e + 1];
                const float size = __builtin_fmaxf(__builtin_fabsf(lo), __builtin_fabsf(__builtin_fmaf(15.0f, s, lo)));
                if (size < __builtin_inff()) top[is_v] = __builtin_fmaxf(top[is_v], size);
            }
        }
    }
#pragma unroll
    for (int is_v = 0; is_v < 2; is_v++) {
#pragma unroll
        for (int o = 32; o; o >>= 1) top[is_v] = __builtin_fmaxf(top[is_v], __shfl_xor(top[is_v], o));
        if ((threadIdx.x & 63) == 0) s_top[is_v][threadIdx.x >> 6] = top[is_v];
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        float t = s_top[threadIdx.x][0];
        for (int w = 1; w < 4; w++) t = __builtin_fmaxf(t, s_top[threadIdx.x][w]);
        a.wide_top[2 * (((long long)b * p.kv_heads + h) * RANGE_PARTS + part) + threadIdx.x] = t;
    }
}

// The visible keys and values, the new ones too, into f16 pages, and the table of those.
// blockIdx.y is the sequence, blockIdx.x and .z deal out its pages and heads.
template <typename T>
__global__ __launch_bounds__(256) void kv4_expand_kernel(Kv4Args a, int group_log) {
    const osh_window_attn &p = a.w.p;
    const int b = blockIdx.y, d = p.head_dim, chunks = d / 8;
    const WinSeq sq = win_seq(p, b);
    if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) a.wide_kl[b] = sq.ok ? sq.kl : -1;
    if (!sq.ok || sq.ql == 0) return;
    const WinKeys keys = win_keys(p, sq, 0, sq.ql - 1);
    const WideBlocks blocks = kv4_blocks(p, sq, keys);
    for (int h = blockIdx.z; h < p.kv_heads; h += gridDim.z)
    for (int at = blockIdx.x; at < a.wide_blocks; at += gridDim.x) {
        const int block = blocks.at(at);
        if (block >= blocks.count) break;
        const long long head = (long long)b * p.kv_heads + h, page = (long long)b * a.wide_blocks + at;
        float by[2];
#pragma unroll
        for (int is_v = 0; is_v < 2; is_v++) {
            float top = a.wide_top[2 * (head * RANGE_PARTS + threadIdx.x % RANGE_PARTS) + is_v];
#pragma unroll
            for (int o = 1; o < RANGE_PARTS; o <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o));
            by[is_v] = __builtin_amdgcn_ldexpf(1.0f, -min(max(__builtin_amdgcn_frexp_expf(top), -120), 126));
        }
        if (threadIdx.x == 0) {
            if (h == 0) a.wide_table[(long long)b * a.wide_width + block] = (int)page;
            if (at == 0) a.wide_by[2 * head] = by[0], a.wide_by[2 * head + 1] = by[1];
        }
        for (int e = threadIdx.x; e < WIDE_PAGE * chunks; e += 256) {
            const int in = e / chunks, c = e - in * chunks;
            const int j = block * WIDE_PAGE + in;
            if (j >= sq.kl || (j < keys.lo && j >= p.sinks)) continue;
            const int slot = j % p.page, id = p.d_table[b * p.table_stride + j / p.page];
            f32x8 k = f32x8{} + __builtin_nanf(""), v = {};
            if ((unsigned)id < (unsigned)p.pages) {
                auto load = [&](const void *codes, const int64_t *st, const void *pairs, const long long *pst, float by) {
                    const unsigned w = *reinterpret_cast<const unsigned *>(static_cast<const char *>(codes) + id * st[0] +
                                                                           slot * st[1] + h * st[2] + 4 * c);
                    const T *pair = static_cast<const T *>(pairs) + id * pst[0] + slot * pst[1] + h * pst[2] +
                                    2 * (8 * c >> group_log);
                    f32x8 f;
#pragma unroll
                    for (int i = 0; i < 8; i++) f[i] = __builtin_fmaf((float)pair[0], (float)(w >> (4 * i) & 15u), (float)pair[1]);
                    return f * by;
                };
                k = load(p.d_k_pages, p.k_stride, a.ks, a.ks_stride, by[0]);
                v = load(p.d_v_pages, p.v_stride, a.vs, a.vs_stride, by[1]);
            }
            const long long to = ((page * p.kv_heads + h) * WIDE_PAGE + in) * d + 8 * c;
            store8(a.k_wide + to, k);
            store8(a.v_wide + to, v);
        }
    }
}

// ----------------------------------------------------------------- few rows

// One workgroup: 16 query rows of one key head, one split of their keys; each wave takes
// every WAVES-th step of 64 keys of the split.
//
// S^T = K Q^T: MFMA row rho of block b is key 16 (rho / 4) + 4 b + rho % 4 of the step, so
// that lane (jl, g) ends with the scores of keys 16 g .. + 15 at query jl, just the operand
// of O^T = V^T P^T.  Codes pass through the wave's own LDS, loaded directly, CP chunks of 16
// bytes a key; K's words are read as they lie, V's by the LDS read that transposes 4-bit
// elements: 16 keys of one value a lane.
//
// The next step's codes are loaded while this one is computed.
// At most N loads in flight.
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ unsigned lds_offset(const void *p) {
    return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void *)p;
}
// 8 bytes to LDS.  By hand: in front of an LDS write of its own the compiler waits for all
// direct loads in flight.  The caller waits for lgkmcnt before it reads.
__device__ __forceinline__ void write_pair(const float2 *to, float2 v) {
    asm volatile("ds_write_b64 %0, %1" ::"v"(lds_offset(to)), "v"(v) : "memory");
}

// Both halves of two or four chunks, transposed among the 16 lanes of a group: a lane's 8
// bytes at a chunk's half become 16 rows' codes of one column.  By hand for the same reason,
// with the wait.
__device__ __forceinline__ void read_transposed4(const void *a, const void *b, unsigned (*to)[2]) {
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    u32x2 r[4];
    asm volatile("ds_read_b64_tr_b4 %0, %4\n\tds_read_b64_tr_b4 %1, %4 offset:8\n\t"
                 "ds_read_b64_tr_b4 %2, %5\n\tds_read_b64_tr_b4 %3, %5 offset:8\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
                 : "v"(lds_offset(a)), "v"(lds_offset(b))
                 : "memory");
#pragma unroll
    for (int i = 0; i < 4; i++) to[i][0] = r[i][0], to[i][1] = r[i][1];
}
__device__ __forceinline__ void read_transposed8(const void *a, const void *b, const void *c, const void *d,
                                                 unsigned (*to)[2]) {
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    u32x2 r[8];
    asm volatile("ds_read_b64_tr_b4 %0, %8\n\tds_read_b64_tr_b4 %1, %8 offset:8\n\t"
                 "ds_read_b64_tr_b4 %2, %9\n\tds_read_b64_tr_b4 %3, %9 offset:8\n\t"
                 "ds_read_b64_tr_b4 %4, %10\n\tds_read_b64_tr_b4 %5, %10 offset:8\n\t"
                 "ds_read_b64_tr_b4 %6, %11\n\tds_read_b64_tr_b4 %7, %11 offset:8\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
                 : "v"(lds_offset(a)), "v"(lds_offset(b)), "v"(lds_offset(c)), "v"(lds_offset(d))
                 : "memory");
#pragma unroll
    for (int i = 0; i < 8; i++) to[i][0] = r[i][0], to[i][1] = r[i][1];
}
// Two words: at a read of a struct the compiler waits too.
__device__ __forceinline__ float2 read_pair(const float2 *from) {
    const unsigned *u = reinterpret_cast<const unsigned *>(from);
    return float2{__uint_as_float(u[0]), __uint_as_float(u[1])};
}

// With SUB 2 or 4 at most 16 / SUB rows are there, and column jl of the products stands for row
// jl % (16 / SUB) over every SUB-th part of each 16 keys: a lane has KPL = 16 / SUB scores a
// step in place of 16, of which most would belong to no row.  Its weights of other keys are 0,
// and its columns' maxima and sums are joined with those of the waves.
template <typename T, int CP, int GS, int WAVES, int SUB>
__global__ __launch_bounds__(64 * WAVES, CP > 4 ? 1 : 2) void kv4_rows_kernel(Kv4Args args) {
    constexpr int RP = 16 / SUB, KPL = 16 / SUB;
    constexpr int NG = CP / GS;        // groups of a head
    constexpr int DP = 32 * CP, OB = 2 * CP, KPI = 64 / CP;
    constexpr int TILE = 64 * CP * 16;
    using H8 = typename Half8<T>::type;
    extern __shared__ __align__(16) unsigned char lds[];
    constexpr int WAVE_LDS = 4 * TILE + 256 + 2 * NG * (256 + 512);
    const WinArgs &a = args.w;
    const osh_window_attn &p = a.p;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int jl = lane & 15, g = lane >> 4;
    const int d = p.head_dim, G = a.group;

    int id = blockIdx.x;
    const int split = id % a.splits;
    id /= a.splits;
    const int unit = id;
    const int tile = id % a.tiles;
    id /= a.tiles;
    const int h = id % p.kv_heads, b = id / p.kv_heads;
    const WinSeq sq = win_seq(p, b);
    const int rows = sq.ql * G, r0 = tile * RP;
    if (!sq.ok) {
        if (tile == 0 && split == 0) {
            win_fill_nan<T>(p, sq, h, G, tid, 64 * WAVES);
            if (args.append) kv4_append<T, 4 * GS>(args, sq, b, h, h + 1, 0, sq.held, tid, 64 * WAVES);  // NaN to the stored values
        }
        return;
    }
    if (r0 >= rows) return;
    T *o = static_cast<T *>(p.d_o);
    const int sub = jl / RP;
    const int my_row = min(r0 + jl % RP, rows - 1), my_tok = my_row / G, my_head = h * G + my_row % G;

    // queries: step t of group e takes of lane (jl, g) the 8 values from 32 GS e + 8 (GS g + t) on
    // of row jl, so that the lane's codes of a group are GS words in a row, in codes8's order;
    // and their sums over a group
    H8 q[CP];
    float qs[NG];
    {
        const T *qr = static_cast<const T *>(p.d_q) + (long long)(sq.c0 + my_tok) * p.q_stride[0] +
                      my_head * p.q_stride[1];
#pragma unroll
        for (int e = 0; e < NG; e++) qs[e] = 0.0f;
#pragma unroll
        for (int s = 0; s < CP; s++) {
            H8 x = {};
            const int from = 32 * GS * (s / GS) + 8 * (GS * g + s % GS);
            if (from < d) __builtin_memcpy(&x, qr + from, 16);
#pragma unroll
            for (int i = 0; i < 8; i++) qs[s / GS] += (float)x[i];
            q[s] = __builtin_shufflevector(x, x, 0, 2, 4, 6, 1, 3, 5, 7);
        }
#pragma unroll
        for (int e = 0; e < NG; e++) {
            qs[e] += __shfl_xor(qs[e], 16);
            qs[e] += __shfl_xor(qs[e], 32);
        }
    }
    const int tok0 = r0 / G, tok1 = min(r0 + RP - 1, rows - 1) / G;
    const WinKeys keys = win_keys(p, sq, tok0, tok1);
    const int nv = keys.count;
    const int steps = cdiv(nv, 64), per = cdiv(steps, a.splits);
    const int s_end = min(steps, (split + 1) * per);
    // the new ones among this workgroup's keys go to the cache first, from where all keys are
    // read; another row block may write the same bytes there
    if (args.append) {
        const int v0 = split * per * 64, v1 = min(nv, s_end * 64);
        const int t0 = max(0, (v0 < nv ? keys.at(v0) : sq.kl) - sq.past), t1 = v1 > v0 ? keys.at(v1 - 1) + 1 - sq.past : 0;
        if (t1 > t0) kv4_append<T, 4 * GS>(args, sq, b, h, h + 1, t0, t1, tid, 64 * WAVES);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
    const int pos0 = sq.past + tok0, pos1 = sq.past + tok1;
    // by key number, this row sees v <= v_hi with v >= v_lo or v < v_sink
    const int shift = keys.sink_end - keys.lo, my_pos = sq.past + my_tok;
    const int v_sink = max(keys.sink_end, win_min(p.sinks, 1 << 30) + shift);
    const int v_hi = my_pos + shift, v_lo = max(my_pos - p.window + 1, keys.lo) + shift;

    float m = -__builtin_inff(), l = 0.0f, zsum[NG];
    f32x4 acc[OB];
#pragma unroll
    for (int i = 0; i < OB; i++) acc[i] = f32x4{0, 0, 0, 0};
    // f16 weights: p scale times a power of two of each group, since f16 has no room for the
    // scales' own range: the scale that sets it becomes 2^9 to 2^10, and none passes 2^15
    constexpr bool UNIT = __is_same(T, _Float16);
    float by[NG];
#pragma unroll
    for (int e = 0; e < NG; e++) zsum[e] = 0.0f, by[e] = 0x1p127f;  // the first scale passes

    unsigned char *mine = lds + wave * WAVE_LDS;
    const float2 *kpair = reinterpret_cast<const float2 *>(mine + 4 * TILE + 256 + 2 * NG * 256), *vpair = kpair + NG * 64;
    auto k_swizzle = [](int key) { return CP == 8 ? (key >> 4 & 3) | (key >> 1 & 1) << 2 : key >> 4 & (CP - 1); };
    auto v_swizzle = [](int key) { return key >> 2 & (CP - 1); };

    // Everything a step reads goes to LDS directly: page ids two steps ahead, codes and scale
    // pairs one.  Always for a key that there is (past the last key its own again), so that no
    // load stands under a condition and the waits, which are written by hand, can count them:
    // loads return in order.
    unsigned char *raw_ids = mine + 4 * TILE, *raw_sc = raw_ids + 256;
    unsigned long long k_row, v_row, k_sc, v_sc;  // of key `lane` of the next step
    bool in = false, bad = false;
    auto position = [&](int st) { return keys.at(min(st * 64 + lane, nv - 1)); };
    auto page_of = [&](int j) { return (int)(__umulhi((unsigned)j << 2, args.page_mul) >> args.page_log); };
    auto load_ids = [&](int st) {
        copy_to_lds<4>(p.d_table + (b * p.table_stride + page_of(position(st))), raw_ids);
        __builtin_amdgcn_sched_barrier(0);  // stays in front of the codes
    };
    auto place = [&](int st) {
        int page_id = reinterpret_cast<const int *>(raw_ids)[lane];
        // in a register before the next ids are on their way: those of a table that the L1
        // holds arrive before a read that waits in a busy LDS
        asm volatile("" : "+v"(page_id)::"memory");
        const int j = position(st), slot = j - page_of(j) * p.page;
        in = st * 64 + lane < nv;
        bad = (unsigned)page_id >= (unsigned)p.pages;
        const unsigned long long zero = (unsigned long long)win_zero_row;
        auto where = [&](const void *base, int e, long long s0, long long s1, long long s2) {
            const unsigned long long at = (unsigned long long)base + e * (h * s2) +
                                          (unsigned long long)(unsigned)page_id * (unsigned)(e * s0) +
                                          (unsigned long long)(unsigned)slot * (unsigned)(e * s1);
            return bad ? zero : at;
        };
        k_row = where(p.d_k_pages, 1, p.k_stride[0], p.k_stride[1], p.k_stride[2]);
        v_row = where(p.d_v_pages, 1, p.v_stride[0], p.v_stride[1], p.v_stride[2]);
        k_sc = where(args.ks, 2, args.ks_stride[0], args.ks_stride[1], args.ks_stride[2]);
        v_sc = where(args.vs, 2, args.vs_stride[0], args.vs_stride[1], args.vs_stride[2]);
    };
    const int last_chunk = d / 32 - 1;  // slots of no value hold a copy of it, and meet queries of 0
    auto load_codes = [&](int buf) {
        unsigned char *kt = mine + buf * 2 * TILE, *vt = kt + TILE;
        const char *kr[CP], *vr[CP];  // all of them before the first copy: one wait for the LDS
#pragma unroll
        for (int i = 0; i < CP; i++) {
            const int key = i * KPI + lane / CP;
            kr[i] = (const char *)__shfl(k_row, key), vr[i] = (const char *)__shfl(v_row, key);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < CP; i++) {
            const int key = i * KPI + lane / CP, slot = lane % CP;
            copy_to_lds<16>(kr[i] + 16 * min(slot ^ k_swizzle(key), last_chunk), kt + i * 1024);
            copy_to_lds<16>(vr[i] + 16 * min(slot ^ v_swizzle(key), last_chunk), vt + i * 1024);
        }
    };
    constexpr int SC_LOADS = 2 * NG;
    const int last_pair = d / (32 * GS) - 1;  // likewise
    auto load_scales = [&] {
#pragma unroll
        for (int e = 0; e < NG; e++) {
            const int from = 4 * min(e, last_pair);
            copy_to_lds<4>((const char *)k_sc + from, raw_sc + e * 256);
            copy_to_lds<4>((const char *)v_sc + from, raw_sc + (NG + e) * 256);
        }
    };
    auto raw_pair = [&](int is_v, int e) {
        return reinterpret_cast<const unsigned *>(raw_sc + (is_v * NG + e) * 256)[lane];
    };
    auto pair_of = [](unsigned u) {
        T t[2];
        __builtin_memcpy(t, &u, 4);
        return float2{(float)t[0], (float)t[1]};
    };
    // a step's pairs in FP32 to LDS: K's times the softmax's scale, V's scale as the weights take it
    auto convert = [&](bool in, bool bad) {
        float2 kp[NG], vp[NG];
#pragma unroll
        for (int e = 0; e < NG; e++) {
            kp[e] = pair_of(raw_pair(0, e)), vp[e] = pair_of(raw_pair(1, e));
            kp[e].x *= a.scale_log2, kp[e].y *= a.scale_log2;
            if (bad) kp[e].x = __builtin_nanf("");
            if (!in) vp[e] = float2{0.0f, 0.0f};
            if constexpr (UNIT) {
                const float scale = vp[e].x;
                vp[e].x *= by[e];
                if (__builtin_amdgcn_ballot_w64(__builtin_fabsf(vp[e].x) > 0x1p15f) != 0) {
                    float top = __builtin_fabsf(scale);
#pragma unroll
                    for (int i = 32; i; i >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, i));
                    const float next = __uint_as_float((263u << 23) - (__float_as_uint(top) & 0x7f800000u));
                    const float fade = next / by[e];
                    by[e] = next, vp[e].x = scale * next;
#pragma unroll
                    for (int i = 2 * GS * e; i < 2 * GS * (e + 1); i++) acc[i] *= fade;
                }
            }
        }
#pragma unroll
        for (int e = 0; e < NG; e++) {
            write_pair(kpair + e * 64 + lane, kp[e]);
            write_pair(vpair + e * 64 + lane, vp[e]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
    // products of the queries with a step's codes of K: they need no scales
    f32x4 prod[4][NG];
    auto multiply = [&](int buf) {
        const unsigned char *kt = mine + buf * 2 * TILE;
        unsigned w[4][CP];
#pragma unroll
        for (int bl = 0; bl < 4; bl++) {
            const int key = 16 * (jl >> 2) + 4 * bl + (jl & 3);
#pragma unroll
            for (int e = 0; e < NG; e++) {
                const int chunk = e * GS + g * GS / 4;
                const unsigned *from = static_cast<const unsigned *>(__builtin_assume_aligned(
                    kt + key * (CP * 16) + ((chunk ^ k_swizzle(key)) << 4) + (g * GS * 4 & 15), GS * 4));
#pragma unroll
                for (int t = 0; t < GS; t++) w[bl][e * GS + t] = from[t];
            }
        }
#pragma unroll
        for (int bl = 0; bl < 4; bl++)
#pragma unroll
            for (int e = 0; e < NG; e++)
#pragma unroll
                for (int t = 0; t < GS; t++) {
                    H8 k;
                    codes8(w[bl][e * GS + t], k);
                    prod[bl][e] = mma16(k, q[e * GS + t], t == 0 ? f32x4{0, 0, 0, 0} : prod[bl][e]);
                }
    };
    auto compute = [&](int st, int buf) {
        const unsigned char *vt = mine + buf * 2 * TILE + TILE;
        float s[KPL];
        const int mine16 = 16 * g + KPL * sub;  // this lane's keys of the step
#pragma unroll
        for (int i = 0; i < KPL; i++) s[i] = 0.0f;
#pragma unroll
        for (int e = 0; e < NG; e++)
#pragma unroll
            for (int i = 0; i < KPL; i++) {
                float c = prod[i / 4][e][i % 4];
                if constexpr (SUB == 2) c = sub ? prod[2 + i / 4][e][i % 4] : c;
                if constexpr (SUB == 4) {
                    const float hi = sub & 1 ? prod[3][e][i] : prod[2][e][i];
                    c = sub & 1 ? prod[1][e][i] : c;
                    c = sub & 2 ? hi : c;
                }
                const float2 kp = read_pair(kpair + e * 64 + mine16 + i);
                s[i] = __builtin_fmaf(kp.x, c, s[i]);
                s[i] = __builtin_fmaf(kp.y, qs[e], s[i]);
            }
        const int v0 = st * 64, j0 = keys.at(v0), j1 = keys.at(v0 + 63);
        const bool all = v0 + 63 < nv && j1 <= pos0 &&
                         (j1 < p.sinks || (v0 >= keys.sink_end && j0 > pos1 - p.window));
        if (!all) {
            const int mine0 = v0 + mine16, hi = v_hi - mine0, lo = v_lo - mine0, sink = v_sink - mine0;
#pragma unroll
            for (int i = 0; i < KPL; i++) {
                const bool hidden = (i > hi) | ((i < lo) & (i >= sink));
                s[i] = hidden ? -__builtin_inff() : s[i];
            }
        }
        float top = s[0];
#pragma unroll
        for (int i = 1; i < KPL; i++) top = __builtin_fmaxf(top, s[i]);
        top = __builtin_fmaxf(top, __shfl_xor(top, 16));
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        if (__builtin_amdgcn_ballot_w64(top > m) != 0) {
            const float old = m;
            m = __builtin_fmaxf(m, top);
            const float fade = old == m ? 1.0f : __builtin_amdgcn_exp2f(old - m);
            l *= fade;
#pragma unroll
            for (int i = 0; i < OB; i++) acc[i] *= fade;
#pragma unroll
            for (int e = 0; e < NG; e++) zsum[e] *= fade;
        }
        // lane jl of 16 reads 16 codes of key 16 g + jl and gets 16 keys' codes of value jl
        unsigned vw[OB][2];
        {
            const int key = 16 * g + jl;
            const unsigned char *row = vt + key * (CP * 16);
            if constexpr (CP == 2) {
                read_transposed4(row + (v_swizzle(key) << 4), row + ((1 ^ v_swizzle(key)) << 4), vw);
            } else {
#pragma unroll
                for (int c = 0; c < CP; c += 4)
                    read_transposed8(row + ((c ^ v_swizzle(key)) << 4), row + (((c + 1) ^ v_swizzle(key)) << 4),
                                     row + (((c + 2) ^ v_swizzle(key)) << 4), row + (((c + 3) ^ v_swizzle(key)) << 4),
                                     vw + 2 * c);
            }
        }
        const float ref = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
        for (int i = 0; i < KPL; i++) {
            s[i] = __builtin_amdgcn_exp2f(s[i] - ref);
            l += s[i];
        }
#pragma unroll
        for (int e = 0; e < NG; e++) {
            if (NG > 2 && SUB == 1) __builtin_amdgcn_sched_barrier(0);
            // weights in the order of codes8: of 8 keys the even ones, then the odd ones; what
            // rounding to T leaves of them is a second operand
            float w[KPL];
#pragma unroll
            for (int i = 0; i < KPL; i++) {
                const float2 vp = read_pair(vpair + e * 64 + mine16 + i);
                w[i] = s[i] * vp.x;
                zsum[e] = __builtin_fmaf(s[i], vp.y, zsum[e]);
            }
            H8 p[2][2];  // by part and 8 keys
#pragma unroll
            for (int part = 0; part < 2; part++) {
                unsigned pw[8];
                auto two = [&](int i, int j) {
                    typedef T T2 __attribute__((ext_vector_type(2)));
                    const T2 v = {(T)w[i], (T)w[j]};
                    if (part == 0) w[i] = __builtin_fmaf((float)v[0], -1.0f, w[i]), w[j] = __builtin_fmaf((float)v[1], -1.0f, w[j]);
                    return __builtin_bit_cast(unsigned, v);
                };
#pragma unroll
                for (int i = 0; i < 8; i++) {  // registers 0..3 are of the first 8 keys
                    if constexpr (SUB == 1) pw[i] = two(8 * (i >> 2) + 4 * (i & 1) + (i >> 1 & 1), 8 * (i >> 2) + 4 * (i & 1) + (i >> 1 & 1) + 2);
                }
                if constexpr (SUB > 1) {
                    unsigned at[KPL / 2];
#pragma unroll
                    for (int i = 0; i < KPL / 2; i++) at[i] = two(4 * (i >> 1) + (i & 1), 4 * (i >> 1) + (i & 1) + 2);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int of = SUB == 2 ? i >> 2 : 2 * (i >> 2) + (i & 1);
                        pw[i] = sub == of ? at[SUB == 2 ? 2 * (i & 1) + (i >> 1 & 1) : i >> 1 & 1] : 0u;
                    }
                }
                __builtin_memcpy(&p[part][0], pw, 16);
                __builtin_memcpy(&p[part][1], pw + 4, 16);
            }
#pragma unroll
            for (int i = 2 * GS * e; i < 2 * GS * (e + 1); i++)
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    H8 v;
                    codes8(vw[i][half], v);
                    acc[i] = mma16(v, p[0][half], acc[i]);
                    acc[i] = mma16(v, p[1][half], acc[i]);
                }
        }
    };
    int st = split * per + wave;
    if (st < s_end) {
        load_ids(st);
        wait_loads<0>();
        place(st);
        load_ids(st + WAVES);
        load_codes(0);
        load_scales();
        int buf = 0;
        for (; st + WAVES < s_end; st += WAVES, buf ^= 1) {
            const bool now_in = in, now_bad = bad;
            wait_loads<2 * CP + SC_LOADS>();
            place(st + WAVES);
            load_ids(st + 2 * WAVES);
            load_codes(buf ^ 1);
            wait_loads<2 * CP + 1>();
            multiply(buf);
            convert(now_in, now_bad);
            load_scales();
            compute(st, buf);
        }
        wait_loads<0>();
        multiply(buf);
        convert(in, bad);
        compute(st, buf);
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
#pragma unroll
    for (int e = 0; e < NG; e++) {
        zsum[e] += __shfl_xor(zsum[e], 16);
        zsum[e] += __shfl_xor(zsum[e], 32);
    }

    // join the waves: [WAVES][16] pairs (m, l), then [WAVES][16][DP + 4] sums
    constexpr int OP = DP + 4;
    __syncthreads();
    float *ml = reinterpret_cast<float *>(lds), *os = ml + WAVES * 32;
    if (g == 0) {
        ml[(wave * 16 + jl) * 2] = m;
        ml[(wave * 16 + jl) * 2 + 1] = l;
    }
#pragma unroll
    for (int i = 0; i < OB; i++) {
        f32x4 f = acc[i];
        if (UNIT) f *= 1.0f / by[i / (2 * GS)];
        f += zsum[i / (2 * GS)];
        *reinterpret_cast<f32x4 *>(os + (wave * 16 + jl) * OP + 16 * i + 4 * g) = f;
    }
    __syncthreads();
    for (int e = tid; e < RP * DP; e += 64 * WAVES) {
        const int r = e / DP, c = e % DP, row = r0 + r;
        if (row >= rows || c >= d) continue;
        float mm = ml[r * 2];
#pragma unroll
        for (int w = 1; w < WAVES * SUB; w++) mm = __builtin_fmaxf(mm, ml[(w * RP + r) * 2]);
        const float base = mm == -__builtin_inff() ? 0.0f : mm;
        float sum = 0.0f, ll = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES * SUB; w++) {
            const float f = __builtin_amdgcn_exp2f(ml[(w * RP + r) * 2] - base);
            ll += f * ml[(w * RP + r) * 2 + 1];
            sum += f * os[(w * RP + r) * OP + c];
        }
        if (a.splits == 1) {
            o[(long long)(sq.c0 + row / G) * p.o_stride[0] + (h * G + row % G) * p.o_stride[1] + c] = (T)(sum / ll);
        } else {
            const long long u = (long long)unit * a.splits + split;
            a.part_o[(u * RP + r) * d + c] = sum;
            if (c == 0) {
                a.part_ml[(u * RP + r) * 2] = mm;
                a.part_ml[(u * RP + r) * 2 + 1] = ll;
            }
        }
    }
}

template <typename T, int CP, int GS, int SUB, int WAVES>
static osh_status kv4_rows_launch_w(const Kv4Args &a, unsigned units, hipStream_t st) {
    constexpr size_t wave_lds = 4 * 64 * CP * 16 + 256 + 2 * (CP / GS) * (256 + 512);
    constexpr size_t lds = std::max<size_t>(WAVES * wave_lds, WAVES * 16 * (32 * CP + 4 + 2) * sizeof(float));
    OSH_LAUNCH((kv4_rows_kernel<T, CP, GS, WAVES, SUB>), dim3(units * a.w.splits), dim3(64 * WAVES), lds, st, a);
    OSH_LAUNCH_CHECK("kv4_rows_kernel");
    return win_join<T>(a.w, units, st);
}

template <typename T, int CP, int GS, int SUB>
static osh_status kv4_rows_launch_s(const Kv4Args &a, unsigned units, hipStream_t st) {
    constexpr int NG = CP / GS;
    if constexpr (SUB > 1 && CP <= 4 && NG <= 2) {
        if (a.w.wide) return kv4_rows_launch_w<T, CP, GS, SUB, 8>(a, units, st);
    }
    return kv4_rows_launch_w<T, CP, GS, SUB, NG == 8 ? 3 : 4>(a, units, st);  // what 160 KB hold
}

template <typename T, int CP, int GS>
static osh_status kv4_rows_launch(const Kv4Args &a, unsigned units, hipStream_t st) {
    if (a.w.tile_rows == 4) return kv4_rows_launch_s<T, CP, GS, 4>(a, units, st);
    if constexpr (CP / GS < 8) {
        if (a.w.tile_rows == 8) return kv4_rows_launch_s<T, CP, GS, 2>(a, units, st);
    }
    if constexpr (CP / GS < 4) return kv4_rows_launch_s<T, CP, GS, 1>(a, units, st);
    return fail(OSH_E_UNSUPPORTED, "Kv4Attention: no kernel for %d rows", a.w.tile_rows);
}

template <typename T, int GL>
static osh_status kv4_append_all(const Kv4Args &a, hipStream_t st) {
    const osh_window_attn &p = a.w.p;
    const long long threads = (long long)p.max_q * p.kv_heads * 2 * (p.head_dim / 8);
    const unsigned x = (unsigned)std::max(1LL, std::min((threads + 255) / 256, std::max(1LL, 65536LL / p.batch)));
    OSH_LAUNCH((kv4_append_kernel<T, GL>), dim3(x, (unsigned)p.batch), dim3(256), 0, st, a);
    OSH_LAUNCH_CHECK("kv4_append_kernel");
    return OSH_OK;
}

template <typename T, int GS>
static osh_status kv4_launch_g(const Kv4Args &a, unsigned units, hipStream_t st) {
    const int d = a.w.p.head_dim;
    if constexpr (GS <= 2) {
        if (d <= 64) return kv4_rows_launch<T, 2, GS>(a, units, st);
    }
    if (d <= 128) return kv4_rows_launch<T, 4, GS>(a, units, st);
    return kv4_rows_launch<T, 8, GS>(a, units, st);
}

static osh_status kv4_wide(const Kv4Args &a, const WinArgs &wide, int group, unsigned units, hipStream_t st) {
    const osh_window_attn &p = a.w.p;
    OSH_LAUNCH(kv4_range_kernel<__bf16>, dim3((unsigned)p.kv_heads * RANGE_PARTS, (unsigned)p.batch), dim3(256), 0, st, a,
               p.head_dim / group);
    OSH_LAUNCH_CHECK("kv4_range_kernel");
    const int x = std::min(a.wide_blocks, std::max(1, 65536 / p.batch));
    OSH_LAUNCH(kv4_expand_kernel<__bf16>, dim3((unsigned)x, (unsigned)p.batch, (unsigned)std::min(p.kv_heads, 256)), dim3(256), 0, st, a, __builtin_ctz(group));
    OSH_LAUNCH_CHECK("kv4_expand_kernel");
    return win_run_expanded(wide, units, st);
}

template <typename T>
static osh_status kv4_launch(const Kv4Args &a, const WinArgs &wide, int group, unsigned units, hipStream_t st) {
    if (!a.append) {
        const osh_status s = group == 32   ? kv4_append_all<T, 4>(a, st)
                             : group == 64 ? kv4_append_all<T, 8>(a, st)
                                           : kv4_append_all<T, 16>(a, st);
        if (s) return s;
    }
    if constexpr (__is_same(T, __bf16)) {
        if (a.wide_blocks) return kv4_wide(a, wide, group, units, st);
    }
    if (group == 32) return kv4_launch_g<T, 1>(a, units, st);
    if (group == 64) return kv4_launch_g<T, 2>(a, units, st);
    return kv4_launch_g<T, 4>(a, units, st);
}

// Where the parts of the scratch lie: a.w's own or, with many rows, `wide`, the 16-bit call.
struct Kv4Room {
    bool wide;
    size_t part, page, by, table, kl, total;  // bytes; page: of K or V
};

// Rows of a key head from which a bf16 call first expands the visible cache to f16, and the room
// that may take.  4096 tokens behind 12288, 32 heads of 128 on 8, window 8192: 690 us so, 1726 as
// f16 blocks of 16 rows (f16 has no type with bits to spare for it); behind 8128, 4 x 64 tokens
// (256 rows) 125 in blocks, 4 x 127 224, 4 x 128 153 so.
constexpr int WIDE_ROWS = 512;
constexpr size_t WIDE_MAX = (size_t)16 << 30;

static osh_status kv4_plan(const osh_kv4_attn *p, Kv4Args &args, WinArgs &wide, Kv4Room &room) {
    if (!p) return fail(OSH_E_INVALID, "Kv4Attention: NULL parameters");
    WinArgs &a = args.w;
    room = {};
    args = {};
    if (const osh_status st = win_plan(&p->w, a, room.part)) return st;
    if (p->group != 32 && p->group != 64 && p->group != 128)
        return fail(OSH_E_UNSUPPORTED, "Kv4Attention: groups of %d (32, 64 or 128)", p->group);
    if (p->w.head_dim % p->group)
        return fail(OSH_E_UNSUPPORTED, "Kv4Attention: heads of %d in groups of %d", p->w.head_dim, p->group);
    if (p->w.batch > 65535) return fail(OSH_E_UNSUPPORTED, "Kv4Attention: %d sequences", p->w.batch);
    const int rows = p->w.max_q * a.group;
    auto align = [](size_t n) { return (n + 255) / 256 * 256; };
    if (rows >= WIDE_ROWS && p->w.batch && p->w.dtype == OSH_T_BF16) {
        const long long most = cdiv(p->w.max_kv, WIDE_PAGE), sinks = cdiv(std::min(p->w.sinks, p->w.max_kv), WIDE_PAGE);
        const long long span = std::min<long long>(p->w.max_kv, (long long)p->w.window - 1 + p->w.max_q);
        args.wide_blocks = (int)std::min(most, sinks + (span + WIDE_PAGE - 1) / WIDE_PAGE + 1);
        args.wide_width = (int)most;
        osh_window_attn w = p->w;
        w.page = WIDE_PAGE;
        w.table_width = args.wide_width;
        w.table_stride = args.wide_width;
        const long long pages = (long long)w.batch * args.wide_blocks, head = (long long)w.head_dim;
        w.pages = (int)std::min<long long>(pages, INT_MAX);
        w.k_stride[0] = w.v_stride[0] = w.kv_heads * WIDE_PAGE * head;
        w.k_stride[1] = w.v_stride[1] = head;
        w.k_stride[2] = w.v_stride[2] = WIDE_PAGE * head;
        if (const osh_status st = win_plan(&w, wide, room.part)) return st;
        room.part = align(room.part);
        room.by = align((size_t)w.batch * w.kv_heads * 8 * (1 + RANGE_PARTS));
        room.table = align((size_t)w.batch * args.wide_width * 4);
        room.kl = align((size_t)w.batch * 4);
        const double bytes = 4.0 * pages * w.kv_heads * WIDE_PAGE * head;
        room.wide = pages <= INT_MAX && w.k_stride[0] <= INT_MAX && bytes <= (double)WIDE_MAX;
        room.page = room.wide ? (size_t)bytes / 2 : 0;
        room.total = room.part + room.by + 2 * room.page + room.table + room.kl;
        if (room.wide) return OSH_OK;
        args.wide_blocks = 0;
    }
    // four or eight groups a head leave no registers for 16 rows' scores: 16 rows of 64 sequences
    // of 5000 keys, 8 heads of 128 in groups of 32, took 465 us in one block (spilled) and take 242 in two
    const int groups = cdiv(p->w.head_dim, 128) * (p->w.head_dim <= 64 ? 64 : 128) / p->group;
    const int most = groups >= 8 ? 4 : groups >= 4 ? 8 : 16;
    a.tile_rows = std::min(most, rows <= 4 ? 4 : rows <= 8 ? 8 : 16);
    a.tiles = cdiv(rows, a.tile_rows);
    const long long units = (long long)p->w.batch * p->w.kv_heads * a.tiles;
    if (units >= (1LL << 22)) return fail(OSH_E_UNSUPPORTED, "Kv4Attention: too many row blocks (%lld)", units);
    // A sequence's few row blocks quantize the new tokens among their keys each for itself, which
    // saves a launch: with 2, 4 and 8 of them, one sequence behind 2000 keys (32 heads of 128 on 8) in
    // groups of 128, 15.4 (18.7 with one launch in front), 17.1 (19.2), 22.9 (22.2) us; 64 of them
    // 70.6 (71.6), 135 (128), 279 (234).  With many it is the square of the new tokens: 4096 f16 ones
    // behind 12288 10065 (1763).
    args.append = a.tiles == 1 || (a.tiles <= 4 && units <= device_cus());
    const long long span = std::min<long long>(p->w.max_kv, (long long)p->w.window + p->w.sinks + 16 / a.group);
    const long long want = units ? std::max(1LL, 2LL * device_cus() / units) : 1;
    a.splits = (int)std::max(1LL, std::min({want, span / 256, (long long)WIN_MAX_SPLITS}));
    // One launch of eight waves for short spans, where 160 KB hold them, else four waves, splits
    // and a join.  Eight against four over 200, 640, 1024 and 1500 keys: one sequence of 12 heads
    // of 64 on 4 in groups of 32: 9.5 (8.9), 10.8 (13.3), 12.0 (12.2), 13.6 (12.2) us; 32 of 32
    // heads of 128 on 8 in groups of 64: 13.1 (12.8), 16.1 (20.0), 18.3 (22.1), 23.2 (26.8).
    a.wide = a.tile_rows < 16 && span <= 1024 && units <= device_cus() && p->w.head_dim <= 128 && groups <= 2;
    if (a.wide) a.splits = 1;
    const long long parts = a.splits > 1 ? units * a.splits : 0;
    room.part = room.total = (size_t)parts * a.tile_rows * (p->w.head_dim + 2) * 4;
    return OSH_OK;
}

}  // namespace osh

extern "C" {

OSH_API osh_status osh_kv4_attention_scratch_bytes(const osh_kv4_attn *p, size_t *bytes) {
    if (!bytes) return fail(OSH_E_INVALID, "Kv4Attention: NULL bytes");
    Kv4Args a;
    WinArgs wide;
    Kv4Room room;
    const osh_status st = kv4_plan(p, a, wide, room);
    *bytes = room.total;
    return st;
}

OSH_API osh_status osh_kv4_attention(const osh_kv4_attn *q, void *d_scratch, osh_stream s) {
    Kv4Args a;
    WinArgs wide;
    Kv4Room room;
    if (const osh_status st = kv4_plan(q, a, wide, room)) return st;
    const size_t scratch = room.total;
    const osh_window_attn *p = &q->w;
    if (p->batch == 0 || p->max_q == 0 || p->tokens == 0) return OSH_OK;
    if (!p->d_q || !p->d_k_new || !p->d_v_new || !p->d_o || !p->d_k_pages || !p->d_v_pages || !p->d_table ||
        !p->d_cu || !p->d_kl || !q->d_k_scales || !q->d_v_scales || (scratch && (!d_scratch || ((uintptr_t)d_scratch & 15))) ||
        !q->d_k_stored != !q->d_v_stored)
        return fail(OSH_E_INVALID, "Kv4Attention: NULL pointer");
    const long long d = p->head_dim, groups = d / q->group;
    const int64_t *two[6] = {p->q_stride,     p->o_stride,        p->k_new_stride,
                             p->v_new_stride, q->k_stored_stride, q->v_stored_stride};
    for (int i = 0; i < 6; i++)
        if (two[i][0] < 0 || two[i][1] < 0) return fail(OSH_E_INVALID, "Kv4Attention: negative stride");
    const int64_t *three[4] = {p->k_stride, p->v_stride, q->k_scale_stride, q->v_scale_stride};
    const void *base[4] = {p->d_k_pages, p->d_v_pages, q->d_k_scales, q->d_v_scales};
    for (int i = 0; i < 4; i++) {
        const int unit = i < 2 ? 16 : 2;
        if ((uintptr_t)base[i] & (i < 2 ? 15 : 3))
            return fail(OSH_E_UNSUPPORTED, "Kv4Attention: codes need 16-byte alignment, scales 4-byte");
        for (int e = 0; e < 3; e++) {
            if (three[i][e] < 0) return fail(OSH_E_INVALID, "Kv4Attention: negative stride");
            if (three[i][e] > INT_MAX) return fail(OSH_E_UNSUPPORTED, "Kv4Attention: a stride above 2^31 - 1");
            if (three[i][e] % unit)
                return fail(OSH_E_UNSUPPORTED, "Kv4Attention: codes need 16-byte alignment, scales 4-byte");
        }
    }
    if (p->table_stride < (p->batch > 1 ? p->table_width : 0))
        return fail(OSH_E_INVALID, "Kv4Attention: table stride below its width");
    auto rows = [&](const void *t, const int64_t *st, int heads) {
        return Strided(t, d * 2).by(p->tokens, (Strided::wide)st[0] * 2).by(heads, (Strided::wide)st[1] * 2);
    };
    auto cache = [&](const void *t, const int64_t *st, int e, long long bytes) {
        return Strided(t, bytes).by(p->pages, st[0] * e).by(p->page, st[1] * e).by(p->kv_heads, st[2] * e);
    };
    // written: o, the four parts of the cache, the stored values, the scratch
    const Strided out[8] = {rows(p->d_o, p->o_stride, p->q_heads),
                            cache(p->d_k_pages, p->k_stride, 1, d / 2),
                            cache(p->d_v_pages, p->v_stride, 1, d / 2),
                            cache(q->d_k_scales, q->k_scale_stride, 2, groups * 4),
                            cache(q->d_v_scales, q->v_scale_stride, 2, groups * 4),
                            rows(q->d_k_stored, q->k_stored_stride, p->kv_heads),
                            rows(q->d_v_stored, q->v_stored_stride, p->kv_heads),
                            Strided(d_scratch, scratch)};
    const Strided in[6] = {rows(p->d_q, p->q_stride, p->q_heads), rows(p->d_k_new, p->k_new_stride, p->kv_heads),
                           rows(p->d_v_new, p->v_new_stride, p->kv_heads),
                           strided_rows(p->d_table, p->batch, p->table_stride * 4, p->table_width * 4LL),
                           Strided(p->d_cu, (p->batch + 1LL) * 4), Strided(p->d_kl, p->batch * 4LL)};
    for (int i = 0; i < 8; i++) {
        if (i < 7 && shares_itself(out[i])) return fail(OSH_E_INVALID, "Kv4Attention: an output's rows share memory");
        for (int e = 0; e < i; e++)
            if (share_bytes(out[i], out[e])) return fail(OSH_E_INVALID, "Kv4Attention: two outputs share memory");
        for (const Strided &t : in)
            if (share_bytes(out[i], t)) return fail(OSH_E_INVALID, "Kv4Attention: an output overlaps an operand");
    }
    WinArgs &call = room.wide ? wide : a.w;
    const long long units = (long long)p->batch * p->kv_heads * call.tiles;
    call.part_ml = static_cast<float *>(d_scratch);
    call.part_o = call.part_ml + units * call.splits * call.tile_rows * 2;
    if (room.wide) {
        char *at = static_cast<char *>(d_scratch) + room.part;
        auto take = [&](size_t n) { return at += n, at - n; };
        wide.expanded = a.wide_by = reinterpret_cast<float *>(take(room.by));
        a.wide_top = a.wide_by + 2LL * p->batch * p->kv_heads;
        wide.p.d_k_pages = a.k_wide = reinterpret_cast<_Float16 *>(take(room.page));
        wide.p.d_v_pages = a.v_wide = reinterpret_cast<_Float16 *>(take(room.page));
        wide.p.d_table = a.wide_table = reinterpret_cast<int32_t *>(take(room.table));
        wide.p.d_kl = a.wide_kl = reinterpret_cast<int32_t *>(take(room.kl));
    }
    a.page_log = 0;
    while ((1LL << a.page_log) < p->page) a.page_log++;
    a.page_mul = (unsigned)(((1LL << (30 + a.page_log)) + p->page - 1) / p->page);
    a.ks = q->d_k_scales;
    a.vs = q->d_v_scales;
    a.k_stored = q->d_k_stored;
    a.v_stored = q->d_v_stored;
    for (int i = 0; i < 3; i++) a.ks_stride[i] = q->k_scale_stride[i], a.vs_stride[i] = q->v_scale_stride[i];
    for (int i = 0; i < 2; i++)
        a.k_stored_stride[i] = q->k_stored_stride[i], a.v_stored_stride[i] = q->v_stored_stride[i];
    return p->dtype == OSH_T_F16 ? kv4_launch<_Float16>(a, wide, q->group, (unsigned)units, to_stream(s))
                                 : kv4_launch<__bf16>(a, wide, q->group, (unsigned)units, to_stream(s));
}

}  // extern "C"
