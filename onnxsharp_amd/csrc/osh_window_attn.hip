// osh_window_attn.hip -- causal attention with a sliding window and sinks over a
// paged cache (osh_window_attention).
//
// The G = q_heads / kv_heads query heads of a key head read the same keys, so a
// sequence's queries at one key head form a matrix of ql * G rows (row = token * G
// + head of the group), taken 16 rows a workgroup where that is all of them, 128 where
// there are more.  For a row block the visible keys are the sinks below the window and one range; "key number" v counts them:
// v < se is key v, the others are key v - se + lo.
//
// Softmax in one pass: each row keeps its running maximum m, the sum l of
// 2^(s - m) and the weighted sum of values; a larger maximum rescales both by
// 2^(m_old - m).  Waves and splits that saw different keys are joined by the same
// rule.  All of it is FP32 but the weights, which the MFMAs take in the type of V: half a
// step each, which adds a quarter to 40% to an output's own rounding.  l sums the FP32
// weights; row blocks of 128 at heads of 65 to 128 sum the rounded ones, which V is weighted
// with, two an instruction.  The two sums are half a step apart at most, all weights rounded
// one way.
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "osh_overlap.h"
#include "osh_window.h"

using namespace osh;

namespace osh {

// ----------------------------------------------------------------- few rows

// One workgroup: 16 query rows of one key head, one split of their keys; each
// wave takes every WAVES-th step of 32 keys of the split.
//
// A step's scores are S^T = K Q^T, two MFMAs' rows of 16 keys.  MFMA row rho of
// block b is key 8 (rho / 4) + 4 b + rho % 4 of the step, so that lane (jl, g) ends
// with the scores of keys 8 g .. 8 g + 7 at query jl: just the operand of
// O^T = V^T P^T, without a move between lanes.  A lane loads ND neighbouring values
// of its 8 keys of V and turns the 8 x ND block around in registers; MFMA i then
// takes values ND jl + i of all lanes.
//
// Memory's latency is what a step waits for, so the next step's K and V are loaded
// before this one is computed (BUFS 2; heads above 128 have no registers for it),
// their addresses pass through the wave's LDS the step before, and the page ids
// they need are loaded the step before that.  The loads in flight bound it: 64 sequences
// to 8192, window 4096, take 191 us (5.1 TB/s, each byte read once; reads alone reach 7.15),
// 234 with one step at a time.
template <typename T, int DP, int WAVES>
__global__ __launch_bounds__(64 * WAVES, DP > 128 ? 1 : 2) void window_attn_rows_kernel(WinArgs a) {
    constexpr int NS = DP > 128 ? 2 : 1;       // sets of up to 128 values
    constexpr int ND = DP >= 128 ? 8 : 4;      // neighbouring values of a lane in a set
    constexpr int KS = DP / 32;                // MFMA steps over the head's values
    constexpr int BUFS = DP > 128 ? 1 : 2;
    using H8 = typename Half8<T>::type;
    extern __shared__ __align__(16) unsigned char lds[];
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
    const int rows = sq.ql * G, r0 = tile * 16;
    if (!sq.ok) {
        if (tile == 0 && split == 0) win_fill_nan<T>(p, sq, h, G, tid, 64 * WAVES);
        return;
    }
    if (r0 >= rows) return;
    T *o = static_cast<T *>(p.d_o);
    const int my_row = r0 + jl, my_tok = min(my_row, rows - 1) / G, my_head = h * G + min(my_row, rows - 1) % G;

    // queries: lane (jl, g) holds values 32 s + 8 g .. + 7 of row jl
    H8 q[KS];
    {
        const T *qr = static_cast<const T *>(p.d_q) + (long long)(sq.c0 + my_tok) * p.q_stride[0] +
                      my_head * p.q_stride[1];
#pragma unroll
        for (int s = 0; s < KS; s++) {
            q[s] = H8{};
            if (32 * s + 8 * g < d) __builtin_memcpy(&q[s], qr + 32 * s + 8 * g, 16);
        }
    }
    const int last = min(r0 + 15, rows - 1);
    const WinKeys keys = win_keys(p, sq, r0 / G, last / G);
    const int nv = keys.count;
    const int steps = cdiv(nv, 32), per = cdiv(steps, a.splits);
    const int s_end = min(steps, (split + 1) * per);
    const int my_pos = sq.past + my_tok;

    float m = -__builtin_inff(), l = 0.0f;
    f32x4 acc[NS][ND];
#pragma unroll
    for (int n = 0; n < NS; n++)
#pragma unroll
        for (int i = 0; i < ND; i++) acc[n][i] = f32x4{0, 0, 0, 0};

    const T **at = reinterpret_cast<const T **>(lds) + wave * 64;  // a step's rows of K, then of V
    struct Step {
        H8 k[2][KS];
        unsigned v[NS][8][ND / 2];
    };
    int page_id = 0;
    auto fetch = [&](int st) {
        if (st < s_end) page_id = win_page(p, sq, keys, b, st * 32 + (lane & 31), a.page_shift);
    };
    auto place = [&](int st) {
        if (st >= s_end) return;
        const WinRows<T> r = win_rows<T>(p, sq, keys, st * 32 + (lane & 31), page_id, a.page_shift, h);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        at[lane] = lane < 32 ? r.k : r.v;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    const T *zero = reinterpret_cast<const T *>(win_zero_row);
    auto load = [&](int st, Step &x) {
        if (st >= s_end) return;
#pragma unroll
        for (int bl = 0; bl < 2; bl++) {
            const T *row = at[8 * (jl >> 2) + 4 * bl + (jl & 3)];
#pragma unroll
            for (int s = 0; s < KS; s++)
                __builtin_memcpy(&x.k[bl][s], 32 * s + 8 * g < d ? row + 32 * s + 8 * g : zero, 16);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const T *row = at[32 + 8 * g + j];
#pragma unroll
            for (int n = 0; n < NS; n++)
                __builtin_memcpy(x.v[n][j], 128 * n + ND * jl < d ? row + 128 * n + ND * jl : zero, 2 * ND);
        }
    };
    auto compute = [&](int st, const Step &x) {
        f32x4 sc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int bl = 0; bl < 2; bl++)
#pragma unroll
            for (int s = 0; s < KS; s++) sc[bl] = mma16(x.k[bl][s], q[s], sc[bl]);
        float s8[8], top = m;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int v = st * 32 + 8 * g + i;
            const bool seen = v < nv && win_sees(p, my_pos, keys.at(v));
            s8[i] = seen ? sc[i >> 2][i & 3] * a.scale_log2 : -__builtin_inff();
            top = __builtin_fmaxf(top, s8[i]);
        }
        top = __builtin_fmaxf(top, __shfl_xor(top, 16));
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        const float base = top == -__builtin_inff() ? 0.0f : top;
        const float fade = __builtin_amdgcn_exp2f(m - base);
        m = top;
        l *= fade;
        f32x8 w;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            w[i] = __builtin_amdgcn_exp2f(s8[i] - base);
            l += w[i];
        }
        const H8 pw = __builtin_convertvector(w, H8);
#pragma unroll
        for (int n = 0; n < NS; n++)
#pragma unroll
            for (int i = 0; i < ND; i++) {
                unsigned vt[4];
#pragma unroll
                for (int e = 0; e < 4; e++)
                    vt[e] = __builtin_amdgcn_perm(x.v[n][2 * e + 1][i / 2], x.v[n][2 * e][i / 2],
                                                  i & 1 ? 0x07060302u : 0x05040100u);
                H8 vh;
                __builtin_memcpy(&vh, vt, 16);
                acc[n][i] *= fade;
                acc[n][i] = mma16(vh, pw, acc[n][i]);
            }
    };
    int st = split * per + wave;
    fetch(st);
    place(st);
    fetch(st + WAVES);
    Step x[BUFS];
    if constexpr (BUFS == 2) {
        load(st, x[0]);
        place(st + WAVES);
        fetch(st + 2 * WAVES);
        for (; st < s_end; st += 2 * WAVES) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int now = st + e * WAVES;
                load(now + WAVES, x[e ^ 1]);
                place(now + 2 * WAVES);
                fetch(now + 3 * WAVES);
                if (now < s_end) compute(now, x[e]);
            }
        }
    } else {
        for (; st < s_end; st += WAVES) {
            load(st, x[0]);
            place(st + WAVES);
            fetch(st + 2 * WAVES);
            compute(st, x[0]);
        }
    }
    if (split == 0) win_append<T>(p, sq, b, h, G, r0, 16, tid, 64 * WAVES);
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // join the waves: [WAVES][16] pairs (m, l), then [WAVES][16][DP] sums
    __syncthreads();
    float *ml = reinterpret_cast<float *>(lds), *os = ml + WAVES * 32;
    if (g == 0) {
        ml[(wave * 16 + jl) * 2] = m;
        ml[(wave * 16 + jl) * 2 + 1] = l;
    }
#pragma unroll
    for (int n = 0; n < NS; n++)
#pragma unroll
        for (int i = 0; i < ND; i++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                os[(wave * 16 + jl) * DP + 128 * n + ND * (4 * g + r) + i] = acc[n][i][r];
    __syncthreads();
    for (int e = tid; e < 16 * DP; e += 64 * WAVES) {
        const int r = e / DP, c = e % DP, row = r0 + r;
        if (row >= rows || c >= d) continue;
        float mm = ml[r * 2];
#pragma unroll
        for (int w = 1; w < WAVES; w++) mm = __builtin_fmaxf(mm, ml[(w * 16 + r) * 2]);
        const float base = mm == -__builtin_inff() ? 0.0f : mm;
        float sum = 0.0f, ll = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float f = __builtin_amdgcn_exp2f(ml[(w * 16 + r) * 2] - base);
            ll += f * ml[(w * 16 + r) * 2 + 1];
            sum += f * os[(w * 16 + r) * DP + c];
        }
        if (a.splits == 1) {
            o[(long long)(sq.c0 + row / G) * p.o_stride[0] + (h * G + row % G) * p.o_stride[1] + c] = (T)(sum / ll);
        } else {
            const long long u = (long long)unit * a.splits + split;
            a.part_o[(u * 16 + r) * d + c] = sum;
            if (c == 0) {
                a.part_ml[(u * 16 + r) * 2] = mm;
                a.part_ml[(u * 16 + r) * 2 + 1] = ll;
            }
        }
    }
}

// ---------------------------------------------------------------- many rows

// 32 NW query rows of one key head and a split of their keys: a wave owns 32 rows,
// and tiles of 64 keys pass through two LDS buffers, loaded directly from the pages.
// S^T = K Q^T leaves a lane the scores of half the keys at one query, and those of
// each 16 keys are the operand that O^T = V^T P^T wants when its keys come in the
// order 4 hl + 0..3, 8 + 4 hl + 0..3 (hl = lane / 32); V's operand is read so, by LDS
// reads that transpose.
//
// C chunks of 16 bytes an LDS row, KS MFMA steps over a head's values, OB blocks of
// 32 of them in the output.  Chunk c of a key's row lies at slot c ^ swizzle: keys'
// rows spread a 16-lane read over all banks, values' rows one of 4 rows x 64 bytes.
//
// Workgroups of 128 rows, two a CU: their phases drift apart, so that one's MFMAs run
// under the other's exponentials (one of 256 rows took 3% more at 8192 tokens and 78% more
// at pieces of prompts).  What bounds it is that a SIMD's two waves still spend 2.4 us on a
// tile each, of which MFMAs are 0.85 and vector instructions 0.9: 8192 tokens, 32 heads of
// 128, window 2048: 293 us (820 TFLOP/s), without a window 591 (930); 8 heads of 256, window
// 2048: 248 (490).  The next tile's scores interleaved with this one's exponentials in one
// wave were 5% slower.
//
// The running maximum moves only when a row's scores pass it by 2^8: weights up to
// 256 are as exact, and most tiles rescale nothing.
//
// EXPANDED: queries and outputs are bf16, keys and values f16 pages that hold the new tokens
// too, taken times a power of two that keeps the largest of a head within 1 (a.expanded); a
// query is taken so as well, and its powers come back with the softmax's scale and at the end.
template <typename T, int C, int KS, int OB, int NW, bool EXPANDED>
__global__ __launch_bounds__(64 * NW, C > 16 ? 1 : 2) void window_attn_tile_kernel(WinArgs a) {
    using H8 = typename Half8<std::conditional_t<EXPANDED, _Float16, T>>::type;
    constexpr int BUF = 64 * C * 16, RPI = 64 / C, IT = 2 * C / NW;  // rows an instruction, instructions a wave
    static_assert(IT * NW == 2 * C, "loads are dealt evenly");
    extern __shared__ __align__(16) unsigned char lds[];  // two of [K tile][V tile]
    const osh_window_attn &p = a.p;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ql32 = lane & 31, hl = lane >> 5;
    const int d = p.head_dim, G = a.group;

    int id = xcd_band(blockIdx.x, gridDim.x);
    const int unit = id / a.splits, split = id - unit * a.splits;
    id = unit;
    const int tile = a.tiles - 1 - id % a.tiles;  // the rows with most keys first
    id /= a.tiles;
    const int h = id % p.kv_heads, b = id / p.kv_heads;
    const WinSeq sq = win_seq(p, b);
    const int rows = sq.ql * G, r0 = tile * 32 * NW;
    if (!sq.ok) {
        if (tile == 0 && split == 0) win_fill_nan<T>(p, sq, h, G, tid, 64 * NW);
        return;
    }
    if (r0 >= rows) return;
    T *o = static_cast<T *>(p.d_o);
    const int row = min(r0 + 32 * wave + ql32, rows - 1), tok = row / G, head = h * G + row % G;
    if (!EXPANDED && split == 0) win_append<T>(p, sq, b, h, G, r0, 32 * NW, tid, 64 * NW);
    WinSeq held = sq;  // for whom all keys lie in pages
    if (EXPANDED) held.past = sq.kl;

    H8 q[KS];
    float scale_log2 = a.scale_log2, back = 1.0f;
    if constexpr (EXPANDED) {
        const T *qr = static_cast<const T *>(p.d_q) + (long long)(sq.c0 + tok) * p.q_stride[0] + head * p.q_stride[1];
        f32x8 f[KS];
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            f[s] = f32x8{};
            if (16 * s + 8 * hl < d) f[s] = load8(qr + 16 * s + 8 * hl);
#pragma unroll
            for (int i = 0; i < 8; i++) top = __builtin_fmaxf(top, __builtin_fabsf(f[s][i]));
        }
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        const int e = top < __builtin_inff() ? min(max(__builtin_amdgcn_frexp_expf(top), -120), 126) : 0;
        const float by = __builtin_amdgcn_ldexpf(1.0f, -e);
#pragma unroll
        for (int s = 0; s < KS; s++) q[s] = __builtin_convertvector(f[s] * by, H8);
        const float *x = a.expanded + 2 * ((long long)b * p.kv_heads + h);
        // by the exponents' sum, kept among normal numbers: at 0 a hidden key's -infinity, and at
        // infinity a score of 0, would make the row NaN
        const int back2 = e + 1 - __builtin_amdgcn_frexp_expf(x[0]);
        scale_log2 = __builtin_fminf(__builtin_fmaxf(__builtin_amdgcn_ldexpf(scale_log2, back2), 0x1p-126f), 0x1p127f);
        back = 1.0f / x[1];
    } else {
        const T *qr = static_cast<const T *>(p.d_q) + (long long)(sq.c0 + tok) * p.q_stride[0] + head * p.q_stride[1];
#pragma unroll
        for (int s = 0; s < KS; s++) {
            q[s] = H8{};
            if (16 * s + 8 * hl < d) __builtin_memcpy(&q[s], qr + 16 * s + 8 * hl, 16);
        }
    }
    const int last = min(r0 + 32 * NW - 1, rows - 1);
    const WinKeys keys = win_keys(p, sq, r0 / G, last / G);
    const int nt_all = cdiv(keys.count, 64), per = cdiv(nt_all, a.splits);
    const int t_end = min(nt_all, (split + 1) * per);
    // by key number: this row sees v <= v_hi with v >= v_lo or v < v_sink, and the wave's
    // rows together none outside [0, w_hi], all of [w_lo, w_all] (and of [0, v_sink))
    const int base = keys.sink_end - keys.lo, pos = sq.past + tok;
    const int v_sink = max(keys.sink_end, win_min(p.sinks, 1 << 30) + base);
    const int v_hi = pos + base, v_lo = max(pos - p.window + 1, keys.lo) + base;
    const int wr = r0 + 32 * wave, tok0 = win_min(wr, rows - 1) / G, tok1 = win_min(wr + 31, rows - 1) / G;
    const int w_hi = sq.past + tok1 + base, w_all = sq.past + tok0 + base;
    const int w_lo = max(sq.past + tok1 - p.window + 1, keys.lo) + base;
    const int w_first = max(sq.past + tok0 - p.window + 1, keys.lo) + base;  // below it only sinks

    // loads: instruction i (K for i < C) covers rows RPI (i % C) + lane / C; a wave has
    // instructions wave + NW e, whose rows repeat for V after C.  The C lanes of a row
    // would all compute its address: lane e of each RW neighbours computes that of the
    // e-th instruction's row and hands it to the others.  A tile of new tokens alone
    // (all of a prompt's) has its rows at one stride.
    constexpr int RW = IT / 2 > 0 ? IT / 2 : 1;  // rows of a lane in a tile
    const int slot = lane % C;
    auto tile_row = [&](int e) { return (wave + NW * e) % C * RPI + lane / C; };
    const int my_tile_row = tile_row(lane % RW);
    const int fresh0 = EXPANDED ? INT_MAX : cdiv(max(sq.past + base, keys.sink_end), 64);  // first tile of new tokens alone
    int page_id = 0;
    auto fetch_pages = [&](int t) {
        if (t < fresh0) page_id = win_page(p, held, keys, b, t * 64 + my_tile_row, a.page_shift);
    };
    // Heads of 65 to 128 keep the byte offsets of a lane's chunks in a tile of new tokens
    // and sum their rounded weights two an instruction (4% of 8192 tokens without a window);
    // above there are no registers for the offsets, below neither gains.
    constexpr bool KEEP = C == 16;
    unsigned k_off[RW], v_off[RW];
    bool k_in[RW], v_in[RW];
    if constexpr (KEEP) {
#pragma unroll
        for (int e = 0; e < RW; e++) {
            const int r = tile_row(e), kc = 8 * (slot ^ win_k_swizzle<C>(r)), vc = 8 * (slot ^ win_v_swizzle<C>(r));
            k_in[e] = kc < d, v_in[e] = vc < d;
            k_off[e] = 2 * (r * (unsigned)p.k_new_stride[0] + kc), v_off[e] = 2 * (r * (unsigned)p.v_new_stride[0] + vc);
        }
    }
    const bool short_strides = max(p.k_new_stride[0], p.v_new_stride[0]) < (1 << 24);  // 32-bit offsets hold
    auto load_tile = [&](int t, int buf) {
        unsigned char *dst = lds + buf * 2 * BUF;
        const bool fresh = t >= fresh0 && t * 64 + 64 <= keys.count;
        if constexpr (KEEP) {
            if (fresh && short_strides) {
                const long long n = sq.c0 + t * 64 - base - sq.past;
                const char *fk =
                    static_cast<const char *>(p.d_k_new) + 2 * (n * p.k_new_stride[0] + h * p.k_new_stride[1]);
                const char *fv =
                    static_cast<const char *>(p.d_v_new) + 2 * (n * p.v_new_stride[0] + h * p.v_new_stride[1]);
#pragma unroll
                for (int e = 0; e < RW; e++) {
                    if (k_in[e]) copy_to_lds(fk + k_off[e], dst + (wave + NW * e) % C * 1024);
                    if (v_in[e]) copy_to_lds(fv + v_off[e], dst + BUF + (wave + NW * e) % C * 1024);
                }
                return;
            }
        }
        const T *fk = nullptr, *fv = nullptr;
        WinRows<T> mine{nullptr, nullptr};
        if (!KEEP && fresh) {
            const long long n = sq.c0 + t * 64 - base - sq.past;
            fk = static_cast<const T *>(p.d_k_new) + n * p.k_new_stride[0] + h * p.k_new_stride[1];
            fv = static_cast<const T *>(p.d_v_new) + n * p.v_new_stride[0] + h * p.v_new_stride[1];
        } else {
            mine = win_rows<T>(p, held, keys, t * 64 + my_tile_row, page_id, a.page_shift, h);
        }
#pragma unroll
        for (int e = 0; e < RW; e++) {
            const int r = tile_row(e);
            const int kc = 8 * (slot ^ win_k_swizzle<C>(r)), vc = 8 * (slot ^ win_v_swizzle<C>(r));
            const T *kr, *vr;
            if (!KEEP && fresh) {
                kr = fk + (unsigned long long)(unsigned)r * (unsigned)p.k_new_stride[0];
                vr = fv + (unsigned long long)(unsigned)r * (unsigned)p.v_new_stride[0];
            } else {
                const int from = lane - lane % RW + e;
                kr = reinterpret_cast<const T *>(__shfl(reinterpret_cast<unsigned long long>(mine.k), from));
                vr = reinterpret_cast<const T *>(__shfl(reinterpret_cast<unsigned long long>(mine.v), from));
            }
            const bool is_k = wave + NW * e < C, is_v = IT > 1 || !is_k;
            if (is_k && kc < d) copy_to_lds(kr + kc, dst + (wave + NW * e) % C * 1024);
            if (is_v && vc < d) copy_to_lds(vr + vc, dst + BUF + (wave + NW * e) % C * 1024);
        }
    };

    if (d < 8 * C) {  // the slots of no value stay zero
        for (int e = tid; e < 4 * BUF / 16; e += 64 * NW) reinterpret_cast<uint4 *>(lds)[e] = uint4{0, 0, 0, 0};
        __syncthreads();
    }
    int t = split * per;
    if (t < t_end) {
        fetch_pages(t);
        load_tile(t, 0);
        if (t + 1 < t_end) fetch_pages(t + 1);
    }
    float m = -__builtin_inff(), l = 0.0f;  // m in units of 2^, after the scale
    f32x16 acc[OB];
#pragma unroll
    for (int i = 0; i < OB; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[i][r] = 0.0f;
    int buf = 0;
    for (; t < t_end; t++, buf ^= 1) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (t + 1 < t_end) {
            load_tile(t + 1, buf ^ 1);
            if (t + 2 < t_end) fetch_pages(t + 2);
        }
        const int v0 = t * 64;
        if (v0 > w_hi || (v0 >= v_sink && v0 + 63 < w_first)) continue;  // the wave sees none
        const unsigned char *kt = lds + buf * 2 * BUF, *vt = kt + BUF;
        // fragments are read ahead of the MFMAs that take them, the first values' before
        // the softmax (3% of a prompt; heads above 128 have no registers for it)
        constexpr bool AHEAD = KS <= 8;
        constexpr int PF = !AHEAD ? 1 : KS < 4 ? KS : 4;
        auto key_frag = [&](int kb, int i) {
            const int r = 32 * kb + ql32;
            H8 k;
            __builtin_memcpy(&k, kt + r * (C * 16) + (((2 * i + hl) ^ win_k_swizzle<C>(r)) << 4), 16);
            return k;
        };
        // this lane reads row key + lane % 16 / 4, values 16 (lane / 16 % 2) + 4 (lane % 4)
        auto value_frag = [&](int e, int i) {
            const int key = 16 * e + 4 * hl + (lane >> 2 & 3), off = (lane >> 4 & 1) * 32 + (lane & 3) * 8;
            const int c = 4 * i + (off >> 4);
            const unsigned char *row = vt + key * (C * 16) + (off & 15);
            const s16x4 x0 = read_transposed(row + ((c ^ win_v_swizzle<C>(key)) << 4));
            const s16x4 x1 = read_transposed(row + 8 * (C * 16) + ((c ^ win_v_swizzle<C>(key + 8)) << 4));
            const s16x8 x = __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
            H8 v;
            __builtin_memcpy(&v, &x, 16);
            return v;
        };
        f32x16 s[2];
        H8 kf[PF], vf[2][OB];
#pragma unroll
        for (int i = 0; i < PF; i++) kf[i] = key_frag(0, i);
        if (AHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int i = 0; i < KS; i++) {
                const int n = kb * KS + i;
                s[kb] = mma32(kf[n % PF], q[i], i == 0 ? f32x16{} : s[kb]);
                if (n + PF < 2 * KS) kf[n % PF] = key_frag((n + PF) / KS, (n + PF) % KS);
            }
#pragma unroll
        for (int i = 0; i < OB; i++)
            if (AHEAD) vf[0][i] = value_frag(0, i);
        if (AHEAD) __builtin_amdgcn_sched_barrier(0);
        if (v0 + 63 > w_all || (v0 + 63 >= v_sink && v0 < w_lo)) {  // some row sees only some
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int v = v0 + 32 * kb + 8 * (r >> 2) + 4 * hl + (r & 3);
                    // selects, not branches: a branch around an element of s moves all of it
                    const bool hidden = (v > v_hi) | ((v < v_lo) & (v >= v_sink));
                    s[kb][r] = hidden ? -__builtin_inff() : s[kb][r];
                }
        }
        float top = s[0][0];
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int r = 0; r < 16; r++) top = __builtin_fmaxf(top, s[kb][r]);
        top = __builtin_fmaxf(top, __shfl_xor(top, 32)) * scale_log2;
        if (__builtin_amdgcn_ballot_w64(top > m + 8.0f) != 0) {
            const float old = m;
            m = __builtin_fmaxf(m, top);
            const float fade = old == m ? 1.0f : __builtin_amdgcn_exp2f(old - m);
            l *= fade;
#pragma unroll
            for (int i = 0; i < OB; i++) acc[i] *= fade;
        }
        const float ref = m == -__builtin_inff() ? 0.0f : m;
        H8 w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            f32x8 f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                f[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 1][8 * (e & 1) + i], scale_log2, -ref));
                if (!KEEP) l += f[i];
            }
            w[e] = __builtin_convertvector(f, H8);
            if (KEEP) l = add8(w[e], l);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
#pragma unroll
            for (int i = 0; i < OB; i++) {
                if (AHEAD && e < 3) vf[(e + 1) & 1][i] = value_frag(e + 1, i);
            }
#pragma unroll
            for (int i = 0; i < OB; i++) acc[i] = mma32(AHEAD ? vf[e & 1][i] : value_frag(e, i), w[e], acc[i]);
            if (AHEAD) __builtin_amdgcn_sched_barrier(0);
        }
    }
    l += __shfl_xor(l, 32);
    // quads of values 8 e + 4 hl + 0..3: exchanging one quad between the halves of the
    // wave leaves a lane 8 neighbouring values
    const bool mine = wr + ql32 < rows;
    const float inv = EXPANDED ? (a.splits == 1 ? back / l : back) : a.splits == 1 ? 1.0f / l : 1.0f;
    const long long u = (long long)unit * a.splits + split;
    const int tr = 32 * wave + ql32;
    if (a.splits > 1 && mine && hl == 0) {
        a.part_ml[(u * 32 * NW + tr) * 2] = m;
        a.part_ml[(u * 32 * NW + tr) * 2 + 1] = l;
    }
#pragma unroll
    for (int i = 0; i < OB; i++)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
            f32x8 f;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[i][4 * e + r] * inv),
                                                                __float_as_uint(acc[i][4 * e + 4 + r] * inv), false,
                                                                false);
                f[r] = __uint_as_float(x[0]), f[r + 4] = __uint_as_float(x[1]);
            }
            const int c = 32 * i + 8 * (e + hl);
            if (!mine || c >= d) continue;
            if (a.splits == 1)
                store8(o + (long long)(sq.c0 + tok) * p.o_stride[0] + head * p.o_stride[1] + c, f);
            else
                store8(a.part_o + (u * 32 * NW + tr) * d + c, f);
        }
}

template <typename T, int C, int KS, int OB, int NW, bool EXPANDED = false>
static osh_status win_tile_launch(const WinArgs &a, unsigned units, hipStream_t st) {
    OSH_LAUNCH((window_attn_tile_kernel<T, C, KS, OB, NW, EXPANDED>), dim3(units * a.splits), dim3(64 * NW), 4 * 64 * C * 16, st, a);
    OSH_LAUNCH_CHECK("window_attn_tile_kernel");
    return win_join<T>(a, units, st);
}

template <typename T, int DP, int WAVES>
static osh_status win_launch(const WinArgs &a, unsigned units, hipStream_t st) {
    constexpr size_t lds = std::max<size_t>(WAVES * 64 * sizeof(void *), WAVES * 16 * (DP + 2) * sizeof(float));
    OSH_LAUNCH((window_attn_rows_kernel<T, DP, WAVES>), dim3(units * a.splits), dim3(64 * WAVES), lds, st, a);
    OSH_LAUNCH_CHECK("window_attn_rows_kernel");
    return win_join<T>(a, units, st);
}

template <typename T>
static osh_status win_launch_t(const WinArgs &a, unsigned units, hipStream_t st) {
    if (a.tile_rows > 16) {
        if (a.p.head_dim <= 32) return win_tile_launch<T, 4, 2, 1, 4>(a, units, st);
        if (a.p.head_dim <= 64) return win_tile_launch<T, 8, 4, 2, 4>(a, units, st);
        if (a.p.head_dim <= 96) return win_tile_launch<T, 16, 6, 3, 4>(a, units, st);
        if (a.p.head_dim <= 128) return win_tile_launch<T, 16, 8, 4, 4>(a, units, st);
        return win_tile_launch<T, 32, 16, 8, 4>(a, units, st);
    }
    if (a.p.head_dim <= 64) return a.wide ? win_launch<T, 64, 8>(a, units, st) : win_launch<T, 64, 4>(a, units, st);
    if (a.p.head_dim <= 128) return a.wide ? win_launch<T, 128, 8>(a, units, st) : win_launch<T, 128, 4>(a, units, st);
    return win_launch<T, 256, 4>(a, units, st);
}

osh_status win_run_expanded(const WinArgs &a, unsigned units, hipStream_t st) {
    const int d = a.p.head_dim;
    if (d <= 32) return win_tile_launch<__bf16, 4, 2, 1, 4, true>(a, units, st);
    if (d <= 64) return win_tile_launch<__bf16, 8, 4, 2, 4, true>(a, units, st);
    if (d <= 96) return win_tile_launch<__bf16, 16, 6, 3, 4, true>(a, units, st);
    if (d <= 128) return win_tile_launch<__bf16, 16, 8, 4, 4, true>(a, units, st);
    return win_tile_launch<__bf16, 32, 16, 8, 4, true>(a, units, st);
}

osh_status win_run(const WinArgs &a, unsigned units, hipStream_t st) {
    return a.p.dtype == OSH_T_F16 ? win_launch_t<_Float16>(a, units, st) : win_launch_t<__bf16>(a, units, st);
}

}  // namespace osh

extern "C" {

OSH_API osh_status osh_window_attention_scratch_bytes(const osh_window_attn *p, size_t *bytes) {
    if (!bytes) return fail(OSH_E_INVALID, "WindowAttention: NULL bytes");
    WinArgs a;
    return win_plan(p, a, *bytes);
}

OSH_API osh_status osh_window_attention(const osh_window_attn *p, void *d_scratch, osh_stream s) {
    WinArgs a;
    size_t scratch = 0;
    if (const osh_status st = win_plan(p, a, scratch)) return st;
    if (p->batch == 0 || p->max_q == 0 || p->tokens == 0) return OSH_OK;
    if (!p->d_q || !p->d_k_new || !p->d_v_new || !p->d_o || !p->d_k_pages || !p->d_v_pages || !p->d_table ||
        !p->d_cu || !p->d_kl || (scratch && !d_scratch))
        return fail(OSH_E_INVALID, "WindowAttention: NULL pointer");
    const long long d = p->head_dim;
    const int64_t *two[4] = {p->q_stride, p->o_stride, p->k_new_stride, p->v_new_stride};
    for (int i = 0; i < 4; i++)
        if (two[i][0] < 0 || two[i][1] < 0) return fail(OSH_E_INVALID, "WindowAttention: negative stride");
    for (int i = 0; i < 3; i++)
        if (p->k_stride[i] < 0 || p->v_stride[i] < 0) return fail(OSH_E_INVALID, "WindowAttention: negative stride");
    for (int i = 0; i < 3; i++)
        if (std::max({p->k_stride[i], p->v_stride[i], p->k_new_stride[i % 2], p->v_new_stride[i % 2]}) > INT_MAX)
            return fail(OSH_E_UNSUPPORTED, "WindowAttention: a stride above 2^31 - 1");
    if (p->table_stride < (p->batch > 1 ? p->table_width : 0))
        return fail(OSH_E_INVALID, "WindowAttention: table stride below its width");
    auto rows = [&](const void *t, const int64_t *st, int heads) {
        return Strided(t, d * 2).by(p->tokens, (Strided::wide)st[0] * 2).by(heads, (Strided::wide)st[1] * 2);
    };
    auto cache = [&](const void *t, const int64_t *st) {
        return Strided(t, d * 2).by(p->pages, st[0] * 2).by(p->page, st[1] * 2).by(p->kv_heads, st[2] * 2);
    };
    const Strided o = rows(p->d_o, p->o_stride, p->q_heads), kc = cache(p->d_k_pages, p->k_stride),
                  vc = cache(p->d_v_pages, p->v_stride), room(d_scratch, scratch);
    const Strided in[6] = {rows(p->d_q, p->q_stride, p->q_heads), rows(p->d_k_new, p->k_new_stride, p->kv_heads),
                           rows(p->d_v_new, p->v_new_stride, p->kv_heads),
                           strided_rows(p->d_table, p->batch, p->table_stride * 4, p->table_width * 4LL),
                           Strided(p->d_cu, (p->batch + 1LL) * 4), Strided(p->d_kl, p->batch * 4LL)};
    if (shares_itself(o)) return fail(OSH_E_INVALID, "WindowAttention: rows of o share memory");
    if (shares_itself(kc) || shares_itself(vc) || share_bytes(kc, vc))
        return fail(OSH_E_INVALID, "WindowAttention: slots of the cache share memory");
    if (share_bytes(o, kc) || share_bytes(o, vc)) return fail(OSH_E_INVALID, "WindowAttention: o overlaps the cache");
    for (const Strided &t : in) {
        if (share_bytes(o, t)) return fail(OSH_E_INVALID, "WindowAttention: o overlaps an operand");
        if (share_bytes(kc, t) || share_bytes(vc, t))
            return fail(OSH_E_INVALID, "WindowAttention: the cache overlaps an operand");
        if (share_bytes(room, t)) return fail(OSH_E_INVALID, "WindowAttention: the scratch overlaps an operand");
    }
    if (share_bytes(room, o) || share_bytes(room, kc) || share_bytes(room, vc))
        return fail(OSH_E_INVALID, "WindowAttention: the scratch overlaps an operand");
    const long long units = (long long)p->batch * p->kv_heads * a.tiles;
    a.part_ml = static_cast<float *>(d_scratch);
    a.part_o = a.part_ml + units * a.splits * a.tile_rows * 2;
    return win_run(a, (unsigned)units, to_stream(s));
}

}  // extern "C"
