// osh_block_norm.hip -- the norms after a block and before the next one, with the
// block's gate and the residual's scale between them:
//
//   n = b / sqrt(mean(b^2) + eps) * post      (n = b without post)
//   h = round(alpha x + beta act(gate) n)     (h = x without b)
//   y = round(h / sqrt(mean(h^2) + eps) * gamma)
//
// One pass over the row: its values stay in registers between the two sums, so memory
// sees x, b, the gate and the gammas once and h and y once.  Sums and everything between
// two roundings are FP32; y is the norm of the h that is stored.
#include <algorithm>
#include <cmath>

#include "osh_lm.h"
#include "osh_overlap.h"

using namespace osh;

namespace osh {

struct BlockNormArgs {
    long long rows, ldx, ldb, ldg, ldh, ldy;  // ldg: 0 for one gate of all rows
    int cols;
    const void *x, *b, *post, *gate, *gamma;
    void *h, *y;
    float eps, alpha, beta;
    int eps_exp;
    bool sigmoid;
};

// Whether a row's squares left FP32's range (mean infinite: inv is 0; or below 2^-100 with
// eps; NaN among what it catches).  Such a row is done again times a power of two.
__device__ __forceinline__ bool inv_is_rare(float inv) {
    return (unsigned)__builtin_amdgcn_readfirstlane(__float_as_uint(inv)) - 1u >= 0x58800000u /* 2^50 */;
}

__device__ __forceinline__ float open_gate(float g, bool sigmoid, bool exact) {
    if (!sigmoid) return g;
    return 1.0f / (1.0f + (exact ? expf(-g) : __builtin_amdgcn_exp2f(g * -1.4426950408889634f)));
}

// WPR waves share a row; a lane holds NV vectors of 8 neighbouring columns, vector v of
// it at column 8 * (thread + 64 WPR v).  The vector that would cross the row's end starts
// at cols - 8 instead: its first `skip` values belong to the vector before, do not count
// in a sum, and are stored with equal values by both.  A row's stores come after all of
// its loads (program order in one wave, a barrier between waves), so h may be x or b.
template <typename T, int WPR, int NV>
__global__ __launch_bounds__(WPR > 4 ? WPR * 64 : 256) void block_norm_kernel(BlockNormArgs a) {
    constexpr int RPB = WPR > 4 ? 1 : 4 / WPR;  // rows of a workgroup
    constexpr int TPR = WPR * 64;
    static_assert(WPR == 1 || RPB == 1, "a barrier joins the waves of one row");
    using V = typename Vec8<T>::type;
    __shared__ float s_red[2][RPB][WPR];
    const int t = threadIdx.x % TPR, wave = t >> 6;
    const int slot = RPB == 1 ? 0 : threadIdx.x / TPR;
    const int cols = a.cols;

    for (long long row0 = (long long)blockIdx.x * RPB; row0 < a.rows; row0 += (long long)gridDim.x * RPB) {
        const long long row = row0 + slot;
        const bool live = row < a.rows;
        const T *x = static_cast<const T *>(a.x) + row * a.ldx;
        const T *b = static_cast<const T *>(a.b) + row * a.ldb;
        const T *gate = static_cast<const T *>(a.gate) + row * a.ldg;
        const T *post = static_cast<const T *>(a.post), *gamma = static_cast<const T *>(a.gamma);
        int col[NV], skip[NV];
        V vx[NV], vb[NV], vp[NV], vg[NV], vw[NV];
        auto get = [&](V &to, const void *base, const T *from, int v) {
            if (base && skip[v] < 8) __builtin_memcpy(&to, from + col[v], sizeof(V));
        };
        // gammas and gates of the longest rows have no registers until they are needed
        constexpr bool EARLY = NV <= 2;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int c = 8 * (t + TPR * v);
            col[v] = min(c, cols - 8);
            skip[v] = live && c < cols ? c - col[v] : 8;
            vx[v] = vb[v] = vp[v] = vg[v] = vw[v] = V{};
            get(vx[v], x, x, v);
            get(vb[v], a.b, b, v);
            if (EARLY) {
                get(vp[v], a.post, post, v);
                get(vg[v], a.gate, gate, v);
                get(vw[v], a.gamma, gamma, v);
            }
        }
        bool turn = false;  // taken in turn: the barrier of a join frees the other's LDS
        auto join = [&](float s, auto op) {
#pragma unroll
            for (int o = 32; o; o >>= 1) s = op(s, __shfl_xor(s, o));
            if constexpr (WPR > 1) {
                float *red = s_red[turn][slot];
                turn = !turn;
                if ((t & 63) == 0) red[wave] = s;
                __syncthreads();
                s = red[0];
#pragma unroll
                for (int w = 1; w < WPR; w++) s = op(s, red[w]);
            }
            return s;
        };
        auto mean_square = [&](const f32x8(&f)[NV]) {
            float sum = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; v++)
#pragma unroll
                for (int i = 0; i < 8; i++) sum = __builtin_fmaf(i >= skip[v] ? f[v][i] : 0.0f, f[v][i], sum);
            return join(sum, [](float p, float q) { return p + q; }) / (float)cols;
        };
        // f over its root mean square; whether it is rare is the same for all waves of a row
        auto normalize = [&](f32x8(&f)[NV]) {
            float inv = 1.0f / __builtin_sqrtf(mean_square(f) + a.eps);
            if (inv_is_rare(inv)) {
                float top = 0.0f;
#pragma unroll
                for (int v = 0; v < NV; v++)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const unsigned u = __float_as_uint(f[v][i]) & 0x7fffffffu;  // NaN above infinity
                        top = __uint_as_float(max(__float_as_uint(top), u));
                    }
                top = join(top, [](float p, float q) {
                    return __uint_as_float(max(__float_as_uint(p), __float_as_uint(q)));
                });
                const float by = row_shift(top, a.eps_exp);
#pragma unroll
                for (int v = 0; v < NV; v++) f[v] *= by;
                inv = row_inv(top, mean_square(f), a.eps * by * by);
            }
#pragma unroll
            for (int v = 0; v < NV; v++) f[v] *= inv;
        };

        f32x8 f[NV];
        if (a.b) {
#pragma unroll
            for (int v = 0; v < NV; v++) f[v] = __builtin_convertvector(vb[v], f32x8);
            if (a.post) {
                normalize(f);
#pragma unroll
                for (int v = 0; v < NV; v++) {
                    if (!EARLY) get(vp[v], a.post, post, v);
                    f[v] *= __builtin_convertvector(vp[v], f32x8);
                }
            }
#pragma unroll
            for (int v = 0; v < NV; v++) {
                if (a.gate) {
                    if (!EARLY) get(vg[v], a.gate, gate, v);
                    const f32x8 g = __builtin_convertvector(vg[v], f32x8);
#pragma unroll
                    for (int i = 0; i < 8; i++) f[v][i] *= open_gate(g[i], a.sigmoid, sizeof(T) == 4);
                }
                f[v] = __builtin_convertvector(vx[v], f32x8) * a.alpha + f[v] * a.beta;
                vx[v] = __builtin_convertvector(f[v], V);
            }
            if (!a.gamma && WPR > 1) __syncthreads();
        }
#pragma unroll
        for (int v = 0; v < NV; v++) f[v] = __builtin_convertvector(vx[v], f32x8);
        if (a.gamma) normalize(f);
#pragma unroll
        for (int v = 0; v < NV; v++) {
            if (skip[v] == 8) continue;
            if (a.b) __builtin_memcpy(static_cast<T *>(a.h) + row * a.ldh + col[v], &vx[v], sizeof(V));
            if (!EARLY) get(vw[v], a.gamma, gamma, v);
            if (a.gamma) store8(static_cast<T *>(a.y) + row * a.ldy + col[v], f[v] * __builtin_convertvector(vw[v], f32x8));
        }
        if constexpr (WPR > 1) __syncthreads();  // s_red is free again
    }
}

// Rows of fewer than 8 columns: a thread a row.
template <typename T>
__global__ __launch_bounds__(256) void block_norm_narrow_kernel(BlockNormArgs a) {
    const T *post = static_cast<const T *>(a.post), *gamma = static_cast<const T *>(a.gamma);
    for (long long row = blockIdx.x * 256LL + threadIdx.x; row < a.rows; row += gridDim.x * 256LL) {
        const T *x = static_cast<const T *>(a.x) + row * a.ldx;
        const T *b = static_cast<const T *>(a.b) + row * a.ldb;
        const T *gate = static_cast<const T *>(a.gate) + row * a.ldg;
        auto normalize = [&](float(&f)[8]) {  // in the steps that hold for every row
            float top = 0.0f, sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++)
                top = __uint_as_float(max(__float_as_uint(top), __float_as_uint(f[i]) & 0x7fffffffu));
            const float by = row_shift(top, a.eps_exp);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                f[i] *= by;
                sum = __builtin_fmaf(f[i], f[i], sum);
            }
            const float inv = row_inv(top, sum / (float)a.cols, a.eps * by * by);
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] *= inv;
        };
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = i < a.cols ? (float)(a.b ? b : x)[i] : 0.0f;
        if (a.b) {
            if (a.post) {
                normalize(f);
#pragma unroll
                for (int i = 0; i < 8; i++) f[i] *= i < a.cols ? (float)post[i] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (i >= a.cols) continue;
                if (a.gate) f[i] *= open_gate((float)gate[i], a.sigmoid, sizeof(T) == 4);
                f[i] = (float)(T)((float)x[i] * a.alpha + f[i] * a.beta);
            }
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < a.cols) static_cast<T *>(a.h)[row * a.ldh + i] = (T)f[i];
        }
        if (!a.gamma) continue;
        normalize(f);
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < a.cols) static_cast<T *>(a.y)[row * a.ldy + i] = (T)(f[i] * (float)gamma[i]);
    }
}

template <typename T>
static osh_status block_norm_launch(const BlockNormArgs &a, hipStream_t st) {
    constexpr long long MAX_GRID = 1 << 20;
    if (a.cols < 8) {
        OSH_LAUNCH(block_norm_narrow_kernel<T>, dim3((unsigned)std::min<long long>((a.rows + 255) / 256, MAX_GRID)),
                   dim3(256), 0, st, a);
        OSH_LAUNCH_CHECK("block_norm_narrow_kernel");
        return OSH_OK;
    }
#define OSH_NORM(WPR, NV)                                                                                     \
    do {                                                                                                      \
        constexpr int RPB = WPR > 4 ? 1 : 4 / WPR;                                                            \
        OSH_LAUNCH((block_norm_kernel<T, WPR, NV>),                                                           \
                   dim3((unsigned)std::min<long long>((a.rows + RPB - 1) / RPB, MAX_GRID)),                   \
                   dim3(WPR > 4 ? WPR * 64 : 256), 0, st, a);                                                 \
    } while (0)
    const int waves = (a.cols + 511) / 512;
    if (waves <= 1) OSH_NORM(1, 1);
    else if (waves <= 4) OSH_NORM(4, 1);
    else if (waves <= 8) OSH_NORM(8, 1);
    else if (waves <= 16) OSH_NORM(8, 2);
    else if (waves <= 32) OSH_NORM(16, 2);
    else OSH_NORM(16, 4);
#undef OSH_NORM
    OSH_LAUNCH_CHECK("block_norm_kernel");
    return OSH_OK;
}

}  // namespace osh

extern "C" {

OSH_API osh_status osh_block_norm(int64_t rows, int cols, int dtype, const void *d_x, int64_t ldx, float alpha,
                                  const void *d_b, int64_t ldb, float beta, const void *d_post, const void *d_gate,
                                  int64_t ldg, int gate_act, const void *d_gamma, float eps, void *d_h, int64_t ldh,
                                  void *d_y, int64_t ldy, osh_stream s) {
    constexpr int MAX_COLS = 32768;  // 16 waves of four vectors a lane
    if (rows < 0 || cols < 0) return fail(OSH_E_INVALID, "BlockNorm: negative sizes");
    if (dtype != OSH_T_F32 && dtype != OSH_T_F16 && dtype != OSH_T_BF16)
        return fail(OSH_E_INVALID, "BlockNorm: rows are f32, f16 or bf16");
    if (!(eps >= 0.0f)) return fail(OSH_E_INVALID, "BlockNorm: eps is negative");
    if (gate_act != OSH_ACT_NONE && gate_act != OSH_ACT_SIGMOID)
        return fail(OSH_E_INVALID, "BlockNorm: a gate is taken as it is or through a sigmoid");
    if (!d_b && (d_post || d_gate)) return fail(OSH_E_INVALID, "BlockNorm: a norm or gate of a branch that is not there");
    if (!d_b && !d_gamma) return fail(OSH_E_INVALID, "BlockNorm: neither a branch nor gamma");
    if (rows == 0) return OSH_OK;
    if (cols == 0) return fail(OSH_E_INVALID, "BlockNorm: rows without columns");
    if (cols > MAX_COLS) return fail(OSH_E_UNSUPPORTED, "BlockNorm: %d columns, at most %d", cols, MAX_COLS);
    if (!d_x || (d_b && !d_h) || (d_gamma && !d_y)) return fail(OSH_E_INVALID, "BlockNorm: NULL pointer");
    if (ldx < cols || (d_b && (ldb < cols || ldh < cols)) || (d_gamma && ldy < cols) || (d_gate && ldg && ldg < cols))
        return fail(OSH_E_INVALID, "BlockNorm: a row pitch below the columns");
    const long long e = elem_bytes(dtype);
    auto matrix = [&](const void *p, long long ld) { return strided_rows(p, rows, ld * e, cols * e); };
    const Strided x = matrix(d_x, ldx), b = matrix(d_b, ldb), h = matrix(d_b ? d_h : nullptr, ldh),
                  y = matrix(d_gamma ? d_y : nullptr, ldy), post(d_post, cols * e), gamma(d_gamma, cols * e),
                  gate = ldg ? matrix(d_gate, ldg) : Strided(d_gate, cols * e);
    if ((share_bytes(h, x) && !(d_h == d_x && ldh == ldx)) || (share_bytes(h, b) && !(d_h == d_b && ldh == ldb)))
        return fail(OSH_E_INVALID, "BlockNorm: h overlaps a row operand without being it");
    for (const Strided &t : {post, gamma, gate})
        if (share_bytes(h, t) || share_bytes(y, t))
            return fail(OSH_E_INVALID, "BlockNorm: an output overlaps another operand");
    if (share_bytes(y, x) || share_bytes(y, b) || share_bytes(y, h))
        return fail(OSH_E_INVALID, "BlockNorm: an output overlaps another operand");
    BlockNormArgs a;
    a.rows = rows;
    a.cols = cols;
    a.ldx = ldx;
    a.ldb = ldb;
    a.ldg = ldg;
    a.ldh = ldh;
    a.ldy = ldy;
    a.x = d_x;
    a.b = d_b;
    a.post = d_post;
    a.gate = d_gate;
    a.gamma = d_gamma;
    a.h = d_h;
    a.y = d_y;
    a.eps = eps;
    a.alpha = alpha;
    a.beta = beta;
    a.eps_exp = eps > 0.0f ? std::min(std::ilogb(std::sqrt(eps)), 127) + 127 : 0;
    a.sigmoid = gate_act == OSH_ACT_SIGMOID;
    if (dtype == OSH_T_F32) return block_norm_launch<float>(a, to_stream(s));
    if (dtype == OSH_T_F16) return block_norm_launch<_Float16>(a, to_stream(s));
    return block_norm_launch<__bf16>(a, to_stream(s));
}

}  // extern "C"
