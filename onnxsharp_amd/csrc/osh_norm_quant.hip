// osh_norm_quant.hip -- RMS norm of a residual stream into 8-bit rows:
//
//   h = round(x + r)                       (h = x without a residual)
//   y = h / sqrt(mean(h^2) + eps) * gamma
//   scale = max|y| / top                   (top = 127 for int8, 448 for e4m3)
//   q = round(y / scale)
//
// One pass over the row: its values stay in registers between the sum, the
// maximum and the rounding, so memory sees x, r and gamma once and h, q and the
// scale once.  Sum, maximum and scale are FP32.  HBM bounds it: 16384 x 4096 bf16 into
// e4m3 with the residual 80.5 us over inputs that no cache holds (5.8 TB/s, two thirds of
// it reads; a copy reaches 4.95, reads alone 7.15); one row 3.2 us, launch and latency.
#include <algorithm>
#include <cmath>

#include "osh_lm.h"
#include "osh_overlap.h"

using namespace osh;

namespace osh {

struct NormArgs {
    long long rows, ldx, ldr, ldh, ldq;
    int cols;
    const void *x, *r, *gamma;
    void *h;
    unsigned char *q;
    float *scale;
    float eps, top;
    int eps_exp, q_int8;
};

// |v| as an integer of the same order, with NaN above infinity: a NaN in gamma, and a NaN or
// an infinity in a row (whose mean is then NaN), reaches the row's scale, and with it every
// value that the row stands for.
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// A row is done again in steps that hold for every finite one where its squares left FP32's
// range (mean of squares infinite: inv and amax are then 0; or below 2^-100 with eps) or its
// scale is not above FP32's normal numbers (amax <= 2^-117): one scalar test of a row, NaN
// among what it catches.  Tests at each step cost 10% of 65536 x 1024 (113 us for 103).
__device__ __forceinline__ bool row_is_rare(float inv, float amax) {
    const unsigned i = __builtin_amdgcn_readfirstlane(__float_as_uint(inv));
    const unsigned m = __builtin_amdgcn_readfirstlane(__float_as_uint(amax));
    return i > 0x58800000u /* 2^50 */ || m <= 0x05000000u /* 2^-117 */ || m > 0x7f800000u;
}
// The steps.  The row is taken times the power of two that brings the larger of its largest
// |h| and sqrt(eps) (of biased exponent eps_exp) to [1, 2), as far as floats go: y is that of
// the row times it, with eps times its square.
__device__ __forceinline__ float row_shift(float hmax, int eps_exp) {
    const int e = max((int)(__float_as_uint(hmax) >> 23), eps_exp);
    return __uint_as_float((unsigned)min(max(254 - e, 1), 253) << 23);
}
// 1 / sqrt; 0 for a row of zeros without eps, NaN for a row that is not finite.
__device__ __forceinline__ float row_inv(float hmax, float mean, float eps) {
    if (!(hmax < __builtin_inff())) return __builtin_nanf("");
    return mean + eps == 0.0f ? 0.0f : 1.0f / __builtin_sqrtf(mean + eps);
}
// Where the scale lies below FP32's normal numbers, y does so too and has few bits: it is
// then taken 2^60 times as large, and `back` is 1 / (2^60 times the scale that is stored), or
// 0 for a scale of 0.
constexpr float ROW_UP = 0x1p60f, ROW_DOWN = 0x1p-60f;
__device__ __forceinline__ bool row_small(float amax) { return !(amax > 0x1p-117f); }
__device__ __forceinline__ float row_back_up(float scale) { return scale > 0.0f ? 1.0f / (scale * ROW_UP) : 0.0f; }

// WPR waves share a row; a lane holds NV vectors of 8 neighbouring columns,
// vector v of it at column 8 * (thread + 64 WPR v).  The vector that would cross
// the row's end starts at cols - 8 instead: its first `skip` values belong to the
// vector before, count in neither sum nor maximum, and are stored with equal
// values by both.  Stores come after every load of the row (program order in one
// wave, the barrier of the sum between waves), so h may be x or r itself.
template <typename T, int WPR, int NV>
__global__ __launch_bounds__(WPR > 4 ? WPR * 64 : 256) void norm_quant_kernel(NormArgs a) {
    constexpr int RPB = WPR > 4 ? 1 : 4 / WPR;  // rows of a workgroup
    constexpr int TPR = WPR * 64;
    __shared__ float s_sum[RPB][WPR];
    __shared__ unsigned s_max[RPB][WPR];
    const int t = threadIdx.x % TPR, wave = t >> 6;
    const int slot = RPB == 1 ? 0 : threadIdx.x / TPR;
    const int cols = a.cols;
    const T *gamma = static_cast<const T *>(a.gamma);

    for (long long row0 = (long long)blockIdx.x * RPB; row0 < a.rows; row0 += (long long)gridDim.x * RPB) {
        const long long row = row0 + slot;
        const bool live = row < a.rows;
        const T *x = static_cast<const T *>(a.x) + row * a.ldx;
        const T *r = static_cast<const T *>(a.r) + row * a.ldr;
        T *h = static_cast<T *>(a.h) + row * a.ldh;
        f32x8 f[NV], g[NV];
        int col[NV], skip[NV];
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int c = 8 * (t + TPR * v);
            col[v] = min(c, cols - 8);
            skip[v] = live && c < cols ? c - col[v] : 8;
            f[v] = f32x8{0, 0, 0, 0, 0, 0, 0, 0};
            g[v] = f[v];
            if (skip[v] < 8) {
                f[v] = load8(x + col[v]);
                g[v] = load8(gamma + col[v]);
                if (a.r) {
                    f[v] += load8(r + col[v]);
                    if constexpr (sizeof(T) == 2)
                        f[v] = __builtin_convertvector(__builtin_convertvector(f[v], typename Vec8<T>::type), f32x8);
                }
            }
        }
        // taken in turn: the barrier of each frees the other's LDS
        auto mean_square = [&](auto value) {
            float sum = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const f32x8 y = value(v);
#pragma unroll
                for (int i = 0; i < 8; i++) sum = __builtin_fmaf(i >= skip[v] ? y[i] : 0.0f, y[i], sum);
            }
#pragma unroll
            for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
            if constexpr (WPR > 1) {
                if ((t & 63) == 0) s_sum[slot][wave] = sum;
                __syncthreads();
                sum = 0.0f;
#pragma unroll
                for (int w = 0; w < WPR; w++) sum += s_sum[slot][w];
            }
            return sum / (float)cols;
        };
        auto largest = [&](auto value) {
            unsigned top_bits = 0;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const f32x8 y = value(v);
#pragma unroll
                for (int i = 0; i < 8; i++) top_bits = max(top_bits, abs_bits(y[i]));
            }
#pragma unroll
            for (int o = 32; o; o >>= 1) top_bits = max(top_bits, (unsigned)__shfl_xor((int)top_bits, o));
            if constexpr (WPR > 1) {
                if ((t & 63) == 0) s_max[slot][wave] = top_bits;
                __syncthreads();
                top_bits = 0;
#pragma unroll
                for (int w = 0; w < WPR; w++) top_bits = max(top_bits, s_max[slot][w]);
            }
            return __uint_as_float(top_bits);
        };
        auto row_f = [&](int v) { return f[v]; };
        float inv = 1.0f / __builtin_sqrtf(mean_square(row_f) + a.eps);
#pragma unroll
        for (int v = 0; v < NV; v++) {
            if (a.r && skip[v] < 8) store8(h + col[v], f[v]);
            f[v] = f[v] * inv * g[v];
        }
        float amax = largest(row_f);
        float scale = amax / a.top, back = a.top / amax;
        if (row_is_rare(inv, amax)) {  // the same for all waves of a row
            if constexpr (WPR > 1) __syncthreads();
            // what this lane stored, or x as it was; no address of it computed ahead of the
            // row's loads
            const T *hr = a.r ? h : x, *gr = gamma;
            asm volatile("" : "+v"(hr), "+v"(gr));
            constexpr f32x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int v = 0; v < NV; v++) f[v] = skip[v] < 8 ? load8(hr + col[v]) : zero;
            const float hmax = largest(row_f), by = row_shift(hmax, a.eps_exp);
#pragma unroll
            for (int v = 0; v < NV; v++) f[v] *= by;
            inv = row_inv(hmax, mean_square(row_f), a.eps * by * by);
            auto y = [&](int v) { return skip[v] < 8 ? f[v] * inv * load8(gr + col[v]) : zero; };
            amax = largest(y), scale = amax / a.top, back = a.top / amax;
            if (row_small(amax)) {
                inv *= ROW_UP;
                if constexpr (WPR > 1) __syncthreads();
                amax = largest(y), scale = amax / a.top * ROW_DOWN, back = row_back_up(scale);
            }
#pragma unroll
            for (int v = 0; v < NV; v++) f[v] = y(v);
        }
        if (live && t == 0) a.scale[row] = scale;
        unsigned char *q = a.q + row * a.ldq;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            if (skip[v] == 8) continue;
            unsigned w[2];
#pragma unroll
            for (int p = 0; p < 2; p++) {
                float s[4];
#pragma unroll
                for (int i = 0; i < 4; i++)
                    s[i] = __builtin_fminf(__builtin_fmaxf(f[v][4 * p + i] * back, -a.top), a.top);
                if (a.q_int8) {
                    w[p] = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) w[p] |= ((unsigned)(int)__builtin_rintf(s[i]) & 255u) << (8 * i);
                } else {
                    w[p] = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
                    w[p] = __builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], w[p], true);
                }
            }
            __builtin_memcpy(q + col[v], w, 8);
        }
        if constexpr (WPR > 1) __syncthreads();  // s_sum and s_max are free again
    }
}

// Rows of fewer than 8 columns: a thread a row.
template <typename T>
__global__ __launch_bounds__(256) void norm_quant_narrow_kernel(NormArgs a) {
    const T *gamma = static_cast<const T *>(a.gamma);
    for (long long row = blockIdx.x * 256LL + threadIdx.x; row < a.rows; row += gridDim.x * 256LL) {
        const T *x = static_cast<const T *>(a.x) + row * a.ldx;
        const T *r = static_cast<const T *>(a.r) + row * a.ldr;
        T *h = static_cast<T *>(a.h) + row * a.ldh;
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            f[i] = 0.0f;
            if (i >= a.cols) continue;
            f[i] = (float)x[i];
            if (a.r) {
                const T s = (T)(f[i] + (float)r[i]);
                h[i] = s;
                f[i] = (float)s;
            }
        }
        auto mean_square = [&] {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) sum = __builtin_fmaf(f[i], f[i], sum);
            return sum / (float)a.cols;
        };
        auto largest = [&](float by, const T *g) {  // of f by g
            unsigned top_bits = 0;
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < a.cols) top_bits = max(top_bits, abs_bits(f[i] * by * (g ? (float)g[i] : 1.0f)));
            return __uint_as_float(top_bits);
        };
        // the steps that hold for every row, for all
        const float hmax = largest(1.0f, nullptr), shift = row_shift(hmax, a.eps_exp);
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] *= shift;
        float inv = row_inv(hmax, mean_square(), a.eps * shift * shift);
        float amax = largest(inv, gamma), scale = amax / a.top, back = a.top / amax;
        if (row_small(amax)) {
            inv *= ROW_UP;
            amax = largest(inv, gamma), scale = amax / a.top * ROW_DOWN, back = row_back_up(scale);
        }
        a.scale[row] = scale;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (i >= a.cols) continue;
            const float s = __builtin_fminf(__builtin_fmaxf(f[i] * inv * (float)gamma[i] * back, -a.top), a.top);
            a.q[row * a.ldq + i] = a.q_int8 ? (unsigned char)(signed char)(int)__builtin_rintf(s)
                                            : (unsigned char)__builtin_amdgcn_cvt_pk_fp8_f32(s, s, 0, false);
        }
    }
}

template <typename T>
static osh_status norm_quant_launch(const NormArgs &a, hipStream_t st) {
    constexpr long long MAX_GRID = 1 << 20;
    if (a.cols < 8) {
        OSH_LAUNCH(norm_quant_narrow_kernel<T>, dim3((unsigned)std::min<long long>((a.rows + 255) / 256, MAX_GRID)),
                   dim3(256), 0, st, a);
        OSH_LAUNCH_CHECK("norm_quant_narrow_kernel");
        return OSH_OK;
    }
#define OSH_NORM(WPR, NV)                                                                                     \
    do {                                                                                                      \
        constexpr int RPB = WPR > 4 ? 1 : 4 / WPR;                                                            \
        OSH_LAUNCH((norm_quant_kernel<T, WPR, NV>),                                                           \
                   dim3((unsigned)std::min<long long>((a.rows + RPB - 1) / RPB, MAX_GRID)),                   \
                   dim3(WPR > 4 ? WPR * 64 : 256), 0, st, a);                                                 \
    } while (0)
    // Waves of one vector a lane that hold a row.  One vector a lane up to eight waves: at
    // 4096 columns 16384 rows take 83.5 us so, 84.4 in four waves of two and 88.9 in two of
    // four, one row 3.5, 3.8 and 4.5; at 8192 columns 8192 rows take 85.6 in eight waves of
    // two, 92.5 in sixteen of one, 91.2 in four of four.
    const int waves = (a.cols + 511) / 512;
    if (waves <= 1) OSH_NORM(1, 1);
    else if (waves <= 4) OSH_NORM(4, 1);
    else if (waves <= 8) OSH_NORM(8, 1);
    else if (waves <= 16) OSH_NORM(8, 2);
    else if (waves <= 32) OSH_NORM(16, 2);
    else OSH_NORM(16, 4);
#undef OSH_NORM
    OSH_LAUNCH_CHECK("norm_quant_kernel");
    return OSH_OK;
}

}  // namespace osh

extern "C" {

OSH_API osh_status osh_rms_norm_quant(int64_t rows, int cols, int dtype, const void *d_x, int64_t ldx,
                                      const void *d_res, int64_t ldr, const void *d_gamma, float eps, void *d_h,
                                      int64_t ldh, int q_type, void *d_q, int64_t ldq, float *d_scale,
                                      osh_stream s) {
    constexpr int MAX_COLS = 32768;  // 16 waves of four vectors a lane
    if (rows < 0 || cols < 0) return fail(OSH_E_INVALID, "RmsNormQuant: negative sizes");
    if (dtype != OSH_T_F32 && dtype != OSH_T_F16 && dtype != OSH_T_BF16)
        return fail(OSH_E_INVALID, "RmsNormQuant: rows are f32, f16 or bf16");
    if (q_type != OSH_T_I8 && q_type != OSH_T_E4M3) return fail(OSH_E_INVALID, "RmsNormQuant: q is int8 or e4m3");
    if (!(eps >= 0.0f)) return fail(OSH_E_INVALID, "RmsNormQuant: eps is negative");
    if (rows == 0) return OSH_OK;
    if (cols == 0) return fail(OSH_E_INVALID, "RmsNormQuant: rows without columns");
    if (cols > MAX_COLS) return fail(OSH_E_UNSUPPORTED, "RmsNormQuant: %d columns, at most %d", cols, MAX_COLS);
    if (!d_x || !d_gamma || !d_q || !d_scale || (d_res && !d_h)) return fail(OSH_E_INVALID, "RmsNormQuant: NULL pointer");
    if (ldx < cols || ldq < cols || (d_res && (ldr < cols || ldh < cols)))
        return fail(OSH_E_INVALID, "RmsNormQuant: a row pitch below the columns");
    const long long e = elem_bytes(dtype);
    const Strided x = strided_rows(d_x, rows, ldx * e, cols * e), r = strided_rows(d_res, rows, ldr * e, cols * e),
                  h = strided_rows(d_res ? d_h : nullptr, rows, ldh * e, cols * e), g(d_gamma, cols * e),
                  q = strided_rows(d_q, rows, ldq, cols), scale(d_scale, rows * 4);
    if (share_bytes(h, x) && !(d_h == d_x && ldh == ldx))
        return fail(OSH_E_INVALID, "RmsNormQuant: h overlaps x without being x");
    if (share_bytes(h, r) && !(d_h == d_res && ldh == ldr))
        return fail(OSH_E_INVALID, "RmsNormQuant: h overlaps the residual without being it");
    if (share_bytes(h, g) || share_bytes(h, q) || share_bytes(h, scale) || share_bytes(q, scale))
        return fail(OSH_E_INVALID, "RmsNormQuant: an output overlaps another operand");
    for (const Strided &t : {x, r, g})
        if (share_bytes(q, t) || share_bytes(scale, t))
            return fail(OSH_E_INVALID, "RmsNormQuant: an output overlaps another operand");
    NormArgs a;
    a.rows = rows;
    a.cols = cols;
    a.ldx = ldx;
    a.ldr = ldr;
    a.ldh = ldh;
    a.ldq = ldq;
    a.x = d_x;
    a.r = d_res;
    a.gamma = d_gamma;
    a.h = d_h;
    a.q = static_cast<unsigned char *>(d_q);
    a.scale = d_scale;
    a.eps = eps;
    a.eps_exp = eps > 0.0f ? std::min(std::ilogb(std::sqrt(eps)), 127) + 127 : 0;
    a.q_int8 = q_type == OSH_T_I8;
    a.top = a.q_int8 ? 127.0f : 448.0f;
    if (dtype == OSH_T_F32) return norm_quant_launch<float>(a, to_stream(s));
    if (dtype == OSH_T_F16) return norm_quant_launch<_Float16>(a, to_stream(s));
    return norm_quant_launch<__bf16>(a, to_stream(s));
}

}  // extern "C"
