// osh_int4_matmul.hip -- product with weights of 4 bits and group scales:
//
//   y[i][j] = act(sum_k a[i][k] (c[j][k] - z[j][k / group]) s[j][k / group] + bias[j]) + res[i][j]
//
// The weights are laid out once (osh_int4_pack): blocks of 16 outputs by 128 k, in a block
// 16 bytes for each lane (jl, g) of a wave, in which word t holds output jl, k 32 t + 8 g ..
// + 7, as the 16x16x32 MFMA takes its A operand.  A wave's load of a block is 1 KB in a row.
//
// The MFMAs multiply the codes, which are exact in 16 bits, and add c - z over a group in
// FP32: sum a c - z sum a, the second sum by an MFMA whose A operand is the constant -8
// or -1.  A group's sum is scaled once, in FP32.  So nothing is rounded between the operands
// and the FP32 sums.  FP32 rows are taken as three bf16 pieces (8 + 8 + 8 bits of 24).
#include <limits.h>

#include <algorithm>

#include "osh_int4.h"
#include "osh_overlap.h"

using namespace osh;

namespace osh {

struct Int4Args {
    int m, n, k, act;
    long long lda, ldr, ldy;
    const void *a;
    const uint4 *codes;  // [n / 16][k / 128][64]
    const void *scales;  // [n / 16][k / 128][groups of a block][16]
    const void *zeros;   // the same, or NULL: 8
    const float *bias;
    const void *res;
    void *y;
};

constexpr int KB = 128;  // k of a block

// The pieces of 8 neighbouring values of a row from k0 on, zero from k on.
template <typename T> constexpr int PIECES = sizeof(T) == 4 ? 3 : 1;
template <typename T>
__device__ __forceinline__ typename Vec8<T>::type load_row8(const T *row, int k0, int k) {
    typename Vec8<T>::type v = {};
    if (k0 + 8 <= k) {
        __builtin_memcpy(&v, row + k0, sizeof(v));
    } else {
#pragma unroll
        for (int i = 0; i < 7; i++)
            if (k0 + i < k) v[i] = row[k0 + i];
    }
    return v;
}
template <typename T, typename H8>
__device__ __forceinline__ void split_row8(const typename Vec8<T>::type &v, H8 (&p)[PIECES<T>]) {
    if constexpr (sizeof(T) == 2) {
        p[0] = v;
    } else {
        // the upper 16 bits of what is left, three times: exact, an infinity apart, whose
        // rest is not taken
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float rest = v[i];
#pragma unroll
            for (int e = 0; e < 3; e++) {
                unsigned top = __float_as_uint(rest) & 0xffff0000u;
                if (e == 0 && rest != rest) top |= 0x00400000u;  // stays a NaN
                p[e][i] = __builtin_bit_cast(__bf16, (unsigned short)(top >> 16));
                rest -= __uint_as_float(top);
                if (e == 0 && (top & 0x7f800000u) == 0x7f800000u) rest = 0.0f;
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ T int4_finish(const Int4Args &p, float v, int row, int col) {
    if (p.bias) v += p.bias[col];
    v = apply_act<sizeof(T) == 4>(p.act, v);
    if (p.res) v += (float)static_cast<const T *>(p.res)[row * p.ldr + col];
    return (T)v;
}

// Eight neighbouring outputs of a row, as far as they are there.
template <typename T>
__device__ __forceinline__ void int4_store8(const Int4Args &p, f32x8 f, int row, int col) {
    if (row >= p.m || col >= p.n) return;
    T *y = static_cast<T *>(p.y) + row * p.ldy + col;
    const T *res = static_cast<const T *>(p.res) + row * p.ldr + col;
    if (col + 8 <= p.n) {
        if (p.bias) f += load8(p.bias + col);
        switch (p.act) {
        case OSH_ACT_RELU: act8<OSH_ACT_RELU, sizeof(T) == 4>(f); break;
        case OSH_ACT_SILU: act8<OSH_ACT_SILU, sizeof(T) == 4>(f); break;
        case OSH_ACT_GELU: act8<OSH_ACT_GELU, sizeof(T) == 4>(f); break;
        default: break;
        }
        if (p.res) f += load8(res);
        store8(y, f);
    } else {
#pragma unroll
        for (int i = 0; i < 7; i++)
            if (col + i < p.n) y[i] = int4_finish<T>(p, f[i], row, col + i);
    }
}

// Few rows: a workgroup takes 16 NB outputs of 16 MB rows, its waves every WAVES-th block
// of k; the weights go from memory to registers, each byte once.  GS steps of 32 k share a
// scale.  The waves' sums meet in LDS, in the order of the waves.
template <typename T, int MB, int NB, int GS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void int4_rows_kernel(Int4Args p) {
    using H8 = typename Half8<T>::type;
    using V = typename Vec8<T>::type;
    typedef T T4 __attribute__((ext_vector_type(4)));
    constexpr int P = PIECES<T>, NG = 4 / GS;
    __shared__ f32x4 part[WAVES][MB * NB][64];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int jl = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * (16 * NB), m0 = blockIdx.y * (16 * MB);
    const int nkb = cdiv(p.k, KB), whole = p.k / KB;
    const T *a[MB];
    long long blk[NB];
    f32x4 acc[MB][NB];
#pragma unroll
    for (int j = 0; j < NB; j++) blk[j] = (long long)min(n0 / 16 + j, cdiv(p.n, 16) - 1) * nkb;
#pragma unroll
    for (int i = 0; i < MB; i++) {
        a[i] = static_cast<const T *>(p.a) + (long long)min(m0 + 16 * i + jl, p.m - 1) * p.lda + 8 * g;
#pragma unroll
        for (int j = 0; j < NB; j++) acc[i][j] = f32x4{0, 0, 0, 0};
    }
    H8 minus;  // sum a times it, in every row of a fragment
#pragma unroll
    for (int e = 0; e < 8; e++) minus[e] = p.zeros ? -1.0f : -8.0f;

    struct Block {
        uint4 w[NB];
        T4 sc[NB][NG], zp[NB][NG];
        V x[MB][4];
    };
    auto load = [&](int kb, Block &v, auto cut) {
#pragma unroll
        for (int j = 0; j < NB; j++) {
            v.w[j] = p.codes[(blk[j] + kb) * 64 + lane];
#pragma unroll
            for (int e = 0; e < NG; e++) {
                const long long at = ((blk[j] + kb) * NG + e) * 16 + 4 * g;
                v.sc[j][e] = *reinterpret_cast<const T4 *>(static_cast<const T *>(p.scales) + at);
                if (p.zeros) v.zp[j][e] = *reinterpret_cast<const T4 *>(static_cast<const T *>(p.zeros) + at);
            }
        }
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
            for (int t = 0; t < 4; t++) {
                if constexpr (decltype(cut)::value) v.x[i][t] = load_row8<T>(a[i] - 8 * g, kb * KB + 32 * t + 8 * g, p.k);
                else __builtin_memcpy(&v.x[i][t], a[i] + kb * KB + 32 * t, sizeof(V));
            }
    };
    auto compute = [&](const Block &v) {
#pragma unroll
        for (int e = 0; e < NG; e++) {
            H8 xs[MB][GS][P];
            f32x4 less[MB];
#pragma unroll
            for (int i = 0; i < MB; i++) {
                less[i] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < GS; t++) {
                    split_row8<T>(v.x[i][e * GS + t], xs[i][t]);
#pragma unroll
                    for (int q = 0; q < P; q++) less[i] = mma16(minus, xs[i][t][q], less[i]);
                }
            }
#pragma unroll
            for (int j = 0; j < NB; j++) {
                f32x4 sum[MB];
#pragma unroll
                for (int i = 0; i < MB; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) sum[i][r] = p.zeros ? less[i][r] * (float)v.zp[j][e][r] : less[i][r];
#pragma unroll
                for (int t = 0; t < GS; t++) {
                    H8 c;
                    codes8(reinterpret_cast<const unsigned *>(&v.w[j])[e * GS + t], c);
#pragma unroll
                    for (int i = 0; i < MB; i++)
#pragma unroll
                        for (int q = 0; q < P; q++) sum[i] = mma16(c, xs[i][t][q], sum[i]);
                }
#pragma unroll
                for (int i = 0; i < MB; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[i][j][r] = __builtin_fmaf((float)v.sc[j][e][r], sum[i][r], acc[i][j][r]);
            }
        }
    };
    int kb = wave;
    Block v;
    for (; kb < whole; kb += WAVES) load(kb, v, IntC<0>{}), compute(v);
    if (kb < nkb) load(kb, v, IntC<1>{}), compute(v);
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int j = 0; j < NB; j++) part[wave][i * NB + j][lane] = acc[i][j];
    __syncthreads();
    for (int e = tid; e < MB * NB * 256; e += 64 * WAVES) {
        // neighbouring threads, neighbouring outputs
        const int c = e % (16 * NB), r16 = e / (16 * NB), col = n0 + c, row = m0 + r16;
        const int f = r16 / 16 * NB + c / 16, from = r16 % 16 + 16 * (c / 4 % 4), r = c % 4;
        float sum = part[0][f][from][r];
#pragma unroll
        for (int v = 1; v < WAVES; v++) sum += part[v][f][from][r];
        if (row < p.m && col < p.n) static_cast<T *>(p.y)[row * p.ldy + col] = int4_finish<T>(p, sum, row, col);
    }
}


// ---------------------------------------------------- few rows, large weights

// A workgroup takes 128 outputs (32 a wave) of up to 16 MB rows over up to KR blocks of k: all its
// codes are on their way before the first one is used, the rows' pieces and the scales pass
// through LDS once for its four waves (chunk c of row r at c ^ r % 16), and one barrier is all.
// The sums of the parts of k go to memory in FP32 and are joined in their order.  In
// int4_rows_kernel each 16 outputs read the rows again, which binds it: 32 rows of 8192 against
// 16384 outputs are 537 MB from the L2.
template <typename T, int MB> constexpr int SLIM_KR = sizeof(T) == 4 ? (MB == 1 ? 4 : 2) : MB == 4 ? 4 : 8;

template <typename T, int MB, int GS>
__global__ __launch_bounds__(256, 2) void int4_slim_kernel(Int4Args p, int kr, float *part, long long pitch) {
    using H8 = typename Half8<T>::type;
    typedef T T4 __attribute__((ext_vector_type(4)));
    constexpr int P = PIECES<T>, NG = 4 / GS, KR = SLIM_KR<T, MB>, ROWS = 16 * MB;
    constexpr int SC = KR * NG * 16;  // scales of 16 outputs
    __shared__ __align__(16) H8 rows[P][ROWS][KR * 16];
    __shared__ __align__(16) T scales[8][SC], zeros[8][SC];
    const int tid = threadIdx.x, lane = tid & 63, jl = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nkb = cdiv(p.k, KB), nblk = cdiv(p.n, 16);
    const int kb0 = blockIdx.y * kr, count = min(kr, nkb - kb0), b0 = blockIdx.x * 8, m0 = blockIdx.z * ROWS;

    // rows and scales first: loads return in order
    constexpr int PER = KR * 16 * ROWS / 256;  // chunks of a thread
    typename Vec8<T>::type x[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = i * 256 + tid, r = e / (KR * 16), c = e % (KR * 16);
        const T *row = static_cast<const T *>(p.a) + (long long)min(m0 + r, p.m - 1) * p.lda;
        x[i] = load_row8<T>(row, kb0 * KB + 8 * c, c < count * 16 ? p.k : 0);
    }
    constexpr int VEC = 16 / sizeof(T);
    for (int e = tid; e < 8 * (SC / VEC); e += 256) {
        const int j = e / (SC / VEC), c = e % (SC / VEC) * VEC;
        if (c >= count * NG * 16) continue;
        const long long at = ((long long)min(b0 + j, nblk - 1) * nkb + kb0) * NG * 16 + c;
        __builtin_memcpy(&scales[j][c], static_cast<const T *>(p.scales) + at, 16);
        if (p.zeros) __builtin_memcpy(&zeros[j][c], static_cast<const T *>(p.zeros) + at, 16);
    }
    uint4 w[KR][2];
#pragma unroll
    for (int kb = 0; kb < KR; kb++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const long long blk = (long long)min(b0 + 2 * wave + j, nblk - 1) * nkb + kb0 + min(kb, count - 1);
            w[kb][j] = p.codes[blk * 64 + lane];
        }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = i * 256 + tid, r = e / (KR * 16), c = e % (KR * 16);
        H8 h[P];
        split_row8<T>(x[i], h);
#pragma unroll
        for (int u = 0; u < P; u++) rows[u][r][c ^ (r & 15)] = h[u];
    }
    __syncthreads();
    H8 minus;
#pragma unroll
    for (int e = 0; e < 8; e++) minus[e] = p.zeros ? -1.0f : -8.0f;
    f32x4 acc[MB][2];
#pragma unroll
    for (int i = 0; i < MB; i++) acc[i][0] = acc[i][1] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int kb = 0; kb < KR; kb++) {
        if (kb >= count) break;
#pragma unroll
        for (int e = 0; e < NG; e++) {
            H8 xs[MB][GS][P];
            f32x4 less[MB];
#pragma unroll
            for (int i = 0; i < MB; i++) {
                less[i] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < GS; s++)
#pragma unroll
                    for (int u = 0; u < P; u++) {
                        xs[i][s][u] = rows[u][16 * i + jl][(kb * 16 + 4 * (e * GS + s) + g) ^ jl];
                        less[i] = mma16(minus, xs[i][s][u], less[i]);
                    }
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const T4 sc = *reinterpret_cast<const T4 *>(&scales[2 * wave + j][(kb * NG + e) * 16 + 4 * g]);
                f32x4 sum[MB];
#pragma unroll
                for (int i = 0; i < MB; i++) sum[i] = less[i];
                if (p.zeros) {
                    const T4 zp = *reinterpret_cast<const T4 *>(&zeros[2 * wave + j][(kb * NG + e) * 16 + 4 * g]);
#pragma unroll
                    for (int i = 0; i < MB; i++)
#pragma unroll
                        for (int r = 0; r < 4; r++) sum[i][r] *= (float)zp[r];
                }
#pragma unroll
                for (int s = 0; s < GS; s++) {
                    H8 c;
                    codes8(reinterpret_cast<const unsigned *>(&w[kb][j])[e * GS + s], c);
#pragma unroll
                    for (int i = 0; i < MB; i++)
#pragma unroll
                        for (int u = 0; u < P; u++) sum[i] = mma16(c, xs[i][s][u], sum[i]);
                }
#pragma unroll
                for (int i = 0; i < MB; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[i][j][r] = __builtin_fmaf((float)sc[r], sum[i][r], acc[i][j][r]);
            }
        }
    }
    // lane (jl, g): outputs 4 g .. + 3 of row jl
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int row = m0 + 16 * i + jl, col = (b0 + 2 * wave + j) * 16 + 4 * g;
            if (row >= p.m) continue;
            if (gridDim.y > 1) {
                *reinterpret_cast<f32x4 *>(part + ((long long)blockIdx.y * p.m + row) * pitch + col) = acc[i][j];
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (col + r < p.n) static_cast<T *>(p.y)[row * p.ldy + col + r] = int4_finish<T>(p, acc[i][j][r], row, col + r);
            }
        }
}

// The parts' sums, four outputs a thread.
template <typename T>
__global__ __launch_bounds__(256) void int4_join_kernel(Int4Args p, int parts, const float *part, long long pitch) {
    const int quads = (int)(pitch / 4);
    const long long at = blockIdx.x * 256LL + threadIdx.x;
    if (at >= (long long)p.m * quads) return;
    const int row = (int)(at / quads), col = (int)(at - (long long)row * quads) * 4;
    const float *from = part + row * pitch + col;
    const long long next = (long long)p.m * pitch;
    f32x4 sum = {0, 0, 0, 0};
    for (int s = 0; s < parts; s += 8) {
        f32x4 v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = *reinterpret_cast<const f32x4 *>(from + min(s + e, parts - 1) * next);
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (s + e < parts) sum += v[e];
    }
#pragma unroll
    for (int r = 0; r < 4; r++)
        if (col + r < p.n) static_cast<T *>(p.y)[row * p.ldy + col + r] = int4_finish<T>(p, sum[r], row, col + r);
}

// ---------------------------------------------------------------- many rows

// What the tile kernel reads of the rows: their 16-bit pieces (the rows themselves where
// they are 16-bit and whole chunks long) and the sums over groups.
struct Int4Prep {
    const unsigned short *a;
    long long pitch, plane;  // of a row and of a piece, in values
    int chunks;              // of 8 values in a row; what lies past them is 0
    int groups;
    const uint2 *sums;       // of 16-bit rows, [m][groups]: -sum a in three bf16 pieces, and 0
};

// The FP32 number v as the sum of three bf16 ones (their bits, in the upper halves).
__device__ __forceinline__ void pieces3(float v, unsigned (&top)[3]) {
    float rest = v;
#pragma unroll
    for (int e = 0; e < 3; e++) {
        top[e] = __float_as_uint(rest) & 0xffff0000u;
        if (e == 0 && rest != rest) top[e] |= 0x00400000u;
        rest -= __uint_as_float(top[e]);
        if (e == 0 && (top[e] & 0x7f800000u) == 0x7f800000u) rest = 0.0f;
    }
}

// Sums of the rows' groups (at most 128 long), and with COPY their pieces [P][m][128 nkb], zero
// past k.  GL lanes a group.
template <typename T, int GL, bool COPY>
__global__ __launch_bounds__(256) void int4_prep_kernel(Int4Args p, int group, int groups, uint2 *sums,
                                                        unsigned short *planes, long long pitch, long long plane) {
    constexpr int P = PIECES<T>;
    const int all = COPY ? max(groups, (int)cdiv((int)pitch, group)) : groups;  // what the copy is padded to
    const long long total = (long long)p.m * all;
    const int sub = threadIdx.x % GL;
    // whole rounds: the lanes of a group stay together
    for (long long i0 = blockIdx.x * (256LL / GL); i0 < total; i0 += gridDim.x * (256LL / GL)) {
        const long long item = i0 + threadIdx.x / GL;
        const bool in = item < total;
        const int row = in ? (int)(item / all) : 0, gr = in ? (int)(item - (long long)row * all) : 0;
        const T *a = static_cast<const T *>(p.a) + row * p.lda;
        float sum = 0.0f;
        for (int c = 8 * sub; c < group; c += 8 * GL) {
            const int k0 = gr * group + c;
            const typename Vec8<T>::type v = load_row8<T>(a, k0, in ? p.k : 0);
#pragma unroll
            for (int i = 0; i < 8; i++) sum += (float)v[i];
            if (COPY && in && k0 < pitch) {
                typename Half8<T>::type h[P];
                split_row8<T>(v, h);
#pragma unroll
                for (int e = 0; e < P; e++) *reinterpret_cast<typename Half8<T>::type *>(planes + e * plane + row * pitch + k0) = h[e];
            }
        }
#pragma unroll
        for (int o = 1; o < GL; o <<= 1) sum += __shfl_xor(sum, o);
        if (P == 1 && in && sub == 0 && gr < groups) {
            unsigned t[3];
            pieces3(-sum, t);
            sums[(long long)row * groups + gr] = uint2{t[0] >> 16 | t[1], t[2] >> 16};
        }
    }
}

static __device__ const uint4 int4_zero_chunk = {0, 0, 0, 0};

// A group's scale s = unit * 2^e: the power of two goes into the codes, which stay exact, and
// the unit (1/2 to 1 in size but at the ends of the type's range) into the sums.
template <typename T>
__device__ __forceinline__ float int4_unit(float s, float &times512) {
    // c 2^e stays a number of T: 15 * 2^12 < 65504, and 2^-24 is f16's smallest
    constexpr bool F16 = __is_same(T, _Float16);
    int e = __builtin_amdgcn_frexp_expf(s);
    e = min(max(e, F16 ? -24 : -100), F16 ? 12 : 100);
    times512 = __builtin_amdgcn_ldexpf(512.0f, e);
    return __builtin_amdgcn_ldexpf(s, -e);
}
// a / b, within 2^-23 of it.
__device__ __forceinline__ float int4_ratio(float a, float b) {
    const float r = __builtin_amdgcn_rcpf(b), q = a * r;
    return __builtin_fmaf(__builtin_fmaf(-q, b, a), r, q);
}

// A workgroup takes 32 MB WM rows by 32 NB WN outputs, a wave 32 MB by 32 NB.  The rows pass
// through two LDS buffers of 128 k, loaded directly (chunk c of row r at c ^ r % 16); codes go
// from memory to registers a block ahead and become 16-bit floats in front of the MFMAs that
// take them.
//
// 16-bit rows: a lane's sums, all of one output j, are kept in the unit of the group at hand
// (int4_unit), so that the MFMAs add onto them directly, and between two groups are taken times
// the ratio of their units: one product a sum, no registers for a group's own sums.  The zero
// points' part, -sum a (three bf16 pieces) times z, goes in front of a group's codes as a matrix
// instruction of its own, so that a sum is never larger than the result so far and one group.
// Added for all of k at the end it takes a few per cent less (8192 x 4096 x 8192 in groups of 128
// 577 us for 589, of 64 700 for 760; of 32 1020 for 945), and leaves rows that do not average zero 50
// to 100 times the error: 1.9e-2 for 2.1e-4 in results of 300, positive rows, k of 8192.
// FP32 rows, three MFMAs a fragment of codes: the zero points come off the codes, which the
// vector unit has time for and which loses nothing to the difference of two sums; a group's
// sum has its own registers and is scaled into the wave's sums.
template <typename T, int MB, int NB, int WM, int WN, int GS>
__global__ __launch_bounds__(64 * WM * WN, 2) void int4_tile_kernel(Int4Args p, Int4Prep q) {
    using H8 = typename Half8<T>::type;
    constexpr int P = PIECES<T>, NG = 4 / GS, WAVES = WM * WN, R = 32 * MB * WM;
    constexpr int STAGE = P * R * 256, COPIES = P * R / 4 / WAVES;
    static_assert(COPIES * 4 * WAVES == P * R, "copies are dealt evenly");
    extern __shared__ __align__(16) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hl = lane >> 5, wm = wave / WN, wn = wave % WN;
    const int nkb = cdiv(p.k, KB);

    // bands of eight row blocks: those that run at once share rows and weights in an L2
    int mt, nt;
    {
        const int tn = cdiv(p.n, 32 * NB * WN), tm = cdiv(p.m, R);
        const int id = xcd_band(blockIdx.x, gridDim.x);
        const int band = id / (8 * tn), high = min(8, tm - 8 * band), in = id - band * 8 * tn;
        mt = 8 * band + in % high;
        nt = in / high;
    }
    const int m0 = mt * R, n0 = nt * 32 * NB * WN;

    const unsigned short *from[COPIES];
    int chunk0[COPIES];
#pragma unroll
    for (int e = 0; e < COPIES; e++) {
        const int i = wave + WAVES * e, r = i % (R / 4) * 4 + (lane >> 4);
        chunk0[e] = (lane & 15) ^ (r & 15);
        from[e] = q.a + i / (R / 4) * q.plane + min(m0 + r, p.m - 1) * q.pitch + 8 * chunk0[e];
    }
    auto load_rows = [&](int kb, int buf) {
#pragma unroll
        for (int e = 0; e < COPIES; e++) {
            const bool in = kb * 16 + chunk0[e] < q.chunks;
            const void *at = from[e] + kb * KB;
            copy_to_lds<16>(in ? at : &int4_zero_chunk, lds + buf * STAGE + (wave + WAVES * e) * 1024);
        }
    };
    long long blk[NB];
#pragma unroll
    for (int j = 0; j < NB; j++)
        blk[j] = (long long)min((n0 + 32 * (wn * NB + j) + l32) / 16, cdiv(p.n, 16) - 1) * nkb;
    const int jl = lane & 15;
    uint4 w[NB][2], w_next[NB][2];
    T sc[NB][NG], sc_next[NB][NG], zp[NB][NG], zp_next[NB][NG];
    const uint2 *sums[MB];
    uint2 less[NG][MB], less_next[NG][MB];
#pragma unroll
    for (int i = 0; i < MB; i++)
        sums[i] = q.sums + (P > 1 ? 0 : (long long)min(m0 + 32 * (wm * MB + i) + l32, p.m - 1) * q.groups);
    auto load_codes = [&](int kb) {
#pragma unroll
        for (int j = 0; j < NB; j++) {
#pragma unroll
            for (int e = 0; e < 2; e++) w_next[j][e] = p.codes[(blk[j] + kb) * 64 + 32 * e + 16 * hl + jl];
#pragma unroll
            for (int e = 0; e < NG; e++) {
                const long long at = ((blk[j] + kb) * NG + e) * 16 + jl;
                sc_next[j][e] = static_cast<const T *>(p.scales)[at];
                zp_next[j][e] = p.zeros ? static_cast<const T *>(p.zeros)[at] : (T)8.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
            for (int e = 0; e < NG; e++)  // a group past the last one has scales of 0
                if (P == 1) less_next[e][i] = sums[i][min(kb * NG + e, q.groups - 1)];
    };
    f32x16 acc[MB][NB];
    float unit[NB], times512[NB];
#pragma unroll
    for (int j = 0; j < NB; j++) {
        unit[j] = 1.0f, times512[j] = 512.0f;
#pragma unroll
        for (int i = 0; i < MB; i++) acc[i][j] = f32x16{};
    }
    // group e of the block at hand: the sums in its unit, and the zero points' part, z in the unit of
    // the codes, which is exact
    auto enter = [&](int j, T scale, T zero, const uint2 (&pieces)[MB]) {
        const float f = (float)scale;
        float t512;
        const float next = int4_unit<T>(f, t512), by = f != 0.0f ? int4_ratio(unit[j], next) : 1.0f;
        unit[j] = f != 0.0f ? next : unit[j];  // a scale of 0 has codes of 0
        times512[j] = t512;
        // the pieces are the lower half of the wave's
        const unsigned z = f != 0.0f && hl == 0 ? __float_as_uint((float)zero * (t512 * 0x1p-9f)) >> 16 : 0u;
        const uint4 zzz = {z | z << 16, z, 0u, 0u};
        bf16x8 b;
        __builtin_memcpy(&b, &zzz, 16);
#pragma unroll
        for (int i = 0; i < MB; i++) {
            const uint4 both = {pieces[i].x, pieces[i].y, 0u, 0u};
            bf16x8 a;
            __builtin_memcpy(&a, &both, 16);
            acc[i][j] *= by;
            acc[i][j] = mma32(a, b, acc[i][j]);
        }
    };
    load_rows(0, 0);
    load_codes(0);
    int buf = 0;
    for (int kb = 0; kb < nkb; kb++, buf ^= 1) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if constexpr (P == 1) {  // the first group in front of the loads, which take its registers
#pragma unroll
            for (int j = 0; j < NB; j++) enter(j, sc_next[j][0], zp_next[j][0], less_next[0]);
        }
#pragma unroll
        for (int j = 0; j < NB; j++) {
#pragma unroll
            for (int e = 0; e < 2; e++) w[j][e] = w_next[j][e];
#pragma unroll
            for (int e = 0; e < NG; e++) {
                sc[j][e] = sc_next[j][e];
                zp[j][e] = zp_next[j][e];
            }
        }
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
            for (int e = 0; e < NG; e++)
                if (P == 1) less[e][i] = less_next[e][i];
        if (kb + 1 < nkb) {
            load_rows(kb + 1, buf ^ 1);
            load_codes(kb + 1);
        }
        const unsigned char *rows = lds + buf * STAGE;
        f32x16 sum[P > 1 ? MB : 1][P > 1 ? NB : 1];
#pragma unroll
        for (int s = 0; s < 8; s++) {
            const int e = s / (2 * GS);
            const bool first = s % (2 * GS) == 0, last = s % (2 * GS) == 2 * GS - 1;
            H8 c[NB];
#pragma unroll
            for (int j = 0; j < NB; j++) {
                const unsigned word = reinterpret_cast<const unsigned *>(&w[j][s & 1])[s >> 1];
                if constexpr (P > 1) {
                    codes8_less(word, zp[j][e], c[j]);
                } else {
                    if (first && e > 0) enter(j, sc[j][e], zp[j][e], less[e]);
                    codes8(word, c[j], times512[j]);
                }
            }
#pragma unroll
            for (int i = 0; i < MB; i++)
#pragma unroll
                for (int u = 0; u < P; u++) {
                    const int r = 32 * (wm * MB + i) + l32;
                    const H8 x = lds_chunk<H8>(rows + u * (R * 256) + r * 256 + (((2 * s + hl) ^ (r & 15)) << 4));
#pragma unroll
                    for (int j = 0; j < NB; j++) {
                        if constexpr (P > 1) sum[i][j] = mma32(x, c[j], first && u == 0 ? f32x16{} : sum[i][j]);
                        else acc[i][j] = mma32(x, c[j], acc[i][j]);
                    }
                }
            if constexpr (P > 1) {
                if (last) {
#pragma unroll
                    for (int j = 0; j < NB; j++)
#pragma unroll
                        for (int i = 0; i < MB; i++)
#pragma unroll
                            for (int r = 0; r < 16; r++)
                                acc[i][j][r] = __builtin_fmaf((float)sc[j][e], sum[i][j][r], acc[i][j][r]);
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NB; j++)
#pragma unroll
        for (int i = 0; i < MB; i++)
            if (P == 1) acc[i][j] *= unit[j];
    // through LDS, 32 rows of a wave at a time, to eight neighbouring outputs a lane
    constexpr int PITCH = 32 * NB + 4;
    float *mine = reinterpret_cast<float *>(lds) + wave * (32 * PITCH);
    const int nw = n0 + 32 * NB * wn;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MB; i++) {
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) mine[(8 * (r >> 2) + 4 * hl + (r & 3)) * PITCH + 32 * j + l32] = acc[i][j][r];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int e = 0; e < 32 * 32 * NB / 8 / 64; e++) {
            const int at = e * 64 + lane, r = at / (4 * NB), c = at % (4 * NB) * 8;
            f32x8 f;
            __builtin_memcpy(&f, mine + r * PITCH + c, 16);
            __builtin_memcpy(reinterpret_cast<float *>(&f) + 4, mine + r * PITCH + c + 4, 16);
            int4_store8<T>(p, f, m0 + 32 * (wm * MB + i) + r, nw + c);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// Codes [n][pitch] two a byte into blocks; codes past n or k are 0 (their scales and the
// values that meet them are 0), and so are those of groups whose scale is 0.
template <typename T>
__global__ __launch_bounds__(256) void int4_pack_codes_kernel(int n, int k, int group, const unsigned char *codes,
                                                              long long pitch, const T *scales, long long lds, uint4 *out) {
    const int nkb = cdiv(k, KB);
    const long long blocks = (long long)cdiv(n, 16) * nkb;
    for (long long e = blockIdx.x * 256LL + threadIdx.x; e < blocks * 64; e += gridDim.x * 256LL) {
        const int lane = (int)(e & 63), jl = lane & 15, g = lane >> 4;
        const long long blk = e >> 6;
        const long long row = blk / nkb * 16 + jl;
        const int k0 = (int)(blk % nkb) * KB;
        unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int at = k0 + 32 * t + 8 * g + i;
                if (row >= n || at >= k || (float)scales[row * lds + at / group] == 0.0f) continue;
                const unsigned code = codes[row * pitch + at / 2] >> (4 * (at & 1)) & 15u;
                w[t] |= code << (4 * (2 * (i & 3) + (i >> 2)));  // 0..3 at even places, 4..7 at odd ones
            }
        out[e] = uint4{w[0], w[1], w[2], w[3]};
    }
}
template <typename T>
__global__ __launch_bounds__(256) void int4_pack_scales_kernel(int n, int k, int group, const T *scales,
                                                               long long lds, const unsigned char *zeros,
                                                               long long ldz, T *out_s, T *out_z) {
    const int per = group < KB ? KB / group : 1, nkb = cdiv(k, KB);
    const long long total = (long long)cdiv(n, 16) * nkb * per * 16;
    for (long long e = blockIdx.x * 256LL + threadIdx.x; e < total; e += gridDim.x * 256LL) {
        const long long blk = e / (16 * per), row = blk / nkb * 16 + e % 16;
        const long long at = (blk % nkb) * KB + e / 16 % per * (KB / per);
        const bool in = row < n && at < k;
        const long long gr = at / group;
        out_s[e] = in ? scales[row * lds + gr] : (T)0.0f;
        if (zeros) out_z[e] = in ? (T)(float)(zeros[row * ldz + gr / 2] >> (4 * (gr & 1)) & 15u) : (T)0.0f;
    }
}

struct Int4Layout {
    size_t codes, scales, total;
};
static Int4Layout int4_layout(int n, int k, int group, int dtype, bool zeros) {
    const size_t blocks = (size_t)cdiv(n, 16) * cdiv(k, KB);
    Int4Layout l;
    l.codes = blocks * 1024;
    l.scales = blocks * (group < KB ? KB / group : 1) * 16 * elem_bytes(dtype);
    l.total = l.codes + l.scales * (zeros ? 2 : 1);
    return l;
}

// Which kernel a call takes, and what it keeps beside its operands.
struct Int4Room {
    bool tile, copy, slim;
    int kr, parts, pitch;       // slim: blocks of k and their number; of a row of sums, or of a piece
    size_t sums, plane, total;  // plane in values
};
static Int4Room int4_room(int m, int n, int k, int group, int dtype) {
    Int4Room r = {};
    const bool f32 = dtype == OSH_T_F32;
    const int nkb = cdiv(k, KB);
    // Small tiles wait for memory once a block of k, the slim kernel once in all but reads the
    // weights again for each 64 rows (32 in FP32).  Tile against slim: 128 rows of 4096 against
    // 4096 outputs 26.3 (22.2) us, 54.4 (39.7) in FP32; of 1024 against 4096 10.8 (16.0), 18.9
    // (16.9); 256 of 8192 against 8192 63.5 (93.7), 144 (286).
    r.tile = m > 64 && (nkb > 65535 || (long long)m * n > (f32 ? 1 << 19 : 1 << 20) || (!f32 && k < 2048));
    if (!r.tile) {
        // Against a launch of int4_rows_kernel, two launches of the slim one cost 4 to 10 us more,
        // by the rows' blocks; it gains what the 16 outputs' own copies of the rows take (20 TB/s as
        // one block of 16, 11 as more) and 0.055 us a MB of weights.  Rows against slim in bf16, every
        // weight out of HBM (1.2 GB of them in turn): 1 row of 8192 on 8192 outputs 11.8 (14.4) us, on
        // 16384 22.9 (22.3), on 32768 43.0 (36.3); of 4096 on 28672 19.3 (19.7); 8 rows of 4096 on
        // 12288 11.4 (13.6), of 8192 on 16384 26.7 (21.0); 16 of 4096 on 4096 6.9 (9.5), on 12288 15.2
        // (14.4); 32 on 4096 10.6 (12.3), on 12288 25.6 (18.1).  Weights that the last cache still
        // holds change it: 1 row on 16384 takes 14 (18).
        // FP32 rows gain where a wave has much to split: 1 on 4096 23 (16), k of 768 on 768 4.8 (9).
        const double copies = (double)cdiv(n, 16) * m * k * 2e-6 / (m <= 16 ? 20 : 11), weights = (double)n * k * 0.5e-6 * 0.055;
        const double cost = m <= 16 ? 4.2 : m <= 32 ? 7.3 : 10.1;
        r.slim = f32 ? (long long)n * k >= 1 << 24 || m > 32 : copies + weights > cost || m > 64;
        if (!r.slim) return r;
        const int mb = m <= 16 ? 1 : m <= 32 || f32 ? 2 : 4;
        const int most = f32 ? (mb == 1 ? 4 : 2) : mb == 4 ? 4 : 8;  // SLIM_KR
        const long long tiles = (long long)cdiv(n, 128) * cdiv(m, 16 * mb);
        r.kr = (int)std::max(1LL, std::min<long long>(most, tiles * nkb / device_cus()));
        r.parts = cdiv(nkb, r.kr);
        if (r.parts > 65535 && m <= 64) {  // more than a grid takes
            r.slim = false;
            return r;
        }
        r.pitch = cdiv(n, 128) * 128;
        r.total = r.parts > 1 ? (size_t)r.parts * m * r.pitch * 4 : 0;
        return r;
    }
    r.copy = f32 || k % 8;
    r.sums = f32 ? 0 : ((size_t)m * cdiv(k, std::min(group, KB)) * 8 + 15) / 16 * 16;
    r.pitch = nkb * KB;
    r.plane = r.copy ? (size_t)m * r.pitch : 0;
    r.total = r.sums + r.plane * (f32 ? 6 : 2);
    return r;
}

template <typename T, int MB, int GS>
static osh_status int4_slim(const Int4Args &p, const Int4Room &room, float *part, hipStream_t st) {
    OSH_LAUNCH((int4_slim_kernel<T, MB, GS>), dim3((unsigned)cdiv(p.n, 128), (unsigned)room.parts, (unsigned)cdiv(p.m, 16 * MB)), dim3(256), 0, st, p,
               room.kr, part, (long long)room.pitch);
    OSH_LAUNCH_CHECK("int4_slim_kernel");
    if (room.parts > 1) {
        const long long threads = (long long)p.m * (room.pitch / 4);
        OSH_LAUNCH(int4_join_kernel<T>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, p, room.parts, part,
                   (long long)room.pitch);
        OSH_LAUNCH_CHECK("int4_join_kernel");
    }
    return OSH_OK;
}

template <typename T, int MB, int NB, int WM, int WN, int GS>
static void int4_tile(const Int4Args &p, const Int4Prep &q, hipStream_t st) {
    constexpr size_t lds = std::max<size_t>(2 * PIECES<T> * 32 * MB * WM * 256, WM * WN * 32 * (32 * NB + 4) * 4);
    OSH_LAUNCH((int4_tile_kernel<T, MB, NB, WM, WN, GS>),
               dim3((unsigned)cdiv(p.m, 32 * MB * WM) * cdiv(p.n, 32 * NB * WN)), dim3(64 * WM * WN), lds, st, p, q);
}

template <typename T, int GS>
static osh_status int4_launch(const Int4Args &p, const Int4Room &room, void *scratch, hipStream_t st) {
    if (room.slim) {
        float *part = static_cast<float *>(scratch);
        if (p.m <= 16) return int4_slim<T, 1, GS>(p, room, part, st);
        if constexpr (sizeof(T) == 2) {
            if (p.m > 32) return int4_slim<T, 4, GS>(p, room, part, st);
        }
        return int4_slim<T, 2, GS>(p, room, part, st);
    }
    if (!room.tile) {
#define OSH_INT4_ROWS(MB)                                                                                        \
    OSH_LAUNCH((int4_rows_kernel<T, MB, 1, GS, 8>), dim3((unsigned)cdiv(p.n, 16), (unsigned)cdiv(p.m, 16 * MB)), \
               dim3(512), 0, st, p)
        if (p.m <= 16) OSH_INT4_ROWS(1);
        else if (p.m <= 32) OSH_INT4_ROWS(2);
        else OSH_INT4_ROWS(4);
#undef OSH_INT4_ROWS
        OSH_LAUNCH_CHECK("int4_rows_kernel");
        return OSH_OK;
    }
    Int4Prep q;
    uint2 *sums = static_cast<uint2 *>(scratch);
    unsigned short *planes = reinterpret_cast<unsigned short *>(static_cast<char *>(scratch) + room.sums);
    q.sums = sums;
    constexpr int group = 32 * GS;  // a longer one's sums in parts of a block
    q.groups = cdiv(p.k, group);
    q.a = room.copy ? planes : static_cast<const unsigned short *>(p.a);
    q.pitch = room.copy ? room.pitch : p.lda;
    q.plane = room.plane;
    q.chunks = (room.copy ? room.pitch : p.k) / 8;
    constexpr int GL = 4 * GS;
    const long long items = (long long)p.m * cdiv(room.pitch, 32 * GS);
    const dim3 grid((unsigned)std::min((items + 256 / GL - 1) / (256 / GL), 1LL << 16));
    if (room.copy) {
        OSH_LAUNCH((int4_prep_kernel<T, GL, true>), grid, dim3(256), 0, st, p, group, q.groups, sums, planes,
                   (long long)room.pitch, (long long)room.plane);
    } else if constexpr (sizeof(T) == 2) {
        OSH_LAUNCH((int4_prep_kernel<T, GL, false>), grid, dim3(256), 0, st, p, group, q.groups, sums, planes,
                   (long long)room.pitch, (long long)room.plane);
    }
    OSH_LAUNCH_CHECK("int4_prep_kernel");
    // 64 x 256 tiles where they fill the card, else 32 x 128 ones: 512 x 4096 x 4096 in bf16 took
    // 56 us as 128 large tiles, 35 as 512 small ones (now 32)
    if ((long long)cdiv(p.m, 64) * cdiv(p.n, 256) >= device_cus()) int4_tile<T, 2, 2, 1, 4, GS>(p, q, st);
    else int4_tile<T, 1, 1, 1, 4, GS>(p, q, st);
    OSH_LAUNCH_CHECK("int4_tile_kernel");
    return OSH_OK;
}

template <typename T>
static osh_status int4_launch_t(const Int4Args &p, int group, const Int4Room &room, void *scratch, hipStream_t st) {
    if (group == 32) return int4_launch<T, 1>(p, room, scratch, st);
    if (group == 64) return int4_launch<T, 2>(p, room, scratch, st);
    return int4_launch<T, 4>(p, room, scratch, st);
}

static osh_status int4_check(int n, int k, int group, int dtype) {
    if (n < 0 || k < 0) return fail(OSH_E_INVALID, "Int4MatMul: negative sizes");
    if (dtype != OSH_T_F32 && dtype != OSH_T_F16 && dtype != OSH_T_BF16)
        return fail(OSH_E_INVALID, "Int4MatMul: rows and scales are f32, f16 or bf16");
    if (group < 1) return fail(OSH_E_INVALID, "Int4MatMul: groups of %d", group);
    if (group != 32 && group != 64 && group % KB)
        return fail(OSH_E_UNSUPPORTED, "Int4MatMul: groups of %d (32, 64 or a multiple of 128)", group);
    if (n > 0 && k == 0) return fail(OSH_E_INVALID, "Int4MatMul: k is 0");
    if (k > (1 << 28) || n > (1 << 28)) return fail(OSH_E_UNSUPPORTED, "Int4MatMul: %d x %d weights", n, k);
    return OSH_OK;
}

}  // namespace osh

extern "C" {

OSH_API osh_status osh_int4_packed_bytes(int n, int k, int group, int dtype, int has_zeros, size_t *bytes) {
    if (!bytes) return fail(OSH_E_INVALID, "Int4MatMul: NULL bytes");
    if (const osh_status st = int4_check(n, k, group, dtype)) return st;
    *bytes = n ? int4_layout(n, k, group, dtype, has_zeros).total : 0;
    return OSH_OK;
}

OSH_API osh_status osh_int4_pack(int n, int k, int group, int dtype, const void *d_codes, int64_t ldc,
                                 const void *d_scales, int64_t lds, const void *d_zeros, int64_t ldz, void *d_packed,
                                 osh_stream s) {
    if (const osh_status st = int4_check(n, k, group, dtype)) return st;
    if (n == 0) return OSH_OK;
    if (!d_codes || !d_scales || !d_packed) return fail(OSH_E_INVALID, "Int4MatMul: NULL pointer");
    const long long groups = cdiv(k, group), e = elem_bytes(dtype);
    if (ldc < cdiv(k, 2) || lds < groups || (d_zeros && ldz < (groups + 1) / 2))
        return fail(OSH_E_INVALID, "Int4MatMul: a row pitch below the columns");
    if ((uintptr_t)d_packed & 15) return fail(OSH_E_INVALID, "Int4MatMul: packed weights need 16-byte alignment");
    const Int4Layout l = int4_layout(n, k, group, dtype, d_zeros);
    const Strided out(d_packed, l.total);
    if (share_bytes(out, strided_rows(d_codes, n, ldc, cdiv(k, 2))) ||
        share_bytes(out, strided_rows(d_scales, n, lds * e, groups * e)) ||
        share_bytes(out, strided_rows(d_zeros, n, ldz, (groups + 1) / 2)))
        return fail(OSH_E_INVALID, "Int4MatMul: the packed weights overlap an operand");
    const hipStream_t st = to_stream(s);
    auto grid = [](size_t threads) { return dim3((unsigned)std::min<size_t>((threads + 255) / 256, 1 << 16)); };
    char *sc = static_cast<char *>(d_packed) + l.codes, *zp = sc + l.scales;
    const unsigned char *c = static_cast<const unsigned char *>(d_codes), *z = static_cast<const unsigned char *>(d_zeros);
#define OSH_PACK(T)                                                                                              \
    do {                                                                                                         \
        const T *from = static_cast<const T *>(d_scales);                                                        \
        OSH_LAUNCH(int4_pack_codes_kernel<T>, grid(l.codes / 16), dim3(256), 0, st, n, k, group, c, (long long)ldc, \
                   from, (long long)lds, static_cast<uint4 *>(d_packed));                                        \
        OSH_LAUNCH(int4_pack_scales_kernel<T>, grid(l.scales / sizeof(T)), dim3(256), 0, st, n, k, group, from,  \
                   (long long)lds, z, (long long)ldz, reinterpret_cast<T *>(sc), reinterpret_cast<T *>(zp));     \
    } while (0)
    if (dtype == OSH_T_F32) OSH_PACK(float);
    else if (dtype == OSH_T_F16) OSH_PACK(_Float16);
    else OSH_PACK(__bf16);
#undef OSH_PACK
    OSH_LAUNCH_CHECK("int4 pack kernels");
    return OSH_OK;
}

OSH_API osh_status osh_int4_matmul_scratch_bytes(int m, int n, int k, int group, int dtype, size_t *bytes) {
    if (!bytes) return fail(OSH_E_INVALID, "Int4MatMul: NULL bytes");
    if (m < 0) return fail(OSH_E_INVALID, "Int4MatMul: negative sizes");
    if (const osh_status st = int4_check(n, k, group, dtype)) return st;
    *bytes = m && n ? int4_room(m, n, k, group, dtype).total : 0;
    return OSH_OK;
}

OSH_API osh_status osh_int4_matmul(int m, int n, int k, int group, int dtype, const void *d_a, int64_t lda,
                                   const void *d_packed, int has_zeros, const float *d_bias, int act,
                                   const void *d_res, int64_t ldr, void *d_y, int64_t ldy, void *d_scratch,
                                   osh_stream s) {
    if (m < 0) return fail(OSH_E_INVALID, "Int4MatMul: negative sizes");
    if (const osh_status st = int4_check(n, k, group, dtype)) return st;
    if (act != OSH_ACT_NONE && act != OSH_ACT_RELU && act != OSH_ACT_SILU && act != OSH_ACT_GELU)
        return fail(OSH_E_INVALID, "Int4MatMul: unknown activation %d", act);
    if (m == 0 || n == 0) return OSH_OK;
    if (!d_a || !d_packed || !d_y) return fail(OSH_E_INVALID, "Int4MatMul: NULL pointer");
    if (lda < k || ldy < n || (d_res && ldr < n)) return fail(OSH_E_INVALID, "Int4MatMul: a row pitch below the columns");
    if ((uintptr_t)d_packed & 15) return fail(OSH_E_INVALID, "Int4MatMul: packed weights need 16-byte alignment");
    if ((long long)cdiv(m, 64) * cdiv(n, 64) >= (1LL << 23) || m > 64 * 65535)
        return fail(OSH_E_UNSUPPORTED, "Int4MatMul: %d x %d outputs", m, n);
    const long long e = elem_bytes(dtype);
    const Int4Layout l = int4_layout(n, k, group, dtype, has_zeros);
    const Int4Room room = int4_room(m, n, k, group, dtype);
    if (room.total && (!d_scratch || ((uintptr_t)d_scratch & 15))) return fail(OSH_E_INVALID, "Int4MatMul: no scratch at 16-byte alignment");
    const Strided y = strided_rows(d_y, m, ldy * e, n * e), res = strided_rows(d_res, m, ldr * e, n * e);
    if (share_bytes(y, strided_rows(d_a, m, lda * e, k * e)) || share_bytes(y, Strided(d_packed, l.total)) ||
        share_bytes(y, Strided(d_bias, n * 4LL)) || (share_bytes(y, res) && !(d_y == d_res && ldy == ldr)))
        return fail(OSH_E_INVALID, "Int4MatMul: y overlaps an operand");
    const Strided own(d_scratch, room.total);
    if (share_bytes(own, y) || share_bytes(own, res) || share_bytes(own, strided_rows(d_a, m, lda * e, k * e)) ||
        share_bytes(own, Strided(d_packed, l.total)) || share_bytes(own, Strided(d_bias, n * 4LL)))
        return fail(OSH_E_INVALID, "Int4MatMul: the scratch overlaps an operand");
    Int4Args p;
    p.m = m;
    p.n = n;
    p.k = k;
    p.act = act;
    p.lda = lda;
    p.ldr = ldr;
    p.ldy = ldy;
    p.a = d_a;
    const char *base = static_cast<const char *>(d_packed);
    p.codes = reinterpret_cast<const uint4 *>(base);
    p.scales = base + l.codes;
    p.zeros = has_zeros ? base + l.codes + l.scales : nullptr;
    p.bias = d_bias;
    p.res = d_res;
    p.y = d_y;
    if (dtype == OSH_T_F32) return int4_launch_t<float>(p, group, room, d_scratch, to_stream(s));
    if (dtype == OSH_T_F16) return int4_launch_t<_Float16>(p, group, room, d_scratch, to_stream(s));
    return int4_launch_t<__bf16>(p, group, room, d_scratch, to_stream(s));
}

}  // extern "C"
