// osh_quant_matmul.hip -- product of 8-bit rows with its epilogue:
//
//   y[i][j] = act(sa[i] sw[j] sum_k a[i][k] w[j][k] + bias[j]) + res[i][j]
//
// with a [m][k] and w [n][k], k contiguous in both.  The weights are the MFMA's
// A operand and the activations its B operand, so a lane ends with four
// neighbouring outputs of one row.
//
// A k-block is 128 bytes of a row, eight chunks of 16.  Lane (l % 16, g = l / 16)
// holds chunks g and g + 4 of its row: int8 multiplies them with two
// v_mfma_i32_16x16x64_i8, e4m3 with one v_mfma_f32_16x16x128_f8f6f4.  Which k
// a byte stands for is the same for both operands, so the sum does not care that
// the hardware numbers a lane's bytes otherwise.
//
// The 8-bit float MFMA (the 32-deep one too) drops what its products have below about
// 2^-16 of an instruction's largest: 1.5e-5 of the result in the 2-norm, for k from 64
// to 16384 alike.  16-bit outputs round by 14 (f16) and 110 (bf16) times that and take
// it.  FP32 outputs take their operands to f16, which holds every e4m3 value (all 256
// codes checked, NaN among them), and v_mfma_f32_16x16x32_f16, whose sums are within
// FP32's roundings: 2.6e-8 at k = 512, 1.2e-7 at 8192.  It has half the rate, and the
// conversions run beside it: 8192 x 8192 x 4096 451 us (1.2 PFLOP/s; with the 8-bit
// instruction 252), 1028 x 5120 x 1280 23.3 (17.6), 24 x 8192 x 4096 10.1 (10.1).
#include <limits.h>

#include <algorithm>

#include "osh_lm.h"
#include "osh_overlap.h"

using namespace osh;

namespace osh {

struct QmmArgs {
    int m, n, k, act;
    long long lda, ldw, ldr, ldy;
    const unsigned char *a, *w;
    const float *sa, *sw, *bias;
    const void *res;
    void *y;
};

constexpr int KB = 128;  // bytes of a k-block

// What Q is in the kernels: an element type of the operands, or e4m3 multiplied in f16.
constexpr int Q_E4M3_AS_F16 = OSH_T_F16;

template <int Q> struct QAcc { using type = f32x4; };
template <> struct QAcc<OSH_T_I8> { using type = i32x4; };

struct Frag {
    i32x4 lo, hi;  // chunks g and g + 4 of a row's k-block
};
struct FragF16 {
    f16x8 v[4];  // the same, 8 bytes of them each
};

// A fragment as the MFMAs take it.
template <int Q> struct QOp { using type = Frag; };
template <> struct QOp<Q_E4M3_AS_F16> { using type = FragF16; };
template <int Q>
__device__ __forceinline__ typename QOp<Q>::type operand(const Frag &f) {
    if constexpr (Q == Q_E4M3_AS_F16) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        FragF16 o;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int word = (i < 2 ? f.lo : f.hi)[(2 * i & 3) + e / 2];
                const auto two = e & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.0f, true)
                                       : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.0f, false);
                const f16x2 v = __builtin_bit_cast(f16x2, two);
                o.v[i][2 * e] = v[0], o.v[i][2 * e + 1] = v[1];
            }
        return o;
    } else {
        return f;
    }
}

template <int Q>
__device__ __forceinline__ typename QAcc<Q>::type mma(const typename QOp<Q>::type &w, const typename QOp<Q>::type &a,
                                                      typename QAcc<Q>::type c) {
    if constexpr (Q == Q_E4M3_AS_F16) {
#pragma unroll
        for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[i], a.v[i], c, 0, 0, 0);
        return c;
    } else if constexpr (Q == OSH_T_I8) {
        c = __builtin_amdgcn_mfma_i32_16x16x64_i8(w.lo, a.lo, c, 0, 0, 0);
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(w.hi, a.hi, c, 0, 0, 0);
    } else {
        const i32x8 w8 = __builtin_shufflevector(w.lo, w.hi, 0, 1, 2, 3, 4, 5, 6, 7);
        const i32x8 a8 = __builtin_shufflevector(a.lo, a.hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, a8, c, 0, 0, 0, 0, 0, 0);
    }
}

// acc[i][j] += w a[i] over FM row fragments; int8 and f16 take a part of all rows
// first, so that no MFMA waits for the one before.
template <int Q, int FM, int FN>
__device__ __forceinline__ void mma_rows(const typename QOp<Q>::type &w, const typename QOp<Q>::type (&a)[FM],
                                         typename QAcc<Q>::type (&acc)[FM][FN], int j) {
    if constexpr (Q == Q_E4M3_AS_F16) {
#pragma unroll
        for (int h = 0; h < 4; h++)
#pragma unroll
            for (int i = 0; i < FM; i++)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[h], a[i].v[h], acc[i][j], 0, 0, 0);
    } else if constexpr (Q == OSH_T_I8) {
#pragma unroll
        for (int i = 0; i < FM; i++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w.lo, a[i].lo, acc[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < FM; i++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w.hi, a[i].hi, acc[i][j], 0, 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < FM; i++) acc[i][j] = mma<Q>(w, a[i], acc[i][j]);
    }
}

// 16 bytes of a row from byte k0, zero from byte k on.
__device__ __forceinline__ i32x4 load_chunk(const unsigned char *row, int k0, int k) {
    i32x4 v = {0, 0, 0, 0};
    if (k0 + 16 <= k) {
        __builtin_memcpy(&v, row + k0, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 15; i++)
            if (k0 + i < k) v[i >> 2] |= (int)row[k0 + i] << (8 * (i & 3));
    }
    return v;
}

// One output from its sum; scale, bias, activation and residual in FP32, one
// rounding to T.
template <typename T>
__device__ __forceinline__ T finish(const QmmArgs &p, float sum, int row, int col, float sa) {
    float v = sum * sa * p.sw[col];
    if (p.bias) v += p.bias[col];
    v = apply_act<sizeof(T) == 4>(p.act, v);
    if (p.res) v += (float)static_cast<const T *>(p.res)[row * p.ldr + col];
    return (T)v;
}

// The epilogue of a wave's FM x FN fragments, rows from row0 and outputs from col0:
// up to four fragments' rows at a time, scaled by row, go to the wave's own LDS, 16 *
// 4 rows of 16 FN sums, and come back eight neighbouring outputs a lane, so that
// residual and output move in 16-byte pieces and a lane's eight scales and biases
// are read once.  The residuals of four passes are loaded while the four before are
// computed (one pass at a time waited for memory 32 times a tile: 88 us of 355 for
// 8192 x 8192 x 4096).  `lds` holds EpiRows * EpiPitch<FN> floats.
constexpr int EpiRows = 64;
template <int FN> constexpr int EpiPitch = 16 * FN + 4;

template <int Q, typename T, int FM, int FN>
__device__ __forceinline__ void qmm_epilogue(const QmmArgs &p, const typename QAcc<Q>::type (&acc)[FM][FN], float *lds,
                                             int row0, int col0) {
    using V = typename Vec8<T>::type;
    constexpr int LPR = 2 * FN, RPP = 64 / LPR;  // lanes of a row, rows of a pass
    constexpr int GROUP = FM < EpiRows / 16 ? FM : EpiRows / 16;
    constexpr int PASSES = FM * 16 / RPP, GPASS = GROUP * 16 / RPP, BATCH = GPASS < 4 ? GPASS : 4;
    static_assert(GPASS % BATCH == 0, "a group is whole batches");
    const int lane = threadIdx.x & 63, jl = lane & 15, g = lane >> 4;
    const int c = lane % LPR * 8, col = col0 + c, cols = p.n - col;
    float sa[FM], sw[8], bias[8];
#pragma unroll
    for (int i = 0; i < FM; i++) sa[i] = p.sa[min(row0 + 16 * i + jl, p.m - 1)];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        sw[i] = i < cols ? p.sw[col + i] : 0.0f;
        bias[i] = i < cols && p.bias ? p.bias[col + i] : 0.0f;
    }
    V res[BATCH];
    auto load_res = [&](int pass) {
#pragma unroll
        for (int e = 0; e < BATCH; e++) {
            const int row = row0 + lane / LPR + (pass + e) * RPP;
            const T *from = static_cast<const T *>(p.res) + row * p.ldr + col;
            if (!p.res || row >= p.m) continue;
            if (cols >= 8) {
                __builtin_memcpy(&res[e], from, sizeof(V));
            } else {
#pragma unroll
                for (int i = 0; i < 7; i++)
                    if (i < cols) res[e][i] = from[i];
            }
        }
    };
#pragma unroll
    for (int e = 0; e < BATCH; e++) res[e] = V{};
    load_res(0);
#pragma unroll
    for (int i0 = 0; i0 < FM; i0 += GROUP) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < GROUP; i++)
#pragma unroll
            for (int j = 0; j < FN; j++) {
                const auto &v = acc[i0 + i][j];
                *reinterpret_cast<f32x4 *>(lds + (16 * i + jl) * EpiPitch<FN> + 16 * j + 4 * g) =
                    f32x4{(float)v[0] * sa[i0 + i], (float)v[1] * sa[i0 + i], (float)v[2] * sa[i0 + i],
                          (float)v[3] * sa[i0 + i]};
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
        for (int q = 0; q < GPASS; q += BATCH) {
            V add[BATCH];
            f32x8 v[BATCH];
#pragma unroll
            for (int e = 0; e < BATCH; e++) {
                add[e] = res[e];
                const f32x4 *from =
                    reinterpret_cast<const f32x4 *>(lds + (lane / LPR + (q + e) * RPP) * EpiPitch<FN> + c);
                const f32x4 v0 = from[0], v1 = from[1];
#pragma unroll
                for (int i = 0; i < 8; i++) v[e][i] = (i < 4 ? v0[i & 3] : v1[i & 3]) * sw[i] + bias[i];
            }
            const int pass = i0 * 16 / RPP + q;
            if (pass + BATCH < PASSES) load_res(pass + BATCH);
            if (p.act == OSH_ACT_GELU) {
#pragma unroll
                for (int e = 0; e < BATCH; e++) act8<OSH_ACT_GELU, sizeof(T) == 4>(v[e]);
            } else if (p.act == OSH_ACT_SILU) {
#pragma unroll
                for (int e = 0; e < BATCH; e++) act8<OSH_ACT_SILU, sizeof(T) == 4>(v[e]);
            } else if (p.act == OSH_ACT_RELU) {
#pragma unroll
                for (int e = 0; e < BATCH; e++) act8<OSH_ACT_RELU, sizeof(T) == 4>(v[e]);
            }
#pragma unroll
            for (int e = 0; e < BATCH; e++) {
                const int row = row0 + lane / LPR + (pass + e) * RPP;
                if (row >= p.m || cols <= 0) continue;
                T *y = static_cast<T *>(p.y) + row * p.ldy + col;
                if (p.res) v[e] += __builtin_convertvector(add[e], f32x8);
                if (cols >= 8) {
                    store8(y, v[e]);
                } else {
#pragma unroll
                    for (int i = 0; i < 7; i++)
                        if (i < cols) y[i] = (T)v[e][i];
                }
            }
        }
    }
}

// Tile (row, column) number id: columns of 8 row tiles one after another, so that
// the 32 tiles an XCD holds at a time share few rows and few weights.
__device__ __forceinline__ int2 qmm_tile_of(int id, int tm, int tn) {
    const int per = 8 * tn, band = id / per, first = band * 8;
    const int rows = min(8, tm - first), in = id - band * per;
    return int2{first + in % rows, in / rows};
}

// 16 bytes a lane from r at byte off + soff to LDS: lane i's to dst + 16 i.
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t r, unsigned char *dst, int off, int soff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)dst, 16, off, soff, 0, 0);
}

// Tile of BM rows by BN outputs, WM x WN waves; k-blocks pass through registers into two
// LDS buffers: operands at any address, and products with fewer tiles than CUs (8192 x 8191
// x 4097 e4m3 486 us, 215 at whole 16-byte chunks; 128 x 4096 x 4096 20.6).  Chunk c of tile row r lies at slot c ^ (r / 2 % 8) of the row's 128
// bytes: the 16 lanes of an operand read then meet all 64 banks once.
template <int Q, typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void qmm_tile_kernel(QmmArgs p) {
    constexpr int THREADS = 64 * WM * WN;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr int CH = (BM + BN) * 8 / THREADS;  // chunks a thread stages
    using Acc = typename QAcc<Q>::type;
    extern __shared__ __align__(16) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int jl = lane & 15, g = lane >> 4;
    const int tiles_m = cdiv(p.m, BM);
    const int id = xcd_band(blockIdx.x, gridDim.x);
    const int m0 = id % tiles_m * BM, n0 = id / tiles_m * BN;
    const int wm = wave % WM, wn = wave / WM;

    const unsigned char *src[CH];
    int dst[CH];
#pragma unroll
    for (int i = 0; i < CH; i++) {
        const int c = tid + THREADS * i, r = c >> 3;
        src[i] = r < BM ? p.a + (long long)min(m0 + r, p.m - 1) * p.lda
                        : p.w + (long long)min(n0 + r - BM, p.n - 1) * p.ldw;
        dst[i] = r * KB + (((c & 7) ^ (r >> 1 & 7)) << 4);
    }
    i32x4 st[CH];
    auto load = [&](int kb) {
#pragma unroll
        for (int i = 0; i < CH; i++) st[i] = load_chunk(src[i], kb * KB + (tid & 7) * 16, p.k);
    };
    auto store = [&](int buf) {
#pragma unroll
        for (int i = 0; i < CH; i++) *reinterpret_cast<i32x4 *>(lds + buf * (BM + BN) * KB + dst[i]) = st[i];
    };
    auto frag = [&](int buf, int r) {
        const unsigned char *row = lds + buf * (BM + BN) * KB + r * KB;
        Frag f;
        f.lo = *reinterpret_cast<const i32x4 *>(row + ((g ^ (r >> 1 & 7)) << 4));
        f.hi = *reinterpret_cast<const i32x4 *>(row + (((g + 4) ^ (r >> 1 & 7)) << 4));
        return operand<Q>(f);
    };

    Acc acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = Acc{0, 0, 0, 0};

    const int nkb = cdiv(p.k, KB);
    load(0);
    store(0);
    __syncthreads();
    for (int kb = 0; kb < nkb; kb++) {
        if (kb + 1 < nkb) load(kb + 1);
        typename QOp<Q>::type fa[FM];
#pragma unroll
        for (int i = 0; i < FM; i++) fa[i] = frag(kb & 1, wm * (BM / WM) + 16 * i + jl);
#pragma unroll
        for (int j = 0; j < FN; j++) {
            const auto fw = frag(kb & 1, BM + wn * (BN / WN) + 16 * j + jl);
#pragma unroll
            for (int i = 0; i < FM; i++) acc[i][j] = mma<Q>(fw, fa[i], acc[i][j]);
        }
        if (kb + 1 < nkb) store((kb + 1) & 1);
        __syncthreads();
    }

    qmm_epilogue<Q, T, FM, FN>(p, acc, reinterpret_cast<float *>(lds) + wave * EpiRows * EpiPitch<FN>,
                               m0 + wm * (BM / WM), n0 + wn * (BN / WN));
}

// Waits written by hand: the compiler does not tie LDS reads to the direct loads that
// fill it.  wait_lds_and_barrier leaves loads and stores of memory in flight.
__device__ __forceinline__ void wait_all() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void wait_all_and_barrier() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
__device__ __forceinline__ void wait_lds_and_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Outputs (or residuals) from element `first` on, and 8 of them at a byte offset.
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t out_rsrc(const void *base, long long first) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)(static_cast<const T *>(base) + first), (short)0, 0x7fffffff,
                                             0x00020000);
}
template <typename T>
__device__ __forceinline__ typename Vec8<T>::type buffer_load8(__amdgpu_buffer_rsrc_t r, int off, int soff) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    u32x4 w[sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) w[i] = __builtin_amdgcn_raw_buffer_load_b128(r, off + 16 * i, soff, 0);
    typename Vec8<T>::type v;
    __builtin_memcpy(&v, w, sizeof(v));
    return v;
}
// No scalar offset: the compiler keeps a vector instruction that reuses a data register
// apart from a 16-byte store only where the store has none.  Right behind stores that had
// one, lanes 12 to 15 of each 16 stored the register's next content now and then (up to
// 400 of 17 million values of a product).
template <typename T>
__device__ __forceinline__ void buffer_store8(typename Vec8<T>::type v, __amdgpu_buffer_rsrc_t r, int off) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    u32x4 w[sizeof(T) / 2];
    __builtin_memcpy(w, &v, sizeof(v));
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) __builtin_amdgcn_raw_buffer_store_b128(w[i], r, off + 16 * i, 0, 0);
}

// Large products: BM x BN tiles of 2 x WN waves, each (BM / 2) x (BN / WN), fed by
// direct loads from global memory to LDS, 16 bytes a lane, two k-blocks deep.
// (Rows at any 16-byte alignment; a k-block that k cuts short goes through
// registers, zeros from byte k on.)
//
// A wave keeps the k-block's FM fragments of its rows in registers and takes the
// FN fragments of the weights one after another, the next read a step ahead.
// Before the last step every wave has read the whole block: there the one barrier
// of a k-block stands, behind it the loads of the block after the next start into
// the buffer just freed, and the row fragments of the next block replace the
// present ones as the last MFMAs use them.
//
// A workgroup takes every gridDim-th tile.  The loads of a tile's first two blocks
// start in the last two steps of the tile before, and the epilogue, from registers
// to memory, needs no LDS, so it runs over them; its stores drain under the next
// tile's first block, whose barrier does not wait for them.
//
// 256 x 256 of eight waves: 8192 x 8192 x 4096 e4m3 215 us (2.56 PFLOP/s; a large
// library product reaches 2.65 here), 288 with a residual, whose 134 MB the CUs all
// want at their tiles' ends.  Bringing it to L2 ahead of the end cost 6 us instead.
// Four waves of 128 x 128 read a quarter less LDS, but their 256 accumulators left
// no register free and the spills cost more (275 us).
template <int Q, typename T, int ACT, int BM, int BN, int WN, bool FAST>
__global__ __launch_bounds__(128 * WN, 2) void qmm_dma_kernel(QmmArgs p) {
    constexpr int THREADS = 128 * WN, RPC = THREADS / 8;  // LDS rows of a staging pass
    constexpr int FM = BM / 32, FN = BN / WN / 16, CH = (BM + BN) / RPC, BUF = (BM + BN) * KB;
    using Acc = typename QAcc<Q>::type;
    using V = typename Vec8<T>::type;
    extern __shared__ __align__(16) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int jl = lane & 15, g = lane >> 4;
    const int tm = cdiv(p.m, BM), tn = cdiv(p.n, BN), tiles = tm * tn;
    const int wm = wave & 1, wn = wave >> 1;
    const int rm = wm * (BM / 2), rn = BM + wn * (BN / WN);
    const int nkb = cdiv(p.k, KB);

    // Opening a tile, its cut k-block and its epilogue start from a thread
    // number that the compiler cannot see through: kept across the k loop, what they
    // compute of it would be spilled, and each reload waits for all loads in flight.
    auto thread = [&] {
        int t = tid;
        asm volatile("" : "+v"(t));
        return t;
    };
    // The tile whose blocks are being loaded.  Chunk (tid & 7) of LDS row tid / 8 + RPC i
    // holds chunk (tid & 7) ^ (tid / 16 & 7) of its row.  A row past the end lies past
    // its buffer, whose loads are then not made; only the vector offset decides it.
    auto chunk = [](int t) { return ((t & 7) ^ (t >> 4 & 7)) * 16; };
    const int src_a = (tid >> 3) * (int)p.lda + chunk(tid), src_w = (tid >> 3) * (int)p.ldw + chunk(tid);
    int lm0, ln0;
    const unsigned char *a0, *w0;
    __amdgpu_buffer_rsrc_t ra, rw;
    auto open_tile = [&](int number) {
        const int2 t = qmm_tile_of(xcd_band(number, tiles), tm, tn);
        lm0 = t.x * BM, ln0 = t.y * BN;
        a0 = p.a + (long long)lm0 * p.lda, w0 = p.w + (long long)ln0 * p.ldw;
        ra = __builtin_amdgcn_make_buffer_rsrc((void *)a0, (short)0, min(p.m - 1 - lm0, BM) * (int)p.lda + p.k, 0x00020000);
        rw = __builtin_amdgcn_make_buffer_rsrc((void *)w0, (short)0, min(p.n - 1 - ln0, BN) * (int)p.ldw + p.k, 0x00020000);
    };
    auto stage1 = [&](int buf, int kb, int i) {  // RPC rows of a whole k-block
        unsigned char *dst = lds + buf * BUF + (RPC * i + wave * 8) * KB;
        if (i < BM / RPC) load_to_lds(ra, dst, src_a + RPC * i * (int)p.lda, kb * KB);
        else load_to_lds(rw, dst, src_w + (RPC * i - BM) * (int)p.ldw, kb * KB);
    };
    auto stage = [&](int buf, int kb) {
        if ((kb + 1) * KB <= p.k) {
#pragma unroll
            for (int i = 0; i < CH; i++) stage1(buf, kb, i);
        } else {
            const int t0 = thread();
#pragma unroll 1
            for (int r = t0 >> 3; r < BM + BN; r += RPC) {
                const unsigned char *row =
                    r < BM ? a0 + min(r, p.m - 1 - lm0) * p.lda : w0 + min(r - BM, p.n - 1 - ln0) * p.ldw;
                *reinterpret_cast<i32x4 *>(lds + buf * BUF + r * KB + (t0 & 7) * 16) =
                    load_chunk(row, kb * KB + chunk(t0), p.k);
            }
        }
    };
    const int sw = jl >> 1;  // fragment rows are jl plus multiples of 16
    const int lo = ((g ^ sw) << 4), hi = (((g + 4) ^ sw) << 4);
    auto frag = [&](int buf, int r) {
        const unsigned char *row = lds + buf * BUF + (r + jl) * KB;
        Frag f;
        f.lo = *reinterpret_cast<const i32x4 *>(row + lo);
        f.hi = *reinterpret_cast<const i32x4 *>(row + hi);
        return operand<Q>(f);
    };
    static_assert(FN % 2 == 0, "the last fragment is in fw[1]");

    int number = blockIdx.x, buf = 0;  // buf holds the present k-block
    open_tile(number);
    stage(0, 0);
    if (nkb > 1) stage(1, 1);
    wait_all_and_barrier();
#pragma unroll 1
    for (bool first = true;; first = false) {
        const int m0 = lm0, n0 = ln0, following = number + gridDim.x;
        const bool more = FAST && following < tiles;
        Acc acc[FM][FN];
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
            for (int j = 0; j < FN; j++) acc[i][j] = Acc{0, 0, 0, 0};
        typename QOp<Q>::type fa[FM], fw[2];
#pragma unroll
        for (int i = 0; i < FM; i++) fa[i] = frag(buf, rm + 16 * i);
        fw[0] = frag(buf, rn);
        // all steps of a k-block but the last one, and its barrier
        auto front = [&](bool wait) {
#pragma unroll
            for (int j = 0; j < FN - 1; j++) {
                fw[(j + 1) & 1] = frag(buf, rn + 16 * (j + 1));
                mma_rows<Q, FM>(fw[j & 1], fa, acc, j);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (wait) wait_all_and_barrier();
            else wait_lds_and_barrier();
        };
        int kb = 0;
        for (const int end = p.k / KB - 2; kb < end; kb++) {  // blocks kb + 2 that are whole
            front(kb > 0 || first);
            fw[0] = frag(buf ^ 1, rn);
#pragma unroll
            for (int i = 0; i < FM; i++) {
                acc[i][FN - 1] = mma<Q>(fw[1], fa[i], acc[i][FN - 1]);
                fa[i] = frag(buf ^ 1, rm + 16 * i);
#pragma unroll
                for (int e = i * CH / FM; e < (i + 1) * CH / FM; e++) stage1(buf, kb + 2, e);
                __builtin_amdgcn_sched_barrier(0);
            }
            buf ^= 1;
        }
#pragma unroll 1
        for (; kb < nkb; kb++) {
            front(true);
            mma_rows<Q, FM>(fw[1], fa, acc, FN - 1);
            int load = kb + 2;
            if (load >= nkb && more) {  // the following tile's first blocks
                if (load == nkb) open_tile(following);
                load -= nkb;
            }
            if (load < nkb) stage(buf, load);
            buf ^= 1;
            if (kb + 1 < nkb) {
                fw[0] = frag(buf, rn);
#pragma unroll
                for (int i = 0; i < FM; i++) fa[i] = frag(buf, rm + 16 * i);
            }
        }
        if constexpr (FAST) {
            // Fragments j and j + 1 at a time: exchanging the odd rows of 16 lanes of one
            // with the even rows of the other leaves a lane eight neighbouring outputs of
            // fragment j + (g & 1).  Rows and outputs past the end get an offset past the
            // buffer: loads return 0, stores are dropped, and with no branch around them
            // waits can count them.
            __builtin_amdgcn_sched_barrier(0);
            const int t0 = thread(), jl = t0 & 15, g = t0 >> 4 & 3;
            const int ec = n0 + rn - BM + 16 * (g & 1) + 8 * (g >> 1);  // of pair 0
            const __amdgpu_buffer_rsrc_t ry = out_rsrc<T>(p.y, m0 * p.ldy), rr = out_rsrc<T>(p.res, m0 * p.ldr);
            auto at = [&](int i, int jp, long long ld) {
                const int r = rm + jl;
                return m0 + r + 16 * i < p.m && ec + 32 * jp < p.n ? (r * (int)ld + ec) * (int)sizeof(T) : INT_MIN;
            };
            float sa[FM];
#pragma unroll
            for (int i = 0; i < FM; i++) sa[i] = p.sa[min(m0 + rm + 16 * i + jl, p.m - 1)];
            f32x8 esw, ebias = {0, 0, 0, 0, 0, 0, 0, 0};
            constexpr int UR = 8 / sizeof(T), UNITS = FM / UR;  // row fragments of a unit
            V eres[UR];
            auto fetch = [&](int jp, int u) {
                if (u == 0) {
                    const int col = min(ec + 32 * jp, p.n - 8);
                    esw = load8(p.sw + col);
                    if (p.bias) ebias = load8(p.bias + col);
                }
                if (p.res) {
#pragma unroll
                    for (int i = 0; i < UR; i++)
                        eres[i] = buffer_load8<T>(rr, at(UR * u + i, jp, p.ldr),
                                                  (16 * (UR * u + i) * (int)p.ldr + 32 * jp) * (int)sizeof(T));
                }
            };
            fetch(0, 0);
#pragma unroll
            for (int s = 0; s < FN / 2 * UNITS; s++) {
                const int jp = s / UNITS, u = s % UNITS;
                V out[UR];
#pragma unroll
                for (int i = 0; i < UR; i++) {
                    f32x8 v;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const auto x = __builtin_amdgcn_permlane16_swap(
                            __float_as_uint((float)acc[UR * u + i][2 * jp][r]),
                            __float_as_uint((float)acc[UR * u + i][2 * jp + 1][r]), false, false);
                        v[r] = __uint_as_float(x[0]), v[r + 4] = __uint_as_float(x[1]);
                    }
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = v[e] * sa[UR * u + i] * esw[e] + ebias[e];
                    act8<ACT, sizeof(T) == 4>(v);
                    if (p.res) v += __builtin_convertvector(eres[i], f32x8);
                    out[i] = __builtin_convertvector(v, V);
                    __builtin_amdgcn_sched_barrier(0);
                }
                // the following tile's second block is here before the first store
                if (s == 0) wait_all();
                if (s + 1 < FN / 2 * UNITS) fetch((s + 1) / UNITS, (s + 1) % UNITS);
#pragma unroll
                for (int i = 0; i < UR; i++)
                    buffer_store8<T>(out[i], ry, at(UR * u + i, jp, p.ldy) +
                                                     (16 * (UR * u + i) * (int)p.ldy + 32 * jp) * (int)sizeof(T));
                __builtin_amdgcn_sched_barrier(0);
            }
            if (!more) break;
            number = following;
        } else {
            __syncthreads();
            qmm_epilogue<Q, T, FM, FN>(p, acc, reinterpret_cast<float *>(lds) + wave * EpiRows * EpiPitch<FN>, m0 + rm,
                                       n0 + rn - BM);
            break;
        }
    }
}

// LDS of a tile kernel: its two buffers, or the epilogue of its waves.
template <int BM, int BN, int WM, int WN>
constexpr int qmm_lds() {
    constexpr int epi = WM * WN * EpiRows * EpiPitch<BN / WN / 16> * 4;
    return epi > 2 * (BM + BN) * KB ? epi : 2 * (BM + BN) * KB;
}

// Few rows: a workgroup takes 16 NB outputs of all rows (up to 16 MB), its waves
// every WAVES-th k-block; the weights go from memory to registers, each byte once.
// What bounds it is how many bytes are in flight: the loads of U k-blocks of a wave
// start together, without a condition around them (24 x 8192 x 4096 e4m3: 13.6 us a
// block at a time, 9.8 so, all of it on the device: the host's part of a call, 9, runs
// beside it).  The waves' sums meet in LDS, in the order of the waves.
template <int Q, typename T, int MB, int NB, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void qmm_rows_kernel(QmmArgs p) {
    using Acc = typename QAcc<Q>::type;
    constexpr int U = MB + NB > 4 ? 2 : 4;
    __shared__ Acc part[WAVES][MB * NB][64];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int jl = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * (16 * NB);
    const unsigned char *w[NB], *a[MB];
    Acc acc[MB][NB];
#pragma unroll
    for (int j = 0; j < NB; j++) w[j] = p.w + (long long)min(n0 + 16 * j + jl, p.n - 1) * p.ldw;
#pragma unroll
    for (int i = 0; i < MB; i++) {
        a[i] = p.a + (long long)min(16 * i + jl, p.m - 1) * p.lda;
#pragma unroll
        for (int j = 0; j < NB; j++) acc[i][j] = Acc{0, 0, 0, 0};
    }
    const int whole = p.k / KB, nkb = cdiv(p.k, KB);
    auto blocks = [&](int kb, auto count, auto cut) {
        constexpr int N = decltype(count)::value;
        Frag fw[N][NB], fa[N][MB];
#pragma unroll
        for (int u = 0; u < N; u++) {
            const int k0 = (kb + u * WAVES) * KB + 16 * g;
            auto get = [&](const unsigned char *row) {
                Frag f;
                if constexpr (decltype(cut)::value) {
                    f.lo = load_chunk(row, k0, p.k), f.hi = load_chunk(row, k0 + 64, p.k);
                } else {
                    __builtin_memcpy(&f.lo, row + k0, 16);
                    __builtin_memcpy(&f.hi, row + k0 + 64, 16);
                }
                return f;
            };
#pragma unroll
            for (int j = 0; j < NB; j++) fw[u][j] = get(w[j]);
#pragma unroll
            for (int i = 0; i < MB; i++) fa[u][i] = get(a[i]);
        }
        __builtin_amdgcn_sched_barrier(0);  // every load in flight before the first MFMA waits
#pragma unroll
        for (int u = 0; u < N; u++)
#pragma unroll
            for (int j = 0; j < NB; j++)
#pragma unroll
                for (int i = 0; i < MB; i++) acc[i][j] = mma<Q>(operand<Q>(fw[u][j]), operand<Q>(fa[u][i]), acc[i][j]);
    };
    int kb = wave;
    for (; kb + (U - 1) * WAVES < whole; kb += U * WAVES) blocks(kb, IntC<U>{}, IntC<0>{});
    if (U > 2 && kb + WAVES < whole) {
        blocks(kb, IntC<2>{}, IntC<0>{});
        kb += 2 * WAVES;
    }
    if (kb < whole) {
        blocks(kb, IntC<1>{}, IntC<0>{});
        kb += WAVES;
    }
    if (kb < nkb) blocks(kb, IntC<1>{}, IntC<1>{});
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int j = 0; j < NB; j++) part[wave][i * NB + j][lane] = acc[i][j];
    __syncthreads();
    for (int e = tid; e < MB * NB * 256; e += 64 * WAVES) {
        // neighbouring threads, neighbouring outputs
        const int c = e % (16 * NB), row = e / (16 * NB), col = n0 + c;
        const int f = row / 16 * NB + c / 16, from = row % 16 + 16 * (c / 4 % 4), r = c % 4;
        auto sum = part[0][f][from][r];
#pragma unroll
        for (int v = 1; v < WAVES; v++) sum += part[v][f][from][r];
        if (row < p.m && col < p.n)
            static_cast<T *>(p.y)[row * p.ldy + col] = finish<T>(p, (float)sum, row, col, p.sa[row]);
    }
}

template <int Q, typename T, int BM, int BN, int WN>
static void qmm_dma_launch(const QmmArgs &p, bool fast, hipStream_t st) {
    const int tiles = cdiv(p.m, BM) * cdiv(p.n, BN);
    if (!fast) {
        OSH_LAUNCH((qmm_dma_kernel<Q, T, 0, BM, BN, WN, false>), dim3((unsigned)tiles), dim3(128 * WN), (qmm_lds<BM, BN, 2, WN>()),
                   st, p);
        return;
    }
    const int grid = std::min(tiles, device_cus() * (BM * BN > 128 * 128 ? 1 : 2));
#define OSH_QMM_ACT(ACT)                                                                                             \
    case ACT:                                                                                                        \
        OSH_LAUNCH((qmm_dma_kernel<Q, T, ACT, BM, BN, WN, true>), dim3((unsigned)grid), dim3(128 * WN), 2 * (BM + BN) * KB, st, p); \
        break
    switch (p.act) {
        OSH_QMM_ACT(OSH_ACT_NONE);
        OSH_QMM_ACT(OSH_ACT_RELU);
        OSH_QMM_ACT(OSH_ACT_SILU);
        OSH_QMM_ACT(OSH_ACT_GELU);
    }
#undef OSH_QMM_ACT
}

template <int Q, typename T>
static osh_status qmm_launch(const QmmArgs &p, hipStream_t st) {
#define OSH_QMM_TILE(BM, BN, WM, WN)                                                                  \
    OSH_LAUNCH((qmm_tile_kernel<Q, T, BM, BN, WM, WN>), dim3((unsigned)(cdiv(p.m, BM) * cdiv(p.n, BN))), \
               dim3(64 * WM * WN), (qmm_lds<BM, BN, WM, WN>()), st, p)
    // direct loads: whole 16-byte chunks; offsets within a tile in 31 bits
    const bool aligned = (((uintptr_t)p.a | (uintptr_t)p.w | p.lda | p.ldw) & 15) == 0 && p.k > KB &&
                         std::max(p.lda, p.ldw) < (1 << 21);
    const int e = 16 / sizeof(T);
    const bool fast = aligned && p.n % 8 == 0 && (((uintptr_t)p.y | (uintptr_t)p.res) & 15) == 0 && p.ldy % e == 0 &&
                      p.ldr % e == 0 && std::max(p.ldy, p.ldr) < (1 << 20);
    // f16 fragments are twice as long: those of a 256 x 256 tile and its accumulators take
    // more registers than a wave has
    constexpr int LARGE = Q == Q_E4M3_AS_F16 ? 128 : 256;
    const bool large = aligned && (long long)cdiv(p.m, LARGE) * cdiv(p.n, LARGE) >= device_cus();
    const bool pairs = p.n >= 32 * device_cus();  // enough workgroups of 32 outputs
#define OSH_QMM_ROWS(MB)                                                                                             \
    do {                                                                                                             \
        if (pairs)                                                                                                   \
            OSH_LAUNCH((qmm_rows_kernel<Q, T, MB, 2, 8>), dim3((unsigned)cdiv(p.n, 32)), dim3(512), 0, st, p);       \
        else                                                                                                         \
            OSH_LAUNCH((qmm_rows_kernel<Q, T, MB, 1, 8>), dim3((unsigned)cdiv(p.n, 16)), dim3(512), 0, st, p);       \
    } while (0)
    if (p.m <= 16) OSH_QMM_ROWS(1);
    else if (p.m <= 32) OSH_QMM_ROWS(2);
    else if (p.m <= 64) OSH_QMM_ROWS(4);
    else if (large)
        qmm_dma_launch<Q, T, LARGE, LARGE, LARGE / 64>(p, fast, st);
    else if (aligned && (long long)cdiv(p.m, 128) * cdiv(p.n, 128) >= device_cus())
        qmm_dma_launch<Q, T, 128, 128, 2>(p, fast, st);
    else if ((long long)cdiv(p.m, 128) * cdiv(p.n, 128) >= device_cus())
        OSH_QMM_TILE(128, 128, 2, 2);
    else
        OSH_QMM_TILE(64, 64, 2, 2);
#undef OSH_QMM_TILE
#undef OSH_QMM_ROWS
    OSH_LAUNCH_CHECK("qmm kernel");
    return OSH_OK;
}

template <int Q>
static osh_status qmm_launch_t(const QmmArgs &p, int dtype, hipStream_t st) {
    if (dtype == OSH_T_F32) return qmm_launch<Q == OSH_T_E4M3 ? Q_E4M3_AS_F16 : Q, float>(p, st);
    if (dtype == OSH_T_F16) return qmm_launch<Q, _Float16>(p, st);
    return qmm_launch<Q, __bf16>(p, st);
}

}  // namespace osh

extern "C" {

OSH_API osh_status osh_quant_matmul(int m, int n, int k, int q_type, const void *d_a, int64_t lda, const float *d_sa,
                                    const void *d_w, int64_t ldw, const float *d_sw, const float *d_bias, int act,
                                    int dtype, const void *d_res, int64_t ldr, void *d_y, int64_t ldy, osh_stream s) {
    if (m < 0 || n < 0 || k < 0) return fail(OSH_E_INVALID, "QuantMatMul: negative sizes");
    if (q_type != OSH_T_I8 && q_type != OSH_T_E4M3) return fail(OSH_E_INVALID, "QuantMatMul: operands are i8 or e4m3");
    if (dtype != OSH_T_F32 && dtype != OSH_T_F16 && dtype != OSH_T_BF16)
        return fail(OSH_E_INVALID, "QuantMatMul: outputs are f32, f16 or bf16");
    if (act != OSH_ACT_NONE && act != OSH_ACT_RELU && act != OSH_ACT_SILU && act != OSH_ACT_GELU)
        return fail(OSH_E_INVALID, "QuantMatMul: unknown activation %d", act);
    if (m == 0 || n == 0) return OSH_OK;
    if (k == 0) return fail(OSH_E_INVALID, "QuantMatMul: k is 0");
    // 131071 products of -128 and -128 stay below 2^31
    if (q_type == OSH_T_I8 && k > 131071) return fail(OSH_E_UNSUPPORTED, "QuantMatMul: k = %d above 131071", k);
    if (k > (1 << 30)) return fail(OSH_E_UNSUPPORTED, "QuantMatMul: k = %d too long", k);
    if (!d_a || !d_sa || !d_w || !d_sw || !d_y) return fail(OSH_E_INVALID, "QuantMatMul: NULL pointer");
    if (lda < k || ldw < k || ldy < n || (d_res && ldr < n))
        return fail(OSH_E_INVALID, "QuantMatMul: a row pitch below the columns");
    if ((long long)cdiv(m, 64) * cdiv(n, 64) >= (1LL << 23))
        return fail(OSH_E_UNSUPPORTED, "QuantMatMul: %d x %d outputs", m, n);
    const long long e = elem_bytes(dtype);
    const Strided y = strided_rows(d_y, m, ldy * e, n * e), res = strided_rows(d_res, m, ldr * e, n * e);
    if (share_bytes(y, strided_rows(d_a, m, lda, k)) || share_bytes(y, strided_rows(d_w, n, ldw, k)) ||
        share_bytes(y, Strided(d_sa, m * 4LL)) || share_bytes(y, Strided(d_sw, n * 4LL)) ||
        share_bytes(y, Strided(d_bias, n * 4LL)) || (share_bytes(y, res) && !(d_y == d_res && ldy == ldr)))
        return fail(OSH_E_INVALID, "QuantMatMul: y overlaps an operand");
    QmmArgs p;
    p.m = m;
    p.n = n;
    p.k = k;
    p.act = act;
    p.lda = lda;
    p.ldw = ldw;
    p.ldr = ldr;
    p.ldy = ldy;
    p.a = static_cast<const unsigned char *>(d_a);
    p.w = static_cast<const unsigned char *>(d_w);
    p.sa = d_sa;
    p.sw = d_sw;
    p.bias = d_bias;
    p.res = d_res;
    p.y = d_y;
    return q_type == OSH_T_I8 ? qmm_launch_t<OSH_T_I8>(p, dtype, to_stream(s))
                              : qmm_launch_t<OSH_T_E4M3>(p, dtype, to_stream(s));
}

}  // extern "C"
