// A matrix product with bias, activation and residual in its epilogue, and its backward pass:
//
//   z = x w^T + b,   y = act(z) + r          x [m x k], w [n x k], b [n], r, z, y [m x n]
//   dz = dy act'(z),   dx = dz w,   dw = dz^T x,   db = column sums of dz        (dr is dy)
//
// in float32, float16 or bfloat16, accumulated in float32 on the matrix cores.  Next to the cosine GEMMs of skm_dense.hip
// (int8 counts with a row-norm epilogue, float64): this one multiplies feature rows by learned weights.  No reference
// counterpart in this form (the reference hands its feature matrices to scikit-learn's estimators, snekmer/model.py).
//
// One kernel computes every product as C[i][j] = sum over c of A[i][c] B[j][c] with both operands contiguous along the
// contraction: x and w are; for the backward pass the operands that are not (w, dz and x read across their rows) are
// transposed once into scratch, as are operands whose rows do not start on 16-byte boundaries (copied with padding).
#include <algorithm>
#include <type_traits>

#include "skm_common.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct __attribute__((packed)) ln_u128 {  // 16 bytes at any address
    uint32_t w[4];
};

// ---- element types
template <int DT>
struct ln_type;
template <>
struct ln_type<0> {
    using T = float;
    using V = f32x4;  // 16 bytes of an operand row
    static constexpr int VE = 4;
    // the two lane halves hold columns 0-3 and 4-7 of a 32-byte step: the i-th product takes columns i and 4 + i of both
    static __device__ __forceinline__ f32x16 mfma(V a, V b, f32x16 c)
    {
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[0], b[0], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[1], b[1], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[2], b[2], c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x2f32(a[3], b[3], c, 0, 0, 0);
    }
};
template <>
struct ln_type<1> {
    using T = _Float16;
    using V = f16x8;
    static constexpr int VE = 8;
    static __device__ __forceinline__ f32x16 mfma(V a, V b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct ln_type<2> {
    using T = __bf16;
    using V = bf16x8;
    static constexpr int VE = 8;
    static __device__ __forceinline__ f32x16 mfma(V a, V b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

// ---- activations (float32)
enum { ACT_NONE = 0, ACT_RELU, ACT_GELU, ACT_GELU_TANH, ACT_SILU, ACT_SIGMOID, ACT_COUNT };

__device__ __forceinline__ float ln_sigmoid(float z) { return 1.0f / (1.0f + __expf(-z)); }  // (exp overflows to inf for z < -88: 0, as it should be)

__device__ __forceinline__ float ln_act(int act, float z)
{
    switch (act) {
    case ACT_RELU:
        return z < 0.0f ? 0.0f : z;  // (NaN stays)
    case ACT_GELU:
        return 0.5f * z * (1.0f + erff(z * 0.707106781186547524f));
    case ACT_GELU_TANH: {
        // 0.5 z (1 + tanh u) = z sigmoid(2 u)
        const float u = 0.797884560802865356f * (z + 0.044715f * z * z * z);
        return z * ln_sigmoid(2.0f * u);
    }
    case ACT_SILU:
        return z * ln_sigmoid(z);
    case ACT_SIGMOID:
        return ln_sigmoid(z);
    default:
        return z;
    }
}

__device__ __forceinline__ float ln_slope(int act, float z)
{
    switch (act) {
    case ACT_RELU:
        return z > 0.0f ? 1.0f : z == z ? 0.0f : z;
    case ACT_GELU:
        return 0.5f * (1.0f + erff(z * 0.707106781186547524f)) + z * __expf(-0.5f * z * z) * 0.398942280401432678f;
    case ACT_GELU_TANH: {
        const float u2 = 1.59576912160573071f * (z + 0.044715f * z * z * z), s = ln_sigmoid(u2);
        return s + z * s * (1.0f - s) * 1.59576912160573071f * (1.0f + 0.134145f * z * z);
    }
    case ACT_SILU: {
        const float s = ln_sigmoid(z);
        return s * (1.0f + z * (1.0f - s));
    }
    case ACT_SIGMOID: {
        const float s = ln_sigmoid(z);
        return s * (1.0f - s);
    }
    default:
        return 1.0f;
    }
}

// ---- the product
struct ln_gemm {
    int64_t m, n, k;            // C [m x n], contraction k
    const uint8_t *a, *b;       // 16-byte aligned rows
    int64_t lda, ldb;           // bytes
    int act;
    const void *bias;           // n values or nullptr
    const void *residual;       // nullptr or [m x n], row stride ldr
    int64_t ldr;
    void *preact;               // nullptr or [m x n], row stride ldp
    int64_t ldp;
    void *out;
    int64_t ldo;                // elements
    float *partial;             // split contraction: [nsplit][m][n] float32, rows of ldq (n rounded up to 4)
    int64_t ldq;
    int nsplit;
    int64_t stages_per_split;
};

__device__ const uint4 ln_zero_block = {0, 0, 0, 0};  // what lanes past the end of the contraction fetch

// bias, activation and residual of VE consecutive cells of one row, and the stores
template <int DT, int VE>
__device__ __forceinline__ void ln_finish(const ln_gemm &g, int64_t i, int64_t j, float (&v)[VE])
{
    using T = typename ln_type<DT>::T;
    const bool whole = j + VE <= g.n;
    T *out = (T *)g.out + i * g.ldo + j;
    if (g.bias) {
        const T *bias = (const T *)g.bias + j;
#pragma unroll
        for (int u = 0; u < VE; ++u)
            if (whole || j + u < g.n)
                v[u] += (float)bias[u];
    }
    auto put = [&](T *to) {
        T o[VE];
#pragma unroll
        for (int u = 0; u < VE; ++u)
            o[u] = (T)v[u];
        if (whole) {
            ln_u128 raw;
            __builtin_memcpy(&raw, o, 16);
            *reinterpret_cast<ln_u128 *>(to) = raw;
        } else {
#pragma unroll
            for (int u = 0; u < VE; ++u)
                if (j + u < g.n)
                    to[u] = o[u];
        }
    };
    if (g.preact)
        put((T *)g.preact + i * g.ldp + j);
    if (g.act != ACT_NONE)
#pragma unroll
        for (int u = 0; u < VE; ++u)
            v[u] = ln_act(g.act, v[u]);
    if (g.residual) {
        const T *res = (const T *)g.residual + i * g.ldr + j;
        if (whole) {
            const ln_u128 raw = *reinterpret_cast<const ln_u128 *>(res);
            T r[VE];
            __builtin_memcpy(r, &raw, 16);
#pragma unroll
            for (int u = 0; u < VE; ++u)
                v[u] += (float)r[u];
        } else {
#pragma unroll
            for (int u = 0; u < VE; ++u)
                if (j + u < g.n)
                    v[u] += (float)res[u];
        }
    }
    put(out);
}

constexpr int LN_BK = 128;  // bytes of contraction per stage: one 128-byte line of every operand row

// Tiles of BM x BN, WM x WN waves of (BM / WM) x (BN / WN).  Operands go to LDS directly (16 bytes a lane, 8 rows of 128
// bytes an instruction), two stages: stage s + 1 is in flight while stage s is multiplied, one barrier a stage.  The
// 16-byte chunk index of a row is XORed with (row >> 1) & 7 on the source address and on the fragment reads, so that the
// 32 rows of a fragment read spread over the banks.
template <int DT, int BM, int BN, int WM, int WN, bool SPLIT>
__global__ __launch_bounds__(WM *WN * 64) void k_linear(ln_gemm g)
{
    using P = ln_type<DT>;
    using V = typename P::V;
    constexpr int NWAVE = WM * WN, TM = BM / WM, TN = BN / WN, FM = TM / 32, FN = TN / 32;
    constexpr int STAGE = (BM + BN) * LN_BK, PER_WAVE = (BM + BN) / 8 / NWAVE;
    constexpr int TROW = TN + 4;  // floats of a buffered output row: 16-byte aligned, spread over the banks
    static_assert((BM + BN) % (8 * NWAVE) == 0 && TM % 32 == 0 && TN % 32 == 0, "tile");
    static_assert(NWAVE * 32 * TROW * 4 <= 2 * STAGE, "the epilogue reuses the stages' memory");
    __shared__ __attribute__((aligned(16))) uint8_t s_t[2 * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);

    // tile of this workgroup: consecutive workgroups go to the eight XCDs in turn, so that each XCD gets a contiguous run
    // of the tile order, which walks groups of 8 tile rows column by column (their operands stay in the XCD's L2)
    const int64_t nty = (g.m + BM - 1) / BM, ntx = (g.n + BN - 1) / BN, tiles = nty * ntx;
    const int64_t bid = blockIdx.x, nwg = gridDim.x, q8 = nwg / 8, r8 = nwg % 8, xcd = bid % 8;
    const int64_t seq = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + bid / 8;
    const int64_t tile = SPLIT ? seq % tiles : seq;
    const int split = SPLIT ? (int)(seq / tiles) : 0;
    const int64_t group = tile / (8 * ntx), first = group * 8, rows_in = min((int64_t)8, nty - first), in_group = tile - group * 8 * ntx;
    const int64_t row0 = (first + in_group % rows_in) * BM, col0 = in_group / rows_in * BN;

    const int64_t kbytes = g.k * (int64_t)sizeof(typename P::T);
    const int64_t nst_all = (kbytes + LN_BK - 1) / LN_BK;
    const int64_t s_lo = SPLIT ? split * g.stages_per_split : 0, s_hi = SPLIT ? min(nst_all, s_lo + g.stages_per_split) : nst_all;

    // staging: instruction q of wave w lands rows [8 (w PER_WAVE + q), + 8) of the stage (A's rows first, then B's)
    const int srow = lane >> 3, schunk = lane & 7;
    const uint8_t *src[PER_WAVE];
    int skb[PER_WAVE];
#pragma unroll
    for (int q = 0; q < PER_WAVE; ++q) {
        const int r = (wid * PER_WAVE + q) * 8 + srow;
        const bool is_a = (wid * PER_WAVE + q) * 8 < BM;
        const int64_t at = is_a ? min(row0 + r, g.m - 1) : min(col0 + (r - BM), g.n - 1);  // rows past the end: any, not stored
        skb[q] = (schunk ^ ((r >> 1) & 7)) * 16;
        src[q] = (is_a ? g.a + at * g.lda : g.b + at * g.ldb) + skb[q];
    }
    auto stage = [&](int64_t s) {
        uint8_t *to = s_t + (int)(s & 1) * STAGE + wid * PER_WAVE * 8 * LN_BK;
        const int64_t k0 = s * LN_BK;
        const bool whole = k0 + LN_BK <= kbytes;
#pragma unroll
        for (int q = 0; q < PER_WAVE; ++q) {
            const uint8_t *p = src[q] + k0;
            if (!whole && k0 + skb[q] >= kbytes)
                p = reinterpret_cast<const uint8_t *>(&ln_zero_block);
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)p, (__attribute__((address_space(3))) void *)(to + q * 8 * LN_BK), 16, 0, 0);
        }
    };

    f32x16 acc[FM][FN];
#pragma unroll
    for (int a = 0; a < FM; ++a)
#pragma unroll
        for (int b = 0; b < FN; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                acc[a][b][r] = 0.0f;

    const int fr = lane & 31, fh = lane >> 5, wr = wid / WN, wc = wid % WN;
    if (s_lo < s_hi)
        stage(s_lo);
    for (int64_t s = s_lo; s < s_hi; ++s) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's part of stage s has landed
        __builtin_amdgcn_s_barrier();                     // everybody's has, and everybody has read stage s - 1
        asm volatile("" ::: "memory");
        if (s + 1 < s_hi)
            stage(s + 1);
        const uint8_t *sa = s_t + (int)(s & 1) * STAGE, *sb = sa + BM * LN_BK;
#pragma unroll
        for (int ks = 0; ks < LN_BK / 32; ++ks) {
            V fa[FM], fb[FN];
#pragma unroll
            for (int t = 0; t < FM; ++t) {
                const int r = wr * TM + t * 32 + fr;
                fa[t] = *reinterpret_cast<const V *>(sa + r * LN_BK + (((ks * 2 + fh) ^ ((r >> 1) & 7)) * 16));
            }
#pragma unroll
            for (int t = 0; t < FN; ++t) {
                const int r = wc * TN + t * 32 + fr;  // (BM is a multiple of 16: the XOR of row BM + r is that of r)
                fb[t] = *reinterpret_cast<const V *>(sb + r * LN_BK + (((ks * 2 + fh) ^ ((r >> 1) & 7)) * 16));
            }
#pragma unroll
            for (int a = 0; a < FM; ++a)
#pragma unroll
                for (int b = 0; b < FN; ++b)
                    acc[a][b] = P::mfma(fa[a], fb[b], acc[a][b]);
        }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __syncthreads();  // the stages have been read: their memory buffers the output

    // A lane holds one column of a 32 x 32 sub-tile (register 4 q + u: row 8 q + 4 (lane / 32) + u).  32 rows at a time go
    // through LDS (this wave's own part) and leave as 16-byte pieces of rows.
    float *buf = reinterpret_cast<float *>(s_t) + wid * 32 * TROW;
#pragma unroll
    for (int a = 0; a < FM; ++a) {
#pragma unroll
        for (int b = 0; b < FN; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                buf[(8 * (r >> 2) + 4 * fh + (r & 3)) * TROW + b * 32 + fr] = acc[a][b][r];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        constexpr int VE = SPLIT ? 4 : P::VE, PIECES = TN / VE, ROWS = 64 / PIECES;
        const int pr = lane / PIECES, pc = lane % PIECES * VE;
        const int64_t j = col0 + wc * TN + pc;
#pragma unroll 1  // (the six activations' code once per 32 rows)
        for (int p = 0; p < 32 / ROWS; ++p) {
            const int64_t i = row0 + wr * TM + a * 32 + p * ROWS + pr;
            float v[VE];
#pragma unroll
            for (int u = 0; u < VE; ++u)
                v[u] = buf[(p * ROWS + pr) * TROW + pc + u];
            if (i < g.m && j < g.n) {
                if constexpr (SPLIT) {
                    *reinterpret_cast<float4 *>(g.partial + ((int64_t)split * g.m + i) * g.ldq + j) = make_float4(v[0], v[1], v[2], v[3]);
                } else {
                    ln_finish<DT, VE>(g, i, j, v);
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// the sums over the splits, in order, and the epilogue
template <int DT>
__global__ __launch_bounds__(256) void k_linear_join(ln_gemm g)
{
    constexpr int VE = ln_type<DT>::VE;
    const int64_t per_row = (g.n + VE - 1) / VE, total = g.m * per_row;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
        const int64_t i = t / per_row, j = (t - i * per_row) * VE;
        float v[VE];
#pragma unroll
        for (int u = 0; u < VE; ++u)
            v[u] = 0.0f;
        for (int s = 0; s < g.nsplit; ++s) {
            const float *from = g.partial + ((int64_t)s * g.m + i) * g.ldq + j;
#pragma unroll
            for (int u = 0; u < VE; u += 4) {
                if (j + u < g.ldq) {
                    const float4 f = *reinterpret_cast<const float4 *>(from + u);
                    v[u] += f.x;
                    v[u + 1] += f.y;
                    v[u + 2] += f.z;
                    v[u + 3] += f.w;
                }
            }
        }
        ln_finish<DT, VE>(g, i, j, v);
    }
}

// ---- operands that have to be laid out anew
// out[r][c] = in[r][c], rows of ldo elements (a multiple of 16 bytes), zeros behind column `cols`
template <int DT>
__global__ __launch_bounds__(256) void k_linear_pad(int64_t rows, int64_t cols, const void *in_, int64_t ld, void *out_, int64_t ldo)
{
    using T = typename ln_type<DT>::T;
    constexpr int VE = ln_type<DT>::VE;
    const T *in = (const T *)in_;
    T *out = (T *)out_;
    const int64_t per_row = ldo / VE, total = rows * per_row;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
        const int64_t i = t / per_row, j = (t - i * per_row) * VE;
        const T *from = in + i * ld + j;
        ln_u128 raw;
        if (j + VE <= cols) {
            raw = *reinterpret_cast<const ln_u128 *>(from);
        } else {
            T v[VE];
#pragma unroll
            for (int u = 0; u < VE; ++u)
                v[u] = j + u < cols ? from[u] : (T)0.0f;
            __builtin_memcpy(&raw, v, 16);
        }
        *reinterpret_cast<uint4 *>(out + t * VE) = *reinterpret_cast<uint4 *>(&raw);
    }
}

// Tiles of 64 x 64 through LDS: outt[c][r] = in[r][c], rows of outt are ldt elements (a multiple of 16 bytes; zeros behind
// row `rows`).  GRAD: in is dy and the value is dz = dy act'(z), rounded to the operands' type once (what the two products
// of the backward pass read); then also out[r][c] = dz (row stride ldo, zeros behind `cols`; nullptr: not wanted) and
// sums[tile row][c] = this tile's column sums of the unrounded dz.
template <int DT, bool GRAD>
__global__ __launch_bounds__(256) void k_linear_transpose(int64_t rows, int64_t cols, const void *in_, int64_t ld, void *outt_, int64_t ldt, int act, const void *z_,
                                                          int64_t ldz, void *out_, int64_t ldo, float *sums)
{
    using T = typename ln_type<DT>::T;
    constexpr int VE = ln_type<DT>::VE, PIECES = 64 / VE, STEP = 256 / PIECES;  // rows a pass
    __shared__ T s_v[64][64 + 16 / sizeof(T) / 2];
    __shared__ float s_sum[GRAD ? 4 : 1][64];
    const T *in = (const T *)in_, *z = (const T *)z_;
    T *outt = (T *)outt_, *out = (T *)out_;
    const int tid = threadIdx.x, pr = tid / PIECES, pc = tid % PIECES * VE;
    const int64_t ntx = (cols + 63) / 64, nty = (rows + 63) / 64, tiles = ntx * nty;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t r0 = tile / ntx * 64, c0 = tile % ntx * 64, c = c0 + pc;
        float sum[VE];
#pragma unroll
        for (int u = 0; u < VE; ++u)
            sum[u] = 0.0f;
#pragma unroll
        for (int p = 0; p < 64 / STEP; ++p) {
            const int rr = p * STEP + pr;
            const int64_t r = r0 + rr;
            T v[VE];
            if (r < rows && c + VE <= cols) {
                const ln_u128 raw = *reinterpret_cast<const ln_u128 *>(in + r * ld + c);
                __builtin_memcpy(v, &raw, 16);
            } else {
#pragma unroll
                for (int u = 0; u < VE; ++u)
                    v[u] = r < rows && c + u < cols ? in[r * ld + c + u] : (T)0.0f;
            }
            if (GRAD) {
                if (act != ACT_NONE) {
                    T zz[VE];
                    if (r < rows && c + VE <= cols) {
                        const ln_u128 raw = *reinterpret_cast<const ln_u128 *>(z + r * ldz + c);
                        __builtin_memcpy(zz, &raw, 16);
                    } else {
#pragma unroll
                        for (int u = 0; u < VE; ++u)
                            zz[u] = r < rows && c + u < cols ? z[r * ldz + c + u] : (T)0.0f;
                    }
#pragma unroll
                    for (int u = 0; u < VE; ++u) {
                        const float d = r < rows && c + u < cols ? (float)v[u] * ln_slope(act, (float)zz[u]) : 0.0f;
                        sum[u] += d;
                        v[u] = (T)d;
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < VE; ++u)
                        sum[u] += (float)v[u];
                }
                if (out && r < rows && c < ldo)
                    __builtin_memcpy(out + r * ldo + c, v, 16);
            }
#pragma unroll
            for (int u = 0; u < VE; ++u)
                s_v[rr][pc + u] = v[u];
        }
        if (GRAD && sums) {  // over the rows that the lanes of a wave hold, then over the waves
#pragma unroll
            for (int u = 0; u < VE; ++u) {
                for (int d = PIECES; d < 64; d <<= 1)
                    sum[u] += __shfl_xor(sum[u], d);
                if ((tid & 63) < PIECES)
                    s_sum[tid >> 6][pc + u] = sum[u];
            }
        }
        __syncthreads();
        if (outt) {
#pragma unroll
            for (int p = 0; p < 64 / STEP; ++p) {
                const int cc = p * STEP + pr;
                if (c0 + cc < cols && r0 + pc < ldt) {
                    T v[VE];
#pragma unroll
                    for (int u = 0; u < VE; ++u)
                        v[u] = s_v[pc + u][cc];
                    __builtin_memcpy(outt + (c0 + cc) * ldt + r0 + pc, v, 16);
                }
            }
        }
        if (GRAD && sums && tid < 64 && c0 + tid < cols)
            sums[tile / ntx * cols + c0 + tid] = s_sum[0][tid] + s_sum[1][tid] + s_sum[2][tid] + s_sum[3][tid];
        __syncthreads();
    }
}

// dbias[c] = the tiles' column sums added up: a wave per 64 columns and quarter of the tiles
template <int DT>
__global__ __launch_bounds__(256) void k_linear_bias_grad(int64_t parts, int64_t cols, const float *sums, void *out_)
{
    using T = typename ln_type<DT>::T;
    __shared__ float s_sum[4][64];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    for (int64_t c0 = (int64_t)blockIdx.x * 64; c0 < cols; c0 += (int64_t)gridDim.x * 64) {
        float v = 0.0f;
        if (c0 + lane < cols)
            for (int64_t p = wid; p < parts; p += 4)
                v += sums[p * cols + c0 + lane];
        s_sum[wid][lane] = v;
        __syncthreads();
        if (wid == 0 && c0 + lane < cols)
            ((T *)out_)[c0 + lane] = (T)(s_sum[0][lane] + s_sum[1][lane] + s_sum[2][lane] + s_sum[3][lane]);
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------- host side
constexpr size_t elem_bytes(int dtype) { return dtype == 0 ? 4 : 2; }

template <int DT, int BM, int BN, int WM, int WN>
int launch_tiles(skm_ctx *ctx, const ln_gemm &g)
{
    const int64_t tiles = skm_ceil_div(g.m, BM) * skm_ceil_div(g.n, BN);
    SKM_REQUIRE(tiles * g.nsplit < ((int64_t)1 << 31), SKM_E_OVERFLOW, "skm_linear: too many tiles");
    if (g.nsplit > 1)
        k_linear<DT, BM, BN, WM, WN, true><<<(unsigned)(tiles * g.nsplit), WM * WN * 64, 0, ctx->stream>>>(g);
    else
        k_linear<DT, BM, BN, WM, WN, false><<<(unsigned)tiles, WM * WN * 64, 0, ctx->stream>>>(g);
    return skm_check_launch("k_linear");
}

// C = A B^T with the epilogue; a and b are ready (16-byte rows).
template <int DT>
int gemm(skm_ctx *ctx, ln_gemm g)
{
    const int64_t stages = skm_ceil_div(g.k * (int64_t)elem_bytes(DT), LN_BK);
    const int64_t big = skm_ceil_div(g.m, 256) * skm_ceil_div(g.n, 256), small = skm_ceil_div(g.m, 128) * skm_ceil_div(g.n, 128);
    const int64_t cus = ctx->usable_cus;
    g.nsplit = 1;
    g.stages_per_split = stages;
    const bool large = big >= cus;
    const int64_t tiles = large ? big : small;
    if (tiles < cus) {
        int64_t s = std::min<int64_t>(skm_ceil_div(cus * 2, tiles), stages / 4);
        s = std::min<int64_t>(s, 64);
        if (s > 1) {
            g.stages_per_split = skm_ceil_div(stages, s);
            g.nsplit = (int)skm_ceil_div(stages, g.stages_per_split);
        }
    }
    if (g.nsplit > 1) {
        void *p;
        g.ldq = skm_ceil_div(g.n, 4) * 4;
        SKM_TRY(skm_ws(ctx, WS_D, sizeof(float) * (size_t)g.nsplit * (size_t)g.m * (size_t)g.ldq, &p));
        g.partial = (float *)p;
    }
    {
        SKM_PROF(ctx, "k_linear");
        if (large)
            SKM_TRY((launch_tiles<DT, 256, 256, 2, 4>(ctx, g)));
        else
            SKM_TRY((launch_tiles<DT, 128, 128, 2, 2>(ctx, g)));
    }
    if (g.nsplit > 1) {
        SKM_PROF(ctx, "k_linear_join");
        k_linear_join<DT><<<skm_grid_cap(ctx, skm_ceil_div(g.m * skm_ceil_div(g.n, ln_type<DT>::VE), 256), 16), 256, 0, ctx->stream>>>(g);
        SKM_TRY(skm_check_launch("k_linear_join"));
    }
    return SKM_OK;
}

// The operand as the product reads it: where it lies if its rows start on 16-byte boundaries and hold whole 16-byte
// pieces, else a padded copy in scratch.
template <int DT>
int ready(skm_ctx *ctx, int slot, int64_t rows, int64_t cols, const void *in, int64_t ld, const uint8_t **out, int64_t *ld_bytes)
{
    constexpr int64_t es = (int64_t)elem_bytes(DT), VE = ln_type<DT>::VE;
    if (((uintptr_t)in & 15) == 0 && (rows == 1 || ld * es % 16 == 0) && cols % VE == 0) {
        *out = (const uint8_t *)in;
        *ld_bytes = rows == 1 ? 0 : ld * es;
        return SKM_OK;
    }
    const int64_t ldo = skm_ceil_div(cols, VE) * VE;
    void *p;
    SKM_TRY(skm_ws(ctx, slot, (size_t)(rows * ldo * es), &p));
    SKM_PROF(ctx, "k_linear_pad");
    k_linear_pad<DT><<<skm_grid_cap(ctx, skm_ceil_div(rows * (ldo / VE), 256), 16), 256, 0, ctx->stream>>>(rows, cols, in, ld, p, ldo);
    SKM_TRY(skm_check_launch("k_linear_pad"));
    *out = (const uint8_t *)p;
    *ld_bytes = ldo * es;
    return SKM_OK;
}

template <int DT>
int transposed(skm_ctx *ctx, int slot, int64_t rows, int64_t cols, const void *in, int64_t ld, const uint8_t **out, int64_t *ld_bytes)
{
    constexpr int64_t es = (int64_t)elem_bytes(DT), VE = ln_type<DT>::VE;
    const int64_t ldt = skm_ceil_div(rows, VE) * VE;
    void *p;
    SKM_TRY(skm_ws(ctx, slot, (size_t)(cols * ldt * es), &p));
    SKM_PROF(ctx, "k_linear_transpose");
    k_linear_transpose<DT, false><<<skm_grid_cap(ctx, skm_ceil_div(rows, 64) * skm_ceil_div(cols, 64), 16), 256, 0, ctx->stream>>>(rows, cols, in, ld, p, ldt, 0, nullptr, 0,
                                                                                                                         nullptr, 0, nullptr);
    SKM_TRY(skm_check_launch("k_linear_transpose"));
    *out = (const uint8_t *)p;
    *ld_bytes = ldt * es;
    return SKM_OK;
}

template <int DT>
int forward(skm_ctx *ctx, int act, int64_t m, int64_t n, int64_t k, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *bias, const void *residual,
            int64_t ldr, void *preact, int64_t ldp, void *y, int64_t ldy)
{
    ln_gemm g = {};
    g.m = m;
    g.n = n;
    g.k = k;
    SKM_TRY(ready<DT>(ctx, WS_A, m, k, x, ldx, &g.a, &g.lda));
    SKM_TRY(ready<DT>(ctx, WS_B, n, k, w, ldw, &g.b, &g.ldb));
    g.act = act;
    g.bias = bias;
    g.residual = residual;
    g.ldr = ldr;
    g.preact = preact;
    g.ldp = ldp;
    g.out = y;
    g.ldo = ldy;
    return gemm<DT>(ctx, g);
}

template <int DT>
int backward(skm_ctx *ctx, int act, int64_t m, int64_t n, int64_t k, const void *dy, int64_t lddy, const void *z, int64_t ldz, const void *x, int64_t ldx, const void *w,
             int64_t ldw, void *dx, int64_t lddx, void *dw, int64_t lddw, void *dbias)
{
    constexpr int64_t es = (int64_t)elem_bytes(DT), VE = ln_type<DT>::VE;
    // dz as dx's left operand: dy itself where it can be read as it lies
    const bool direct = act == ACT_NONE && ((uintptr_t)dy & 15) == 0 && (m == 1 || lddy * es % 16 == 0) && n % VE == 0;
    const uint8_t *dz = (const uint8_t *)dy, *dzt = nullptr;
    int64_t lddz = m == 1 ? 0 : lddy * es, lddzt = 0;
    if (dw || dbias || (dx && !direct)) {
        const int64_t ldo = skm_ceil_div(n, VE) * VE, ldt = skm_ceil_div(m, VE) * VE, parts = skm_ceil_div(m, 64);
        void *p, *to = nullptr, *tot = nullptr;
        float *sums = nullptr;
        if (dx && !direct) {
            SKM_TRY(skm_ws(ctx, WS_A, (size_t)(m * ldo * es), &to));
            dz = (const uint8_t *)to;
            lddz = ldo * es;
        }
        if (dw) {
            SKM_TRY(skm_ws(ctx, WS_B, (size_t)(n * ldt * es), &tot));
            dzt = (const uint8_t *)tot;
            lddzt = ldt * es;
        }
        if (dbias) {
            SKM_TRY(skm_ws(ctx, WS_C, sizeof(float) * (size_t)(parts * n), &p));
            sums = (float *)p;
        }
        {
            SKM_PROF(ctx, "k_linear_transpose");
            k_linear_transpose<DT, true><<<skm_grid_cap(ctx, parts * skm_ceil_div(n, 64), 16), 256, 0, ctx->stream>>>(m, n, dy, lddy, tot, ldt, act, z, ldz, to, ldo, sums);
            SKM_TRY(skm_check_launch("k_linear_transpose"));
        }
        if (dbias) {
            k_linear_bias_grad<DT><<<skm_grid_cap(ctx, skm_ceil_div(n, 64), 16), 256, 0, ctx->stream>>>(parts, n, sums, dbias);
            SKM_TRY(skm_check_launch("k_linear_bias_grad"));
        }
    }
    if (dx) {
        ln_gemm g = {};
        g.m = m;
        g.n = k;
        g.k = n;
        g.a = dz;
        g.lda = lddz;
        SKM_TRY(transposed<DT>(ctx, WS_E, n, k, w, ldw, &g.b, &g.ldb));
        g.out = dx;
        g.ldo = lddx;
        SKM_TRY(gemm<DT>(ctx, g));
    }
    if (dw) {
        ln_gemm g = {};
        g.m = n;
        g.n = k;
        g.k = m;
        g.a = dzt;
        g.lda = lddzt;
        SKM_TRY(transposed<DT>(ctx, WS_F, m, k, x, ldx, &g.b, &g.ldb));
        g.out = dw;
        g.ldo = lddw;
        SKM_TRY(gemm<DT>(ctx, g));
    }
    return SKM_OK;
}

int check_matrix(const char *who, const char *what, const void *p, int64_t rows, int64_t cols, int64_t ld, int64_t es)
{
    SKM_REQUIRE(ld >= cols, SKM_E_BADARG, "%s: the row stride of %s (%lld) is less than its %lld columns", who, what, (long long)ld, (long long)cols);
    SKM_REQUIRE((uintptr_t)p % (uintptr_t)es == 0, SKM_E_BADARG, "%s: %s is not aligned to its type", who, what);
    return SKM_OK;
}

}  // namespace

extern "C" int skm_linear(skm_ctx *ctx, int dtype, int activation, int64_t m, int64_t n, int64_t k, const void *d_x, int64_t ldx, const void *d_w, int64_t ldw,
                          const void *d_bias, const void *d_residual, int64_t ldr, void *d_preact, int64_t ldp, void *d_y, int64_t ldy)
{
    const char *who = "skm_linear";
    SKM_REQUIRE(ctx, SKM_E_BADARG, "%s: null context", who);
    SKM_REQUIRE(dtype >= 0 && dtype <= 2, SKM_E_BADARG, "%s: dtype must be 0 (float32), 1 (float16) or 2 (bfloat16)", who);
    SKM_REQUIRE(activation >= 0 && activation < ACT_COUNT, SKM_E_BADARG, "%s: unknown activation %d", who, activation);
    SKM_REQUIRE(m >= 0 && n >= 0 && k >= 0, SKM_E_BADARG, "%s: negative size", who);
    if (m == 0 || n == 0)
        return SKM_OK;
    const int64_t es = (int64_t)elem_bytes(dtype);
    SKM_REQUIRE(d_y && (k == 0 || (d_x && d_w)), SKM_E_BADARG, "%s: null array", who);
    SKM_TRY(check_matrix(who, "x", d_x, m, k, ldx, es));
    SKM_TRY(check_matrix(who, "w", d_w, n, k, ldw, es));
    SKM_TRY(check_matrix(who, "y", d_y, m, n, ldy, es));
    SKM_REQUIRE((uintptr_t)d_bias % (uintptr_t)es == 0, SKM_E_BADARG, "%s: bias is not aligned to its type", who);
    if (d_residual)
        SKM_TRY(check_matrix(who, "residual", d_residual, m, n, ldr, es));
    if (d_preact)
        SKM_TRY(check_matrix(who, "preact", d_preact, m, n, ldp, es));
    void *const outs[2] = {d_y, d_preact};
    const int64_t ldos[2] = {ldy, ldp};
    for (int o = 0; o < 2; ++o) {
        SKM_REQUIRE(!skm_overlap(outs[o], m, n, ldos[o], d_x, m, k, ldx, es) && !skm_overlap(outs[o], m, n, ldos[o], d_w, n, k, ldw, es) &&
                        !skm_overlap(outs[o], m, n, ldos[o], d_bias, 1, n, n, es),
                    SKM_E_BADARG, "%s: an output shares memory with x, w or bias", who);
        // (a cell of the residual is read by the lane that writes that cell: the output may BE the residual)
        SKM_REQUIRE((outs[o] == d_residual && ldos[o] == ldr && o == 0) || !skm_overlap(outs[o], m, n, ldos[o], d_residual, m, n, ldr, es), SKM_E_BADARG,
                    "%s: an output shares memory with the residual without being it", who);
    }
    SKM_REQUIRE(!skm_overlap(d_y, m, n, ldy, d_preact, m, n, ldp, es), SKM_E_BADARG, "%s: y and preact share memory", who);
    SKM_HIP(hipSetDevice(ctx->device));
    if (dtype == 0)
        return forward<0>(ctx, activation, m, n, k, d_x, ldx, d_w, ldw, d_bias, d_residual, ldr, d_preact, ldp, d_y, ldy);
    if (dtype == 1)
        return forward<1>(ctx, activation, m, n, k, d_x, ldx, d_w, ldw, d_bias, d_residual, ldr, d_preact, ldp, d_y, ldy);
    return forward<2>(ctx, activation, m, n, k, d_x, ldx, d_w, ldw, d_bias, d_residual, ldr, d_preact, ldp, d_y, ldy);
}

extern "C" int skm_linear_backward(skm_ctx *ctx, int dtype, int activation, int64_t m, int64_t n, int64_t k, const void *d_dy, int64_t lddy, const void *d_preact,
                                   int64_t ldp, const void *d_x, int64_t ldx, const void *d_w, int64_t ldw, void *d_dx, int64_t lddx, void *d_dw, int64_t lddw,
                                   void *d_dbias)
{
    const char *who = "skm_linear_backward";
    SKM_REQUIRE(ctx, SKM_E_BADARG, "%s: null context", who);
    SKM_REQUIRE(dtype >= 0 && dtype <= 2, SKM_E_BADARG, "%s: dtype must be 0 (float32), 1 (float16) or 2 (bfloat16)", who);
    SKM_REQUIRE(activation >= 0 && activation < ACT_COUNT, SKM_E_BADARG, "%s: unknown activation %d", who, activation);
    SKM_REQUIRE(m >= 0 && n >= 0 && k >= 0, SKM_E_BADARG, "%s: negative size", who);
    SKM_REQUIRE(d_dx || d_dw || d_dbias || (m == 0 && n == 0), SKM_E_BADARG, "%s: no gradient is asked for", who);
    const int64_t es = (int64_t)elem_bytes(dtype);
    const bool cells = m > 0 && n > 0;
    SKM_REQUIRE(!cells || d_dy, SKM_E_BADARG, "%s: null dy", who);
    SKM_REQUIRE(!cells || activation == ACT_NONE || d_preact, SKM_E_BADARG, "%s: the activation's slope needs the pre-activation values", who);
    SKM_REQUIRE(!d_dx || n == 0 || k == 0 || d_w, SKM_E_BADARG, "%s: dx needs w", who);
    SKM_REQUIRE(!d_dw || m == 0 || k == 0 || d_x, SKM_E_BADARG, "%s: dw needs x", who);
    if (cells)
        SKM_TRY(check_matrix(who, "dy", d_dy, m, n, lddy, es));
    if (cells && activation != ACT_NONE)
        SKM_TRY(check_matrix(who, "preact", d_preact, m, n, ldp, es));
    if (d_dx) {
        SKM_TRY(check_matrix(who, "w", d_w, n, k, ldw, es));
        SKM_TRY(check_matrix(who, "dx", d_dx, m, k, lddx, es));
    }
    if (d_dw) {
        SKM_TRY(check_matrix(who, "x", d_x, m, k, ldx, es));
        SKM_TRY(check_matrix(who, "dw", d_dw, n, k, lddw, es));
    }
    SKM_REQUIRE((uintptr_t)d_dbias % (uintptr_t)es == 0, SKM_E_BADARG, "%s: dbias is not aligned to its type", who);
    struct part {
        const void *p;
        int64_t rows, cols, ld;
    };
    const part in[4] = {{d_dy, m, n, lddy}, {activation != ACT_NONE ? d_preact : nullptr, m, n, ldp}, {d_dw ? d_x : nullptr, m, k, ldx}, {d_dx ? d_w : nullptr, n, k, ldw}};
    const part out[3] = {{d_dx, m, k, lddx}, {d_dw, n, k, lddw}, {d_dbias, 1, n, n}};
    for (int o = 0; o < 3; ++o) {
        for (const part &i : in)
            SKM_REQUIRE(!skm_overlap(out[o].p, out[o].rows, out[o].cols, out[o].ld, i.p, i.rows, i.cols, i.ld, es), SKM_E_BADARG, "%s: a gradient shares memory with an input", who);
        for (int q = 0; q < o; ++q)
            SKM_REQUIRE(!skm_overlap(out[o].p, out[o].rows, out[o].cols, out[o].ld, out[q].p, out[q].rows, out[q].cols, out[q].ld, es), SKM_E_BADARG,
                        "%s: two gradients share memory", who);
    }
    SKM_HIP(hipSetDevice(ctx->device));
    // (k = 0: dx and dw have no cells, the bias's gradient is what is left; m or n = 0: what has cells is an empty sum)
    void *dx = m && k ? d_dx : nullptr, *dw = n && k ? d_dw : nullptr, *db = n ? d_dbias : nullptr;
    if (!dx && !dw && !db)
        return SKM_OK;
    if (dtype == 0)
        return backward<0>(ctx, activation, m, n, k, d_dy, lddy, d_preact, ldp, d_x, ldx, d_w, ldw, dx, lddx, dw, lddw, db);
    if (dtype == 1)
        return backward<1>(ctx, activation, m, n, k, d_dy, lddy, d_preact, ldp, d_x, ldx, d_w, ldw, dx, lddx, dw, lddw, db);
    return backward<2>(ctx, activation, m, n, k, d_dy, lddy, d_preact, ldp, d_x, ldx, d_w, ldw, dx, lddx, dw, lddw, db);
}
