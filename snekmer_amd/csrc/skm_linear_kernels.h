// A matrix product with bias, activation and residual in its epilogue, and its backward pass:
//
//   z = x w^T + b,   y = act(z) + r          x [m x k], w [n x k], b [n], r, z, y [m x n]
//   dz = dy act'(z),   dx = dz w,   dw = dz^T x,   db = column sums of dz        (dr is dy)
//
// in float32, float16 or bfloat16, accumulated in float32 on the matrix cores.  Next to the cosine GEMMs of skm_dense.hip
// (int8 counts with a row-norm epilogue, float64): this one multiplies feature rows by learned weights.  No reference
// counterpart in this form (the reference hands its feature matrices to scikit-learn's estimators, snekmer/model.py).
//
// One kernel computes every product as C[i][j] = sum over c of A[i][c] B[j][c].  x and w lie along the contraction; the backward pass's
// w, dz and x lie across it and are read so, transposed on the way from LDS to the registers.  Operands whose rows do not
// hold whole words on 4-byte boundaries are copied with padding first.
//
// Compiled once for each element type (skm_linear_f32.hip, skm_linear_f16.hip, skm_linear_bf16.hip).
#pragma once
#include <algorithm>
#include <type_traits>
#include <utility>

#include "skm_linear.h"

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
    // the two lane halves hold columns 0-3 and 4-7 of a 32-byte step: part i takes columns i and 4 + i of both
    static constexpr int PARTS = 4;
    static __device__ __forceinline__ f32x16 mfma(V a, V b, f32x16 c, int i) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0); }
};
template <>
struct ln_type<1> {
    using T = _Float16;
    using V = f16x8;
    static constexpr int VE = 8;
    static constexpr int PARTS = 1;
    static __device__ __forceinline__ f32x16 mfma(V a, V b, f32x16 c, int) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct ln_type<2> {
    using T = __bf16;
    using V = bf16x8;
    static constexpr int VE = 8;
    static constexpr int PARTS = 1;
    static __device__ __forceinline__ f32x16 mfma(V a, V b, f32x16 c, int) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

// ---- activations (in float32)
// FINE: for float32 outputs, which keep that type's precision however small they are (4096 x 4096 cells of k = 1024 with residual and
// pre-activation: 272 us without activation, 274 with silu, 279 with gelu).  16-bit outputs are off by up to 2^-8 or 2^-11 of
// themselves, by their rounding: the plain exponential, off by |x| u (u = 2^-24: 6e-6 at x = -100), is exact enough for them.

// exp(x + x_lo) for x <= 0 (NaN stays) to 8 u: the rounding of x log2(e) is put back, and the square of exp(x / 2) reaches below
// 2^-126, where the instruction's own results end
__device__ __forceinline__ float ln_exp_fine(float x, float x_lo = 0.0f)
{
    x = __builtin_elementwise_maximum(x, -110.0f);  // (0 from -104 on)
    const float t = x * 0.721347511f;               // log2(e) / 2, and what that float leaves out
    const float lo = __builtin_fmaf(x_lo, 0.721347511f, __builtin_fmaf(x, 9.62981495e-09f, __builtin_fmaf(x, 0.721347511f, -t)));
    const float h = __builtin_amdgcn_exp2f(t), f = __builtin_fmaf(h, lo * 0.693147181f, h);
    return f * f;
}

// (fast: exp overflows to inf for z < -88: 0, as it should be; the reciprocal instruction is good to 1 ulp, a rounded division costs ten more)
template <bool FINE>
__device__ __forceinline__ float ln_sigmoid(float z)
{
    if (!FINE)
        return __builtin_amdgcn_rcpf(1.0f + __expf(-z));
    const float e = ln_exp_fine(-fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + e);
    return z > 0.0f ? r : e * r;
}

// The normal distribution's lower tail at -|z|, bell = exp(-z z / 2): tail / (t bell) with t = 1 / (1 + 0.27 |z|) is smooth over all z, a
// polynomial of degree 8 in t fitted to it (least maximum error over |z| < 14.5) is off by 3.9e-8 of its value, evaluated in float32
// by 2.6e-7.  So gelu keeps its relative precision in the tail, where 1 + erf cancels (4e-6 at z = -12), for one exponential: 4096 x
// 4096 cells of k = 1024 with residual and pre-activation in 63 us where erff took 74 (bfloat16).
template <bool FINE>
__device__ __forceinline__ float ln_normal_tail(float z, float &bell)
{
    // (FINE: bell is 0 from 15 on; NaN stays)
    const float a = FINE ? __builtin_elementwise_minimum(fabsf(z), 15.0f) : fabsf(z), t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.27f, a, 1.0f));
    float p = 0.0289610978f;
    p = __builtin_fmaf(p, t, -0.126485839f);
    p = __builtin_fmaf(p, t, 0.169786125f);
    p = __builtin_fmaf(p, t, -0.0692107156f);
    p = __builtin_fmaf(p, t, 0.107825592f);
    p = __builtin_fmaf(p, t, 0.0720496252f);
    p = __builtin_fmaf(p, t, 0.101810604f);
    p = __builtin_fmaf(p, t, 0.107542872f);
    p = __builtin_fmaf(p, t, 0.107720658f);
    const float q = -0.5f * a * a;
    bell = FINE ? ln_exp_fine(q, __builtin_fmaf(-0.5f * a, a, -q)) : __expf(q);
    return p * t * bell;
}

template <bool FINE>
__device__ __forceinline__ float ln_act(int act, float z)
{
    switch (act) {
    case ACT_RELU:
        return z < 0.0f ? 0.0f : z;  // (NaN stays)
    case ACT_GELU: {
        float bell;
        const float tail = ln_normal_tail<FINE>(z, bell);
        return z * (z > 0.0f ? 1.0f - tail : tail);
    }
    case ACT_GELU_TANH: {
        // 0.5 z (1 + tanh u) = z sigmoid(2 u)
        const float u = 0.797884560802865356f * (z + 0.044715f * z * z * z);
        return z * ln_sigmoid<FINE>(2.0f * u);
    }
    case ACT_SILU:
        return z * ln_sigmoid<FINE>(z);
    case ACT_SIGMOID:
        return ln_sigmoid<FINE>(z);
    default:
        return z;
    }
}

template <bool FINE>
__device__ __forceinline__ float ln_slope(int act, float z)
{
    switch (act) {
    case ACT_RELU:
        return z > 0.0f ? 1.0f : z == z ? 0.0f : z;
    case ACT_GELU: {
        float bell;
        const float tail = ln_normal_tail<FINE>(z, bell);
        return (z > 0.0f ? 1.0f - tail : tail) + z * bell * 0.398942280401432678f;
    }
    case ACT_GELU_TANH: {
        const float u2 = 1.59576912160573071f * (z + 0.044715f * z * z * z), s = ln_sigmoid<FINE>(u2);
        const float bell = s * (1.0f - s);  // (0 from |z| = 11 on, where z z may be infinite)
        return bell == 0.0f ? s : s + z * bell * 1.59576912160573071f * (1.0f + 0.134145f * z * z);
    }
    case ACT_SILU: {
        const float s = ln_sigmoid<FINE>(z);
        return s * (1.0f + z * (1.0f - s));
    }
    case ACT_SIGMOID: {
        // s (1 - s) = e / (1 + e)^2, e = exp(-|z|): 1 - s would keep nothing of itself where s is next to 1 (17 % off at z = 15, 0 from 17 on)
        const float e = FINE ? ln_exp_fine(-fabsf(z)) : __expf(-fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + e);
        return e * r * r;
    }
    default:
        return 1.0f;
    }
}

// ---- the product
struct ln_gemm {
    int64_t m, n, k;            // C [m x n], contraction k
    const uint8_t *a, *b;       // rows on 4-byte boundaries
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
    int64_t stages, stages_per_split;  // of the contraction, LN_BK bytes each
};

__device__ const uint4 ln_zero_block = {0, 0, 0, 0};  // what lanes past the end of the contraction fetch

// 16 bytes of a row, `whole` if all of them are columns of the matrix
template <int DT, int VE>
__device__ __forceinline__ void ln_read(const typename ln_type<DT>::T *from, bool whole, int64_t left, typename ln_type<DT>::T (&v)[VE])
{
    static_assert(VE * sizeof(v[0]) == 16, "16 bytes");
    if (whole) {
        const ln_u128 raw = *reinterpret_cast<const ln_u128 *>(from);
        __builtin_memcpy(v, &raw, 16);
    } else {
#pragma unroll
        for (int u = 0; u < VE; ++u)
            v[u] = u < left ? from[u] : (typename ln_type<DT>::T)0.0f;
    }
}
// v in the type, as it is stored.  (Words that the compiler cannot look into: it would move the arithmetic behind the
// branches of every store, each waiting for its own results.)
template <int DT, int VE>
__device__ __forceinline__ ln_u128 ln_pack(const float (&v)[VE])
{
    typename ln_type<DT>::T o[VE];
#pragma unroll
    for (int u = 0; u < VE; ++u)
        o[u] = (typename ln_type<DT>::T)v[u];
    ln_u128 raw;
    __builtin_memcpy(&raw, o, 16);
    asm volatile("" : "+v"(raw.w[0]), "+v"(raw.w[1]), "+v"(raw.w[2]), "+v"(raw.w[3]));
    return raw;
}

// VE consecutive cells from (i, j) on: bias, activation and residual; the pre-activation and the output as stored
template <int DT, int VE>
struct ln_done {
    ln_u128 z, y;
};
template <int DT, int VE>
__device__ __forceinline__ ln_done<DT, VE> ln_cells(const ln_gemm &g, int act, const float (&bias)[VE], const typename ln_type<DT>::T (&res)[VE], float (&v)[VE])
{
    ln_done<DT, VE> d;
#pragma unroll
    for (int u = 0; u < VE; ++u)
        v[u] += bias[u];
    if (g.preact)
        d.z = ln_pack<DT, VE>(v);
#pragma unroll
    for (int u = 0; u < VE; ++u)
        v[u] = ln_act<DT == 0>(act, v[u]) + (float)res[u];
    d.y = ln_pack<DT, VE>(v);
    return d;
}
// `left` of them are cells of the matrix
template <int DT, int VE>
__device__ __forceinline__ void ln_put(const ln_gemm &g, int64_t i, int64_t j, int64_t left, const ln_done<DT, VE> &d)
{
    using T = typename ln_type<DT>::T;
    T *z = (T *)g.preact + i * g.ldp + j, *y = (T *)g.out + i * g.ldo + j;
    if (left >= VE) {
        if (g.preact)
            *reinterpret_cast<ln_u128 *>(z) = d.z;
        *reinterpret_cast<ln_u128 *>(y) = d.y;
    } else if (left > 0) {
        T o[VE];
        if (g.preact) {
            __builtin_memcpy(o, &d.z, 16);
#pragma unroll
            for (int u = 0; u < VE; ++u)
                if (u < left)
                    z[u] = o[u];
        }
        __builtin_memcpy(o, &d.y, 16);
#pragma unroll
        for (int u = 0; u < VE; ++u)
            if (u < left)
                y[u] = o[u];
    }
}

// calls f with the activation as a compile-time constant
template <typename F>
__device__ __forceinline__ void ln_with_act(int act, F &&f)
{
    switch (act) {
    case ACT_RELU:
        return f(std::integral_constant<int, ACT_RELU>());
    case ACT_GELU:
        return f(std::integral_constant<int, ACT_GELU>());
    case ACT_GELU_TANH:
        return f(std::integral_constant<int, ACT_GELU_TANH>());
    case ACT_SILU:
        return f(std::integral_constant<int, ACT_SILU>());
    case ACT_SIGMOID:
        return f(std::integral_constant<int, ACT_SIGMOID>());
    default:
        return f(std::integral_constant<int, ACT_NONE>());
    }
}

template <int... I, typename F>
__device__ __forceinline__ void ln_each(std::integer_sequence<int, I...>, F &&f)  // f of 0, 1, ... as constants
{
    (f(std::integral_constant<int, I>()), ...);
}

constexpr int LN_BK = 128;  // bytes of contraction per stage: one 128-byte line of every operand row

// Where a workgroup works.  Consecutive workgroups go to the eight XCDs in turn, so that each XCD gets a contiguous run of
// the tile order, which walks groups of 8 tile rows column by column (their operands stay in the XCD's L2).
struct ln_place {
    int64_t row0, col0, s_lo, s_hi;  // the tile's first cell, the stages of the contraction
    int split;
};
template <int BM, int BN>
__device__ __forceinline__ ln_place ln_tile_of(const ln_gemm &g)
{
    // (32-bit: the launcher keeps the workgroups below 2^24; 64-bit divisions cost microseconds at the start of every tile)
    const uint32_t nty = (uint32_t)((g.m + BM - 1) / BM), ntx = (uint32_t)((g.n + BN - 1) / BN), tiles = nty * ntx;
    const uint32_t bid = blockIdx.x, nwg = gridDim.x, q8 = nwg / 8, r8 = nwg % 8, xcd = bid % 8;
    const uint32_t seq = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + bid / 8;
    const uint32_t split = seq / tiles, tile = seq - split * tiles;
    const uint32_t group = tile / (8 * ntx), first = group * 8, rows_in = min(8u, nty - first), in_group = tile - group * 8 * ntx;
    const uint32_t col = in_group / rows_in;
    ln_place p;
    p.row0 = (int64_t)(first + in_group - col * rows_in) * BM;
    p.col0 = (int64_t)col * BN;
    p.split = (int)split;
    p.s_lo = p.split * g.stages_per_split;
    p.s_hi = min(g.stages, p.s_lo + g.stages_per_split);
    return p;
}

// A wave's FM x FN sub-tiles of 32 x 32, at (wrow, wcol) of the workgroup's tile.  B is the products' left operand, so that a
// lane holds cells of one row (row lane % 32, register 4 q + u: column 8 q + 4 (lane / 32) + u); 32 rows at a time go through LDS (this wave's own part of `s_f`) and leave
// as 16-byte pieces of rows.  The residual's pieces of the next rows are under way while these are worked on: with one wave
// a SIMD nothing else hides their latency (8192 x 4096 outputs of k = 4096 with silu, residual and pre-activation: 353 us
// without, 286 with).
template <int FN>
constexpr int ln_trow = FN * 32 + 4;  // floats of a buffered row: 16-byte aligned, spread over the banks
template <int DT, int FM, int FN, bool SPLIT>
__device__ __forceinline__ void ln_store_tile(const ln_gemm &g, const ln_place &at, const f32x16 (&acc)[FM][FN], float *s_f, int wid, int wrow, int wcol, int lane)
{
    using T = typename ln_type<DT>::T;
    constexpr int TROW = ln_trow<FN>, VE = SPLIT ? 4 : ln_type<DT>::VE, PIECES = FN * 32 / VE, ROWS = 64 / PIECES, PASSES = 32 / ROWS;
    const int fr = lane & 31, fh = lane >> 5, pr = lane / PIECES, pc = lane % PIECES * VE;
    float *buf = s_f + wid * 32 * TROW;
    const int64_t j = at.col0 + wcol + pc, left = g.n - j;
    auto put = [&](auto A) {
        constexpr int aa = decltype(A)::value;
        // (the two comments keep the branches of to_lds apart: merged, they would index the registers at run time, in scratch memory)
        asm volatile("; rows %0" ::"n"(aa * 32));
#pragma unroll
        for (int b = 0; b < FN; ++b)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<float4 *>(buf + fr * TROW + b * 32 + 8 * q + 4 * fh) = make_float4(acc[aa][b][4 * q], acc[aa][b][4 * q + 1], acc[aa][b][4 * q + 2], acc[aa][b][4 * q + 3]);
        asm volatile("; rows %0 done" ::"n"(aa * 32) : "memory");
    };
    auto to_lds = [&](int a) {
        if constexpr (FM == 4) {
            if (a == 0)
                put(std::integral_constant<int, 0>());
            else if (a == 1)
                put(std::integral_constant<int, 1>());
            else if (a == 2)
                put(std::integral_constant<int, 2>());
            else
                put(std::integral_constant<int, 3>());
        } else if constexpr (FM == 2) {
            if (a == 0)
                put(std::integral_constant<int, 0>());
            else
                put(std::integral_constant<int, 1>());
        } else {
            static_assert(FM == 1, "rows of sub-tiles");
            put(std::integral_constant<int, 0>());
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    auto from_lds = [&](int p, float (&v)[VE]) {
#pragma unroll
        for (int u = 0; u < VE; u += 4) {
            const float4 f = *reinterpret_cast<const float4 *>(buf + (p * ROWS + pr) * TROW + pc + u);
            v[u] = f.x;
            v[u + 1] = f.y;
            v[u + 2] = f.z;
            v[u + 3] = f.w;
        }
    };
    if constexpr (SPLIT) {
#pragma unroll 1
        for (int a = 0; a < FM; ++a) {
            to_lds(a);
#pragma unroll
            for (int p = 0; p < PASSES; ++p) {
                const int64_t i = at.row0 + wrow + a * 32 + p * ROWS + pr;
                float v[VE];
                from_lds(p, v);
                if (i < g.m && left > 0)
                    *reinterpret_cast<float4 *>(g.partial + ((int64_t)at.split * g.m + i) * g.ldq + j) = make_float4(v[0], v[1], v[2], v[3]);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    } else {
        constexpr int CHUNK = PASSES < 8 ? PASSES : 8, CHUNKS = PASSES / CHUNK;
        const bool whole = left >= VE;
        float bias[VE];
        {
            T b[VE];
#pragma unroll
            for (int u = 0; u < VE; ++u)
                b[u] = (T)0.0f;
            if (g.bias && left > 0)
                ln_read<DT, VE>((const T *)g.bias + j, whole, left, b);
#pragma unroll
            for (int u = 0; u < VE; ++u)
                bias[u] = (float)b[u];
        }
        T res[CHUNK][VE], next[CHUNK][VE];
        auto fetch = [&](int it, T (&r)[CHUNK][VE]) {  // the residual of chunk `it` of FM * CHUNKS
#pragma unroll
            for (int p = 0; p < CHUNK; ++p) {
                const int64_t i = at.row0 + wrow + (it * CHUNK + p) * ROWS + pr;
                if (g.residual && i < g.m && left > 0)
                    ln_read<DT, VE>((const T *)g.residual + i * g.ldr + j, whole, left, r[p]);
                else
#pragma unroll
                    for (int u = 0; u < VE; ++u)
                        r[p][u] = (T)0.0f;
            }
        };
        fetch(0, res);
#pragma unroll 1  // (the activations' code once)
        for (int it = 0; it < FM * CHUNKS; ++it) {
            const int c = it % CHUNKS;
            if (c == 0)
                to_lds(it / CHUNKS);
            if (g.residual && it + 1 < FM * CHUNKS)
                fetch(it + 1, next);
            ln_with_act(g.act, [&](auto ACT) {
                constexpr int BATCH = CHUNK < 4 ? CHUNK : 4;  // pieces worked on side by side
#pragma unroll
                for (int p0 = 0; p0 < CHUNK; p0 += BATCH) {
                    float v[BATCH][VE];
                    ln_done<DT, VE> d[BATCH];
#pragma unroll
                    for (int p = 0; p < BATCH; ++p)
                        from_lds(c * CHUNK + p0 + p, v[p]);
#pragma unroll
                    for (int p = 0; p < BATCH; ++p)
                        d[p] = ln_cells<DT, VE>(g, decltype(ACT)::value, bias, res[p0 + p], v[p]);
#pragma unroll
                    for (int p = 0; p < BATCH; ++p) {
                        const int64_t i = at.row0 + wrow + (it * CHUNK + p0 + p) * ROWS + pr;
                        ln_put<DT, VE>(g, i, j, i < g.m ? left : 0, d[p]);
                    }
                }
            });
            if (g.residual)
#pragma unroll
                for (int p = 0; p < CHUNK; ++p)
#pragma unroll
                    for (int u = 0; u < VE; ++u)
                        res[p][u] = next[p][u];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
}

// The LDS's transposing read: lane i of 16 gets value i % 4 of the 8 bytes at lane (4 u + i / 4)'s address as its value u.
// (The restrict says that nothing writes there during the read, as the barriers see to; without it the compiler would wait
// for every fetch under way, into whatever slot, before each of these reads: 604 us for a product that takes 215.)
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 ln_lds_s16x4;
__device__ __forceinline__ s16x4 ln_read_tr(const ln_lds_s16x4 *__restrict__ p)
{
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(const_cast<ln_lds_s16x4 *>(p));
}

// Tiles of BM x BN, 2 x 2 waves of (BM / 2) x (BN / 2).  Operands go to LDS directly (16 bytes a lane, 8 rows of 128 bytes an
// instruction), in stages of 128 bytes of contraction: A(0), B(0), A(1), B(1), ... through a ring of five slots, so that two
// and a half stages are held.  The 16-byte chunk index of a row is XORed with (row >> 1) & 7 on the source address and on the
// fragment reads, so that the 32 rows of a fragment read spread over the banks.
//
// A wave keeps its matrix unit fed by itself: while the FM x FN products of a 32-byte step run, the fragments of the next
// step are read into the other of two register sets and a quarter of a stage is fetched, one instruction at a time between
// the products.  One barrier a stage, before its last step: by then everybody has read the stage (its slots are free) and the
// next stage has landed (its first fragments are read during the last step).  In stage s the steps fetch the second half of
// B(s+1), A(s+2), and after the barrier the first half of B(s+2): what is fetched has two steps or more to arrive, and all
// four steps load the memory pipe alike.  bfloat16, 256 x 256 tiles, all compute units busy: 1.46 us a stage; with two whole
// stages in memory, fetching in two of the steps 1.59, in one of them 1.66, all between the barriers of a simpler loop 1.8.
//
// CA, CB: that operand lies across the contraction (its rows are the contraction's columns: w and dz, x in the backward
// pass).  A slot then holds 128 bytes' worth of contraction rows of BM (BN) values, fetched in whole lines as they lie, and
// the fragments are read transposed: 16-bit types by the LDS's transposing reads (16 lanes give four rows of 16 values
// and get four values of one column each), float32 one value a read, which its slower products hide.  The 64-byte blocks of a row
// are XORed with the row so that the four rows of a transposing read lie in different banks.
template <int DT, int BM, int BN, bool CA, bool CB, typename OFF>
__global__ __launch_bounds__(256, (BM + BN) > 256 ? 1 : 2) void k_linear(ln_gemm g)
{
    using P = ln_type<DT>;
    using T = typename P::T;
    using V = typename P::V;
    constexpr int TM = BM / 2, TN = BN / 2, FM = TM / 32, FN = TN / 32, KS = LN_BK / 32, RING = 5;
    constexpr int NA = BM / 32, NB = BN / 32;  // fetches of a wave for an operand's stage
    constexpr int SLOT = (BM > BN ? BM : BN) * LN_BK;
    constexpr int KROWS = LN_BK / (int)sizeof(T);  // contraction columns of a stage
    static_assert(NA % 2 == 0 && NB % 2 == 0 && TM % 32 == 0 && TN % 32 == 0 && KS == 4, "tile");
    static_assert(4 * 32 * ln_trow<FN> * 4 <= RING * SLOT && RING * SLOT <= 160 * 1024, "memory");
    __shared__ __attribute__((aligned(16))) uint8_t s_t[RING * SLOT];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const ln_place at = ln_tile_of<BM, BN>(g);
    const int64_t row0 = at.row0, col0 = at.col0, s_lo = at.s_lo, s_hi = at.s_hi, kbytes = g.k * (int64_t)sizeof(T);

    // Instruction q of wave w fetches 1 KiB of A's stage, or B's, from byte (w NA + q) 1024 of the slot on.  OFF is 64-bit
    // where a tile's rows may span 2^32 bytes.
    const uint8_t *const a0 = CA ? g.a + row0 * (int64_t)sizeof(T) : g.a + row0 * g.lda, *const b0 = CB ? g.b + col0 * (int64_t)sizeof(T) : g.b + col0 * g.ldb;
    const int64_t stepa = CA ? KROWS * g.lda : LN_BK, stepb = CB ? KROWS * g.ldb : LN_BK;  // bytes from stage to stage
    const int srow = lane >> 3, schunk = lane & 7;
    auto chunk_of = [&](int r) { return (schunk ^ ((r >> 1) & 7)) * 16; };
    // across: the contraction row of a stage that this lane fetches, and the XOR of a row's 64-byte blocks
    auto krow_of = [&](int q, int n, int width) { return ((wid * n + q) * 1024 + lane * 16) / (width * (int)sizeof(T)); };
    auto blocks_of = [](int krow, int width) { return sizeof(T) == 4 ? 0 : width >= 128 ? krow & 3 : (krow >> 1) & 1; };
    auto place = [&](auto &off, auto ACROSS, auto COUNT, int width, int64_t first, int64_t rows, int64_t ld) {
        constexpr int n = decltype(COUNT)::value;
#pragma unroll
        for (int q = 0; q < n; ++q) {
            if (decltype(ACROSS)::value) {
                const int k = krow_of(q, n, width), byte = ((wid * n + q) * 1024 + lane * 16) % (width * (int)sizeof(T)) ^ (blocks_of(k, width) * 64);
                // values past the end: any, not stored
                off[q] = (OFF)(k * ld) + (OFF)(first * (int64_t)sizeof(T) + byte < rows * (int64_t)sizeof(T) ? byte : 0);
            } else {
                const int r = (wid * n + q) * 8 + srow;
                off[q] = (OFF)(min((int64_t)r, rows - 1 - first) * ld) + (OFF)chunk_of(r);
            }
        }
    };
    OFF offa[NA], offb[NB];
    place(offa, std::integral_constant<bool, CA>(), std::integral_constant<int, NA>(), BM, row0, g.m, g.lda);
    place(offb, std::integral_constant<bool, CB>(), std::integral_constant<int, NB>(), BN, col0, g.n, g.ldb);
    const int64_t last = kbytes % LN_BK ? kbytes / LN_BK : -1;  // the stage that the contraction ends in, if it does not fill it
    auto fetch = [&](auto WHOLE, auto IS_A, int64_t s, int q, int slot) {
        constexpr bool is_a = decltype(IS_A)::value, across = is_a ? CA : CB;
        constexpr int n = is_a ? NA : NB;
        const uint8_t *p = (is_a ? a0 + offa[is_a ? q : 0] : b0 + offb[is_a ? 0 : q]) + s * (is_a ? stepa : stepb);
        if (!decltype(WHOLE)::value && s == last) {
            if constexpr (across) {
                if ((s * KROWS + krow_of(q, n, is_a ? BM : BN)) * (int64_t)sizeof(T) >= kbytes)
                    p = reinterpret_cast<const uint8_t *>(&ln_zero_block);
            } else {
                // by words of 4 bytes, 2 rows an instruction: the contraction may end inside a 16-byte piece
                const int64_t rows = is_a ? g.m - 1 - row0 : g.n - 1 - col0, ld = is_a ? g.lda : g.ldb;
                int l = lane;
                asm volatile("" : "+v"(l));  // (worked out here, not held in registers all along)
#pragma unroll 1
                for (int d = 0; d < 4; ++d) {
                    const int r = (wid * n + q) * 8 + d * 2 + (l >> 5), byte = (((l >> 2) & 7) ^ ((r >> 1) & 7)) * 16 + (l & 3) * 4;
                    const int64_t c = s * LN_BK + byte;
                    const uint8_t *from = (is_a ? a0 : b0) + min((int64_t)r, rows) * ld + c;
                    if (c >= kbytes)
                        from = reinterpret_cast<const uint8_t *>(&ln_zero_block);
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from, (__attribute__((address_space(3))) void *)(s_t + slot + (wid * n + q) * 1024 + d * 256), 4, 0, 0);
                }
                return;
            }
        }
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)p, (__attribute__((address_space(3))) void *)(s_t + slot + (wid * n + q) * 1024), 16, 0, 0);
    };
    auto fwd = [](int slot, int by) {  // `by` slots on
        slot += by * SLOT;
        return slot >= RING * SLOT ? slot - RING * SLOT : slot;
    };

    f32x16 acc[FM][FN];
#pragma unroll
    for (int a = 0; a < FM; ++a)
#pragma unroll
        for (int b = 0; b < FN; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                acc[a][b][r] = 0.0f;

    const int fr = lane & 31, fh = lane >> 5, wr = wid >> 1, wc = wid & 1;
    V fa[2][FM], fb[2][FN];
    // (the waves' rows are multiples of 16: the XOR of every row of a fragment is that of fr)
    const int swz = (fr >> 1) & 7;
    const uint8_t *const la = s_t + (wr * TM + fr) * LN_BK, *const lb = s_t + (wc * TN + fr) * LN_BK;
    // across: where this lane's part of fragment i starts (row 0 of a step)
    auto across_at = [&](int width, int first) {  // first: the fragment's first value
        if (sizeof(T) == 4)
            return (4 * fh) * width * 4 + (first + fr) * 4;
        const int k = 8 * fh + ((lane & 15) >> 2);
        return k * width * 2 + ((first / 32) ^ blocks_of(k, width)) * 64 + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
    };
    int xa[FM], xb[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
        xa[i] = CA ? across_at(BM, wr * TM + i * 32) : 0;
#pragma unroll
    for (int i = 0; i < FN; ++i)
        xb[i] = CB ? across_at(BN, wc * TN + i * 32) : 0;
    auto read_across = [&](const uint8_t *from, int width) {
        V v;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = *reinterpret_cast<const float *>(from + i * width * 4);
        } else {
            v = __builtin_bit_cast(V, __builtin_shufflevector(ln_read_tr((const ln_lds_s16x4 *)from), ln_read_tr((const ln_lds_s16x4 *)(from + 4 * width * 2)), 0, 1, 2, 3, 4, 5, 6, 7));
        }
        return v;
    };
    auto frag = [&](auto SET, int slot, int ks, int i) {  // the i-th of FM + FN fragments of step ks of the stage whose A is at `slot`
        constexpr int set = decltype(SET)::value;
        const int c = ((ks * 2 + fh) ^ swz) * 16;
        if (i < FM) {
            if (CA)
                fa[set][i] = read_across(s_t + slot + xa[i] + ks * (KROWS / KS) * BM * (int)sizeof(T), BM);
            else
                fa[set][i] = *reinterpret_cast<const V *>(la + slot + c + i * 32 * LN_BK);
        } else {
            if (CB)
                fb[set][i - FM] = read_across(s_t + fwd(slot, 1) + xb[i - FM] + ks * (KROWS / KS) * BN * (int)sizeof(T), BN);
            else
                fb[set][i - FM] = *reinterpret_cast<const V *>(lb + fwd(slot, 1) + c + (i - FM) * 32 * LN_BK);
        }
    };
    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;
    // the products of set SET; between them the fragments of step `ks` (of the stage at `slot`) into the other set and half of the
    // fetches of an operand's stage `sf`, from the q0-th on, into slot `to`
    auto step = [&](auto SET, auto WHOLE, bool reading, int slot, int ks, bool fetching, auto IS_A, int64_t sf, int q0, int to) {
        constexpr int set = decltype(SET)::value;
        using OTHER = std::integral_constant<int, 1 - set>;
        constexpr bool is_a = decltype(IS_A)::value;
        // (parts outside: no product waits for the one before it)
        constexpr int NP = FM * FN, NT = NP * P::PARTS, NR = FM + FN, HALF = (is_a ? NA : NB) / 2;
        // (a fold, not a loop: 64 products of float32 would not be unrolled, and their fragments lie in scratch memory)
        ln_each(std::make_integer_sequence<int, NT>(), [&](auto TT) {
            constexpr int t = decltype(TT)::value, a = t % NP / FN, b = t % NP % FN;
#pragma unroll
            for (int i = t * NR / NT; i < (t + 1) * NR / NT; ++i)
                if (reading)
                    frag(OTHER(), slot, ks, i);
            acc[a][b] = P::mfma(fb[set][b], fa[set][a], acc[a][b], t / NP);
#pragma unroll
            for (int q = t * HALF / NT; q < (t + 1) * HALF / NT; ++q)
                if (fetching)
                    fetch(WHOLE, IS_A, sf, q0 + q, to);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    using OF_A = std::true_type;
    using OF_B = std::false_type;
    // stage s, its A at `slot`; WHOLE: stages s + 1 and s + 2 exist and are filled by the contraction
    auto body = [&](auto WHOLE, int64_t s, int slot) {
        constexpr bool whole = decltype(WHOLE)::value;
        const bool more = whole || s + 1 < s_hi, more2 = whole || s + 2 < s_hi;
        step(S0(), WHOLE, true, slot, 1, more, OF_B(), s + 1, NB / 2, fwd(slot, 3));
        step(S1(), WHOLE, true, slot, 2, more2, OF_A(), s + 2, 0, fwd(slot, 4));
        step(S0(), WHOLE, true, slot, 3, more2, OF_A(), s + 2, NA / 2, fwd(slot, 4));
        // this wave has read stage s, and its part of s + 1 has landed (A(s+2), the last NA fetches, may be under way)
        if (more2)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(NA) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        step(S1(), WHOLE, more, fwd(slot, 2), 0, more2, OF_B(), s + 2, 0, slot);
    };

    if (s_lo < s_hi) {
        using ANY = std::false_type;
#pragma unroll
        for (int q = 0; q < NA; ++q)
            fetch(ANY(), OF_A(), s_lo, q, 0);
#pragma unroll
        for (int q = 0; q < NB; ++q)
            fetch(ANY(), OF_B(), s_lo, q, SLOT);
        if (s_lo + 1 < s_hi) {
#pragma unroll
            for (int q = 0; q < NA; ++q)
                fetch(ANY(), OF_A(), s_lo + 1, q, 2 * SLOT);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NA) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (s_lo + 1 < s_hi)
#pragma unroll
            for (int q = 0; q < NB / 2; ++q)
                fetch(ANY(), OF_B(), s_lo + 1, q, 3 * SLOT);
#pragma unroll
        for (int i = 0; i < FM + FN; ++i)
            frag(S0(), 0, 0, i);
        const int64_t s_fast = min(s_hi, last < 0 ? s_hi : last) - 2;
        int64_t s = s_lo;
        int slot = 0;
        for (; s < s_fast; ++s, slot = fwd(slot, 2))
            body(std::true_type(), s, slot);
        for (; s < s_hi; ++s, slot = fwd(slot, 2))
            body(ANY(), s, slot);
    }
    __syncthreads();  // the stages have been read: their memory buffers the output
    if (g.nsplit > 1)
        ln_store_tile<DT, FM, FN, true>(g, at, acc, reinterpret_cast<float *>(s_t), wid, wr * TM, wc * TN, lane);
    else
        ln_store_tile<DT, FM, FN, false>(g, at, acc, reinterpret_cast<float *>(s_t), wid, wr * TM, wc * TN, lane);
}

// ---- few rows: the weights are read once, and that is the time
// A workgroup computes 16 columns of up to 16 MB rows: its NW waves share the contraction in 128-byte lines, both operands
// come straight from memory into the matrix operands (16 x 16 products; 16 bytes a lane, rows of any alignment), and the
// waves' sums are added up in LDS in order.  One launch and no scratch: what a single query costs is a launch and the
// weights' way through memory.
template <int DT>
struct ln_small;
template <>
struct ln_small<0> {
    static __device__ __forceinline__ f32x4 mfma(f32x4 a, f32x4 b, f32x4 c)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i)  // (lane quarter h holds columns 4 h .. 4 h + 3: the i-th product takes columns 4 h + i)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};
template <>
struct ln_small<1> {
    static __device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct ln_small<2> {
    static __device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

template <int DT, int MB, int NW>
__global__ __launch_bounds__(NW * 64) void k_linear_few(ln_gemm g)
{
    using P = ln_type<DT>;
    using T = typename P::T;
    using V = typename P::V;
    constexpr int VE = P::VE, LINE = 128 / (int)sizeof(T), HALVES = LINE / (4 * VE);
    static_assert(HALVES == 2, "a line is two steps of four 16-byte pieces");
    constexpr int AHEAD = MB == 1 ? 4 : 2;  // lines whose loads are under way together
    __shared__ f32x4 s_sum[NW][MB][64];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, piece = lane >> 4;
    const int64_t col0 = (int64_t)blockIdx.x * 16;
    const T *const w = reinterpret_cast<const T *>(g.b + min(col0 + r, g.n - 1) * g.ldb);  // (rows past the end: any, not stored)
    const T *x[MB];
#pragma unroll
    for (int q = 0; q < MB; ++q)
        x[q] = reinterpret_cast<const T *>(g.a + min((int64_t)q * 16 + r, g.m - 1) * g.lda);
    f32x4 acc[MB];
#pragma unroll
    for (int q = 0; q < MB; ++q)
        acc[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // 16 bytes of a row from column c on, zeros behind the contraction's end: a piece that would reach past it starts earlier, at
    // the last whole one, and what that repeats is dropped (from both operands alike: which lane holds a column is all one)
    auto read = [&](const T *row, int64_t c) {
        V v;
        if (g.k >= VE) {
            const int64_t start = min(c, g.k - VE), drop = c - start;
            const ln_u128 raw = *reinterpret_cast<const ln_u128 *>(row + start);
            __builtin_memcpy(&v, &raw, 16);
#pragma unroll
            for (int u = 0; u < VE; ++u)
                v[u] = u < drop ? (T)0.0f : v[u];
        } else {
#pragma unroll
            for (int u = 0; u < VE; ++u)
                v[u] = c + u < g.k ? row[c + u] : (T)0.0f;
        }
        return v;
    };
    const int64_t lines = (g.k + LINE - 1) / LINE, whole = g.k / LINE;
    int64_t l = wid;
    for (; l + (AHEAD - 1) * NW < whole; l += AHEAD * NW) {
        V vw[AHEAD][2], vx[AHEAD][2][MB];
#pragma unroll
        for (int d = 0; d < AHEAD; ++d)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t c = (l + d * NW) * LINE + (h * 4 + piece) * VE;
                ln_u128 raw = *reinterpret_cast<const ln_u128 *>(w + c);
                __builtin_memcpy(&vw[d][h], &raw, 16);
#pragma unroll
                for (int q = 0; q < MB; ++q) {
                    raw = *reinterpret_cast<const ln_u128 *>(x[q] + c);
                    __builtin_memcpy(&vx[d][h][q], &raw, 16);
                }
            }
#pragma unroll
        for (int d = 0; d < AHEAD; ++d)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int q = 0; q < MB; ++q)
                    acc[q] = ln_small<DT>::mfma(vw[d][h], vx[d][h][q], acc[q]);
    }
    for (; l < lines; l += NW)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t c = l * LINE + (h * 4 + piece) * VE;
            const V vw = read(w, c);
#pragma unroll
            for (int q = 0; q < MB; ++q)
                acc[q] = ln_small<DT>::mfma(vw, read(x[q], c), acc[q]);
        }
#pragma unroll
    for (int q = 0; q < MB; ++q)
        s_sum[wid][q][lane] = acc[q];
    __syncthreads();
    // cell (row 16 q + r, column 4 piece + u) of the tile is register u of lane (piece, r)
    for (int t = threadIdx.x; t < MB * 256; t += NW * 64) {
        const int q = t >> 8, row = (t >> 4) & 15, col = t & 15;
        const int64_t i = q * 16 + row, j = col0 + col;
        if (i >= g.m || j >= g.n)
            continue;
        float v = 0.0f;
#pragma unroll
        for (int s = 0; s < NW; ++s)
            v += reinterpret_cast<const float *>(&s_sum[s][q][(col >> 2) * 16 + row])[col & 3];
        if (g.bias)
            v += (float)((const T *)g.bias)[j];
        if (g.preact)
            ((T *)g.preact)[i * g.ldp + j] = (T)v;
        v = ln_act<DT == 0>(g.act, v);
        if (g.residual)
            v += (float)((const T *)g.residual)[i * g.ldr + j];
        ((T *)g.out)[i * g.ldo + j] = (T)v;
    }
}

// the sums over the splits, in order, and the epilogue
template <int DT>
__global__ __launch_bounds__(256) void k_linear_join(ln_gemm g)
{
    using T = typename ln_type<DT>::T;
    constexpr int VE = ln_type<DT>::VE;
    const int64_t per_row = (g.n + VE - 1) / VE, total = g.m * per_row;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
        const int64_t i = t / per_row, j = (t - i * per_row) * VE, left = g.n - j;
        const bool whole = left >= VE;
        T b[VE], res[VE];
        float v[VE], bias[VE];
#pragma unroll
        for (int u = 0; u < VE; ++u) {
            v[u] = 0.0f;
            b[u] = res[u] = (T)0.0f;
        }
        if (g.bias)
            ln_read<DT, VE>((const T *)g.bias + j, whole, left, b);
        if (g.residual)
            ln_read<DT, VE>((const T *)g.residual + i * g.ldr + j, whole, left, res);
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
#pragma unroll
        for (int u = 0; u < VE; ++u)
            bias[u] = (float)b[u];
        ln_with_act(g.act, [&](auto ACT) { ln_put<DT, VE>(g, i, j, left, ln_cells<DT, VE>(g, decltype(ACT)::value, bias, res, v)); });
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

// out[r][c] = dz = dy act'(z), rounded to the operands' type once (what the two products of the backward pass read; rows of
// ldo elements, zeros behind `cols`; nullptr: not wanted), and sums[tile row][c] = the column sums of the unrounded dz
// over a tile's 64 rows (nullptr: not wanted).  Bound by memory: 8192 x 4096 bfloat16 with silu (201 MB) in 46 us (a copy
// of as many bytes takes 42).
template <int DT>
__global__ __launch_bounds__(256) void k_linear_dz(int64_t rows, int64_t cols, const void *dy_, int64_t ld, int act, const void *z_, int64_t ldz, void *out_, int64_t ldo, float *sums)
{
    using T = typename ln_type<DT>::T;
    constexpr int VE = ln_type<DT>::VE, PIECES = 64 / VE, STEP = 256 / PIECES, PASSES = 64 / STEP;  // rows a pass
    __shared__ float s_sum[4][64];
    const T *dy = (const T *)dy_, *z = (const T *)z_;
    T *out = (T *)out_;
    const int tid = threadIdx.x, pr = tid / PIECES, pc = tid % PIECES * VE;
    const int64_t ntx = (cols + 63) / 64, nty = (rows + 63) / 64, tiles = ntx * nty;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t ty = tile / ntx, r0 = ty * 64, c0 = (tile - ty * ntx) * 64, c = c0 + pc;
        const bool whole = c + VE <= cols;
        T v[PASSES][VE], zz[PASSES][VE];
        auto read = [&](const T *from, int64_t stride, T(&to)[PASSES][VE]) {
#pragma unroll
            for (int p = 0; p < PASSES; ++p) {
                const int64_t r = r0 + p * STEP + pr;
                if (r < rows && c < cols) {
                    ln_read<DT, VE>(from + r * stride + c, whole, cols - c, to[p]);
                } else {
#pragma unroll
                    for (int u = 0; u < VE; ++u)
                        to[p][u] = (T)0.0f;
                }
            }
        };
        read(dy, ld, v);
        if (act != ACT_NONE)
            read(z, ldz, zz);
        float sum[VE];
#pragma unroll
        for (int u = 0; u < VE; ++u)
            sum[u] = 0.0f;
        ln_with_act(act, [&](auto ACT) {
#pragma unroll
            for (int p = 0; p < PASSES; ++p) {
                const int64_t r = r0 + p * STEP + pr;
#pragma unroll
                for (int u = 0; u < VE; ++u) {
                    float d = (float)v[p][u];
                    if (decltype(ACT)::value != ACT_NONE)
                        d = r < rows && c + u < cols ? d * ln_slope<DT == 0>(decltype(ACT)::value, (float)zz[p][u]) : 0.0f;
                    sum[u] += d;
                    v[p][u] = (T)d;
                }
                if (out && r < rows && c < ldo)
                    __builtin_memcpy(__builtin_assume_aligned(out + r * ldo + c, 16), v[p], 16);
            }
        });
        if (sums) {  // over the rows that the lanes of a wave hold, then over the waves
#pragma unroll
            for (int u = 0; u < VE; ++u) {
                for (int d = PIECES; d < 64; d <<= 1)
                    sum[u] += __shfl_xor(sum[u], d);
                if ((tid & 63) < PIECES)
                    s_sum[tid >> 6][pc + u] = sum[u];
            }
            __syncthreads();
            if (tid < 64 && c0 + tid < cols)
                sums[ty * cols + c0 + tid] = s_sum[0][tid] + s_sum[1][tid] + s_sum[2][tid] + s_sum[3][tid];
            __syncthreads();
        }
    }
}

// dbias[c] = the tiles' column sums added up, in one order: a wave per 64 columns and sixteenth of the tiles, eight loads under way
// (4096 columns, 128 tiles: 11 us by four waves and a load at a time, 5 so)
template <int DT>
__global__ __launch_bounds__(1024) void k_linear_bias_grad(int64_t parts, int64_t cols, const float *sums, void *out_)
{
    using T = typename ln_type<DT>::T;
    constexpr int W = 16, AHEAD = 8;
    __shared__ float s_sum[W][64];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    for (int64_t c0 = (int64_t)blockIdx.x * 64; c0 < cols; c0 += (int64_t)gridDim.x * 64) {
        float v = 0.0f;
        if (c0 + lane < cols) {
            const float *from = sums + c0 + lane;
            for (int64_t p = wid; p < parts; p += W * AHEAD) {
                float part[AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i)
                    part[i] = p + i * W < parts ? from[(p + i * W) * cols] : 0.0f;
#pragma unroll
                for (int i = 0; i < AHEAD; ++i)
                    v += part[i];
            }
        }
        s_sum[wid][lane] = v;
        __syncthreads();
        if (wid == 0 && c0 + lane < cols) {
            v = 0.0f;
#pragma unroll
            for (int i = 0; i < W; ++i)
                v += s_sum[i][lane];
            ((T *)out_)[c0 + lane] = (T)v;
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------- host side
constexpr int64_t LN_MAX_TILES = (int64_t)1 << 24;  // a launch holds less than 2^32 threads
template <int DT, int BM, int BN, bool CA, bool CB, typename OFF = uint32_t>
int launch_tiles(skm_ctx *ctx, const ln_gemm &g)
{
    const int64_t tiles = skm_ceil_div(g.m, BM) * skm_ceil_div(g.n, BN);
    SKM_REQUIRE(tiles * g.nsplit < LN_MAX_TILES, SKM_E_OVERFLOW, "skm_linear: too many tiles");
    k_linear<DT, BM, BN, CA, CB, OFF><<<(unsigned)(tiles * g.nsplit), 256, 0, ctx->stream>>>(g);
    return skm_check_launch("k_linear");
}

// What a workgroup of each tile costs, in microseconds measured on MI355X: a 128-byte stage of the contraction with the chip
// idle around it, the same with every compute unit busy (then the clock, held down by the chip's power, and what the units
// share bound it), and the rest of the tile (first fetch, epilogue).  16-bit types / float32 (bound by its matrix rate).
// The plan with the least estimate is taken; e.g. k = 6592 (16 bits), m x n = 3383 x 1000, measured in all: 256 x 256 in 4 parts 58,
// 256 x 128 in 2 parts 53, 128 x 128 59, 128 x 64 57, 64 x 64 74; 512 x 512, k = 4096: 26 / 19 / 16 / 14 / 12 at the best number of
// parts of each; 4096 x 4096, k = 4096: 108 / 133 / 151 / 192 / 208; float32 10000 x 1000, k = 6561, at the best number
// of parts of each: 1060 / 1044 / 1022 / 1059 / 1074.
struct ln_tile {
    int bm, bn;
    float idle[2], busy[2], rest;
};
const ln_tile LN_TILES[] = {
    {256, 256, {1.03f, 7.25f}, {1.44f, 7.4f}, 10.0f},
    {256, 128, {0.53f, 3.72f}, {0.75f, 3.82f}, 5.0f},
    {128, 128, {0.29f, 1.93f}, {0.53f, 1.94f}, 1.5f},
    {128, 64, {0.21f, 1.04f}, {0.30f, 1.01f}, 1.2f},
    {64, 64, {0.16f, 0.59f}, {0.20f, 0.51f}, 0.7f},
};

struct ln_plan {
    int tile = 2, nsplit = 1;
    int64_t stages_per_split = 0;
};

ln_plan plan_of(int dtype, int64_t cus, int64_t m, int64_t n, int64_t stages)
{
    ln_plan best;
    double best_us = 1e300;
    const int kind = dtype == 0;
    for (int t = 0; t < 5; ++t) {
        const ln_tile &c = LN_TILES[t];
        const int64_t tiles = skm_ceil_div(m, c.bm) * skm_ceil_div(n, c.bn);
        if (t && tiles >= LN_MAX_TILES)
            continue;
        for (int64_t want = 1; want <= 32; ++want) {
            const int64_t per = std::max<int64_t>(skm_ceil_div(stages, want), 1), parts = std::max<int64_t>(skm_ceil_div(stages, per), 1);
            if (parts != want || (want > 1 && (per < 4 || tiles * want > 16 * cus)))
                continue;
            const double blocks = (double)tiles * want, load = std::min(1.0, blocks / (double)cus);
            const double stage = c.idle[kind] + (c.busy[kind] - c.idle[kind]) * load;
            double us = (double)skm_ceil_div((int64_t)blocks, cus) * ((double)per * stage + c.rest);
            if (want > 1)  // the parts' sums travel through the caches, and a second kernel starts
                us += 4.0 + 8.0 * (double)want * (double)m * (double)n / 12e6;
            if (us < best_us) {
                best_us = us;
                best.tile = t;
                best.nsplit = (int)want;
                best.stages_per_split = per;
            }
        }
    }
    return best;
}

// C = A B^T with the epilogue; a and b are as `ready` leaves them, CA / CB: across the contraction.
template <int DT, bool CA = false, bool CB = false>
int gemm(skm_ctx *ctx, ln_gemm g)
{
    const int64_t stages = skm_ceil_div(g.k * (int64_t)elem_bytes(DT), LN_BK);
    ln_plan plan = plan_of(DT, ctx->usable_cus, g.m, g.n, stages);
    const bool wide = std::max(g.lda, g.ldb) >= ((int64_t)1 << 24);  // 256 rows may span 2^32 bytes
    g.stages = stages;
    g.nsplit = plan.nsplit;
    g.stages_per_split = plan.stages_per_split;
    if (g.nsplit > 1) {
        void *p;
        g.ldq = skm_ceil_div(g.n, 4) * 4;
        SKM_TRY(skm_ws(ctx, WS_D, sizeof(float) * (size_t)g.nsplit * (size_t)g.m * (size_t)g.ldq, &p));
        g.partial = (float *)p;
    }
    {
        SKM_PROF(ctx, "k_linear");
        if (wide)
            SKM_TRY((launch_tiles<DT, 128, 128, CA, CB, uint64_t>(ctx, g)));
        else if (plan.tile == 0)
            SKM_TRY((launch_tiles<DT, 256, 256, CA, CB>(ctx, g)));
        else if (plan.tile == 1)
            SKM_TRY((launch_tiles<DT, 256, 128, CA, CB>(ctx, g)));
        else if (plan.tile == 2)
            SKM_TRY((launch_tiles<DT, 128, 128, CA, CB>(ctx, g)));
        else if (plan.tile == 3)
            SKM_TRY((launch_tiles<DT, 128, 64, CA, CB>(ctx, g)));
        else
            SKM_TRY((launch_tiles<DT, 64, 64, CA, CB>(ctx, g)));
    }
    if (g.nsplit > 1) {
        SKM_PROF(ctx, "k_linear_join");
        k_linear_join<DT><<<skm_grid_cap(ctx, skm_ceil_div(g.m * skm_ceil_div(g.n, ln_type<DT>::VE), 256), 16), 256, 0, ctx->stream>>>(g);
        SKM_TRY(skm_check_launch("k_linear_join"));
    }
    return SKM_OK;
}

// Few rows read the weights straight from memory.  Measured, microseconds, 1 / 16 / 32 rows of k = 4096, n = 1000, bfloat16: 6.8 / 9.0 /
// 12.9 against 11.2 / 13.2 / 13.2 by tiles; k = 16384, n = 4096: 26 / 32 / 44 against 30 / 30 / 31; k = 300, 64 rows: 6.8 against 12.7.
// (A launch holds less than 2^32 threads: 2^25 columns are 2^21 workgroups of up to 2^10.)
bool few_rows(int64_t m, int64_t n, int64_t kbytes) { return (m <= 16 || (m <= 64 && kbytes <= 1024)) && n <= (int64_t)1 << 25; }

template <int DT, int MB>
int launch_few(skm_ctx *ctx, const ln_gemm &g)
{
    const int64_t groups = skm_ceil_div(g.n, 16);
    SKM_PROF(ctx, "k_linear_few");
    if (g.k * (int64_t)elem_bytes(DT) >= 4096)
        k_linear_few<DT, MB, 16><<<(unsigned)groups, 1024, 0, ctx->stream>>>(g);
    else
        k_linear_few<DT, MB, 4><<<(unsigned)groups, 256, 0, ctx->stream>>>(g);
    return skm_check_launch("k_linear_few");
}

template <int DT>
int launch_few(skm_ctx *ctx, const ln_gemm &g)
{
    if (g.m <= 16)
        return launch_few<DT, 1>(ctx, g);
    if (g.m <= 32)
        return launch_few<DT, 2>(ctx, g);
    return launch_few<DT, 4>(ctx, g);
}

// Rows of scratch copies start on 128-byte lines, as a stage of a row is one: bfloat16 3383 x 1000, k = 6561, 54 us of product; with rows of
// 13136 bytes (16-byte pieces) 63.
constexpr int64_t row_elems(int64_t cols, int64_t es) { return skm_ceil_div(cols * es, 128) * 128 / es; }

// The operand as the product reads it: where it lies if its rows start on 4-byte boundaries and hold whole units (words of 4 bytes,
// across the contraction 16-byte pieces), else (16-bit types with odd strides or addresses, odd lengths) a padded copy in scratch.
// Reading 4-byte rows as they lie: bfloat16 8192 x 4096, k = 4096: 252 us against 234 for 16-byte rows and 277 by way of a
// copy; float32 10000 x 1000, k = 6561: the same time within 1 %, where the copies took 104 us of 1136.
template <int DT>
int ready(skm_ctx *ctx, int slot, bool across, int64_t rows, int64_t cols, const void *in, int64_t ld, const uint8_t **out, int64_t *ld_bytes)
{
    constexpr int64_t es = (int64_t)elem_bytes(DT), VE = ln_type<DT>::VE;
    if (((uintptr_t)in & 3) == 0 && (rows == 1 || ld * es % 4 == 0) && cols * es % (across ? 16 : 4) == 0) {
        *out = (const uint8_t *)in;
        *ld_bytes = rows == 1 ? 0 : ld * es;
        return SKM_OK;
    }
    const int64_t ldo = row_elems(cols, es);
    void *p;
    SKM_TRY(skm_ws(ctx, slot, (size_t)(rows * ldo * es), &p));
    SKM_PROF(ctx, "k_linear_pad");
    k_linear_pad<DT><<<skm_grid_cap(ctx, skm_ceil_div(rows * (ldo / VE), 256), 16), 256, 0, ctx->stream>>>(rows, cols, in, ld, p, ldo);
    SKM_TRY(skm_check_launch("k_linear_pad"));
    *out = (const uint8_t *)p;
    *ld_bytes = ldo * es;
    return SKM_OK;
}

}  // namespace

template <int DT>
int skm_linear_forward(skm_ctx *ctx, int act, int64_t m, int64_t n, int64_t k, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *bias, const void *residual,
            int64_t ldr, void *preact, int64_t ldp, void *y, int64_t ldy)
{
    ln_gemm g = {};
    g.m = m;
    g.n = n;
    g.k = k;
    g.act = act;
    g.bias = bias;
    g.residual = residual;
    g.ldr = ldr;
    g.preact = preact;
    g.ldp = ldp;
    g.out = y;
    g.ldo = ldy;
    if (few_rows(m, n, k * (int64_t)elem_bytes(DT))) {
        constexpr int64_t es = (int64_t)elem_bytes(DT);
        g.a = (const uint8_t *)x;
        g.lda = ldx * es;
        g.b = (const uint8_t *)w;
        g.ldb = ldw * es;
        return launch_few<DT>(ctx, g);
    }
    SKM_TRY(ready<DT>(ctx, WS_A, false, m, k, x, ldx, &g.a, &g.lda));
    SKM_TRY(ready<DT>(ctx, WS_B, false, n, k, w, ldw, &g.b, &g.ldb));
    return gemm<DT>(ctx, g);
}

template <int DT>
int skm_linear_gradients(skm_ctx *ctx, int act, int64_t m, int64_t n, int64_t k, const void *dy, int64_t lddy, const void *z, int64_t ldz, const void *x, int64_t ldx, const void *w,
             int64_t ldw, void *dx, int64_t lddx, void *dw, int64_t lddw, void *dbias)
{
    constexpr int64_t es = (int64_t)elem_bytes(DT);
    // dz: dy itself where nothing changes it and the products can read it as it lies
    const bool make_dz = (dx || dw) && (act != ACT_NONE || ((uintptr_t)dy & 3) || (m > 1 && lddy * es % 4) || n * es % (dw ? 16 : 4));
    const uint8_t *dz = (const uint8_t *)dy;
    int64_t lddz = m == 1 ? 0 : lddy * es;
    if (dbias || make_dz) {
        const int64_t ldo = row_elems(n, es), parts = skm_ceil_div(m, 64);
        void *to = nullptr, *sums = nullptr;
        if (make_dz) {
            SKM_TRY(skm_ws(ctx, WS_A, (size_t)(m * ldo * es), &to));
            dz = (const uint8_t *)to;
            lddz = ldo * es;
        }
        if (dbias)
            SKM_TRY(skm_ws(ctx, WS_C, sizeof(float) * (size_t)(parts * n), &sums));
        {
            SKM_PROF(ctx, "k_linear_dz");
            k_linear_dz<DT><<<skm_grid_cap(ctx, parts * skm_ceil_div(n, 64), 64), 256, 0, ctx->stream>>>(m, n, dy, lddy, act, z, ldz, to, ldo, (float *)sums);
            SKM_TRY(skm_check_launch("k_linear_dz"));
        }
        if (dbias) {
            k_linear_bias_grad<DT><<<skm_grid_cap(ctx, skm_ceil_div(n, 64), 16), 1024, 0, ctx->stream>>>(parts, n, (const float *)sums, dbias);
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
        g.out = dx;
        g.ldo = lddx;
        SKM_TRY(ready<DT>(ctx, WS_B, true, n, k, w, ldw, &g.b, &g.ldb));
        SKM_TRY((gemm<DT, false, true>(ctx, g)));
    }
    if (dw) {
        ln_gemm g = {};
        g.m = n;
        g.n = k;
        g.k = m;
        g.a = dz;
        g.lda = lddz;
        g.out = dw;
        g.ldo = lddw;
        SKM_TRY(ready<DT>(ctx, WS_E, true, m, k, x, ldx, &g.b, &g.ldb));
        SKM_TRY((gemm<DT, true, true>(ctx, g)));
    }
    return SKM_OK;
}
