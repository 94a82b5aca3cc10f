// Log probabilities of given labels under a row of class scores, with the entropy, the best alternatives and the gradient:
// what follows a materialised score block (skm_cosine_csr against family totals, skm_linear) where skm_row_top2 only
// ranks it.  No reference counterpart in this form: the reference turns the difference of the two best scores into a
// confidence by a table (snekmer/rules/apply.smk:312-328, rules/learn.smk:831-849).
//
//   allowed classes of a row: mask != 0 and s > -inf;   m = max s;   d_j = (s_j - m) / T
//   S = sum over d_j < 0 of exp(d_j);   c = number of d_j == 0;   l = log1p(S + c - 1)
//   log p_j = d_j - l;   H = l - (sum of exp(d_j) d_j) / (S + c)
//
// The largest entries are counted (c), not added: where one class holds nearly all of the mass, S is what is left and
// log1p keeps it to its own precision; l and -sum(e d) have one sign, so H does not cancel either.  Differences are taken
// before the scale 1 / T (s - m cannot overflow where s / T would) and the exponentials are powers of two of
// d * (log2 e / T).
//
// One pass over the scores, a wave at a time: a tile of 1024 scores in registers (16 a lane, from 16-byte loads of any
// alignment), its maximum, then the running (m, c, S, Q) of an online softmax - m and c the wave's, S and Q the lanes' -
// and the running list of the k best.  Rows with many tiles are shared by the waves of a workgroup, few long rows by
// several workgroups whose partial states a second kernel joins.
//
// The k best of a tile: its lanes form G >= k groups (4, 8, 16, 32 for k up to 4, 8, 12, 16; the single lanes for k = 2), and no
// element below the k-th largest of the group maxima can be among them, so only those above it (hardly more than k) are collected in LDS and ranked; equal ones
// are taken in index order until k are held.  After the first tile only elements above the list's last one are looked at,
// which costs one comparison a tile.
//
// Many short rows (the learn / apply block) are bound by instructions, not by memory: a wave takes up to eight rows, holds
// row r's state in lane r, and does logarithms, divisions and label look-ups for all of them at once.
#include <algorithm>
#include <cmath>

#include "skm_common.h"
#include "skm_logprob.h"

namespace {

constexpr int LP_E = 16;            // scores a lane holds of a tile
constexpr int LP_TILE = 64 * LP_E;  // 1024
constexpr int LP_KMAX = 16;
constexpr int LP_BUF = 64 + LP_TILE / 2 + 2 * LP_KMAX;  // candidates a wave can hold: 64, half a tile, and the list that comes of them
constexpr int LP_MAX_SPLITS = 64;
constexpr float LP_INF = __builtin_inff();

struct lp_args {
    int64_t rows, cols;
    const void *scores;
    int64_t ld;
    const uint8_t *mask;
    int64_t ldmask;  // 0: one row for all
    const void *labels;
    int label64, k;
    float c2, inv_t;  // log2(e) / T, 1 / T
    float *logp, *entropy, *stats;
    int32_t *top_index;
    float *top_logp;
    uint32_t *err;
    // split rows only
    int nsplit;
    int64_t tiles_per_split;
    float4 *part;       // [rows][nsplit]: m, S, Q, c (negative: a score that has no distribution)
    uint2 *part_lists;  // [rows][nsplit][LP_KMAX]: (score, index), index 0xFFFFFFFF behind the last
};

// ---- wave helpers: results uniform over the wave
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lp_dpp(uint32_t old, uint32_t x)
{
    return (uint32_t)__builtin_amdgcn_update_dpp((int)old, (int)x, CTRL, ROWS, 0xF, false);
}

template <typename F>
__device__ __forceinline__ uint32_t lp_reduce(uint32_t x, uint32_t identity, F &&op)
{
    x = op(x, lp_dpp<0xB1, 0xF>(identity, x));   // lane ^ 1
    x = op(x, lp_dpp<0x4E, 0xF>(identity, x));   // lane ^ 2
    x = op(x, lp_dpp<0x141, 0xF>(identity, x));  // 7 - lane within 8
    x = op(x, lp_dpp<0x140, 0xF>(identity, x));  // 15 - lane within 16
    x = op(x, lp_dpp<0x142, 0xA>(identity, x));  // lane 15 of rows 0, 2 into rows 1, 3
    x = op(x, lp_dpp<0x143, 0xC>(identity, x));  // lane 31 into rows 2, 3
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

// NaN wins
__device__ __forceinline__ float lp_wave_max(float v)
{
    return __uint_as_float(lp_reduce(__float_as_uint(v), 0xFF800000u, [](uint32_t a, uint32_t b) {
        return __float_as_uint(__builtin_elementwise_maximum(__uint_as_float(a), __uint_as_float(b)));
    }));
}
__device__ __forceinline__ float lp_wave_sum(float v)
{
    return __uint_as_float(lp_reduce(__float_as_uint(v), 0u, [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
__device__ __forceinline__ float lp_wave_min(float v)
{
    return __uint_as_float(lp_reduce(__float_as_uint(v), 0x7F800000u, [](uint32_t a, uint32_t b) { return __float_as_uint(fminf(__uint_as_float(a), __uint_as_float(b))); }));
}
__device__ __forceinline__ uint32_t lp_wave_umax(uint32_t v)
{
    return lp_reduce(v, 0u, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

__device__ __forceinline__ uint64_t lp_readlane64(uint64_t v, int lane)
{
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
    return ((uint64_t)hi << 32) | lo;
}

__device__ __forceinline__ int lp_below(uint64_t mask)  // set bits below this lane
{
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// (score, index) as one word whose order is the alternatives': larger scores first, lower indices first among equals
__device__ __forceinline__ uint64_t lp_key(float v, uint32_t index)
{
    uint32_t b = __float_as_uint(v + 0.0f);  // -0 and 0 are equal scores
    b ^= (b >> 31) ? 0xFFFFFFFFu : 0x80000000u;
    return ((uint64_t)b << 32) | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ float lp_key_score(uint64_t key)
{
    uint32_t b = (uint32_t)(key >> 32);
    b ^= (b >> 31) ? 0x80000000u : 0xFFFFFFFFu;
    return __uint_as_float(b);
}
__device__ __forceinline__ uint32_t lp_key_index(uint64_t key) { return 0xFFFFFFFFu - (uint32_t)key; }

// ---- loads
struct __attribute__((packed)) lp_u128 {  // 16 bytes at any address
    uint32_t w[4];
};
struct __attribute__((packed)) lp_u64 {
    uint32_t w[2];
};
struct __attribute__((packed)) lp_u32 {
    uint32_t w[1];
};

template <int DT>
struct lp_type;
template <>
struct lp_type<0> {
    using T = float;
    static constexpr int VE = 4;
    static __device__ __forceinline__ float one(T v) { return v; }
    static __device__ __forceinline__ float pick(const lp_u128 &r, int u) { return __uint_as_float(r.w[u]); }
    static __device__ __forceinline__ T round(float v) { return v; }
};
template <>
struct lp_type<1> {
    using T = _Float16;
    static constexpr int VE = 8;
    static __device__ __forceinline__ float one(T v) { return (float)v; }
    static __device__ __forceinline__ float pick(const lp_u128 &r, int u) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(r.w[u >> 1] >> (16 * (u & 1)))); }
    static __device__ __forceinline__ T round(float v) { return (_Float16)v; }
};
template <>
struct lp_type<2> {
    using T = __bf16;
    static constexpr int VE = 8;
    static __device__ __forceinline__ float one(T v) { return (float)v; }
    static __device__ __forceinline__ float pick(const lp_u128 &r, int u) { return __uint_as_float((u & 1) ? r.w[u >> 1] & 0xFFFF0000u : r.w[u >> 1] << 16); }
    static __device__ __forceinline__ T round(float v) { return (__bf16)v; }
};

// One tile of a row on its way: vector v of a lane holds classes (v * 64 + lane) * VE .. of the tile.
template <int DT, int MASK>
struct lp_raw {
    static constexpr int VE = lp_type<DT>::VE, NV = LP_E / VE;
    lp_u128 v[NV];
    uint32_t mask[MASK ? NV : 1][VE / 4];
};

// Where vector v of a lane starts in a tile of which `rem` classes are left: vectors that would reach past the row's end
// start earlier, at its last whole vector (their first elements, which another lane holds, are dropped in lp_unpack): all
// loads are whole, unconditional and inside the row.
template <int VE>
__device__ __forceinline__ int lp_start(int v, int lane, int rem)
{
    return min((v * 64 + lane) * VE, rem - VE);
}

// at, mat: the tile's first score and mask byte; rem <= LP_TILE classes are left there; the row has `cols`
template <int DT, int MASK>
__device__ __forceinline__ void lp_fetch(const typename lp_type<DT>::T *at, const uint8_t *mat, int rem, int64_t cols, int lane, lp_raw<DT, MASK> &raw)
{
    using T = typename lp_type<DT>::T;
    constexpr int VE = lp_raw<DT, MASK>::VE, NV = lp_raw<DT, MASK>::NV;
    if (cols >= VE) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int off = lp_start<VE>(v, lane, rem);
            raw.v[v] = *reinterpret_cast<const lp_u128 *>(at + off);
            if constexpr (MASK && VE == 4) {
                raw.mask[v][0] = reinterpret_cast<const lp_u32 *>(mat + off)->w[0];
            } else if constexpr (MASK) {
                const lp_u64 w = *reinterpret_cast<const lp_u64 *>(mat + off);
                raw.mask[v][0] = w.w[0];
                raw.mask[v][1] = w.w[1];
            }
        }
    } else {  // rows shorter than a vector: as the last elements of one
        T one[VE];
        uint8_t m[VE];
#pragma unroll
        for (int u = 0; u < VE; ++u) {
            const int j = u - (VE - rem);
            one[u] = j >= 0 ? at[j] : (T)0.0f;
            m[u] = MASK && j >= 0 ? mat[j] : 0;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            __builtin_memcpy(&raw.v[v], one, 16);
            if (MASK)
                __builtin_memcpy(raw.mask[v], m, VE);
        }
    }
}

// x[v * VE + u] = the score at lp_start(v) + u, -inf where masked, past the end or held by another lane
template <int DT, int MASK>
__device__ __forceinline__ void lp_unpack(lp_raw<DT, MASK> raw, int rem, int lane, float (&x)[LP_E])
{
    constexpr int VE = lp_raw<DT, MASK>::VE, NV = lp_raw<DT, MASK>::NV;
    // (words that the compiler cannot look into: it would cut the 16-byte loads into the pieces that are used)
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        asm volatile("" : "+v"(raw.v[v].w[0]), "+v"(raw.v[v].w[1]), "+v"(raw.v[v].w[2]), "+v"(raw.v[v].w[3]));
        if (MASK)
#pragma unroll
            for (int h = 0; h < VE / 4; ++h)
                asm volatile("" : "+v"(raw.mask[v][h]));
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int u = 0; u < VE; ++u) {
            float f = lp_type<DT>::pick(raw.v[v], u);
            if (MASK)
                f = ((raw.mask[v][u >> 2] >> (8 * (u & 3))) & 0xFFu) ? f : -LP_INF;
            x[v * VE + u] = f;
        }
    if (rem < LP_TILE) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int drop = (v * 64 + lane) * VE - lp_start<VE>(v, lane, rem);
            if (rem % VE == 0) {  // (all or none of a vector)
#pragma unroll
                for (int u = 0; u < VE; ++u)
                    x[v * VE + u] = drop > 0 ? -LP_INF : x[v * VE + u];
            } else {
#pragma unroll
                for (int u = 0; u < VE; ++u)
                    x[v * VE + u] = u < drop ? -LP_INF : x[v * VE + u];
            }
        }
    }
}

// ---- the running state of a wave
struct lp_state {
    float m = -LP_INF;  // uniform: the largest allowed score so far
    int c = 0;          // uniform: how many scores equal it
    float S = 0.0f, Q = 0.0f;  // this lane's sums of 2^t and 2^t t over t = (s - m) * log2(e) / T < 0
    bool bad = false;   // uniform: a NaN or +inf was allowed: the row has no distribution
    int len = 0;        // uniform: alternatives held, best first, in the wave's buffer
    float tau = -LP_INF;  // the score of the last of k
};

// The n candidates of the buffer as (score, index), of which the first st.len are the sorted list so far: ranked, the best k
// stay.  TIES: equal scores are to be expected (16-bit types).
template <bool TIES>
__device__ __forceinline__ void lp_rank(uint2 *buf, int n, int k, int lane, lp_state &st)
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (n <= 64) {  // a lane a candidate
        const uint2 q = buf[lane];
        const uint64_t key = lane < n ? lp_key(__uint_as_float(q.x), q.y) : 0;
        int rank = 0;
        bool done = false;
        if (st.len == k) {  // a full list and some that may enter it: only those are compared with everybody
            rank = lane < k ? lane : 0;
            for (int j = k; j < n; ++j) {
                const uint64_t s = lp_readlane64(key, j);
                rank += s > key;
                const int behind = __popcll(__ballot(lane < k && key > s));  // (of the list, ahead of candidate j)
                rank += lane == j ? behind : 0;
            }
            done = true;
        } else if (!TIES) {
            const float v = lane < n ? __uint_as_float(q.x) : -LP_INF;
            for (int j = 0; j < n; j += 4)  // (lanes past the end hold -inf)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    rank += __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(v), j + i)) > v;
            const bool mine = lane < n && rank < k;
            if (mine)
                buf[rank] = q;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            done = __ballot(mine && buf[rank].y != q.y) == 0;  // (else equal scores met in one place)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        if (!done) {
            rank = 0;
            for (int j = 0; j < n; ++j)
                rank += lp_readlane64(key, j) > key;
        }
        if (lane < n && rank < k)
            buf[rank] = q;
    } else {  // (rows in rising order, scores that are nearly all equal) one after the other
        uint2 *out = buf + n;  // (n + k stays below the buffer's end: see lp_collect)
#pragma unroll 1
        for (int r = 0; r < k; ++r) {
            uint64_t best = 0;
            int which = 0;
            for (int i = lane; i < n; i += 64) {
                const uint2 q = buf[i];
                const uint64_t a = q.y != 0xFFFFFFFFu ? lp_key(__uint_as_float(q.x), q.y) : 0;
                which = a > best ? i : which;
                best = a > best ? a : best;
            }
            const uint32_t hi = lp_wave_umax((uint32_t)(best >> 32));
            const uint32_t lo = lp_wave_umax((uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
            if (best == (((uint64_t)hi << 32) | lo)) {  // one lane: the indices differ
                out[r] = buf[which];
                buf[which].y = 0xFFFFFFFFu;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        if (lane < k)
            buf[lane] = out[lane];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    st.len = n < k ? n : k;
    if (st.len == k)
        st.tau = __uint_as_float(__builtin_amdgcn_readfirstlane((int)buf[k - 1].x));
}

// A score that at least k elements of the tile reach, close to the k-th largest; -inf if fewer are allowed.
__device__ __forceinline__ float lp_threshold(float lane_max, int k)
{
    // the maxima of G lane groups ...
    float g = lane_max;
    auto up = [&](uint32_t other) { g = fmaxf(g, __uint_as_float(other)); };
    int width = 64;  // lanes of a group
    if (k > 12) {
        width = 2;
    } else if (k > 8) {
        width = 4;
    } else if (k > 4) {
        width = 8;
    } else if (k > 2) {
        width = 16;
    }
    if (k > 2) {
        up(lp_dpp<0xB1, 0xF>(0, __float_as_uint(g)));
        if (width >= 4)
            up(lp_dpp<0x4E, 0xF>(0, __float_as_uint(g)));
        if (width >= 8)
            up(lp_dpp<0x141, 0xF>(0, __float_as_uint(g)));
        if (width >= 16)
            up(lp_dpp<0x140, 0xF>(0, __float_as_uint(g)));
        // ... without the smallest G - k of them
        float thr;
        if (k * width == 64) {
            thr = lp_wave_min(g);
        } else {
            int above = 0;  // groups with a larger maximum
            if (width == 2) {
#pragma unroll
                for (int i = 0; i < 64; i += 2)
                    above += __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(g), i)) > g;
            } else if (width == 4) {
#pragma unroll
                for (int i = 0; i < 64; i += 4)
                    above += __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(g), i)) > g;
            } else if (width == 8) {
#pragma unroll
                for (int i = 0; i < 64; i += 8)
                    above += __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(g), i)) > g;
            } else {
#pragma unroll
                for (int i = 0; i < 64; i += 16)
                    above += __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(g), i)) > g;
            }
            thr = lp_wave_min(above < k ? g : LP_INF);
        }
        if (thr > -LP_INF)
            return thr;
    }
    // k is 1 or 2, or some groups are empty (short rows, few allowed): the k-th largest lane maximum
    float cur = lane_max, thr;
    for (int r = 0;; ++r) {
        thr = lp_wave_max(cur);
        if (r == k - 1 || thr == -LP_INF)
            return thr;
        const int at = __ffsll((unsigned long long)__ballot(cur == thr)) - 1;
        if (((int)threadIdx.x & 63) == at)
            cur = -LP_INF;
    }
}

// the largest float below v (v finite or -inf, which stays)
__device__ __forceinline__ float lp_below_value(float v)
{
    const uint32_t b = __float_as_uint(v + 0.0f);
    return v == -LP_INF ? v : __uint_as_float(b == 0 ? 0x80000001u : (b >> 31) ? b + 1 : b - 1);
}

template <int VE>
__device__ __forceinline__ void lp_collect(const float (&x)[LP_E], float lane_max, float tile_max, uint32_t base, int rem, int k, int lane, uint2 *buf, lp_state &st)
{
    constexpr int NV = LP_E / VE;
    const bool full = st.len == k;
    if (full && !(tile_max > st.tau))
        return;  // ties with the last one lose: their indices are higher
    // what is taken: larger scores than the last of a full list, or those from the threshold on
    const float thr = full ? st.tau : k == 1 ? tile_max : lp_threshold(lane_max, k);
    const float over = full ? thr : lp_below_value(thr);
    uint32_t first[NV];  // indices of the lane's vectors
#pragma unroll
    for (int v = 0; v < NV; ++v)
        first[v] = base + lp_start<VE>(v, lane, rem);
    int n = st.len;
    auto gather = [&](int e, float limit) {
        const bool take = x[e] > limit;
        const uint64_t at = __ballot(take);
        if (at == 0)
            return;
        if (take)
            buf[n + lp_below(at)] = make_uint2(__float_as_uint(x[e]), first[e / VE] + e % VE);
        n += __popcll(at);
    };
#pragma unroll
    for (int e = 0; e < LP_E / 2; ++e)
        gather(e, over);
    if (n <= 64) {
#pragma unroll
        for (int e = LP_E / 2; e < LP_E; ++e)
            gather(e, over);
    }
    // Many at once: scores equal to the threshold, of which only the first that are needed may be taken, or rows in rising
    // order.  Half a tile at a time, ranked in between.
    if (n > 64) {
        n = st.len;
        int above = 0;
#pragma unroll
        for (int e = 0; e < LP_E; ++e) {
            above += __popcll(__ballot(x[e] > thr));
            gather(e, thr);
            if (e == LP_E / 2 - 1 && n > 64) {
                lp_rank<VE == 8>(buf, n, k, lane, st);
                n = st.len;
            }
        }
        int need = full || !(thr > -LP_INF) ? 0 : k - above;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            int before = 0, total = 0;
#pragma unroll
            for (int u = 0; u < VE; ++u) {
                const uint64_t at = __ballot(x[v * VE + u] == thr);
                before += lp_below(at);
                total += __popcll(at);
            }
            if (need > 0 && total > 0) {
#pragma unroll
                for (int u = 0; u < VE; ++u)
                    if (x[v * VE + u] == thr) {
                        if (before < need)
                            buf[n + before] = make_uint2(__float_as_uint(thr), first[v] + u);
                        ++before;
                    }
                n += total < need ? total : need;
                need -= total;
            }
        }
    }
    lp_rank<VE == 8>(buf, n, k, lane, st);
}

template <int VE>
__device__ __forceinline__ void lp_tile(const float (&x)[LP_E], uint32_t base, int rem, float c2, int k, int lane, uint2 *buf, lp_state &st)
{
    float lm = x[0];
#pragma unroll
    for (int e = 1; e < LP_E; ++e)
        lm = __builtin_elementwise_maximum(lm, x[e]);
    const float tm = lp_wave_max(lm);
    if (!(tm < LP_INF)) {
        st.bad = true;
        return;
    }
    if (tm > st.m) {
        if (st.m > -LP_INF) {  // the sums so far, and the former largest ones among them, relative to the new maximum
            const float d = (st.m - tm) * c2, f = __builtin_amdgcn_exp2f(d);
            const float w = st.S + (lane == 0 ? (float)st.c : 0.0f);
            st.S = w * f;
            st.Q = f > 0.0f ? __builtin_fmaf(w, d, st.Q) * f : 0.0f;
        }
        st.m = tm;
        st.c = 0;
    } else if (tm == -LP_INF) {
        return;
    }
#pragma unroll
    for (int e = 0; e < LP_E; ++e) {
        const float t = x[e] - st.m;
        const bool less = t < 0.0f;
        const float t2 = t * c2;
        const float p = less ? __builtin_amdgcn_exp2f(t2) : 0.0f;
        st.c += 64 - __popcll(__ballot(less));
        st.S += p;
        st.Q = __builtin_fmaf(p, fmaxf(t2, -1e30f), st.Q);  // (0 times -inf)
    }
    if (k)
        lp_collect<VE>(x, lm, tm, base, rem, k, lane, buf, st);
}

// Joins n <= 64 partial states: lane p < n holds state p and its sorted list of `len` at lists + p * LP_KMAX (LDS).
// Results uniform (m, c, S, Q, bad, len); the k best go to `out`.
__device__ __forceinline__ void lp_join(float m, float S, float Q, float c, bool bad, int len, const uint2 *lists, int k, float c2, int lane, lp_state &st, uint2 *out)
{
    st = lp_state();
    st.bad = __ballot(bad) != 0;
    if (st.bad)
        return;
    st.m = lp_wave_max(m);
    const bool has = m > -LP_INF;
    const float d = has ? (m - st.m) * c2 : 0.0f, f = __builtin_amdgcn_exp2f(d);
    const bool top = has && m == st.m;
    const float w = S + c;
    st.c = (int)lp_wave_sum(top ? c : 0.0f);
    st.S = lp_wave_sum(top ? S : has ? w * f : 0.0f);
    st.Q = lp_wave_sum(top ? Q : has && f > 0.0f ? (Q + w * d) * f : 0.0f);
    int at = 0;
    auto head_of = [&](int i) {
        const uint2 q = lists[lane * LP_KMAX + i];
        return lp_key(__uint_as_float(q.x), q.y);
    };
    uint64_t head = len > 0 ? head_of(0) : 0;
    for (; st.len < k; ++st.len) {
        const uint32_t hi = lp_wave_umax((uint32_t)(head >> 32));
        if (hi == 0)
            break;  // (no key of a score has a zero upper word)
        const uint32_t lo = lp_wave_umax((uint32_t)(head >> 32) == hi ? (uint32_t)head : 0u);
        const uint64_t best = ((uint64_t)hi << 32) | lo;
        if (head == best) {  // one lane: the indices differ
            out[st.len] = make_uint2(__float_as_uint(lp_key_score(best)), lp_key_index(best));
            ++at;
            head = at < len ? head_of(at) : 0;
        }
    }
}

// The kernel's arguments (its first parameter), read when they are needed: those of the last step would otherwise sit in
// registers, and in spill space, from the start.
__device__ __forceinline__ const lp_args &lp_late_args()
{
    auto *p = (const __attribute__((address_space(4))) lp_args *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const lp_args *)p;
}

// What is written of rows row0 .. row0 + nrows - 1: lane r holds row r's sums (S and Q of the whole row), its list lies at
// lists + r * LP_KMAX.
template <int DT>
__device__ __forceinline__ void lp_finish(int64_t row0, int nrows, float m, float S, float Q, int c, bool bad, int len, const uint2 *lists, int lane)
{
    using P = lp_type<DT>;
    const lp_args &a = lp_late_args();
    const float nan = __builtin_nanf("");
    const float l = m > -LP_INF ? log1pf(S + (float)(c - 1)) : -LP_INF;
    if (lane < nrows) {
        const int64_t row = row0 + lane;
        if (a.stats)
            reinterpret_cast<lp_u64 *>(a.stats)[row] = lp_u64{{__float_as_uint(bad ? nan : m), __float_as_uint(bad ? nan : l)}};
        if (a.entropy)
            a.entropy[row] = bad ? nan : m > -LP_INF ? l - 0.693147180559945f * (Q / (S + (float)c)) : 0.0f;
        if (a.logp) {
            float v = 0.0f;
            const int64_t y = a.label64 ? ((const int64_t *)a.labels)[row] : (int64_t)((const int32_t *)a.labels)[row];
            if (y < -1 || y >= a.cols) {
                v = nan;
                if (a.err)
                    __hip_atomic_store(a.err, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            } else if (y >= 0) {
                if (bad) {
                    v = nan;
                } else if (a.mask && a.mask[row * a.ldmask + y] == 0) {
                    v = -LP_INF;
                } else {
                    const float s = P::one(((const typename P::T *)a.scores)[row * a.ld + y]);
                    v = s > -LP_INF ? (s - m) * a.inv_t - l : -LP_INF;
                }
            }
            a.logp[row] = v;
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int i0 = 0; i0 < nrows * a.k; i0 += 64) {
        const int i = i0 + lane, r = min(i / max(a.k, 1), nrows - 1), at = i - r * a.k;
        const float mr = __shfl(m, r), lr = __shfl(l, r);
        const int lenr = __shfl(len, r);
        const bool badr = __shfl((int)bad, r) != 0;
        if (i < nrows * a.k) {
            const bool there = !badr && at < lenr;
            const uint2 q = there ? lists[r * LP_KMAX + at] : make_uint2(0, 0xFFFFFFFFu);
            if (a.top_index)
                a.top_index[row0 * a.k + i] = (int32_t)q.y;
            if (a.top_logp)
                a.top_logp[row0 * a.k + i] = there ? (__uint_as_float(q.x) - mr) * a.inv_t - lr : badr ? nan : -LP_INF;
        }
    }
}

// classes of a row from tile t on, at most a tile's; opaque, so that what follows from it is not computed ahead of the loops
__device__ __forceinline__ int lp_left(int64_t cols, int64_t t)
{
    int rem = (int)min(cols - t * LP_TILE, (int64_t)LP_TILE);
    rem = __builtin_amdgcn_readfirstlane(rem);
    asm volatile("" : "+s"(rem));
    return rem;
}

// The tiles t0, t0 + step, .. < t1 of one row, each under way while the one before it is worked on.  `next` holds the first
// one; after the last it holds tile 0 of row `then` (no row: below 0).
template <int DT, int MASK>
__device__ __forceinline__ void lp_fetch_tile(const lp_args &a, int64_t row, int64_t t, int lane, lp_raw<DT, MASK> &raw)
{
    using T = typename lp_type<DT>::T;
    lp_fetch<DT, MASK>((const T *)a.scores + row * a.ld + t * LP_TILE, MASK ? a.mask + row * a.ldmask + t * LP_TILE : nullptr,
                       lp_left(a.cols, t), a.cols, lane, raw);
}
template <int DT, int MASK>
__device__ __forceinline__ void lp_walk(const lp_args &a, int64_t row, int64_t t0, int64_t t1, int step, int64_t then, int lane, uint2 *buf, lp_state &st,
                                        lp_raw<DT, MASK> &next)
{
    for (int64_t t = t0; t < t1; t += step) {
        float x[LP_E];
        const int rem = lp_left(a.cols, t);
        lp_unpack<DT, MASK>(next, rem, lane, x);
        if (t + step < t1)
            lp_fetch_tile<DT, MASK>(a, row, t + step, lane, next);
        else if (then >= 0)
            lp_fetch_tile<DT, MASK>(a, then, 0, lane, next);
        if (!st.bad)
            lp_tile<lp_type<DT>::VE>(x, (uint32_t)(t * LP_TILE), rem, a.c2, a.k, lane, buf, st);
    }
    st.S = lp_wave_sum(st.S);
    st.Q = lp_wave_sum(st.Q);
}

// A wave a row, `rows_per_wave` <= LP_ROWS rows one after the other.
constexpr int LP_ROWS = 8;
template <int DT, int MASK>
__global__ __launch_bounds__(256, 5) void k_log_probabilities_rows(lp_args a, int rows_per_wave)
{
    __shared__ uint2 s_buf[4][LP_BUF];
    __shared__ uint2 s_lists[4][LP_ROWS * LP_KMAX];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t tiles = (a.cols + LP_TILE - 1) / LP_TILE;
    const int64_t row0 = ((int64_t)blockIdx.x * 4 + wid) * rows_per_wave;
    if (row0 >= a.rows)
        return;
    const int nrows = (int)min((int64_t)rows_per_wave, a.rows - row0);
    float m = 0.0f, S = 0.0f, Q = 0.0f;
    int c = 0, len = 0;
    bool bad = false;
    lp_raw<DT, MASK> next;
    lp_fetch_tile<DT, MASK>(a, row0, 0, lane, next);
#pragma unroll 1
    for (int r = 0; r < nrows; ++r) {
        lp_state st;
        lp_walk<DT, MASK>(a, row0 + r, 0, tiles, 1, r + 1 < nrows ? row0 + r + 1 : -1, lane, s_buf[wid], st, next);
        if (lane < st.len)
            s_lists[wid][r * LP_KMAX + lane] = s_buf[wid][lane];
        if (lane == r) {
            m = st.m;
            S = st.S;
            Q = st.Q;
            c = st.c;
            len = st.len;
            bad = st.bad;
        }
    }
    lp_finish<DT>(row0, nrows, m, S, Q, c, bad, len, s_lists[wid], lane);
}

// W waves a row; SPLIT: a workgroup takes tiles_per_split tiles of a row and leaves its state.
template <int DT, int MASK, int W, bool SPLIT>
__global__ __launch_bounds__(W * 64, W == 4 ? 5 : 4) void k_log_probabilities(lp_args a)
{
    __shared__ uint2 s_buf[W][LP_BUF];
    __shared__ uint2 s_lists[W * LP_KMAX];
    __shared__ float4 s_state[W];
    __shared__ int s_len[W];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t unit = blockIdx.x, tiles = (a.cols + LP_TILE - 1) / LP_TILE;
    const int64_t row = SPLIT ? (uint32_t)unit / (uint32_t)a.nsplit : unit;
    const int64_t t0 = SPLIT ? (unit - row * a.nsplit) * a.tiles_per_split : 0, t1 = SPLIT ? min(tiles, t0 + a.tiles_per_split) : tiles;
    lp_state st;
    uint2 *buf = s_buf[wid];
    lp_raw<DT, MASK> next;
    if (t0 + wid < t1)
        lp_fetch_tile<DT, MASK>(a, row, t0 + wid, lane, next);
    lp_walk<DT, MASK>(a, row, t0 + wid, t1, W, -1, lane, buf, st, next);
    if (lane == 0) {
        s_state[wid] = make_float4(st.m, st.S, st.Q, st.bad ? -1.0f : (float)st.c);
        s_len[wid] = st.len;
    }
    if (lane < st.len)
        s_lists[wid * LP_KMAX + lane] = buf[lane];
    __syncthreads();
    if (wid != 0)
        return;
    const bool own = lane < W;
    const float4 q = own ? s_state[lane] : make_float4(-LP_INF, 0.0f, 0.0f, 0.0f);
    lp_join(q.x, q.y, q.z, fmaxf(q.w, 0.0f), q.w < 0.0f, own ? s_len[lane] : 0, s_lists, a.k, a.c2, lane, st, buf);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (SPLIT) {
        if (lane == 0)
            a.part[unit] = make_float4(st.m, st.S, st.Q, st.bad ? -1.0f : (float)st.c);
        if (lane < LP_KMAX)
            a.part_lists[unit * LP_KMAX + lane] = lane < st.len ? buf[lane] : make_uint2(0, 0xFFFFFFFFu);
    } else {
        lp_finish<DT>(row, 1, st.m, st.S, st.Q, st.c, st.bad, st.len, buf, lane);
    }
}

// The states of a row's splits, joined: a wave a row.
template <int DT>
__global__ __launch_bounds__(64) void k_log_probabilities_join(lp_args a)
{
    __shared__ uint2 s_lists[LP_MAX_SPLITS * LP_KMAX];
    __shared__ uint2 s_out[LP_KMAX];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const bool own = lane < a.nsplit;
    const float4 q = own ? a.part[row * a.nsplit + lane] : make_float4(-LP_INF, 0.0f, 0.0f, 0.0f);
    int len = 0;
    if (a.k) {
        for (int i = lane; i < a.nsplit * LP_KMAX; i += 64)
            s_lists[i] = a.part_lists[row * a.nsplit * LP_KMAX + i];
        __syncthreads();
        if (own)
            for (int i = 0; i < LP_KMAX; ++i)
                len += s_lists[lane * LP_KMAX + i].y != 0xFFFFFFFFu;
    }
    lp_state st;
    lp_join(q.x, q.y, q.z, fmaxf(q.w, 0.0f), q.w < 0.0f, len, s_lists, a.k, a.c2, lane, st, s_out);
    __syncthreads();
    lp_finish<DT>(row, 1, st.m, st.S, st.Q, st.c, st.bad, st.len, s_out, lane);
}

// ---------------------------------------------------------------------------- gradient
//   p = exp(d - l);   ds_j = [gl ((j == y) - p_j) - gh p_j (d_j - l + H)] / T, 0 for classes that are not allowed
// One pass: a score in, its gradient out (they may be the same array).  At the label 1 - p is -expm1(d - l): where the
// label holds nearly all of the mass the difference would keep nothing.
struct lp_grad_args {
    int64_t rows, cols;
    const void *scores;
    int64_t ld;
    const uint8_t *mask;
    int64_t ldmask;
    const void *labels;
    int label64;
    float c2, inv_t;
    const float *stats, *entropy, *d_logp, *d_entropy;
    void *out;
    int64_t ldo;
    uint32_t *err;
};

template <int DT, int MASK>
__global__ __launch_bounds__(256) void k_log_probabilities_grad(lp_grad_args a)
{
    using P = lp_type<DT>;
    using T = typename P::T;
    constexpr int VE = P::VE, NV = LP_E / VE;
    const int lane = threadIdx.x & 63;
    const int64_t tiles = (a.cols + LP_TILE - 1) / LP_TILE, units = a.rows * tiles;
    for (int64_t unit = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); unit < units; unit += (int64_t)gridDim.x * 4) {
        const int64_t row = unit / tiles, base = (unit - row * tiles) * LP_TILE;
        const T *srow = (const T *)a.scores + row * a.ld;
        T *orow = (T *)a.out + row * a.ldo;
        const int rem = (int)min(a.cols - base, (int64_t)LP_TILE);
        float x[LP_E];
        {  // (in place: what is read of other lanes' elements may be their gradients already, and is dropped)
            lp_raw<DT, MASK> raw;
            lp_fetch<DT, MASK>(srow + base, MASK ? a.mask + row * a.ldmask + base : nullptr, rem, a.cols, lane, raw);
            lp_unpack<DT, MASK>(raw, rem, lane, x);
        }
        const int64_t y = !a.d_logp ? -1 : a.label64 ? ((const int64_t *)a.labels)[row] : (int64_t)((const int32_t *)a.labels)[row];
        const bool wrong = y < -1 || y >= a.cols;
        if (wrong && a.err && lane == 0)
            __hip_atomic_store(a.err, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        const float gl = wrong ? __builtin_nanf("") : y >= 0 ? a.d_logp[row] : 0.0f;
        const float gh = a.d_entropy ? a.d_entropy[row] : 0.0f;
        const float m = a.stats[2 * row], l = a.stats[2 * row + 1], hl = (a.d_entropy ? a.entropy[row] : 0.0f) - l;
        const float l2 = l * 1.44269504088896f;
        // p is 0 in float32 from d = -104 on (l is not negative), however far the scaled difference goes: cut off at -1000 it
        // changes no product, and gh times it stays finite for every gh below 3e35 - 0 times infinity would be NaN.  1 / T comes
        // last for the same reason: gh / T times it need not be finite.
        auto far = [](float d) { return fmaxf(d, -1e3f); };
#pragma unroll
        for (int e = 0; e < LP_E; ++e) {
            const float t = x[e] - m;
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(t, a.c2, -l2));
            const float r = -p * __builtin_fmaf(gh, far(t * a.inv_t) + hl, gl) * a.inv_t;
            x[e] = x[e] == -LP_INF ? 0.0f : r;
        }
        // the label's entry again, by the lane that holds it
        const int off = lp_entry_of(y, base, rem);
        if (off >= 0 && ((off / VE) & 63) == lane) {
            const float s = P::one(srow[y]);
            const bool allowed = s != -LP_INF && (!MASK || a.mask[row * a.ldmask + y] != 0);
            const float z = (s - m) * a.inv_t - l;
            const float p = __builtin_amdgcn_exp2f(z * 1.44269504088896f);
            const float d = allowed ? -(gl * expm1f(z) + p * gh * (far((s - m) * a.inv_t) + hl)) * a.inv_t : 0.0f;
#pragma unroll
            for (int e = 0; e < LP_E; ++e)
                if (off / VE / 64 == e / VE && off - lp_start<VE>(e / VE, lane, rem) == e % VE)
                    x[e] = d;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int at = lp_start<VE>(v, lane, rem), drop = (v * 64 + lane) * VE - at;
            T o[VE];
#pragma unroll
            for (int u = 0; u < VE; ++u)
                o[u] = P::round(x[v * VE + u]);
            if (drop == 0) {
                lp_u128 raw;
                __builtin_memcpy(&raw, o, 16);
                *reinterpret_cast<lp_u128 *>(orow + base + at) = raw;
            } else {
#pragma unroll
                for (int u = 0; u < VE; ++u)
                    if (u >= drop)
                        orow[base + at + u] = o[u];
            }
        }
    }
}

// How a row is cut: a wave a row where that fills the chip, else several waves of a workgroup, else several workgroups.
struct lp_cut {
    int waves, rows_per_wave, nsplit;
    int64_t tiles_per_split;
};

lp_cut lp_plan(const skm_ctx *ctx, int64_t rows, int64_t cols)
{
    const int64_t tiles = skm_ceil_div(cols, LP_TILE), cus = ctx->usable_cus, want = cus * 16;  // waves
    lp_cut c = {1, 1, 1, tiles};
    if (tiles == 1 || rows >= want / 2) {
        c.rows_per_wave = (int)std::min<int64_t>(LP_ROWS, std::max<int64_t>(1, rows / (want * 2)));
        return c;
    }
    // one workgroup a row: four waves, or sixteen where they have no more than four tiles each
    c.waves = tiles <= 8 || tiles > 64 || rows * 4 >= want ? 4 : 16;
    if (tiles > 64) {  // several a row: what the compute units hold at once (four workgroups each), two tiles a wave at least
        const int64_t s = std::min<int64_t>(std::min<int64_t>(4 * cus / rows, tiles / 8), LP_MAX_SPLITS);
        if (s > 1) {
            c.tiles_per_split = skm_ceil_div(tiles, s);
            c.nsplit = (int)skm_ceil_div(tiles, c.tiles_per_split);
        }
    }
    return c;
}

// `rows` rows from row0 on: a launch holds at most 2^32 work-items
lp_args lp_rows_from(const lp_args &whole, int64_t row0, int64_t rows, int64_t elem)
{
    lp_args a = whole;
    a.rows = rows;
    a.scores = (const uint8_t *)whole.scores + row0 * whole.ld * elem;
    a.mask = whole.mask ? whole.mask + row0 * whole.ldmask : nullptr;
    a.labels = whole.labels ? (const uint8_t *)whole.labels + row0 * (whole.label64 ? 8 : 4) : nullptr;
    a.logp = whole.logp ? whole.logp + row0 : nullptr;
    a.entropy = whole.entropy ? whole.entropy + row0 : nullptr;
    a.stats = whole.stats ? whole.stats + 2 * row0 : nullptr;
    a.top_index = whole.top_index ? whole.top_index + row0 * whole.k : nullptr;
    a.top_logp = whole.top_logp ? whole.top_logp + row0 * whole.k : nullptr;
    return a;
}

template <int DT, int MASK>
int lp_launch(skm_ctx *ctx, const lp_args &whole, const lp_cut &cut)
{
    constexpr int64_t MOST = (int64_t)1 << 21;  // workgroups
    if (cut.nsplit > 1) {                       // (only where rows are few)
        k_log_probabilities<DT, MASK, 4, true><<<(unsigned)(whole.rows * cut.nsplit), 256, 0, ctx->stream>>>(whole);
        SKM_TRY(skm_check_launch("k_log_probabilities"));
        k_log_probabilities_join<DT><<<(unsigned)whole.rows, 64, 0, ctx->stream>>>(whole);
        return skm_check_launch("k_log_probabilities_join");
    }
    const int64_t step = cut.waves == 1 ? MOST * 4 * cut.rows_per_wave : MOST;
    for (int64_t row0 = 0; row0 < whole.rows; row0 += step) {
        const lp_args a = lp_rows_from(whole, row0, std::min(step, whole.rows - row0), sizeof(typename lp_type<DT>::T));
        if (cut.waves == 1)
            k_log_probabilities_rows<DT, MASK><<<(unsigned)skm_ceil_div(a.rows, 4 * cut.rows_per_wave), 256, 0, ctx->stream>>>(a, cut.rows_per_wave);
        else if (cut.waves == 4)
            k_log_probabilities<DT, MASK, 4, false><<<(unsigned)a.rows, 256, 0, ctx->stream>>>(a);
        else
            k_log_probabilities<DT, MASK, 16, false><<<(unsigned)a.rows, 1024, 0, ctx->stream>>>(a);
        SKM_TRY(skm_check_launch("k_log_probabilities"));
    }
    return SKM_OK;
}

// rows of bytes
struct lp_span {
    const void *p;
    int64_t rows, bytes, stride;
};
bool lp_share(const lp_span &a, const lp_span &b) { return skm_overlap(a.p, a.rows, a.bytes, a.stride, b.p, b.rows, b.bytes, b.stride, 1); }

// float32 and integer arrays are read and written as such
struct lp_vector {
    const char *what;
    const void *p;
    int bytes;
};
template <int N>
int lp_check_aligned(const char *who, const lp_vector (&vectors)[N])
{
    for (const lp_vector &v : vectors)
        SKM_REQUIRE((uintptr_t)v.p % (uintptr_t)v.bytes == 0, SKM_E_BADARG, "%s: %s is not aligned to its type", who, v.what);
    return SKM_OK;
}

// what both entry points check
int lp_check(const char *who, skm_ctx *ctx, int dtype, int64_t rows, int64_t cols, const void *d_scores, int64_t ld, const uint8_t *d_mask, int64_t ldmask,
             int label_bits, double temperature)
{
    SKM_REQUIRE(ctx, SKM_E_BADARG, "%s: null context", who);
    SKM_REQUIRE(dtype >= 0 && dtype <= 2, SKM_E_BADARG, "%s: dtype must be 0 (float32), 1 (float16) or 2 (bfloat16)", who);
    SKM_REQUIRE(rows >= 0 && cols >= 1, SKM_E_BADARG, "%s: %lld rows of %lld classes", who, (long long)rows, (long long)cols);
    SKM_REQUIRE(cols < ((int64_t)1 << 31), SKM_E_OVERFLOW, "%s: %lld classes (indices are 32-bit)", who, (long long)cols);
    SKM_REQUIRE(ld >= cols, SKM_E_BADARG, "%s: ld (%lld) < cols (%lld)", who, (long long)ld, (long long)cols);
    SKM_REQUIRE(ldmask == 0 || ldmask >= cols, SKM_E_BADARG, "%s: ldmask (%lld) must be 0 (one mask for all rows) or at least cols", who, (long long)ldmask);
    SKM_REQUIRE(label_bits == 32 || label_bits == 64, SKM_E_BADARG, "%s: label_bits must be 32 or 64", who);
    SKM_REQUIRE(temperature > 0.0 && temperature < 1e30 && temperature > 1e-30, SKM_E_BADARG, "%s: temperature %g (want a positive number between 1e-30 and 1e30)", who,
                temperature);
    SKM_REQUIRE(rows == 0 || d_scores, SKM_E_BADARG, "%s: null scores", who);
    const uintptr_t align = dtype == 0 ? 3 : 1;
    SKM_REQUIRE(((uintptr_t)d_scores & align) == 0, SKM_E_BADARG, "%s: scores are not aligned to their type", who);
    return SKM_OK;
}

}  // namespace

extern "C" int skm_log_probabilities(skm_ctx *ctx, int dtype, int64_t rows, int64_t cols, const void *d_scores, int64_t ld, const uint8_t *d_mask, int64_t ldmask,
                                     const void *d_labels, int label_bits, int k, double temperature, float *d_logp, float *d_entropy, float *d_stats,
                                     int32_t *d_top_index, float *d_top_logp)
{
    const char *who = "skm_log_probabilities";
    SKM_TRY(lp_check(who, ctx, dtype, rows, cols, d_scores, ld, d_mask, ldmask, label_bits, temperature));
    SKM_REQUIRE(k >= 0 && k <= LP_KMAX, SKM_E_BADARG, "%s: k (%d) must be 0..%d", who, k, LP_KMAX);
    SKM_REQUIRE(k > 0 || (!d_top_index && !d_top_logp), SKM_E_BADARG, "%s: arrays for alternatives, but k is 0", who);
    SKM_REQUIRE(!d_logp || d_labels || rows == 0, SKM_E_BADARG, "%s: log probabilities need labels", who);
    if (rows == 0)
        return SKM_OK;
    SKM_TRY(lp_check_aligned(who, {{"labels", d_labels, label_bits / 8}, {"logp", d_logp, 4}, {"entropy", d_entropy, 4}, {"stats", d_stats, 4}, {"top_index", d_top_index, 4}, {"top_logp", d_top_logp, 4}}));
    const int64_t es = dtype == 0 ? 4 : 2;
    const lp_span in[3] = {{d_scores, rows, cols * es, ld * es}, {d_mask, ldmask ? rows : 1, cols, ldmask ? ldmask : cols}, {d_logp ? d_labels : nullptr, 1, rows * (label_bits / 8), rows * (label_bits / 8)}};
    const lp_span out[5] = {{d_logp, 1, rows * 4, rows * 4}, {d_entropy, 1, rows * 4, rows * 4}, {d_stats, 1, rows * 8, rows * 8}, {d_top_index, 1, rows * k * 4, rows * k * 4}, {d_top_logp, 1, rows * k * 4, rows * k * 4}};
    for (int o = 0; o < 5; ++o) {
        for (const lp_span &i : in)
            SKM_REQUIRE(!lp_share(out[o], i), SKM_E_BADARG, "%s: an output shares memory with the scores, the mask or the labels", who);
        for (int q = 0; q < o; ++q)
            SKM_REQUIRE(!lp_share(out[o], out[q]), SKM_E_BADARG, "%s: two outputs share memory", who);
    }
    SKM_ON_DEVICE(ctx);
    lp_args a = {};
    a.rows = rows;
    a.cols = cols;
    a.scores = d_scores;
    a.ld = ld;
    a.mask = d_mask;
    a.ldmask = ldmask;
    a.labels = d_labels;
    a.label64 = label_bits == 64;
    a.k = d_top_index || d_top_logp ? k : 0;
    a.c2 = (float)(1.4426950408889634 / temperature);
    a.inv_t = (float)(1.0 / temperature);
    a.logp = d_logp;
    a.entropy = d_entropy;
    a.stats = d_stats;
    a.top_index = d_top_index;
    a.top_logp = d_top_logp;
    a.err = skm_err_word(ctx, SKM_DEVERR_LABEL);
    const lp_cut cut = lp_plan(ctx, rows, cols);
    a.nsplit = cut.nsplit;
    a.tiles_per_split = cut.tiles_per_split;
    if (cut.nsplit > 1) {
        void *p;
        const size_t units = (size_t)rows * (size_t)cut.nsplit;
        SKM_TRY(skm_ws(ctx, WS_A, units * (sizeof(float4) + LP_KMAX * sizeof(uint2)), &p));
        a.part = (float4 *)p;
        a.part_lists = (uint2 *)((uint8_t *)p + units * sizeof(float4));
    }
    SKM_PROF(ctx, "k_log_probabilities");
    switch (dtype * 2 + (d_mask ? 1 : 0)) {
    case 0:
        return lp_launch<0, 0>(ctx, a, cut);
    case 1:
        return lp_launch<0, 1>(ctx, a, cut);
    case 2:
        return lp_launch<1, 0>(ctx, a, cut);
    case 3:
        return lp_launch<1, 1>(ctx, a, cut);
    case 4:
        return lp_launch<2, 0>(ctx, a, cut);
    default:
        return lp_launch<2, 1>(ctx, a, cut);
    }
}

extern "C" int skm_log_probabilities_backward(skm_ctx *ctx, int dtype, int64_t rows, int64_t cols, const void *d_scores, int64_t ld, const uint8_t *d_mask,
                                              int64_t ldmask, const void *d_labels, int label_bits, double temperature, const float *d_stats,
                                              const float *d_entropy, const float *d_grad_logp, const float *d_grad_entropy, void *d_grad_scores, int64_t ldg)
{
    const char *who = "skm_log_probabilities_backward";
    SKM_TRY(lp_check(who, ctx, dtype, rows, cols, d_scores, ld, d_mask, ldmask, label_bits, temperature));
    SKM_REQUIRE(ldg >= cols, SKM_E_BADARG, "%s: ldg (%lld) < cols (%lld)", who, (long long)ldg, (long long)cols);
    if (rows == 0)
        return SKM_OK;
    SKM_REQUIRE(d_grad_logp || d_grad_entropy, SKM_E_BADARG, "%s: neither a gradient of the log probabilities nor one of the entropies", who);
    SKM_REQUIRE(d_stats && d_grad_scores && (!d_grad_logp || d_labels) && (!d_grad_entropy || d_entropy), SKM_E_BADARG,
                "%s: null array (stats, the output, labels for grad_logp, entropy for grad_entropy)", who);
    SKM_TRY(lp_check_aligned(who, {{"labels", d_labels, label_bits / 8}, {"stats", d_stats, 4}, {"entropy", d_entropy, 4}, {"grad_logp", d_grad_logp, 4}, {"grad_entropy", d_grad_entropy, 4}}));
    SKM_REQUIRE(((uintptr_t)d_grad_scores & (dtype == 0 ? 3 : 1)) == 0, SKM_E_BADARG, "%s: the output is not aligned to its type", who);
    const int64_t es = dtype == 0 ? 4 : 2;
    SKM_REQUIRE((d_grad_scores == d_scores && ldg == ld) || !skm_overlap(d_grad_scores, rows, cols, ldg, d_scores, rows, cols, ld, es), SKM_E_BADARG,
                "%s: the output shares memory with the scores without being them", who);
    const lp_span out = {d_grad_scores, rows, cols * es, ldg * es};
    const lp_span in[6] = {{d_mask, ldmask ? rows : 1, cols, ldmask ? ldmask : cols}, {d_grad_logp ? d_labels : nullptr, 1, rows * (label_bits / 8), rows * (label_bits / 8)}, {d_stats, 1, rows * 8, rows * 8},
                           {d_grad_entropy ? d_entropy : nullptr, 1, rows * 4, rows * 4}, {d_grad_logp, 1, rows * 4, rows * 4}, {d_grad_entropy, 1, rows * 4, rows * 4}};
    for (const lp_span &i : in)
        SKM_REQUIRE(!lp_share(out, i), SKM_E_BADARG, "%s: the output shares memory with another input than the scores", who);
    SKM_ON_DEVICE(ctx);
    lp_grad_args a = {};
    a.rows = rows;
    a.cols = cols;
    a.scores = d_scores;
    a.ld = ld;
    a.mask = d_mask;
    a.ldmask = ldmask;
    a.labels = d_labels;
    a.label64 = label_bits == 64;
    a.c2 = (float)(1.4426950408889634 / temperature);
    a.inv_t = (float)(1.0 / temperature);
    a.stats = d_stats;
    a.entropy = d_entropy;
    a.d_logp = d_grad_logp;
    a.d_entropy = d_grad_entropy;
    a.out = d_grad_scores;
    a.ldo = ldg;
    a.err = skm_err_word(ctx, SKM_DEVERR_LABEL);
    const int64_t units = rows * skm_ceil_div(cols, LP_TILE);
    const unsigned grid = (unsigned)std::min<int64_t>((int64_t)1 << 23, skm_ceil_div(units, 4));
    SKM_PROF(ctx, "k_log_probabilities_grad");
#define LP_GRAD(DT, MASK) k_log_probabilities_grad<DT, MASK><<<grid, 256, 0, ctx->stream>>>(a)
    switch (dtype * 2 + (d_mask ? 1 : 0)) {
    case 0:
        LP_GRAD(0, 0);
        break;
    case 1:
        LP_GRAD(0, 1);
        break;
    case 2:
        LP_GRAD(1, 0);
        break;
    case 3:
        LP_GRAD(1, 1);
        break;
    case 4:
        LP_GRAD(2, 0);
        break;
    default:
        LP_GRAD(2, 1);
    }
#undef LP_GRAD
    return skm_check_launch("k_log_probabilities_grad");
}
