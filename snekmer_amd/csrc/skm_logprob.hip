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
// The k best of a tile: no element below the k-th largest of the 64 lane maxima can be among them, so only those above
// it (about as many as k) are collected in LDS and ranked; equal ones are taken in index order until k are held.  After
// the first tile only elements above the list's last one are looked at, which costs one comparison a tile.
#include <algorithm>
#include <cmath>

#include "skm_common.h"

namespace {

constexpr int LP_E = 16;            // scores a lane holds of a tile
constexpr int LP_TILE = 64 * LP_E;  // 1024
constexpr int LP_KMAX = 16;
constexpr int LP_BUF = 128;  // candidates a wave holds before it ranks them (after ranking: at most 16, and 64 may follow)
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
    uint64_t *part_keys;  // [rows][nsplit][LP_KMAX]
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

// One tile of a row: x[v * VE + u] = score of class base + (v * 64 + lane) * VE + u, -inf where masked or past the end.
// MASK: 0 none, 1 present.
template <int DT, int MASK>
__device__ __forceinline__ void lp_load_tile(const typename lp_type<DT>::T *row, const uint8_t *mrow, int64_t base, int64_t cols, int lane, float (&x)[LP_E])
{
    using P = lp_type<DT>;
    constexpr int VE = P::VE, NV = LP_E / VE;
    if (base + LP_TILE <= cols) {
        lp_u128 raw[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v)
            raw[v] = *reinterpret_cast<const lp_u128 *>(row + base + (v * 64 + lane) * VE);
        uint32_t mk[NV][VE / 4];
        if (MASK) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const uint8_t *at = mrow + base + (v * 64 + lane) * VE;
                if constexpr (VE == 4) {
                    mk[v][0] = reinterpret_cast<const lp_u32 *>(at)->w[0];
                } else {
                    const lp_u64 w = *reinterpret_cast<const lp_u64 *>(at);
                    mk[v][0] = w.w[0];
                    mk[v][1] = w.w[1];
                }
            }
        }
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int u = 0; u < VE; ++u) {
                float f = P::pick(raw[v], u);
                if (MASK)
                    f = ((mk[v][u >> 2] >> (8 * (u & 3))) & 0xFFu) ? f : -LP_INF;
                x[v * VE + u] = f;
            }
    } else {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int64_t at = base + (v * 64 + lane) * VE;
            if (at + VE <= cols) {
                const lp_u128 raw = *reinterpret_cast<const lp_u128 *>(row + at);
#pragma unroll
                for (int u = 0; u < VE; ++u)
                    x[v * VE + u] = P::pick(raw, u);
            } else {
#pragma unroll
                for (int u = 0; u < VE; ++u)
                    x[v * VE + u] = at + u < cols ? P::one(row[at + u]) : -LP_INF;
            }
            if (MASK)
#pragma unroll
                for (int u = 0; u < VE; ++u)
                    if (at + u < cols && mrow[at + u] == 0)
                        x[v * VE + u] = -LP_INF;
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

// The n candidates of the buffer, best first; the first k stay.
__device__ __forceinline__ void lp_rank(uint64_t *buf, int n, int k, int lane, lp_state &st)
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const uint64_t a = lane < n ? buf[lane] : 0, b = lane + 64 < n ? buf[lane + 64] : 0;
    int ra = 0, rb = 0;
    const int first = n < 64 ? n : 64;
    for (int j = 0; j < first; ++j) {
        const uint64_t s = lp_readlane64(a, j);
        ra += s > a;
        rb += s > b;
    }
    for (int j = 64; j < n; ++j) {
        const uint64_t s = lp_readlane64(b, j - 64);
        ra += s > a;
        rb += s > b;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (lane < n && ra < k)
        buf[ra] = a;
    if (lane + 64 < n && rb < k)
        buf[rb] = b;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    st.len = n < k ? n : k;
    if (st.len == k)
        st.tau = lp_key_score(buf[k - 1]);
}

template <int VE>
__device__ __forceinline__ void lp_collect(const float (&x)[LP_E], float lane_max, float tile_max, int64_t base, int k, int lane, uint64_t *buf, lp_state &st)
{
    constexpr int NV = LP_E / VE;
    const bool full = st.len == k;
    if (full && !(tile_max > st.tau))
        return;  // ties with the last one lose: their indices are higher
    float thr = st.tau;
    if (!full) {  // the k-th largest lane maximum
        float cur = lane_max;
        for (int r = 0;; ++r) {
            thr = lp_wave_max(cur);
            if (r == k - 1 || thr == -LP_INF)
                break;
            const uint64_t at = __ballot(cur == thr);
            if (lane == __ffsll((unsigned long long)at) - 1)
                cur = -LP_INF;
        }
    }
    int n = st.len, above = 0;
    uint64_t floor_key = 0;
#pragma unroll
    for (int e = 0; e < LP_E; ++e) {
        bool take = x[e] > thr;
        uint64_t at = __ballot(take);
        if (at == 0)
            continue;
        above += __popcll(at);
        if (n + __popcll(at) > LP_BUF) {
            lp_rank(buf, n, k, lane, st);
            n = st.len;
            floor_key = n == k ? buf[k - 1] : 0;
        }
        const uint64_t key = lp_key(x[e], (uint32_t)(base + ((e / VE) * 64 + lane) * VE + e % VE));
        if (floor_key) {
            take = take && key > floor_key;
            at = __ballot(take);
        }
        if (take)
            buf[n + lp_below(at)] = key;
        n += __popcll(at);
    }
    if (!full && thr > -LP_INF && above < k) {  // those equal to the threshold, lowest indices first
        int need = k - above;
        for (int v = 0; v < NV && need > 0; ++v) {
            uint64_t eq[VE];
            int before = 0, total = 0, own = 0;
#pragma unroll
            for (int u = 0; u < VE; ++u) {
                float xe = x[u];  // (x[v * VE + u] without a run-time register index)
#pragma unroll
                for (int w = 1; w < NV; ++w)
                    xe = v == w ? x[w * VE + u] : xe;
                eq[u] = __ballot(xe == thr);
                before += lp_below(eq[u]);
                total += __popcll(eq[u]);
            }
#pragma unroll
            for (int u = 0; u < VE; ++u) {
                if ((eq[u] >> lane) & 1) {
                    if (before + own < need)
                        buf[n + before + own] = lp_key(thr, (uint32_t)(base + (v * 64 + lane) * VE + u));
                    ++own;
                }
            }
            const int got = total < need ? total : need;
            n += got;
            need -= got;
        }
    }
    lp_rank(buf, n, k, lane, st);
}

template <int VE>
__device__ __forceinline__ void lp_tile(const float (&x)[LP_E], int64_t base, float c2, int k, int lane, uint64_t *buf, lp_state &st)
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
            st.Q = f > 0.0f ? (st.Q + w * d) * f : 0.0f;
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
        st.Q += p * fmaxf(t2, -1e30f);  // (0 times -inf)
    }
    if (k)
        lp_collect<VE>(x, lm, tm, base, k, lane, buf, st);
}

// Joins n <= 64 partial states: lane p < n holds state p and, in LDS, its sorted list of `len` keys at lists + p * LP_KMAX.
// Results uniform (m, c, S, Q, bad); the k best keys to `out`.  Returns how many there are.
__device__ __forceinline__ int lp_join(float m, float S, float Q, float c, bool bad, int len, const uint64_t *lists, int k, float c2, int lane, lp_state &st, uint64_t *out)
{
    st.bad = __ballot(bad) != 0;
    if (st.bad)
        return 0;
    st.m = lp_wave_max(m);
    const bool has = m > -LP_INF;
    const float d = has ? (m - st.m) * c2 : 0.0f, f = __builtin_amdgcn_exp2f(d);
    const bool top = has && m == st.m;
    const float w = S + c;
    st.c = (int)lp_wave_sum(top ? c : 0.0f);
    st.S = lp_wave_sum(top ? S : has ? w * f : 0.0f);
    st.Q = lp_wave_sum(top ? Q : has && f > 0.0f ? (Q + w * d) * f : 0.0f);
    int held = 0, at = 0;
    uint64_t head = len > 0 ? lists[lane * LP_KMAX] : 0;
    for (; held < k; ++held) {
        const uint32_t hi = lp_wave_umax((uint32_t)(head >> 32));
        if (hi == 0)
            break;  // (no key of a score has a zero upper word)
        const uint32_t lo = lp_wave_umax((uint32_t)(head >> 32) == hi ? (uint32_t)head : 0u);
        const uint64_t best = ((uint64_t)hi << 32) | lo;
        if (head == best) {  // one lane: the indices differ
            out[held] = best;
            ++at;
            head = at < len ? lists[lane * LP_KMAX + at] : 0;
        }
    }
    return held;
}

template <int DT>
__device__ __forceinline__ void lp_finish(const lp_args &a, int64_t row, const lp_state &st, const uint64_t *buf, int lane)
{
    using P = lp_type<DT>;
    const float nan = __builtin_nanf("");
    const float l = st.m > -LP_INF ? log1pf(st.S + (float)(st.c - 1)) : -LP_INF;
    if (lane == 0) {
        if (a.stats) {
            a.stats[2 * row] = st.bad ? nan : st.m;
            a.stats[2 * row + 1] = st.bad ? nan : l;
        }
        if (a.entropy)
            a.entropy[row] = st.bad ? nan : st.m > -LP_INF ? l - 0.693147180559945f * (st.Q / (st.S + (float)st.c)) : 0.0f;
        if (a.logp) {
            float v = 0.0f;
            const int64_t y = a.label64 ? ((const int64_t *)a.labels)[row] : (int64_t)((const int32_t *)a.labels)[row];
            if (y < -1 || y >= a.cols) {
                v = nan;
                if (a.err)
                    __hip_atomic_store(a.err, SKM_DEVERR_LABEL, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            } else if (y >= 0) {
                if (st.bad) {
                    v = nan;
                } else if (a.mask && a.mask[row * a.ldmask + y] == 0) {
                    v = -LP_INF;
                } else {
                    const float s = P::one(((const typename P::T *)a.scores)[row * a.ld + y]);
                    v = s > -LP_INF ? (s - st.m) * a.inv_t - l : -LP_INF;
                }
            }
            a.logp[row] = v;
        }
    }
    if (lane < a.k) {
        const bool there = !st.bad && lane < st.len;
        const uint64_t key = there ? buf[lane] : 0;
        if (a.top_index)
            a.top_index[row * a.k + lane] = there ? (int32_t)lp_key_index(key) : -1;
        if (a.top_logp)
            a.top_logp[row * a.k + lane] = there ? (lp_key_score(key) - st.m) * a.inv_t - l : st.bad ? nan : -LP_INF;
    }
}

// W waves a row (workgroups of max(4, W) waves); SPLIT: a workgroup takes tiles_per_split tiles of a row and leaves its state.
template <int DT, int MASK, int W, bool SPLIT>
__global__ __launch_bounds__(W == 16 ? 1024 : 256) void k_log_probabilities(lp_args a)
{
    using P = lp_type<DT>;
    constexpr int NW = W == 16 ? 16 : 4, ROWS = NW / W;
    __shared__ uint64_t s_buf[NW][LP_BUF];
    __shared__ uint64_t s_lists[W > 1 ? NW : 1][LP_KMAX];
    __shared__ float4 s_state[NW];
    __shared__ int s_len[NW];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part = W == 1 ? 0 : wid;
    const int64_t units = SPLIT ? a.rows * a.nsplit : a.rows;
    for (int64_t unit0 = (int64_t)blockIdx.x * ROWS; unit0 < units; unit0 += (int64_t)gridDim.x * ROWS) {
        const int64_t unit = unit0 + (W == 1 ? wid : 0);
        const int64_t row = SPLIT ? unit / a.nsplit : unit;
        const int split = SPLIT ? (int)(unit % a.nsplit) : 0;
        lp_state st;
        uint64_t *buf = s_buf[wid];
        if (unit < units) {
            const typename P::T *srow = (const typename P::T *)a.scores + row * a.ld;
            const uint8_t *mrow = MASK ? a.mask + row * a.ldmask : nullptr;
            const int64_t tiles = (a.cols + LP_TILE - 1) / LP_TILE;
            const int64_t t0 = SPLIT ? split * a.tiles_per_split : 0, t1 = SPLIT ? min(tiles, t0 + a.tiles_per_split) : tiles;
            for (int64_t t = t0 + part; t < t1 && !st.bad; t += W) {
                float x[LP_E];
                lp_load_tile<DT, MASK>(srow, mrow, t * LP_TILE, a.cols, lane, x);
                lp_tile<P::VE>(x, t * LP_TILE, a.c2, a.k, lane, buf, st);
            }
            st.S = lp_wave_sum(st.S);
            st.Q = lp_wave_sum(st.Q);
        }
        if (W > 1) {
            if (lane == 0) {
                s_state[wid] = make_float4(st.m, st.S, st.Q, st.bad ? -1.0f : (float)st.c);
                s_len[wid] = st.len;
            }
            if (lane < st.len)
                s_lists[wid][lane] = buf[lane];
            __syncthreads();
            if (wid == 0) {
                const bool own = lane < W;
                const float4 q = own ? s_state[lane] : make_float4(-LP_INF, 0.0f, 0.0f, 0.0f);
                st = lp_state();
                st.len = lp_join(q.x, q.y, q.z, q.w < 0.0f ? 0.0f : q.w, q.w < 0.0f, own ? s_len[lane] : 0, &s_lists[0][0], a.k, a.c2, lane, st, buf);
            }
        }
        if (unit < units && (W == 1 || wid == 0)) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (SPLIT) {
                if (lane == 0)
                    a.part[unit] = make_float4(st.m, st.S, st.Q, st.bad ? -1.0f : (float)st.c);
                if (lane < LP_KMAX)
                    a.part_keys[unit * LP_KMAX + lane] = lane < st.len ? buf[lane] : 0;
            } else {
                lp_finish<DT>(a, row, st, buf, lane);
            }
        }
        if (W > 1)
            __syncthreads();  // the lists are read before the next row's are written
    }
}

// The states of a row's splits, joined: a wave a row.
template <int DT>
__global__ __launch_bounds__(64) void k_log_probabilities_join(lp_args a)
{
    __shared__ uint64_t s_lists[LP_MAX_SPLITS * LP_KMAX];
    __shared__ uint64_t s_out[LP_KMAX];
    const int lane = threadIdx.x;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const bool own = lane < a.nsplit;
        const float4 q = own ? a.part[row * a.nsplit + lane] : make_float4(-LP_INF, 0.0f, 0.0f, 0.0f);
        int len = 0;
        if (a.k) {
            for (int i = lane; i < a.nsplit * LP_KMAX; i += 64)
                s_lists[i] = a.part_keys[row * a.nsplit * LP_KMAX + i];
            __syncthreads();
            if (own)
                for (int i = 0; i < LP_KMAX; ++i)
                    len += s_lists[lane * LP_KMAX + i] != 0;
        }
        lp_state st;
        st.len = lp_join(q.x, q.y, q.z, q.w < 0.0f ? 0.0f : q.w, q.w < 0.0f, len, s_lists, a.k, a.c2, lane, st, s_out);
        __syncthreads();
        lp_finish<DT>(a, row, st, s_out, lane);
        __syncthreads();
    }
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
        float x[LP_E];
        lp_load_tile<DT, MASK>(srow, MASK ? a.mask + row * a.ldmask : nullptr, base, a.cols, lane, x);
        const int64_t y = !a.d_logp ? -1 : a.label64 ? ((const int64_t *)a.labels)[row] : (int64_t)((const int32_t *)a.labels)[row];
        const bool wrong = y < -1 || y >= a.cols;
        if (wrong && a.err && lane == 0)
            __hip_atomic_store(a.err, SKM_DEVERR_LABEL, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        const float gl = wrong ? __builtin_nanf("") : y >= 0 ? a.d_logp[row] : 0.0f;
        const float gh = a.d_entropy ? a.d_entropy[row] : 0.0f;
        const float m = a.stats[2 * row], l = a.stats[2 * row + 1], hl = (a.d_entropy ? a.entropy[row] : 0.0f) - l;
        const float l2 = l * 1.44269504088896f, gi = gl * a.inv_t, hi = gh * a.inv_t;
#pragma unroll
        for (int e = 0; e < LP_E; ++e) {
            const float t = x[e] - m;
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(t, a.c2, -l2));
            // (p is 0 where the scaled difference is beyond float32: the clamp keeps 0 times infinity out)
            const float r = -p * __builtin_fmaf(hi, fmaxf(t * a.inv_t, -1e30f) + hl, gi);
            x[e] = x[e] == -LP_INF ? 0.0f : r;
        }
        // the label's entry again, by the lane that holds it
        const int64_t off = y - base;
        if (y >= 0 && off >= 0 && off < LP_TILE && (int)((off / VE) & 63) == lane) {
            const float s = P::one(srow[y]);
            const bool allowed = s != -LP_INF && (!MASK || a.mask[row * a.ldmask + y] != 0);
            const float z = (s - m) * a.inv_t - l;
            const float v = allowed ? -gi * expm1f(z) - __builtin_amdgcn_exp2f(z * 1.44269504088896f) * hi * (fmaxf((s - m) * a.inv_t, -1e30f) + hl) : 0.0f;
#pragma unroll
            for (int e = 0; e < LP_E; ++e)
                if ((int)((off / VE) / 64) == e / VE && (int)(off % VE) == e % VE)
                    x[e] = v;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int64_t at = base + (v * 64 + lane) * VE;
            if (at + VE <= a.cols) {
                lp_u128 raw;
                T o[VE];
#pragma unroll
                for (int u = 0; u < VE; ++u)
                    o[u] = P::round(x[v * VE + u]);
                __builtin_memcpy(&raw, o, 16);
                *reinterpret_cast<lp_u128 *>(orow + at) = raw;
            } else {
#pragma unroll
                for (int u = 0; u < VE; ++u)
                    if (at + u < a.cols)
                        orow[at + u] = P::round(x[v * VE + u]);
            }
        }
    }
}

// How a row is cut.  A wave's tile costs about as much as a wave's join, so rows are only cut where whole rows would not
// keep the chip's waves busy.
struct lp_cut {
    int waves, nsplit;
    int64_t tiles_per_split;
};

lp_cut lp_plan(const skm_ctx *ctx, int64_t rows, int64_t cols)
{
    const int64_t tiles = skm_ceil_div(cols, LP_TILE), want = (int64_t)ctx->usable_cus * 8;
    lp_cut c = {1, 1, tiles};
    if (tiles == 1 || rows >= want)
        return c;
    c.waves = tiles <= 4 || rows * 4 >= want ? 4 : 16;
    const int64_t per_wave = 2;  // tiles, at least
    if (c.waves == 16 && rows * 16 < want && tiles > 16 * per_wave) {
        int64_t s = skm_ceil_div(want, rows * 16);
        s = std::min<int64_t>(s, tiles / (16 * per_wave));
        s = std::min<int64_t>(s, LP_MAX_SPLITS);
        if (s > 1) {
            c.tiles_per_split = skm_ceil_div(tiles, s);
            c.nsplit = (int)skm_ceil_div(tiles, c.tiles_per_split);
        }
    }
    return c;
}

template <int DT, int MASK>
int lp_launch(skm_ctx *ctx, const lp_args &a, const lp_cut &cut)
{
    const int64_t most = (int64_t)1 << 30;
    if (cut.nsplit > 1) {
        k_log_probabilities<DT, MASK, 16, true><<<(unsigned)std::min(most, a.rows * cut.nsplit), 1024, 0, ctx->stream>>>(a);
        SKM_TRY(skm_check_launch("k_log_probabilities"));
        k_log_probabilities_join<DT><<<(unsigned)std::min(most, a.rows), 64, 0, ctx->stream>>>(a);
        return skm_check_launch("k_log_probabilities_join");
    }
    if (cut.waves == 1)
        k_log_probabilities<DT, MASK, 1, false><<<(unsigned)std::min(most, skm_ceil_div(a.rows, 4)), 256, 0, ctx->stream>>>(a);
    else if (cut.waves == 4)
        k_log_probabilities<DT, MASK, 4, false><<<(unsigned)std::min(most, a.rows), 256, 0, ctx->stream>>>(a);
    else
        k_log_probabilities<DT, MASK, 16, false><<<(unsigned)std::min(most, a.rows), 1024, 0, ctx->stream>>>(a);
    return skm_check_launch("k_log_probabilities");
}

// what both entry points check; sets *elem to the bytes of a score
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
    SKM_HIP(hipSetDevice(ctx->device));
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
    a.err = ctx->d_err;
    const lp_cut cut = lp_plan(ctx, rows, cols);
    a.nsplit = cut.nsplit;
    a.tiles_per_split = cut.tiles_per_split;
    if (cut.nsplit > 1) {
        void *p;
        const size_t units = (size_t)rows * (size_t)cut.nsplit;
        SKM_TRY(skm_ws(ctx, WS_A, units * (sizeof(float4) + LP_KMAX * sizeof(uint64_t)), &p));
        a.part = (float4 *)p;
        a.part_keys = (uint64_t *)((uint8_t *)p + units * sizeof(float4));
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
    SKM_REQUIRE(d_grad_logp || d_grad_entropy, SKM_E_BADARG, "%s: neither a gradient of the log probabilities nor one of the entropies", who);
    if (rows == 0)
        return SKM_OK;
    SKM_REQUIRE(d_stats && d_grad_scores && (!d_grad_logp || d_labels) && (!d_grad_entropy || d_entropy), SKM_E_BADARG,
                "%s: null array (stats, the output, labels for grad_logp, entropy for grad_entropy)", who);
    SKM_REQUIRE(((uintptr_t)d_grad_scores & (dtype == 0 ? 3 : 1)) == 0, SKM_E_BADARG, "%s: the output is not aligned to its type", who);
    const int64_t es = dtype == 0 ? 4 : 2;
    SKM_REQUIRE((d_grad_scores == d_scores && ldg == ld) || !skm_overlap(d_grad_scores, rows, cols, ldg, d_scores, rows, cols, ld, es), SKM_E_BADARG,
                "%s: the output shares memory with the scores without being them", who);
    SKM_HIP(hipSetDevice(ctx->device));
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
    a.err = ctx->d_err;
    const int64_t units = rows * skm_ceil_div(cols, LP_TILE);
    const unsigned grid = (unsigned)std::min<int64_t>((int64_t)1 << 30, skm_ceil_div(units, 4));
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
