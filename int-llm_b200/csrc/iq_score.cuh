// iq_score.cuh -- log probabilities of given tokens, entropy and top
// alternatives of rows of logits (iq_logprobs_dev).
//
// Arithmetic (every step a whole-number operation, floors throughout):
//   E(d) = e^-d in Q16.48, 0 from d = 34 on: y = floor(d log2(e)), k and f its
//   whole and fractional parts, j the top 6 bits of f, r the rest;
//   h = 2^-r by a polynomial of degree 5 (coefficients ln2^i / i!), and
//   E = floor(2^(-j/64) h) >> k. Truncation is below 2^-48.7 and the five floors
//   below 2^-46 in all, before the shift.
//   ln S: log2 of S by 50 squarings of its mantissa, times ln 2.
#pragma once
#include <cooperative_groups.h>
#include "iq_ops.cuh"

namespace iq {

#define IQ_LP_LOG2E_60 1663314137230540311ll   // log2(e) 2^60
#define IQ_LP_LN2_60 799144290325165979ll     // ln(2) 2^60
#define IQ_LP_MAX_TOP 32

// 2^(-j/64) in Q16.48
__constant__ int64_t c_lp_pow[64] = {
    281474976710656ll, 278442931975303ll, 275443548385834ll, 272476474116817ll,
    269541361132679ll, 266637865146880ll, 263765645581531ll, 260924365527444ll,
    258113691704612ll, 255333294423116ll, 252582847544451ll, 249862028443274ll,
    247170517969557ll, 244508000411151ll, 241874163456754ll, 239268698159280ll,
    236691298899613ll, 234141663350766ll, 231619492442411ll, 229124490325803ll,
    226656364339077ll, 224214824972914ll, 221799585836591ll, 219410363624378ll,
    217046878082311ll, 214708851975319ll, 212396011054705ll, 210108084025971ll,
    207844802517004ll, 205605901046590ll, 203391116993276ll, 201200190564561ll,
    199032864766430ll, 196888885373201ll, 194768000897708ll, 192669962561802ll,
    190594524267169ll, 188541442566463ll, 186510476634748ll, 184501388241253ll,
    182513941721425ll, 180547903949287ll, 178603044310089ll, 176679134673265ll,
    174775949365665ll, 172893265145088ll, 171030861174094ll, 169188518994104ll,
    167366022499769ll, 165563157913624ll, 163779713761015ll, 162015480845287ll,
    160270252223250ll, 158543823180903ll, 156835991209421ll, 155146555981404ll,
    153475319327372ll, 151822085212527ll, 150186659713755ll, 148568850996877ll,
    146968469294152ll, 145385326882014ll, 143819238059052ll, 142270019124227ll};

#define IQ_LP_C0 281474976710656.0   // ln2^i / i! 2^48
#define IQ_LP_C1 195103586505167.0
#define IQ_LP_C2 67617750451595.0
#define IQ_LP_C3 15623017693776.0
#define IQ_LP_C4 2707262666570.0
#define IQ_LP_C5 375306296874.0

// E(d) in Q16.48, d = max - logit as an unsigned difference; pw: the table of powers,
// as doubles. The floors are those of fma.rd in the binade of 2^52 (one unit = one
// ulp): g = M + floor(h r 2^-48), and c - floor(h r 2^-48) = (c + M) - g exactly.
__device__ __forceinline__ uint64_t lp_exp(uint64_t d, const double *pw) {
    const double M = 4503599627370496.0;
    // y = d log2e >> 60 from 32-bit pieces (d < 2^54, log2e < 2^61)
    const uint32_t dl = (uint32_t)d, dh = (uint32_t)(d >> 32);
    uint64_t y = __umulhi(dl, (uint32_t)IQ_LP_LOG2E_60);
    madu(y, dh, (uint32_t)IQ_LP_LOG2E_60);
    madu(y, dl, (uint32_t)(IQ_LP_LOG2E_60 >> 32));
    y >>= 28;
    madu(y, dh << 4, (uint32_t)(IQ_LP_LOG2E_60 >> 32));
    // r 2^-48 from the low 42 bits of y, j the next 6, k = y >> 48
    const double r = __hiloint2double((int)(((uint32_t)(y >> 32) & 0x3FF) | 0x43300000), (int)(uint32_t)y) * 0x1p-48 - M * 0x1p-48;
    double h = IQ_LP_C5;
    h = (IQ_LP_C4 + M) - __fma_rd(h, r, M);
    h = (IQ_LP_C3 + M) - __fma_rd(h, r, M);
    h = (IQ_LP_C2 + M) - __fma_rd(h, r, M);
    h = (IQ_LP_C1 + M) - __fma_rd(h, r, M);
    h = (IQ_LP_C0 + M) - __fma_rd(h, r, M);
    const uint32_t hi = (uint32_t)(y >> 32);
    const uint64_t e = (uint64_t)__double_as_longlong(__fma_rd(pw[hi >> 10 & 63], h, M)) & 0xFFFFFFFFFFFFFull;   // pw: 2^(-j/64)
    return dh < (34u << 16) ? e >> (hi >> 16) : 0;
}

__device__ __forceinline__ int u128_bits(u128 x) {
    const uint64_t hi = (uint64_t)(x >> 64);
    return hi ? 128 - d_clz64(hi) : 64 - d_clz64((uint64_t)x);
}

// ln(S / 2^48) in Q16.48 for S >= 2^48
__device__ __forceinline__ int64_t lp_ln(u128 S) {
    const int bl = u128_bits(S);
    uint64_t y = (uint64_t)(bl <= 62 ? S << (62 - bl) : S >> (bl - 62)), z = 0;
    for (int i = 0; i < 50; i++) {
        y = (__umul64hi(y, y) << 3) | ((y * y) >> 61);
        const uint64_t bit = y >> 62;
        z = 2 * z + bit;
        y >>= bit;
    }
    const uint64_t a = ((uint64_t)(bl - 49) << 50) + z;
    return (int64_t)((__umul64hi(a, (uint64_t)IQ_LP_LN2_60) << 2) | ((a * (uint64_t)IQ_LP_LN2_60) >> 62));
}

// -d - z, INT64_MIN where it is below that
__device__ __forceinline__ int64_t lp_of(uint64_t d, int64_t z) {
    if (d > (uint64_t)INT64_MAX - (uint64_t)z) return INT64_MIN;
    return -(int64_t)d - z;
}

// z + A / S
__device__ __forceinline__ int64_t lp_entropy(u128 S, u128 A, int64_t z) {
    const int n = max(0, u128_bits(S > A ? S : A) - 61);
    return z + (int64_t)(uint64_t)d_udiv128_64((u128)(uint64_t)(A >> n) << 48, (uint64_t)(S >> n));
}

struct LpArgs {
    const int64_t *lg;
    int64_t ld;
    int rows, V, top;
    const int *tok;
    int64_t *logp, *ent;
    int *ids;
    int64_t *tl;
    int cs;   // CTAs a row
};

// A cluster of CTAs takes a row, each a slice of it held in shared memory (SM; else read
// again, from L2): one pass over the logits from HBM gives the maximum (distributed
// shared memory joins the slices') and each thread's own maximum, a second one
// the sums. Alternatives: the n-th largest of 32 groups' maxima is a lower bound
// of the slice's n-th largest logit; the few logits not below it are ranked by
// counting. Where more than LP_CAND reach it (many equal logits) the slice is searched
// n times instead. CTA 0 ranks the slices' lists the same way. Measured: one row of
// 32000 15 us, the latency of its steps in turn; 512 rows 89 us: 40 M warp
// instructions (35 us at full issue) in chains of doubles and 256 MB read in two passes (39 us), which hardly
// overlap, since all rows are on the GPU at once and read and compute in step.
#define LP_T 256
#define LP_CAND 512

__device__ __forceinline__ bool lp_before(int64_t v, int i, int64_t w, int k) { return v > w || (v == w && i < k); }

// The `top` first of n <= cap (value, index) pairs in falling order by counting, into ov, oi (smem)
__device__ __forceinline__ void lp_rank(const int64_t *v, const int *ix, int n, int top, int64_t *ov, int *oi) {
    for (int a = threadIdx.x; a < n; a += LP_T) {
        const int64_t w = v[a];
        const int k = ix[a];
        int c = 0;
        for (int b = 0; b < n; b++) c += lp_before(v[b], ix[b], w, k);
        if (c < top) { ov[c] = w; oi[c] = k; }
    }
}

template <bool SM>
__global__ void __launch_bounds__(LP_T) k_logprobs(const __grid_constant__ LpArgs a) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) int64_t lp_buf[];
    __shared__ int64_t tmax[LP_T], cv[LP_CAND], lv[IQ_LP_MAX_TOP], gv[8 * IQ_LP_MAX_TOP];
    __shared__ int ci[LP_CAND], li[IQ_LP_MAX_TOP], gi[8 * IQ_LP_MAX_TOP], cnt, last_i;
    __shared__ uint64_t wred[4 * (LP_T / 32)], part[4];
    __shared__ double pw[64];
    __shared__ int64_t cmax, last_v, tau_s;
    cg::cluster_group cl = cg::this_cluster();
    const int cs = a.cs, rank = blockIdx.x % cs, row = blockIdx.x / cs, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t *l = a.lg + (int64_t)row * a.ld;
    const int per = (a.V + cs - 1) / cs, b0 = min(a.V, rank * per), n = min(per, a.V - b0);
    if (tid < 64) pw[tid] = (double)c_lp_pow[tid] * 0x1p-48;
    if (tid == 0) cnt = 0;

    // the given token's logit, early
    int64_t given = 0;
    bool has = false;
    if (rank == 0 && tid == 32 && a.tok) {
        const int t = a.tok[row];
        has = index_ok(t, a.V);
        if (has) given = l[t];
    }

    // the maximum
    int64_t m = INT64_MIN;
    const int64_t *src = l + b0;
    const int skew = (int)(((uintptr_t)src >> 3) & 1);   // pairs from the first 16-byte boundary on
    const longlong2 *s2 = reinterpret_cast<const longlong2 *>(src + skew);
    const int n2 = n > skew ? (n - skew) >> 1 : 0;
    for (int i0 = 0; i0 < n2; i0 += 4 * LP_T) {
        longlong2 u[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = i0 + k * LP_T + tid;
            u[k] = i < n2 ? __ldg(s2 + i) : make_longlong2(INT64_MIN, INT64_MIN);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = i0 + k * LP_T + tid;
            m = max(m, (int64_t)max(u[k].x, u[k].y));
            if (SM && i < n2) reinterpret_cast<longlong2 *>(lp_buf)[i] = u[k];
        }
    }
    const int odd = n - 2 * n2;   // 0 .. 2 elements outside the pairs: the first (skew) and the last
    int64_t ov = INT64_MIN;
    if (tid < odd) {
        const int i = skew && n > 0 && tid == 0 ? 0 : n - 1;
        ov = __ldg(src + i);
        m = max(m, ov);
    }
    const longlong2 *x2 = SM ? reinterpret_cast<const longlong2 *>(lp_buf) : s2;
    // f(logit, its place in the row) for each of the thread's logits
    auto each = [&](auto f) {
        int i = tid;
        for (; i + 3 * LP_T < n2; i += 4 * LP_T) {
            longlong2 u[4];
#pragma unroll
            for (int k = 0; k < 4; k++) u[k] = x2[i + k * LP_T];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                f(u[k].x, b0 + skew + 2 * (i + k * LP_T));
                f(u[k].y, b0 + skew + 2 * (i + k * LP_T) + 1);
            }
        }
        for (; i < n2; i += LP_T) {
            const longlong2 u = x2[i];
            f(u.x, b0 + skew + 2 * i);
            f(u.y, b0 + skew + 2 * i + 1);
        }
        if (tid < odd) f(ov, b0 + (skew && tid == 0 ? 0 : n - 1));
    };
    tmax[tid] = m;
    for (int k = 16; k >= 1; k >>= 1) m = max(m, (int64_t)__shfl_xor_sync(0xffffffffu, m, k));
    if (lane == 0) wred[warp] = (uint64_t)m;
    __syncthreads();
    m = (int64_t)wred[0];
#pragma unroll
    for (int k = 1; k < LP_T / 32; k++) m = max(m, (int64_t)wred[k]);
    if (tid == 0) cmax = m;
    // the bound for the alternatives: the top-th largest of 32 maxima of LP_T / 32 threads each
    const int top = min(a.top, n);
    if (warp == 0 && top) {
        int64_t g = INT64_MIN;
        for (int k = 0; k < LP_T / 32; k++) g = max(g, tmax[k * 32 + lane]);
        int c = 0;
        for (int k = 0; k < 32; k++) {
            const int64_t o = __shfl_sync(0xffffffffu, g, k);
            c += lp_before(o, k, g, lane);
        }
        if (c == top - 1) tau_s = g;
    }
    if (cs > 1) {
        cl.sync();
        int64_t o = lane < cs ? *cl.map_shared_rank(&cmax, lane) : INT64_MIN;
        for (int k = 4; k >= 1; k >>= 1) o = max(o, (int64_t)__shfl_xor_sync(0xffffffffu, o, k));
        m = __shfl_sync(0xffffffffu, o, 0);
    } else {
        __syncthreads();
    }

    // the sums: S and A in two words each (a thread's own stay below 2^64: at most 2^15 terms of 2^48)
    uint64_t S = 0, A = 0, Sh = 0, Ah = 0;
    const bool ent = a.ent != nullptr;
    const int64_t tau = top ? tau_s : INT64_MAX;
    each([&](int64_t v, int i) {
        const uint64_t d = (uint64_t)m - (uint64_t)v, e = lp_exp(d, pw);
        S += e;
        if (ent) {   // floor(e d / 2^48), e <= 2^48 and 0 from d = 34 on: from 32-bit pieces
            const uint32_t el = (uint32_t)e, eh = (uint32_t)(e >> 32), dl = (uint32_t)d, dh = (uint32_t)(d >> 32);
            uint64_t t = __umulhi(el, dl);
            madu(t, eh, dl);
            madu(t, el, dh);
            t >>= 16;
            madu(t, eh << 8, dh << 8);
            A += t;
        }
        if (v >= tau && top) {
            const int c = atomicAdd(&cnt, 1);
            if (c < LP_CAND) { cv[c] = v; ci[c] = i; }
        }
    });
    Sh = S >> 32;
    S &= 0xFFFFFFFFull;
    Ah = A >> 32;
    A &= 0xFFFFFFFFull;
    for (int k = 16; k >= 1; k >>= 1) {
        S += __shfl_xor_sync(0xffffffffu, S, k);
        Sh += __shfl_xor_sync(0xffffffffu, Sh, k);
        A += __shfl_xor_sync(0xffffffffu, A, k);
        Ah += __shfl_xor_sync(0xffffffffu, Ah, k);
    }
    __syncthreads();
    if (lane == 0) { wred[4 * warp] = S; wred[4 * warp + 1] = Sh; wred[4 * warp + 2] = A; wred[4 * warp + 3] = Ah; }
    __syncthreads();
    if (tid < 4) {
        uint64_t t = 0;
        for (int k = 0; k < LP_T / 32; k++) t += wred[4 * k + tid];
        part[tid] = t;
    }
    if (top) {
        if (cnt <= LP_CAND) {
            lp_rank(cv, ci, cnt, top, lv, li);
        } else {
            int64_t pv = INT64_MAX;
            int pi = -1;
            for (int k = 0; k < top; k++) {   // the first after (pv, pi)
                int64_t best = INT64_MIN;
                int idx = 0x7fffffff;
                each([&](int64_t v, int p) {
                    if (lp_before(pv, pi, v, p) && (idx == 0x7fffffff || lp_before(v, p, best, idx))) { best = v; idx = p; }
                });
                for (int o = 16; o >= 1; o >>= 1) {
                    const int64_t w = __shfl_xor_sync(0xffffffffu, best, o);
                    const int j = __shfl_xor_sync(0xffffffffu, idx, o);
                    if (lp_before(w, j, best, idx)) { best = w; idx = j; }
                }
                __syncthreads();
                if (lane == 0) { cv[warp] = best; ci[warp] = idx; }
                __syncthreads();
                if (tid == 0) {
                    for (int w = 1; w < LP_T / 32; w++)
                        if (lp_before(cv[w], ci[w], best, idx)) { best = cv[w]; idx = ci[w]; }
                    lv[k] = last_v = best;
                    li[k] = last_i = idx;
                }
                __syncthreads();
                pv = last_v;
                pi = last_i;
            }
        }
    }
    if (tid >= top && tid < IQ_LP_MAX_TOP) { lv[tid] = INT64_MIN; li[tid] = 0x7fffffff; }   // a short slice's missing ones
    if (cs > 1) cl.sync();
    else __syncthreads();
    if (rank == 0) {
        if (cs > 1) {
            for (int e = tid; e < cs * a.top; e += LP_T) {
                const int r = e / a.top, k = e - r * a.top;
                gv[e] = cl.map_shared_rank(lv, r)[k];
                gi[e] = cl.map_shared_rank(li, r)[k];
            }
            if (tid >= 32 && tid < 36) {
                uint64_t t = 0;
                for (int r = 0; r < cs; r++) t += cl.map_shared_rank(part, r)[tid - 32];
                wred[tid - 32] = t;
            }
        } else {
            if (tid < a.top) { gv[tid] = lv[tid]; gi[tid] = li[tid]; }
            if (tid >= 32 && tid < 36) wred[tid - 32] = part[tid - 32];
        }
    }
    if (cs > 1) cl.sync();   // CTA 0 holds the others' lists and sums: they are done
    else __syncthreads();
    if (rank != 0) return;
    if (cs > 1) {
        lp_rank(gv, gi, cs * a.top, a.top, cv, ci);
        __syncthreads();
    }
    const u128 St = ((u128)wred[1] << 32) + wred[0];
    if (warp < 2) {
        const int64_t z = lp_ln(St);
        if (has) a.logp[row] = lp_of((uint64_t)m - (uint64_t)given, z);
        if (tid == 33 && ent) a.ent[row] = lp_entropy(St, ((u128)wred[3] << 32) + wred[2], z);
        if (tid < a.top) {
            a.ids[(size_t)row * a.top + tid] = cs > 1 ? ci[tid] : gi[tid];
            a.tl[(size_t)row * a.top + tid] = lp_of((uint64_t)m - (uint64_t)(cs > 1 ? cv[tid] : gv[tid]), z);
        }
    }
}

}  // namespace iq
