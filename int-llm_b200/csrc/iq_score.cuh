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

// floor(e^-d) in Q16.48, d = max - logit as an unsigned difference
__device__ __forceinline__ int64_t lp_exp(uint64_t d, const int64_t *pw) {
    if (d >= (34ull << 48)) return 0;
    const uint64_t y = __umul64hi(d << 4, (uint64_t)IQ_LP_LOG2E_60);   // (d log2e) >> 60
    const int64_t f = (int64_t)(y & ((1ull << 48) - 1)), r = f & ((1ll << 42) - 1);
    int64_t h = 375306296874ll;
    h = 2707262666570ll - d_mul(h, r);
    h = 15623017693776ll - d_mul(h, r);
    h = 67617750451595ll - d_mul(h, r);
    h = 195103586505167ll - d_mul(h, r);
    h = 281474976710656ll - d_mul(h, r);
    return d_mul(pw[f >> 42], h) >> (y >> 48);
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
};

// One CTA a row; the top alternatives by one search of the row for each.
__global__ void __launch_bounds__(1024) k_logprobs_simple(LpArgs a) {
    __shared__ uint64_t red[64];
    __shared__ int64_t bv[32];
    __shared__ int bi[32];
    const int row = blockIdx.x;
    const int64_t *l = a.lg + row * a.ld;
    int64_t m = INT64_MIN;
    for (int i = threadIdx.x; i < a.V; i += blockDim.x) m = max(m, l[i]);
    m = cta_max_i64(m, (int64_t *)red);
    u128 S = 0, A = 0;
    for (int i = threadIdx.x; i < a.V; i += blockDim.x) {
        const uint64_t d = (uint64_t)m - (uint64_t)l[i];
        const int64_t e = lp_exp(d, c_lp_pow);
        S += (uint64_t)e;
        if (e) A += (uint64_t)d_mul(e, (int64_t)d);
    }
    S = (u128)cta_sum_i128((i128)S, red);
    A = (u128)cta_sum_i128((i128)A, red);
    const int64_t z = lp_ln(S);
    if (threadIdx.x == 0) {
        if (a.tok && index_ok(a.tok[row], a.V)) a.logp[row] = lp_of((uint64_t)m - (uint64_t)l[a.tok[row]], z);
        if (a.ent) a.ent[row] = lp_entropy(S, A, z);
    }
    int64_t pv = INT64_MAX;
    int pi = -1;
    for (int k = 0; k < a.top; k++) {   // the first after (pv, pi) in falling value, rising index
        int64_t best = INT64_MIN;
        int idx = 0x7fffffff;
        for (int i = threadIdx.x; i < a.V; i += blockDim.x) {
            const int64_t v = l[i];
            if ((v < pv || (v == pv && i > pi)) && (v > best || (v == best && i < idx))) { best = v; idx = i; }
        }
        for (int o = 16; o >= 1; o >>= 1) {
            const int64_t ov = __shfl_xor_sync(0xffffffffu, best, o);
            const int oi = __shfl_xor_sync(0xffffffffu, idx, o);
            if (ov > best || (ov == best && oi < idx)) { best = ov; idx = oi; }
        }
        __syncthreads();
        if ((threadIdx.x & 31) == 0) { bv[threadIdx.x >> 5] = best; bi[threadIdx.x >> 5] = idx; }
        __syncthreads();
        for (int w = 0; w < 32; w++)
            if (bv[w] > best || (bv[w] == best && bi[w] < idx)) { best = bv[w]; idx = bi[w]; }
        if (threadIdx.x == 0) {
            a.ids[(size_t)row * a.top + k] = idx;
            a.tl[(size_t)row * a.top + k] = lp_of((uint64_t)m - (uint64_t)best, z);
        }
        pv = best;
        pi = idx;
    }
}

}  // namespace iq
