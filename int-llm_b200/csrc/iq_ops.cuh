// iq_ops.cuh -- rotary tables and rotation, cache rows written and read back
// (the operator forms of rope_init / rope_apply, llama_int.c:960-1008, and of
// kv_pack_vector / kv_unpack_vector, llama_int.c:1197-1235).
#pragma once
#include "iq_layer.cuh"

namespace iq {

// acc += x y, unsigned
__device__ __forceinline__ void madu(uint64_t &acc, uint32_t x, uint32_t y) {
    asm("mad.wide.u32 %0, %1, %2, %0;" : "+l"(acc) : "r"(x), "r"(y));
}

// A bad index of a device array (not the -1 of a padding row): left out and recorded.
__device__ __forceinline__ bool index_ok(int i, int n) {
    if (i >= 0 && i < n) return true;
    if (i >= n) atomicExch(&g_iq_err, (int)IQ_ERR_RANGE);
    return false;
}

// ------------------------------------------------------------ rotary tables

struct RopeTab {
    int half, rot, n_pos, kind, orig_len;
    int64_t ln_theta, factor, low, span, mscale;   // span = high - low
};

// One frequency a pair (see iq_rope_scaling in iq.h).
__device__ __forceinline__ int64_t rope_freq(const RopeTab &t, int i, int64_t pi) {
    const int64_t y = d_mul(-d_div(d_from_int(2 * i), d_from_int(t.rot)), t.ln_theta);
    int64_t th;
    if (y < -10 * IQ_ONE) {   // fp_exp squares up to e^10.4 only
        th = d_exp(y >> 1);
        th = d_mul(th, th);
    } else {
        th = d_exp(y);
    }
    if (t.kind == IQ_ROPE_SCALE_LINEAR) return d_div(th, t.factor);
    if (t.kind == IQ_ROPE_SCALE_PARTS) {
        const uint64_t turns = (uint64_t)d_udiv128_64((u128)((u128)(uint64_t)t.orig_len * (uint64_t)th) << 48,
                                                      (uint64_t)(2 * pi));
        int64_t w = (int64_t)turns - t.low;
        w = d_div(min(max(w, (int64_t)0), t.span), t.span);
        return d_mul(th, w) + d_mul(d_div(th, t.factor), IQ_ONE - w);
    }
    return th;
}

// cos, sin [n_pos][half] of p th_i. The angle is reduced mod 2 pi from the exact
// product (p < 2^24, th <= 2^48): a double estimate of the quotient is within
// one of it, and the wrapped remainder is exact, so it equals fp_sincos's
// repeated subtraction (fp_math.h:861-902) at the positions where that has no
// overflow. Issue-bound on the 48 integer CORDIC steps, not on the 16 bytes an
// entry writes.
__global__ void __launch_bounds__(256) k_rope_tables(int64_t *__restrict__ cs, int64_t *__restrict__ sn, RopeTab t) {
    __shared__ int64_t th[128];
    const CordicTables &ct = g_cordic;
    const int64_t pi = ct.pi, w = 2 * pi;
    for (int i = threadIdx.x; i < t.half; i += blockDim.x) th[i] = rope_freq(t, i, pi);
    __syncthreads();
    const int64_t n = (int64_t)t.n_pos * t.half, step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t e = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; e < n; e += step) {
        const int p = (int)(e / t.half);
        const int64_t f = th[(int)(e - (int64_t)p * t.half)];
        const int64_t q = (int64_t)((double)p * (double)f / (double)w);
        int64_t a = (int64_t)((uint64_t)p * (uint64_t)f - (uint64_t)q * (uint64_t)w);
        if (a < 0) a += w;
        else if (a >= w) a -= w;
        if (a > pi) a -= w;
        int64_t c, s;
        d_sincos(ct, a, &c, &s);
        if (t.mscale) { c = d_mul(c, t.mscale); s = d_mul(s, t.mscale); }
        cs[e] = c;
        sn[e] = s;
    }
}

// ---------------------------------------------------------------- rotation

struct RopeArgs {
    const int64_t *cos, *sin;
    const int *pos;
    int n_pos, rot, layout;
};

// Elements (e0, e1) of pair p of a head: rotation pairs first, then the
// unrotated rest two by two (e1 may be hd when the rest is odd).
__device__ __forceinline__ void rope_pair(const RopeArgs &r, int p, int &e0, int &e1) {
    const int half = r.rot >> 1;
    if (p >= half) { e0 = 2 * p; e1 = e0 + 1; }
    else if (r.layout == IQ_ROPE_HALF) { e0 = p; e1 = p + half; }
    else { e0 = 2 * p; e1 = e0 + 1; }
}
__device__ __forceinline__ void rope_turn(int64_t &a, int64_t &b, int64_t c, int64_t s) {
    const int64_t u = (int64_t)((uint64_t)d_mul(a, c) - (uint64_t)d_mul(b, s));
    b = (int64_t)((uint64_t)d_mul(b, c) + (uint64_t)d_mul(a, s));
    a = u;
}

// One thread a pair; blockDim.y rows a block, blockIdx.y steps over the pairs
// of a row. Memory-bound: 8 bytes read and 8 written an element.
__global__ void __launch_bounds__(256)
k_rope(int64_t *__restrict__ out, const int64_t *__restrict__ x, RopeArgs r, int rows, int heads, int hd,
       int64_t xs, int64_t os) {
    const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= rows) return;
    const int pos = r.pos[row];
    if (!index_ok(pos, r.n_pos)) return;
    const int half = r.rot >> 1, np = (hd + 1) >> 1;
    const int64_t *c = r.cos + (size_t)pos * half, *s = r.sin + (size_t)pos * half;
    const int64_t *xr = x + row * xs;
    int64_t *orow = out + row * os;
    for (int it = blockIdx.y * blockDim.x + threadIdx.x; it < heads * np; it += gridDim.y * blockDim.x) {
        const int h = it / np, p = it - h * np;
        int e0, e1;
        rope_pair(r, p, e0, e1);
        e0 += h * hd;
        e1 += h * hd;
        if (p < half) {
            int64_t a = xr[e0], b = xr[e1];
            rope_turn(a, b, c[p], s[p]);
            orow[e0] = a;
            orow[e1] = b;
        } else {
            orow[e0] = xr[e0];
            if (2 * p + 1 < hd) orow[e1] = xr[e1];
        }
    }
}

// ------------------------------------------------------------------- cache

// b-bit code of x against the magnitude M (kv_pack_vector, llama_int.c:1197-1218):
// ((x + M) 2^b) / (2M) truncated, clamped to [0, 2^b - 1]. For M < 2^61 a double
// estimate (inv = 2^b / 2M; the quotient is below 2^17, so three roundings move
// it by less than 2^-34) is corrected by its exact remainder.
__device__ __forceinline__ int kv_code(int64_t x, int64_t M, int bits, double inv) {
    if (M == 0) return 0;
    const int64_t top = ((int64_t)1 << bits) - 1;
    if (M < (1ll << 61)) {
        const int64_t u = x + M, D = 2 * M;   // 0 <= u <= D
        int64_t q = (int64_t)((double)u * inv);
        const int64_t rem = (int64_t)(((uint64_t)u << bits) - (uint64_t)q * (uint64_t)D);
        if (rem < 0) q--;
        else if (rem >= D) q++;
        return (int)min(q, top);
    }
    const i128 num = (i128)(int64_t)((uint64_t)x + (uint64_t)M) * ((i128)1 << bits);
    i128 t = d_sdiv128_64(num, (int64_t)((uint64_t)M * 2));
    if (t < 0) t = 0;
    if (t > top) t = top;
    return (int)t;
}

// ((2q + 1) M >> b) - M (kv_unpack_vector, llama_int.c:1226-1235) from 32-bit halves of M:
// c M = c Mh 2^32 + c Ml with c < 2^17, and 2^32 is a multiple of 2^b.
__device__ __forceinline__ int64_t kv_value(int q, int64_t M, int bits) {
    const uint32_t c = 2 * q + 1;
    const uint64_t lo = (uint64_t)c * (uint32_t)M;
    const int64_t hi = (int64_t)(int)c * (int)(M >> 32);
    return (int64_t)(((uint64_t)hi << (32 - bits)) + (lo >> bits) - (uint64_t)M);
}

struct KVArgs {
    int64_t *k, *v;
    uint8_t *kq;
    uint16_t *vq;
    int64_t *kmag, *vmag;
    int seqs, max_seq, nkv, hd, kbits, vbits;
};

// One warp a vector of (row, kv head, K or V), the vector in registers (hd <=
// 256: up to 4 pairs a lane): rotate, take the magnitude, write the codes.
template <bool PACKED>
__global__ void __launch_bounds__(256)
k_kv_write(KVArgs c, const int64_t *__restrict__ k, const int64_t *__restrict__ v, const int *__restrict__ seq,
           const int *__restrict__ slot, int rows, int64_t ks, int64_t vs, RopeArgs r) {
    const int64_t gw = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (gw >= (int64_t)rows * c.nkv * 2) return;
    const int which = (int)(gw & 1);
    const int64_t row = (gw >> 1) / c.nkv;
    const int h = (int)((gw >> 1) - row * c.nkv);
    const int sq = seq ? seq[row] : 0, t = slot[row];
    if (!index_ok(sq, c.seqs) || !index_ok(t, c.max_seq)) return;
    int pos = 0;
    if (r.cos) {   // both vectors of a row without a position are left out
        pos = r.pos[row];
        if (!index_ok(pos, r.n_pos)) return;
    }
    RopeArgs rr = r;
    if (which || !r.cos) rr.rot = 0;
    const int half = rr.rot >> 1, np = (c.hd + 1) >> 1;
    const int64_t *src = which ? v + row * vs + (int64_t)h * c.hd : k + row * ks + (int64_t)h * c.hd;
    const int64_t *cs = rr.rot ? r.cos + (size_t)pos * half : nullptr, *sn = rr.rot ? r.sin + (size_t)pos * half : nullptr;
    const size_t vec = ((size_t)sq * c.max_seq + t) * c.nkv + h, e0v = vec * c.hd;
    int64_t a[4], b[4], M = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int p = lane + 32 * j;
        a[j] = b[j] = 0;
        if (p >= np) continue;
        int e0, e1;
        rope_pair(rr, p, e0, e1);
        a[j] = src[e0];
        if (e1 < c.hd) b[j] = src[e1];
        if (p < half) rope_turn(a[j], b[j], cs[p], sn[p]);
        if (PACKED) {   // |INT64_MIN| wraps to itself, below every magnitude, as in the reference
            const int64_t ma = a[j] < 0 ? (int64_t)(0 - (uint64_t)a[j]) : a[j];
            const int64_t mb = b[j] < 0 ? (int64_t)(0 - (uint64_t)b[j]) : b[j];
            M = max(M, max(ma, mb));
        }
    }
    double inv = 0;
    const int bits = which ? c.vbits : c.kbits;
    if (PACKED) {
        for (int m = 16; m >= 1; m >>= 1) M = max(M, (int64_t)__shfl_xor_sync(0xffffffffu, M, m));
        if (lane == 0) (which ? c.vmag : c.kmag)[vec] = M;
        if (M && M < (1ll << 61)) inv = (double)(1 << bits) / (double)(2 * M);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int p = lane + 32 * j;
        if (p >= np) continue;
        int e0, e1;
        rope_pair(rr, p, e0, e1);
        if (PACKED) {
            const int q0 = kv_code(a[j], M, bits, inv), q1 = kv_code(b[j], M, bits, inv);
            if (which) {
                c.vq[e0v + e0] = (uint16_t)q0;
                if (e1 < c.hd) c.vq[e0v + e1] = (uint16_t)q1;
            } else {
                c.kq[e0v + e0] = (uint8_t)q0;
                if (e1 < c.hd) c.kq[e0v + e1] = (uint8_t)q1;
            }
        } else {
            int64_t *dst = (which ? c.v : c.k) + e0v;
            dst[e0] = a[j];
            if (e1 < c.hd) dst[e1] = b[j];
        }
    }
}

// One warp a vector, as k_kv_write.
__global__ void __launch_bounds__(256)
k_kv_read(int64_t *__restrict__ k, int64_t *__restrict__ v, KVArgs c, const int *__restrict__ seq,
          const int *__restrict__ slot, int rows) {
    const int64_t gw = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (gw >= (int64_t)rows * c.nkv * 2) return;
    const int which = (int)(gw & 1);
    const int64_t row = (gw >> 1) / c.nkv;
    const int h = (int)((gw >> 1) - row * c.nkv);
    const int sq = seq ? seq[row] : 0, t = slot[row];
    if (!index_ok(sq, c.seqs) || !index_ok(t, c.max_seq)) return;
    const size_t vec = ((size_t)sq * c.max_seq + t) * c.nkv + h, e0 = vec * c.hd;
    int64_t *dst = (which ? v : k) + (row * c.nkv + h) * c.hd;
    if (c.kbits) {
        const int64_t M = (which ? c.vmag : c.kmag)[vec];
        const int bits = which ? c.vbits : c.kbits;
        for (int d = lane; d < c.hd; d += 32) dst[d] = kv_value(which ? c.vq[e0 + d] : c.kq[e0 + d], M, bits);
    } else {
        const int64_t *src = (which ? c.v : c.k) + e0;
        for (int d = lane; d < c.hd; d += 32) dst[d] = src[d];
    }
}

}  // namespace iq
