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

// 1 / x by two Newton steps, relative error below 2^-51
__device__ __forceinline__ double f64_rcp(double x) {
    double y;
    asm("rcp.approx.ftz.f64 %0, %1;" : "=d"(y) : "d"(x));
    y = __fma_rn(y, __fma_rn(-x, y, 1.0), y);
    return __fma_rn(y, __fma_rn(-x, y, 1.0), y);
}
// the positive 64-bit x as a double (one rounding)
__device__ __forceinline__ double f64_u64(uint64_t x) {
    return (__longlong_as_double((long long)((x >> 32) | 0x4530000000000000ull)) - 19342813118337666422669312.0) +
           __longlong_as_double((long long)((x & 0xFFFFFFFFull) | 0x4330000000000000ull));
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
    int64_t pi, gain, angles[25];                  // of the CORDIC; from step 25 on the angle is 2^(48 - i)
};

// One frequency a pair (see iq_rope_scaling in iq.h).
__device__ __forceinline__ int64_t rope_freq(const RopeTab &t, int i) {
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
                                                      (uint64_t)(2 * t.pi));
        int64_t w = (int64_t)turns - t.low;
        w = d_div(min(max(w, (int64_t)0), t.span), t.span);
        return d_mul(th, w) + d_mul(d_div(th, t.factor), IQ_ONE - w);
    }
    return th;
}

// CORDIC steps I .. 47 of (x, y) by the angle z (fp_sincos, fp_math.h:861-902). From step
// 18 on the shifted values and the angle fit 32 bits (|x|, |y| stay below 2^48.1), so
// that sign and sum are one wide multiply-add: 7 instructions a step against 17.
template <int I>
__device__ __forceinline__ void cordic(const RopeTab &t, int64_t &x, int64_t &y, int64_t &z) {
    if constexpr (I < 48) {
        if constexpr (I < 18) {
            const int64_t xs = x >> I, ys = y >> I, a = t.angles[I];
            if (z >= 0) { x -= ys; y += xs; z -= a; }
            else        { x += ys; y -= xs; z += a; }
        } else {
            const int sg = (int)(z >> 63) | 1, xs = (int)(x >> I), ys = (int)(y >> I);
            const int a = I < 25 ? (int)t.angles[I] : (int)(IQ_ONE >> I);
            madw(x, -sg, ys);
            madw(y, sg, xs);
            madw(z, -sg, a);
        }
        cordic<I + 1>(t, x, y, z);
    }
}

// cos, sin [n_pos][half] of p th_i. The angle is reduced mod 2 pi from the exact
// product (p < 2^24, th <= 2^48): a double estimate of the quotient is within
// one of it, and the wrapped remainder is exact, so it equals fp_sincos's
// repeated subtraction at the positions where that has no overflow.
// Bound by the 48 CORDIC steps, each waiting for the one before, not by the 16 bytes an
// entry writes: 65536 positions of 64 pairs 154 us (67 MB would take 10; 109 M warp
// instructions, 62 % of the issue slots), with 64-bit steps throughout 199.
__global__ void __launch_bounds__(256) k_rope_tables(int64_t *__restrict__ cs, int64_t *__restrict__ sn,
                                                     const __grid_constant__ RopeTab t) {
    __shared__ int64_t th[128];
    const int64_t pi = t.pi, w = 2 * pi, half_pi = pi >> 1;
    for (int i = threadIdx.x; i < t.half; i += blockDim.x) th[i] = rope_freq(t, i);
    __syncthreads();
    const int64_t n = (int64_t)t.n_pos * t.half, step = (int64_t)gridDim.x * blockDim.x;
    const double inv_w = 1.0 / (double)w;
    for (int64_t e = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; e < n; e += step) {
        const int p = (int)((uint32_t)e / (uint32_t)t.half);   // n <= 2^31
        const int64_t f = th[(int)(e - (int64_t)p * t.half)];
        const int64_t q = (int64_t)((double)p * (double)f * inv_w);
        int64_t a = (int64_t)((uint64_t)p * (uint64_t)f - (uint64_t)q * (uint64_t)w);
        if (a < 0) a += w;
        else if (a >= w) a -= w;
        if (a > pi) a -= w;
        const bool neg = a > half_pi || a < -half_pi;
        int64_t z = a > half_pi ? pi - a : a < -half_pi ? -pi - a : a, x = t.gain, y = 0;
        cordic<0>(t, x, y, z);
        if (neg) x = -x;
        if (t.mscale) { x = d_mul(x, t.mscale); y = d_mul(y, t.mscale); }
        cs[e] = x;
        sn[e] = y;
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

// Wide form (hd and rot multiples of 4, everything 16-byte aligned): item q of a
// head is the four elements ea, ea + 1, eb, eb + 1, moved as two pieces of 16 bytes.
struct RopeItem { int ea, eb, turn; };
__device__ __forceinline__ RopeItem rope_item(const RopeArgs &r, int q) {
    RopeItem it;
    it.turn = 4 * q < r.rot;
    if (it.turn && r.layout == IQ_ROPE_HALF) { it.ea = 2 * q; it.eb = 2 * q + (r.rot >> 1); }
    else { it.ea = 4 * q; it.eb = 4 * q + 2; }
    return it;
}
// fp_mul for |x| < 2^59 and |c| < 2^49: with both halves signed, x = xh 2^32 + xl and
// c = ch 2^32 + cl, every product is one wide multiply-add:
// floor(x c / 2^48) = 8 xh 2^13 ch + floor((xh cl + xl ch + floor(xl cl / 2^32)) / 2^16).
// A negative low half carries into the high one, so |xh| <= 2^27 and |ch| <= 2^17 with
// both ends: 8 xh and 2^13 ch stay within 2^30.
struct Half { int h, l; };
__device__ __forceinline__ Half halves(int64_t x) {
    const int l = (int)(uint32_t)x;
    return Half{(int)(x >> 32) - (l >> 31), l};
}
__device__ __forceinline__ int64_t mul_small(const Half &x, const Half &c) {
    int64_t t = __mulhi(x.l, c.l);
    madw(t, x.h, c.l);
    madw(t, x.l, c.h);
    t >>= 16;
    madw(t, x.h * 8, c.h * (1 << 13));
    return t;
}
__device__ __forceinline__ void turn_small(int64_t &a, int64_t &b, int64_t c, int64_t s) {
    const Half x = halves(a), y = halves(b), u = halves(c), v = halves(s);
    a = mul_small(x, u) - mul_small(y, v);
    b = mul_small(y, u) + mul_small(x, v);
}
// 0 where -2^(32 + k) <= x < 2^(32 + k)
__device__ __forceinline__ uint32_t beyond(int64_t x, int k) { return ((uint32_t)(x >> 32) + (1u << k)) >> (k + 1); }

// (a, b) and the row's tables c, s of the item's two pairs
__device__ __forceinline__ void rope_turn4(const RopeArgs &r, longlong2 &a, longlong2 &b, const longlong2 &c, const longlong2 &s) {
    int64_t v[4] = {a.x, a.y, b.x, b.y};
    if (r.layout == IQ_ROPE_HALF) { v[1] = b.x; v[2] = a.y; }   // pairs (0, 1), (2, 3)
    if ((beyond(a.x, 27) | beyond(a.y, 27) | beyond(b.x, 27) | beyond(b.y, 27) | beyond(c.x, 17) | beyond(c.y, 17) |
         beyond(s.x, 17) | beyond(s.y, 17)) == 0) {
        turn_small(v[0], v[1], c.x, s.x);
        turn_small(v[2], v[3], c.y, s.y);
    } else {
        rope_turn(v[0], v[1], c.x, s.x);
        rope_turn(v[2], v[3], c.y, s.y);
    }
    if (r.layout == IQ_ROPE_HALF) {
        const int64_t w = v[1];
        v[1] = v[2];
        v[2] = w;
    }
    a = make_longlong2(v[0], v[1]);
    b = make_longlong2(v[2], v[3]);
}

// One thread an item (W) or a pair; blockDim.y rows a block, blockIdx.y steps
// over the items of a row. Memory-bound: 8 bytes read and 8 written an element (2048
// rows of 64 heads of 128: 57 us, 4.7 TB/s, issue 60 %; pair by pair 96 us).
template <bool W>
__global__ void __launch_bounds__(256)
k_rope(int64_t *__restrict__ out, const int64_t *__restrict__ x, RopeArgs r, int rows, int heads, int hd,
       int64_t xs, int64_t os) {
    const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= rows) return;
    const int pos = r.pos[row];
    if (!index_ok(pos, r.n_pos)) return;
    const int half = r.rot >> 1, np = W ? hd >> 2 : (hd + 1) >> 1;
    const int64_t *c = r.cos + (size_t)pos * half, *s = r.sin + (size_t)pos * half;
    const int64_t *xr = x + row * xs;
    int64_t *orow = out + row * os;
    for (int it = blockIdx.y * blockDim.x + threadIdx.x; it < heads * np; it += gridDim.y * blockDim.x) {
        const int h = it / np, p = it - h * np;
        if (W) {
            const RopeItem q = rope_item(r, p);
            longlong2 a = *reinterpret_cast<const longlong2 *>(xr + h * hd + q.ea);
            longlong2 b = *reinterpret_cast<const longlong2 *>(xr + h * hd + q.eb);
            if (q.turn)
                rope_turn4(r, a, b, __ldg(reinterpret_cast<const longlong2 *>(c) + p),
                           __ldg(reinterpret_cast<const longlong2 *>(s) + p));
            *reinterpret_cast<longlong2 *>(orow + h * hd + q.ea) = a;
            *reinterpret_cast<longlong2 *>(orow + h * hd + q.eb) = b;
            continue;
        }
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
// ((x + M) 2^b) / (2M) truncated, clamped to [0, 2^b - 1]. For M < 2^61 the quotient
// (at most 2^16) by a double factor (kv_mag: three roundings, then lowered, so
// that its floor is q or q - 1); the exact remainder's sign tells which.
struct KVMag {
    int64_t M;
    uint64_t D;     // 2M, or 1 where M is 0 (every code is 0 then)
    double inv;     // 2^b / D lowered by 2^-50
    int bits, top;
};
__device__ __forceinline__ KVMag kv_mag(int64_t M, int bits) {
    KVMag m;
    m.M = M;
    m.D = M ? 2 * (uint64_t)M : 1;
    m.inv = f64_rcp(f64_u64(m.D)) * ((double)(1 << bits) * (1.0 - 0x1p-50));
    m.bits = bits;
    m.top = (1 << bits) - 1;
    return m;
}
__device__ __forceinline__ int kv_code(int64_t x, const KVMag &m) {   // |x| <= M < 2^61
    const uint64_t u = (uint64_t)(x + m.M);   // u <= D
    // the floored quotient in the binade of 2^52
    const uint32_t q = (uint32_t)__double_as_longlong(__fma_rd(f64_u64(u), m.inv, 4503599627370496.0));
    // sign of (q + 1) D - u 2^b - 1
    uint64_t t = m.D - 1 - (u << m.bits);
    madu(t, q, (uint32_t)m.D);
    const uint32_t h = (uint32_t)(t >> 32) + q * (uint32_t)(m.D >> 32);
    return min((int)(q + (h >> 31)), m.top);
}
// the same for any x and M, as the reference's int64 wraps
__device__ __noinline__ int kv_code_any(int64_t x, int64_t M, int bits) {
    if (M == 0) return 0;
    const int64_t top = ((int64_t)1 << bits) - 1;
    const i128 num = (i128)(int64_t)((uint64_t)x + (uint64_t)M) * ((i128)1 << bits);
    i128 t = d_sdiv128_64(num, (int64_t)((uint64_t)M * 2));
    if (t < 0) t = 0;
    if (t > top) t = top;
    return (int)t;
}

// The magnitude of x as the reference takes it: |INT64_MIN| wraps to itself, below every
// other, so that an element can lie below -M. `hi` gathers the high words, for kv_fits.
__device__ __forceinline__ int64_t kv_abs(int64_t x, uint32_t &hi) {
    const int64_t a = x < 0 ? (int64_t)(0 - (uint64_t)x) : x;
    hi |= (uint32_t)(a >> 32);
    return a;
}
// whether the elements of which kv_abs gathered hi, of a vector of magnitude M, may take kv_code
__device__ __forceinline__ bool kv_fits(uint32_t hi, int64_t M) { return M < (1ll << 61) && (int)hi >= 0; }

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

// Wide form: L lanes (a power of two) a vector of (row, kv head, K or V), each with
// NJ items of four elements: rotate, take the magnitude, write the codes. One item a
// lane up to 128-wide heads (2048 rows of 32 heads of 128 written as codes: 82 us,
// issue-bound at 68 %, two products a rotated element and an exact quotient; two items a
// lane and a divided reciprocal 103 us, the narrow form 123).
template <bool PACKED, int NJ>
__global__ void __launch_bounds__(256)
k_kv_write_wide(KVArgs c, const int64_t *__restrict__ k, const int64_t *__restrict__ v, const int *__restrict__ seq,
                const int *__restrict__ slot, int rows, int64_t ks, int64_t vs, RopeArgs r, int log_l) {
    const int L = 1 << log_l;
    const int64_t gv = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> log_l;
    const int lane = threadIdx.x & (L - 1);
    bool live = gv < (int64_t)rows * c.nkv * 2;
    const int which = (int)(gv & 1);
    const uint32_t rh = (uint32_t)(gv >> 1), row = rh / (uint32_t)c.nkv, h = rh - row * c.nkv;
    int sq = 0, t = 0, pos = 0;
    if (live) {
        sq = seq ? seq[row] : 0;
        t = slot[row];
        if (r.cos) pos = r.pos[row];   // both vectors of a row without a position are left out
        live = index_ok(sq, c.seqs) && index_ok(t, c.max_seq) && (!r.cos || index_ok(pos, r.n_pos));
    }
    if (which || !r.cos) r.rot = 0;
    const int half = r.rot >> 1, np = c.hd >> 2;
    const int64_t *src = which ? v + row * vs + (int64_t)h * c.hd : k + row * ks + (int64_t)h * c.hd;
    const longlong2 *cs = reinterpret_cast<const longlong2 *>(r.cos + (size_t)pos * half);
    const longlong2 *sn = reinterpret_cast<const longlong2 *>(r.sin + (size_t)pos * half);
    const size_t vec = ((size_t)sq * c.max_seq + t) * c.nkv + h, e0 = vec * c.hd;
    longlong2 a[NJ], b[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const int q = lane + j * L;
        a[j] = b[j] = make_longlong2(0, 0);
        if (live && q < np) {
            const RopeItem it = rope_item(r, q);
            a[j] = __ldg(reinterpret_cast<const longlong2 *>(src + it.ea));
            b[j] = __ldg(reinterpret_cast<const longlong2 *>(src + it.eb));
        }
    }
    int64_t M = 0;
    uint32_t hi = 0;
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const int q = lane + j * L;
        if (live && q < np && 4 * q < r.rot) rope_turn4(r, a[j], b[j], __ldg(cs + q), __ldg(sn + q));
        if (PACKED) {
            const int64_t w[4] = {a[j].x, a[j].y, b[j].x, b[j].y};
#pragma unroll
            for (int i = 0; i < 4; i++) M = max(M, kv_abs(w[i], hi));
        }
    }
    const int bits = which ? c.vbits : c.kbits;
    KVMag km = {};
    bool fits = true;
    if (PACKED) {
        for (int m = L >> 1; m >= 1; m >>= 1) M = max(M, (int64_t)__shfl_xor_sync(0xffffffffu, M, m));
        if (live && lane == 0) (which ? c.vmag : c.kmag)[vec] = M;
        km = kv_mag(M, bits);
        fits = kv_fits(hi, M);
    }
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const int q = lane + j * L;
        if (!live || q >= np) continue;
        const RopeItem it = rope_item(r, q);
        if (PACKED) {
            int c0, c1, c2, c3;
            if (fits) {
                c0 = kv_code(a[j].x, km);
                c1 = kv_code(a[j].y, km);
                c2 = kv_code(b[j].x, km);
                c3 = kv_code(b[j].y, km);
            } else {
                c0 = kv_code_any(a[j].x, M, bits);
                c1 = kv_code_any(a[j].y, M, bits);
                c2 = kv_code_any(b[j].x, M, bits);
                c3 = kv_code_any(b[j].y, M, bits);
            }
            if (which) {
                *reinterpret_cast<ushort2 *>(c.vq + e0 + it.ea) = make_ushort2(c0, c1);
                *reinterpret_cast<ushort2 *>(c.vq + e0 + it.eb) = make_ushort2(c2, c3);
            } else {
                *reinterpret_cast<uchar2 *>(c.kq + e0 + it.ea) = make_uchar2(c0, c1);
                *reinterpret_cast<uchar2 *>(c.kq + e0 + it.eb) = make_uchar2(c2, c3);
            }
        } else {
            int64_t *dst = (which ? c.v : c.k) + e0;
            *reinterpret_cast<longlong2 *>(dst + it.ea) = a[j];
            *reinterpret_cast<longlong2 *>(dst + it.eb) = b[j];
        }
    }
}

// One warp a vector, any hd <= 256 and alignment: up to 4 pairs a lane.
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
    uint32_t hi = 0;
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
        if (PACKED) {
            M = max(M, kv_abs(a[j], hi));
            M = max(M, kv_abs(b[j], hi));
        }
    }
    KVMag km = {};
    bool fits = true;
    const int bits = which ? c.vbits : c.kbits;
    if (PACKED) {
        for (int m = 16; m >= 1; m >>= 1) M = max(M, (int64_t)__shfl_xor_sync(0xffffffffu, M, m));
        if (lane == 0) (which ? c.vmag : c.kmag)[vec] = M;
        km = kv_mag(M, bits);
        fits = kv_fits(hi, M);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int p = lane + 32 * j;
        if (p >= np) continue;
        int e0, e1;
        rope_pair(rr, p, e0, e1);
        if (PACKED) {
            const int q0 = fits ? kv_code(a[j], km) : kv_code_any(a[j], M, bits);
            const int q1 = fits ? kv_code(b[j], km) : kv_code_any(b[j], M, bits);
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

// A thread four elements (W: hd a multiple of 4, aligned) or one, K and V in turn
// (2048 rows of 4 heads of 64 codes to int64: 7.7 us).
template <bool W>
__global__ void __launch_bounds__(256)
k_kv_read(int64_t *__restrict__ k, int64_t *__restrict__ v, KVArgs c, const int *__restrict__ seq,
          const int *__restrict__ slot, int rows) {
    const uint32_t np = W ? c.hd >> 2 : c.hd;
    const int64_t n = (int64_t)rows * c.nkv * 2 * np;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t gv = n >> 32 ? i / np : (uint32_t)i / np;
        const int d = (int)(i - gv * np) * (W ? 4 : 1), which = (int)(gv & 1);
        const uint32_t rh = (uint32_t)(gv >> 1), row = rh / (uint32_t)c.nkv, h = rh - row * c.nkv;
        const int sq = seq ? seq[row] : 0, t = slot[row];
        if (!index_ok(sq, c.seqs) || !index_ok(t, c.max_seq)) continue;
        const size_t vec = ((size_t)sq * c.max_seq + t) * c.nkv + h, e = vec * c.hd + d;
        int64_t *dst = (which ? v : k) + (size_t)rh * c.hd + d;
        const int64_t M = c.kbits ? __ldg((which ? c.vmag : c.kmag) + vec) : 0;
        const int bits = which ? c.vbits : c.kbits;
        if (!W) {
            *dst = c.kbits ? kv_value(which ? c.vq[e] : c.kq[e], M, bits) : (which ? c.v : c.k)[e];
            continue;
        }
        longlong2 a, b;
        if (c.kbits) {
            ushort4 q;
            if (which) q = __ldg(reinterpret_cast<const ushort4 *>(c.vq + e));
            else {
                const uchar4 u = __ldg(reinterpret_cast<const uchar4 *>(c.kq + e));
                q = make_ushort4(u.x, u.y, u.z, u.w);
            }
            a = make_longlong2(kv_value(q.x, M, bits), kv_value(q.y, M, bits));
            b = make_longlong2(kv_value(q.z, M, bits), kv_value(q.w, M, bits));
        } else {
            const longlong2 *p = reinterpret_cast<const longlong2 *>((which ? c.v : c.k) + e);
            a = p[0];
            b = p[1];
        }
        reinterpret_cast<longlong2 *>(dst)[0] = a;
        reinterpret_cast<longlong2 *>(dst)[1] = b;
    }
}

}  // namespace iq
