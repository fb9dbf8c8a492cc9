// iq_tree.cuh -- attention of drafted tokens over the cache (iq_attn_tree_dev).
// Per node row r and query head h, over the positions t it sees (all before
// the draft, its ancestors, itself), in the reference's order (llama_int.c:1432-1529):
//   s_t = fp_mul((int64)(sum_d (i128)q[d] k_t[d] >> 48), fp_inv_sqrt(hd))
//   m = max s;  e_t = fp_safe_exp(s_t - m);  S = sum e;  p_t = S > 0 ? fp_div(e_t, S) : e_t
//   out[d] = sum_t fp_mul(p_t, v_t[d])   (wrapping int64)
//
// One cluster of CTAs takes NC = 8 NT columns (node, query head of one kv head)
// of a sequence; its CTAs split the positions, so K and V are read once for all
// the columns and the scores stay in shared memory (in the workspace when they
// do not fit). Maxima, sums and partial outputs meet over distributed shared
// memory; all of them are whole numbers, so the split changes nothing.
//
// 1. Scores on the int8 tensor cores: byte planes of K (A: 16 positions x 32 d)
//    and Q (B: 32 d x 8 columns), the pairs of each diagonal i + j in one s32
//    (see k_attn_scores_tc). Where every |x| < 2^55 (128.0) on both sides
//    plane 6 is the signed top and 49 of the 63 products remain.
// 2. fp_safe_exp and fp_div in doubles with directed rounding. With r = 2^48 + f,
//    floor(r^2 / 2^48) = 2^48 + 2f + floor(f^2 / 2^48), and as long as the result is below
//    2^52 an fma that rounds down at M = 2^52 (one unit = one ulp) gives the
//    floor: g = M + f -> fma.rd(f 2^-24, f 2^-24, M + 2f). 12 of the 14 squarings
//    fit (r <= e^2.5); the last two take 32-bit pieces.
// 3. sum_t floor(p_t v_t / 2^48) as one chain of fma.rd per output at 1.5 2^52: with p
//    and v exact in doubles and the running sum within 2^51, each step adds
//    exactly floor(p v 2^-48). As sum p <= 2^48 that holds for |v| <= 2^51 - 2^16
//    (8.0). Up to |v| < 2^54 (64.0), v = n 2^51 + f with |f| <= 2^50 and
//    floor(p v / 2^48) = 8 p n + floor(p f / 2^48): a second, exact chain. Larger values take
//    fp_mul term by term. One DFMA a term against six integer instructions of
//    the remainder form (k_attn_pv_tc).
#pragma once
#include <cooperative_groups.h>
#include "iq_ops.cuh"

namespace iq {

#define TREE_MAX_NODES 256

struct TreeArgs {
    int64_t *out;
    const int64_t *q;
    KVArgs c;
    const int *seq, *len, *start, *parent;
    int n_seq, rows, max_nodes, max_len, nh;
    int64_t qs, scale;
    int64_t *sc;   // [CTA][NC][Ts] scores where they do not fit shared memory, else null
    int cs, blocks, Ts, vec;   // CTAs a cluster, column blocks a kv head, row stride of the scores, wide loads
};

struct TreeSeq { int row0, n, len, sq; };

// Sequence b's rows and lengths; false (and recorded) when they leave the call's bounds.
__device__ __forceinline__ bool tree_seq(const TreeArgs &a, int b, TreeSeq &s) {
    s.sq = a.seq ? a.seq[b] : b;
    s.len = a.len[b];
    s.row0 = a.start[b];
    s.n = a.start[b + 1] - s.row0;
    if (s.n == 0) return false;
    const bool ok = s.sq >= 0 && s.sq < a.c.seqs && s.row0 >= 0 && s.n > 0 && s.n <= a.max_nodes &&
                    s.row0 <= a.rows - s.n && s.len >= 0 && s.len <= a.max_len - s.n;
    if (!ok && s.sq != -1) atomicExch(&g_iq_err, (int)IQ_ERR_RANGE);
    return ok;
}

// ---- exponentials and quotients

#define TREE_M 4503599627370496.0            // 2^52
#define TREE_MB 0x4330000000000000ull        // its bits
#define TREE_A 6755399441055744.0            // 1.5 2^52
#define TREE_AB 0x4338000000000000ull

__device__ __forceinline__ double tree_u52(uint64_t x) {   // exact for x < 2^52
    return __longlong_as_double((long long)(x | TREE_MB)) - TREE_M;
}
// floor(r^2 / 2^48) for r < 2^56
__device__ __forceinline__ uint64_t tree_sqr(uint64_t r) {
    const uint32_t l = (uint32_t)r, h = (uint32_t)(r >> 32);
    return (((uint64_t)h * h) << 16) + ((((uint64_t)h * l << 1) + __umulhi(l, l)) >> 16);
}
// fp_exp(-d) (fp_math.h:714-732) for 0 <= d <= 10
__device__ __forceinline__ int64_t tree_exp(uint64_t d) {
    double g = __longlong_as_double((long long)((d >> 14) | TREE_MB));
#pragma unroll
    for (int i = 0; i < 12; i++) {
        const double u = __fma_rn(g, 0x1p-24, -TREE_M * 0x1p-24);
        g = __fma_rd(u, u, __fma_rn(g, 2.0, -TREE_M));
    }
    const uint64_t r12 = IQ_ONE + ((uint64_t)__double_as_longlong(g) & 0xFFFFFFFFFFFFFull);
    const uint64_t r = tree_sqr(tree_sqr(r12));   // 2^48 <= r < 2^62.5
    // floor(2^96 / r): reciprocal by two Newton steps (relative error below
    // 2^-51, so the quotient, at most 2^48, is off by less than 1/8), floored,
    // then one exact remainder (2^96 = 0 mod 2^64)
    const double rd = (__longlong_as_double((long long)((r >> 32) | 0x4530000000000000ull)) - 19342813118337666422669312.0) +
                      __longlong_as_double((long long)((r & 0xFFFFFFFFull) | TREE_MB));
    double y;
    asm("rcp.approx.ftz.f64 %0, %1;" : "=d"(y) : "d"(rd));
    y = __fma_rn(y, __fma_rn(-rd, y, 1.0), y);
    y = __fma_rn(y, __fma_rn(-rd, y, 1.0), y);
    uint64_t q = (uint64_t)__double_as_longlong(__fma_rd(y, 0x1p96, TREE_M)) & 0xFFFFFFFFFFFFFull;
    const int64_t rem = (int64_t)(0 - q * r);
    if (rem < 0) q--;
    else if ((uint64_t)rem >= r) q++;
    return (int64_t)q;
}
// fp_div(e, S) for 0 <= e <= 2^48 <= S < 2^63, e <= S, inv = 2^48 / S
__device__ __forceinline__ uint64_t tree_prob(int64_t e, int64_t S, double inv) {
    uint64_t q = (uint64_t)__double_as_longlong(__fma_rd(tree_u52((uint64_t)e), inv, TREE_M)) & 0xFFFFFFFFFFFFFull;
    const int64_t rem = (int64_t)(((uint64_t)e << 48) - q * (uint64_t)S);
    if (rem < 0) q--;
    else if (rem >= S) q++;
    return q;
}
// fp_mul(s, c) for 0 <= c <= 2^48 (the score scale)
__device__ __forceinline__ int64_t tree_scale(int64_t s, uint64_t c) {
    const uint32_t sl = (uint32_t)s, cl = (uint32_t)c, ch = (uint32_t)(c >> 32);
    const int64_t sh = s >> 32;
    const int64_t t = (int64_t)((uint64_t)sl * ch + __umulhi(sl, cl)), u = sh * (int64_t)cl;
    return (int64_t)((uint64_t)(sh * (int64_t)ch) << 16) + (t >> 16) + (u >> 16) + (((t & 0xFFFF) + (u & 0xFFFF)) >> 16);
}

// ---- the kernel

#define TREE_V 4096   // doubles of a staged value tile

template <bool PK>
__device__ __forceinline__ int64_t tree_at(const KVArgs &c, bool val, size_t vec, int d) {
    const size_t e = vec * c.hd + d;
    if (!PK) return (val ? c.v : c.k)[e];
    return val ? kv_value(c.vq[e], c.vmag[vec], c.vbits) : kv_value(c.kq[e], c.kmag[vec], c.kbits);
}
// elements d .. d + 3 of a vector, zero from hd on
template <bool PK>
__device__ __forceinline__ void tree_at4(const TreeArgs &a, bool val, size_t vec, int d, int64_t (&x)[4]) {
    const KVArgs &c = a.c;
    if (a.vec && d < c.hd) {   // hd a multiple of 4, aligned bases
        const size_t e = vec * c.hd + d;
        if (!PK) {
            const longlong2 *p = reinterpret_cast<const longlong2 *>((val ? c.v : c.k) + e);
            const longlong2 u = __ldg(p), w = __ldg(p + 1);
            x[0] = u.x; x[1] = u.y; x[2] = w.x; x[3] = w.y;
        } else if (val) {
            const ushort4 q = __ldg(reinterpret_cast<const ushort4 *>(c.vq + e));
            const int64_t M = __ldg(c.vmag + vec);
            x[0] = kv_value(q.x, M, c.vbits); x[1] = kv_value(q.y, M, c.vbits);
            x[2] = kv_value(q.z, M, c.vbits); x[3] = kv_value(q.w, M, c.vbits);
        } else {
            const uchar4 q = __ldg(reinterpret_cast<const uchar4 *>(c.kq + e));
            const int64_t M = __ldg(c.kmag + vec);
            x[0] = kv_value(q.x, M, c.kbits); x[1] = kv_value(q.y, M, c.kbits);
            x[2] = kv_value(q.z, M, c.kbits); x[3] = kv_value(q.w, M, c.kbits);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = d + i < c.hd ? tree_at<PK>(c, val, vec, d + i) : 0;
}

// All plane pairs of one 16 x 8 x 32 step into the diagonals; P planes, the last signed.
template <int P>
__device__ __forceinline__ void tree_mma(int (&acc)[14][4], const uint32_t (&A)[4][8], const uint2 *B, int lane) {
#pragma unroll
    for (int j = 0; j < P; j++) {
        const uint2 b = B[j * 32 + lane];
#pragma unroll
        for (int i = 0; i < P; i++) {
            if (i + j > 13) continue;
            if (i == P - 1 && j == P - 1) mma_s32<true, true>(acc[i + j], A[0][i], A[1][i], A[2][i], A[3][i], b.x, b.y);
            else if (i == P - 1) mma_s32<true, false>(acc[i + j], A[0][i], A[1][i], A[2][i], A[3][i], b.x, b.y);
            else if (j == P - 1) mma_s32<false, true>(acc[i + j], A[0][i], A[1][i], A[2][i], A[3][i], b.x, b.y);
            else mma_s32<false, false>(acc[i + j], A[0][i], A[1][i], A[2][i], A[3][i], b.x, b.y);
        }
    }
}

__device__ __forceinline__ bool tree_big(int64_t x) { return (uint64_t)(x + (1ll << 55)) >= (1ull << 56); }

__host__ __device__ constexpr int tree_hdp(int hd) { return (hd + 63) / 64 * 64; }
// bytes of shared memory beside the scores: query planes, or value tile and partial outputs
__host__ __device__ constexpr size_t tree_side(int NT, int hd) {
    const size_t q = (size_t)NT * ((hd + 31) / 32) * 8 * 32 * 8;
    const size_t v = (size_t)TREE_V * 8 + (size_t)8 * NT * tree_hdp(hd) * 8;
    return q > v ? q : v;
}

template <int NT, bool PK, bool SM>
__global__ void __launch_bounds__(256, 2) k_tree(const __grid_constant__ TreeArgs a) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) char tree_smem[];
    constexpr int NC = 8 * NT;
    __shared__ int64_t cmax[NC], csum[NC], gmax[NC], gsum[NC];
    __shared__ double ginv[NC];
    __shared__ uint32_t anc[TREE_MAX_NODES][TREE_MAX_NODES / 32];   // nodes that a node sees
    __shared__ int up[TREE_MAX_NODES];
    __shared__ int weird_s;
    const int rank = blockIdx.x % a.cs, rest = blockIdx.x / a.cs;
    const int blk = rest % a.blocks, g = rest / a.blocks % a.c.nkv, b = rest / a.blocks / a.c.nkv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    TreeSeq s;
    const int grp = a.nh / a.c.nkv, hd = a.c.hd;
    // uniform over the cluster: every CTA of it leaves here or none
    if (!tree_seq(a, b, s) || blk * NC >= s.n * grp) return;
    const int cols = min(NC, s.n * grp - blk * NC), c0 = blk * NC, T = s.len + s.n;
    const int per = ((T + a.cs - 1) / a.cs + 15) & ~15;
    const int tb = min(T, rank * per), Tl = min(per, T - tb), Tp = (Tl + 15) & ~15;   // this CTA's positions
    const size_t v0 = (size_t)s.sq * a.c.max_seq + tb;
    int64_t *sc = SM ? reinterpret_cast<int64_t *>(tree_smem) : a.sc + (size_t)blockIdx.x * NC * a.Ts;
    char *side = SM ? tree_smem + (size_t)NC * a.Ts * 8 : tree_smem;
    uint2 *qp = reinterpret_cast<uint2 *>(side);   // [NT][KS][8][32]
    const int KS = (hd + 31) / 32;

    // ---- query planes in B-fragment order, node masks
    int qbig = 0;
    for (int e = tid; e < NT * KS * 64; e += 256) {   // (nt, ks, fragment half, lane)
        const int ln = e & 31, f = (e >> 5) & 1, ks = (e >> 6) % KS, nt = (e >> 6) / KS;
        const int col = nt * 8 + (ln >> 2), d = ks * 32 + (ln & 3) * 4 + f * 16;
        int64_t x[4] = {0, 0, 0, 0};
        if (col < cols) {
            const int64_t *q = a.q + (int64_t)(s.row0 + (c0 + col) / grp) * a.qs + (int64_t)(g * grp + (c0 + col) % grp) * hd;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[i] = d + i < hd ? q[d + i] : 0;
                qbig |= tree_big(x[i]);
            }
        }
        uint32_t o[8];
        byte_planes4(x, o);
        uint32_t *dst = reinterpret_cast<uint32_t *>(qp + (size_t)(nt * KS + ks) * 256 + ln) + f;
#pragma unroll
        for (int j = 0; j < 8; j++) dst[j * 64] = o[j];
    }
    // ancestors by pointer doubling: after k rounds a node knows 2^k of its path
    constexpr int AW = TREE_MAX_NODES / 32;
    const int nw = (s.n + 31) >> 5;
    if (tid < s.n) {
        for (int i = 0; i < nw; i++) anc[tid][i] = i == tid >> 5 ? 1u << (tid & 31) : 0;
        const int p = a.parent[s.row0 + tid];
        up[tid] = p < tid ? p : -1;
    }
    __syncthreads();
    for (int k = 1; k < s.n; k <<= 1) {
        uint32_t m[AW];
        int nu = -1;
        const int p = tid < s.n ? up[tid] : -1;
        if (p >= 0) {
            for (int i = 0; i < AW; i++) m[i] = i < nw ? anc[p][i] : 0;
            nu = up[p];
        }
        if (!__syncthreads_or(p >= 0)) break;
        if (p >= 0) {
            for (int i = 0; i < AW; i++)
                if (i < nw) anc[tid][i] |= m[i];
            up[tid] = nu;
        }
        __syncthreads();
    }
    if (tid == 0) weird_s = 0;
    qbig = __syncthreads_or(qbig);

    // ---- 1. scores
    const int gq = lane >> 2, tq = lane & 3;
    for (int u = warp; u < (Tp >> 4) * NT; u += 8) {
        const int nt = u % NT, t0 = u / NT * 16;
        if (nt * 8 >= cols) continue;
        int acc[14][4];
#pragma unroll
        for (int k = 0; k < 14; k++) acc[k][0] = acc[k][1] = acc[k][2] = acc[k][3] = 0;
        for (int ks = 0; ks < KS; ks++) {
            uint32_t A[4][8];
            int big = qbig;
            int64_t x[4][4];
#pragma unroll
            for (int f = 0; f < 4; f++) {   // rows gq (+8), columns tq*4 (+16)
                const int t = t0 + gq + (f & 1) * 8, d = ks * 32 + tq * 4 + (f >> 1) * 16;
                x[f][0] = x[f][1] = x[f][2] = x[f][3] = 0;
                if (t < Tl) tree_at4<PK>(a, false, (v0 + t) * a.c.nkv + g, d, x[f]);
            }
#pragma unroll
            for (int f = 0; f < 4; f++) {
                big |= tree_big(x[f][0]) | tree_big(x[f][1]) | tree_big(x[f][2]) | tree_big(x[f][3]);
                byte_planes4(x[f], A[f]);
            }
            const uint2 *B = qp + (size_t)(nt * KS + ks) * 256;
            if (__any_sync(0xffffffffu, big)) tree_mma<8>(acc, A, B, lane);
            else tree_mma<7>(acc, A, B, lane);
        }
#pragma unroll
        for (int c = 0; c < 4; c++) {   // positions t0 + gq (+8), columns 2 tq + {0, 1}
            int64_t G[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                G[k] = acc[4 * k][c];
#pragma unroll
                for (int m = 1; m < 4; m++)
                    if (4 * k + m < 14) madw(G[k], acc[4 * k + m][c], 1 << (8 * m));
            }
            // (G0 + G1 2^32 + G2 2^64 + G3 2^96) >> 48, nested floors
            const int64_t lo = (G[0] >> 32) + G[1];
            const int64_t dot = (int64_t)((uint64_t)(lo >> 16) + ((uint64_t)G[2] << 16) + ((uint64_t)G[3] << 48));
            const int t = t0 + gq + (c < 2 ? 0 : 8), col = nt * 8 + 2 * tq + (c & 1);
            sc[(size_t)col * a.Ts + t] = tree_scale(dot, (uint64_t)a.scale);
        }
    }
    __syncthreads();

    // ---- 2. maxima, exponentials, sums: a warp a column
    auto sees = [&](int node, int t) {   // local position t
        const int j = tb + t - s.len;
        return t < Tl && (j < 0 || (anc[node][j >> 5] >> (j & 31) & 1));
    };
    auto cluster_wait = [&]() {
        if (a.cs > 1) cg::this_cluster().sync();
        else __syncthreads();
    };
    for (int col = warp; col < cols; col += 8) {
        const int node = (c0 + col) / grp;
        int64_t m = INT64_MIN;
        for (int t = lane; t < Tl; t += 32)
            if (sees(node, t)) m = max(m, sc[(size_t)col * a.Ts + t]);
        for (int k = 16; k >= 1; k >>= 1) m = max(m, (int64_t)__shfl_xor_sync(0xffffffffu, m, k));
        if (lane == 0) cmax[col] = m;
    }
    cluster_wait();
    if (tid < cols) {
        int64_t m = cmax[tid];
        for (int r = 0; r < a.cs && a.cs > 1; r++)
            m = max(m, cg::this_cluster().map_shared_rank(cmax, r)[tid]);
        gmax[tid] = m;
    }
    __syncthreads();
    int weird = 0;
    for (int col = warp; col < cols; col += 8) {
        const int64_t m = gmax[col];
        int64_t *row = sc + (size_t)col * a.Ts;
        const int node = (c0 + col) / grp;
        uint64_t sum = 0;
        for (int t = lane; t < Tp; t += 32) {
            int64_t e = 0;
            if (sees(node, t)) {
                const uint64_t d = (uint64_t)m - (uint64_t)row[t];
                if ((int64_t)d < 0) {   // the difference wraps: the reference's value all the same
                    weird = 1;
                    e = d_safe_exp((int64_t)(0 - d));
                } else if (d <= 10 * (uint64_t)IQ_ONE) {
                    e = tree_exp(d);
                }
            }
            row[t] = e;
            sum += (uint64_t)e;
        }
        for (int k = 16; k >= 1; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
        if (lane == 0) csum[col] = (int64_t)sum;
    }
    if (weird) weird_s = 1;
    cluster_wait();
    weird = weird_s;
    for (int r = 0; r < a.cs && a.cs > 1; r++) weird |= *cg::this_cluster().map_shared_rank(&weird_s, r);
    if (tid < cols) {
        uint64_t S = (uint64_t)csum[tid];
        if (a.cs > 1) {
            S = 0;
            for (int r = 0; r < a.cs; r++) S += (uint64_t)cg::this_cluster().map_shared_rank(csum, r)[tid];
        }
        gsum[tid] = (int64_t)S;
        ginv[tid] = 281474976710656.0 / (double)(int64_t)S;
    }
    __syncthreads();
    for (int col = warp; col < NC; col += 8) {
        int64_t *row = sc + (size_t)col * a.Ts;
        if (col >= cols) {
            for (int t = lane; t < Tp; t += 32) row[t] = 0;
            continue;
        }
        const int64_t S = gsum[col];
        const double inv = ginv[col];
        for (int t = lane; t < Tp; t += 32) {
            const int64_t e = row[t];
            if (weird) row[t] = S > 0 ? d_div(e, S) : e;
            else row[t] = __double_as_longlong(tree_u52(e ? tree_prob(e, S, inv) : 0));
        }
    }

    // ---- 3. probabilities times values
    const int hdp = tree_hdp(hd), TV = TREE_V / hdp, nd = hdp >> 6;
    double *vt = reinterpret_cast<double *>(side);                                    // [TV][hdp]
    unsigned long long *part = reinterpret_cast<unsigned long long *>(side + TREE_V * 8);   // [NC][hdp]
    for (int e = tid; e < NC * hdp; e += 256) part[e] = 0;
    const int units = NT * nd, tg_n = 8 / units;      // units <= 8
    const int unit = warp % units, tg = warp / units;   // warps beyond units * tg_n idle
    const int pc = (unit / nd) * 8 + (lane >> 4) * 4, pd = (unit % nd) * 64 + (lane & 15) * 2;
    const int per_t = (TV + tg_n - 1) / tg_n;
    double o[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = TREE_A;
    const bool on = tg < tg_n && (unit / nd) * 8 < cols;
    for (int st = 0; st < Tl; st += TV) {
        int64_t x[4][4];
        int big = 0;   // 1: beyond the single chain, 2: beyond both
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int e = (k * 256 + tid) * 4, t = e / hdp, d = e - t * hdp;
            x[k][0] = x[k][1] = x[k][2] = x[k][3] = 0;
            if (st + t < Tl) tree_at4<PK>(a, true, (v0 + st + t) * a.c.nkv + g, d, x[k]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int64_t lim = (1ll << 51) - (1 << 16);
                if ((uint64_t)(x[k][i] + lim) > (uint64_t)(2 * lim)) big |= 1;
                if ((uint64_t)(x[k][i] + (1ll << 54)) >= (1ull << 55)) big |= 2;
            }
        }
        // the previous tile is consumed
        big = __syncthreads_or(big & 2) ? 2 : __syncthreads_or(big) ? 1 : 0;
        const int n = min(TV, Tl - st);
        if (big == 2 || weird) {   // term by term
            int64_t *vi = reinterpret_cast<int64_t *>(vt);
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) vi[(k * 256 + tid) * 4 + i] = x[k][i];
            __syncthreads();
            for (int e = tid; e < cols * hdp; e += 256) {
                const int col = e / hdp, d = e - col * hdp;
                uint64_t acc = 0;
                for (int t = 0; t < n; t++) {
                    const int64_t pv = sc[(size_t)col * a.Ts + st + t];
                    const int64_t p = weird ? pv : (int64_t)((uint64_t)__double_as_longlong(
                                                        __longlong_as_double(pv) + TREE_M) & 0xFFFFFFFFFFFFFull);
                    acc += (uint64_t)d_mul(p, vi[t * hdp + d]);
                }
                atomicAdd(&part[e], (unsigned long long)acc);
            }
            continue;
        }
        for (int half = 0; half <= big; half++) {   // v, or its low part f, then n = (v - f) / 2^51
            if (half) __syncthreads();
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    int64_t v = x[k][i];
                    if (big) {
                        const int64_t f = (int64_t)((uint64_t)v << 13) >> 13;
                        v = half ? (v - f) >> 51 : f;
                    }
                    const double w = __longlong_as_double((long long)((uint64_t)v + TREE_AB)) - TREE_A;
                    vt[(k * 256 + tid) * 4 + i] = half ? w : w * 0x1p-48;
                }
            __syncthreads();
            if (!on) continue;
            const int te = min(n, (tg + 1) * per_t);
            const double *pp = reinterpret_cast<const double *>(sc) + (size_t)pc * a.Ts + st;
            if (!half) {
#pragma unroll 2
                for (int t = tg * per_t; t < te; t++) {
                    const double2 va = *reinterpret_cast<const double2 *>(vt + t * hdp + pd);
                    const double2 vb = *reinterpret_cast<const double2 *>(vt + t * hdp + pd + 32);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const double p = pp[(size_t)i * a.Ts + t];
                        o[i][0] = __fma_rd(p, va.x, o[i][0]);
                        o[i][1] = __fma_rd(p, va.y, o[i][1]);
                        o[i][2] = __fma_rd(p, vb.x, o[i][2]);
                        o[i][3] = __fma_rd(p, vb.y, o[i][3]);
                    }
                }
            } else {   // 8 sum p n, exact: below 2^48 2^3
                double m[4][4];
#pragma unroll
                for (int i = 0; i < 4; i++) m[i][0] = m[i][1] = m[i][2] = m[i][3] = TREE_A;
                for (int t = tg * per_t; t < te; t++) {
                    const double2 va = *reinterpret_cast<const double2 *>(vt + t * hdp + pd);
                    const double2 vb = *reinterpret_cast<const double2 *>(vt + t * hdp + pd + 32);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const double p = pp[(size_t)i * a.Ts + t];
                        m[i][0] = __fma_rn(p, va.x, m[i][0]);
                        m[i][1] = __fma_rn(p, va.y, m[i][1]);
                        m[i][2] = __fma_rn(p, vb.x, m[i][2]);
                        m[i][3] = __fma_rn(p, vb.y, m[i][3]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        atomicAdd(&part[(pc + i) * hdp + pd + (k & 1) + (k >> 1) * 32],
                                  ((unsigned long long)__double_as_longlong(m[i][k]) - TREE_AB) << 3);
            }
        }
    }
    __syncthreads();
    if (on)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int k = 0; k < 4; k++)
                atomicAdd(&part[(pc + i) * hdp + pd + (k & 1) + (k >> 1) * 32],
                          (unsigned long long)__double_as_longlong(o[i][k]) - TREE_AB);
    cluster_wait();
    for (int e = rank * 256 + tid; e < cols * hdp; e += 256 * a.cs) {
        const int col = e / hdp, d = e - col * hdp;
        if (d >= hd) continue;
        uint64_t t = 0;
        if (a.cs == 1) t = part[e];
        else
            for (int r = 0; r < a.cs; r++) t += cg::this_cluster().map_shared_rank(part, r)[e];
        a.out[((size_t)(s.row0 + (c0 + col) / grp) * a.nh + g * grp + (c0 + col) % grp) * hd + d] = (int64_t)t;
    }
    if (a.cs > 1) cg::this_cluster().sync();   // the others may still read this CTA's part
}

}  // namespace iq
