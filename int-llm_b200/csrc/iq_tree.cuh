// iq_tree.cuh -- attention of drafted tokens over the cache (iq_attn_tree_dev).
// Per node row r and query head h, over the positions t it sees (all before
// the draft, its ancestors, itself), in the reference's order (llama_int.c:1432-1529):
//   s_t = fp_mul((int64)(sum_d (i128)q[d] k_t[d] >> 48), fp_inv_sqrt(hd))
//   m = max s;  e_t = fp_safe_exp(s_t - m);  S = sum e;  p_t = S > 0 ? fp_div(e_t, S) : e_t
//   out[d] = sum_t fp_mul(p_t, v_t[d])   (wrapping int64)
// The columns of a (sequence, kv head) are its (node, query head) pairs. Three
// kernels over scores in the workspace: p needs S, and S the maximum of the whole
// row, and each step has its own best shape. Every reduction is of whole
// numbers, so neither tiles nor splits change a result.
//
// 1. k_tree_scores, on the tensor cores (tcgen05 kind::i8). With x_u = x + 2^63 in 8
//    unsigned bytes, q.k = sum_(i,j) 2^(8(i+j)) sum_d q_j k_i - 2^63 (sum q_u + sum k_u) +
//    hd 2^126, and (q.k >> 48) mod 2^64 needs the diagonals i + j <= 13 and, of the rest,
//    only -2^15 (sum q + sum k). A: 128 positions x 32 d of one key plane; B: the 8
//    planes of NC queries (N = 8 NC rows, plane-major). Plane i accumulates into
//    TMEM from column i NC on, so that all pairs of a diagonal land on the same
//    NC columns: 8 instructions a step for the 64 pairs, 15 NC columns of s32
//    (each below 8 pairs x hd x 255^2 < 2^28). The epilogue reads 14 diagonals.
// 2. k_tree_softmax, a CTA a row and head: fp_safe_exp and fp_div in doubles with
//    directed rounding. With r / 2^24 exact in a double and M = 2^52 (one unit = one
//    ulp up to 2^53), fma.rd(r 2^-24, r 2^-24, M) = M + floor(r^2 / 2^48) while that floor is
//    below 2^52. 12 of the 14 squarings fit (r <= e^2.5 < 16); the last two
//    take 32-bit pieces.
// 3. k_tree_pv: sum_t floor(p_t v_t / 2^48) as one chain of fma.rd per output at
//    1.5 2^52: with p and v exact in doubles and the running sum within 2^51, each
//    step adds exactly floor(p v 2^-48). As sum p <= 2^48 that holds for
//    |v| <= 2^51 - 2^32 (8.0). Beyond, v = n 2^51 + f with |f| <= 2^50 and floor(p v / 2^48) =
//    8 p n + floor(p f / 2^48): f takes the chain, 8 p n (mod 2^64) whole numbers beside it.
//    The chain runs on the FP64 tensor cores (m8n8k4, .rm: every product is
//    added and rounded down in its turn), 256 terms an instruction; plain fma.rd
//    would wait for its operands (a load returns 16 doubles a clock, the pipe
//    takes 64 terms). Six integer instructions a term is what the remainder form
//    of k_attn_pv_tc costs.
#pragma once
#include <type_traits>
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
    int64_t *sc;    // workspace [rows][nh][Tw]: scores, then p 2^-48 as doubles
    int Tw;
    int tiles, tpc, groups, passes;   // k_tree_scores: CTAs along the positions, tiles each, groups of column blocks, blocks a group
    int chunk, chunks, cg, cblocks, tp;   // k_tree_pv: positions a CTA, their number, groups of 8 CB columns a block, blocks, positions a tile
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
    if (!ok && s.sq >= 0) atomicExch(&g_iq_err, (int)IQ_ERR_RANGE);
    return ok;
}

// The d (of a 32-wide step) of element e of a half h. Any order serves as long as keys
// and queries share it: exact keys take 16-byte pieces in turn, so that the two
// halves read full sectors, packed ones 16 codes in a row.
template <bool PK>
__device__ __forceinline__ int tree_d(int h, int e) {
    return PK ? h * 16 + e : (e >> 1) * 4 + 2 * h + (e & 1);
}

// The K or V vectors of one (sequence, kv head) from a first position on. The
// loads never branch: a position or d beyond the end is clamped into the
// vectors (such keys meet a query plane of zeros or a score that no row sees,
// such values a probability of zero or an output column that is not kept).
// W: whole 32-wide steps in aligned pieces; else element by element.
struct TreeRows {
    const char *x;         // exact elements or codes
    const int64_t *mag;    // packed
    uint32_t rs, ms;       // bytes of a position, magnitudes of a position
    int T, hd, bits;
};
template <bool PK>
__device__ __forceinline__ TreeRows tree_rows(const TreeArgs &a, bool val, size_t vec0, int T) {
    const KVArgs &c = a.c;
    const size_t e = vec0 * c.hd;
    TreeRows r;
    const int es = !PK ? 8 : val ? 2 : 1;
    r.x = (!PK ? (const char *)(val ? c.v : c.k) : val ? (const char *)c.vq : (const char *)c.kq) + e * es;
    r.mag = PK ? (val ? c.vmag : c.kmag) + vec0 : nullptr;
    r.rs = (uint32_t)c.nkv * c.hd * es;
    r.ms = c.nkv;
    r.T = T;
    r.hd = c.hd;
    r.bits = val ? c.vbits : c.kbits;
    return r;
}
// Half h of one position's 32-wide key step from d0 on, as loaded.
template <bool PK, bool W> struct TreeKeys;
template <bool W> struct TreeKeys<false, W> {
    longlong2 x[8];
    __device__ __forceinline__ void load(const TreeRows &r, int t, int d0, int h) {
        const int64_t *p = reinterpret_cast<const int64_t *>(r.x + (size_t)(uint32_t)min(t, r.T - 1) * r.rs);
        if constexpr (W) {
            const longlong2 *q = reinterpret_cast<const longlong2 *>(p + d0 + 2 * h);
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = __ldg(q + 2 * j);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                x[j] = make_longlong2(__ldg(p + min(d0 + tree_d<false>(h, 2 * j), r.hd - 1)),
                                      __ldg(p + min(d0 + tree_d<false>(h, 2 * j + 1), r.hd - 1)));
        }
    }
    // elements 4w .. 4w + 3
    __device__ __forceinline__ void get(const TreeRows &, int w, int64_t (&o)[4]) const {
        o[0] = x[2 * w].x; o[1] = x[2 * w].y; o[2] = x[2 * w + 1].x; o[3] = x[2 * w + 1].y;
    }
};
template <bool W> struct TreeKeys<true, W> {
    uint32_t q[4];
    int64_t m;
    __device__ __forceinline__ void load(const TreeRows &r, int t, int d0, int h) {
        t = min(t, r.T - 1);
        const uint8_t *p = reinterpret_cast<const uint8_t *>(r.x) + (size_t)(uint32_t)t * r.rs;
        m = __ldg(r.mag + (size_t)(uint32_t)t * r.ms);
        if constexpr (W) {
            const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p + d0 + h * 16));
            q[0] = u.x; q[1] = u.y; q[2] = u.z; q[3] = u.w;
        } else {
#pragma unroll
            for (int w = 0; w < 4; w++) {
                q[w] = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) q[w] |= (uint32_t)__ldg(p + min(d0 + h * 16 + 4 * w + i, r.hd - 1)) << (8 * i);
            }
        }
    }
    __device__ __forceinline__ void get(const TreeRows &r, int w, int64_t (&o)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = kv_value((q[w] >> (8 * i)) & 0xFF, m, r.bits);
    }
};
// key or value d < hd of position t < T
template <bool PK>
__device__ __forceinline__ int64_t tree_key(const TreeRows &r, int t, int d) {
    const char *p = r.x + (size_t)(uint32_t)t * r.rs;
    return PK ? kv_value(reinterpret_cast<const uint8_t *>(p)[d], r.mag[(size_t)(uint32_t)t * r.ms], r.bits)
              : reinterpret_cast<const int64_t *>(p)[d];
}
template <bool PK>
__device__ __forceinline__ int64_t tree_val(const TreeRows &r, int t, int d) {
    const char *p = r.x + (size_t)(uint32_t)t * r.rs;
    return PK ? kv_value(reinterpret_cast<const uint16_t *>(p)[d], r.mag[(size_t)(uint32_t)t * r.ms], r.bits)
              : reinterpret_cast<const int64_t *>(p)[d];
}

// c0, c1 of an 8 x 8 tile += A (8 x 4, row) B (4 x 8, col), each product added and
// rounded down in its turn
__device__ __forceinline__ void dmma_rd(double &c0, double &c1, double x, double y) {
    asm volatile("wmma.mma.sync.aligned.row.col.m8n8k4.rm.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
                 : "+d"(c0), "+d"(c1) : "d"(x), "d"(y));
}

// Byte planes of four elements' words w: o[i] holds byte i of w[0] .. w[3].
__device__ __forceinline__ void tree_bytes4(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t (&o)[4]) {
    const uint32_t x01 = __byte_perm(w0, w1, 0x5140), x23 = __byte_perm(w2, w3, 0x5140);
    const uint32_t y01 = __byte_perm(w0, w1, 0x7362), y23 = __byte_perm(w2, w3, 0x7362);
    o[0] = __byte_perm(x01, x23, 0x5410);
    o[1] = __byte_perm(x01, x23, 0x7632);
    o[2] = __byte_perm(y01, y23, 0x5410);
    o[3] = __byte_perm(y01, y23, 0x7632);
}
// byte offset of 16-byte piece c of row r in a tile of 128-byte rows with the 128-byte swizzle
__device__ __forceinline__ uint32_t tree_sw(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

// 4 TMEM columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_ld4(uint32_t taddr, uint32_t (&v)[4]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(taddr));
}
__device__ __forceinline__ void tmem_zero4(uint32_t taddr) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %1, %1, %1};" :: "r"(taddr), "r"(0) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// this thread's shared-memory writes before the tensor cores' reads
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Range check from the high words, gathered with a maximum: hi + b as unsigned stays
// below 2b exactly when -b <= hi < b.
__device__ __forceinline__ void tree_hi(uint32_t &m, int64_t x, uint32_t b) { m = max(m, (uint32_t)(x >> 32) + b); }
#define TREE_V1 ((1u << 19) - 1)    // |x| <= 2^51 - 2^32: one chain

// Work that the kernel launched before this one may still be doing is waited for here.
__device__ __forceinline__ void tree_prev_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// fp_mul(s, c) for 0 <= c <= 2^48 (the score scale). With s = sh 2^32 + sl and c = ch 2^32 + cl =
// ch' 2^32 + cl', cl' signed (so that |sh cl'| <= 2^62):
// floor(s c / 2^48) = sh ch' 2^16 + floor((sh cl' + floor(sl c / 2^32)) / 2^16).
struct TreeScale {
    uint32_t ch, cl;
    int hs, ls;   // ch', cl'
};
__device__ __forceinline__ TreeScale tree_scale_of(int64_t c) {
    TreeScale r;
    r.ch = (uint32_t)((uint64_t)c >> 32);
    r.cl = (uint32_t)c;
    r.ls = (int)r.cl;
    r.hs = (int)r.ch + (r.ls < 0);
    return r;
}
__device__ __forceinline__ int64_t tree_scale(int64_t s, const TreeScale &c) {
    const uint32_t sl = (uint32_t)s;
    const int sh = (int)(s >> 32);
    uint64_t t = __umulhi(sl, c.cl);
    madu(t, sl, c.ch);
    int64_t u = (int64_t)t;
    madw(u, sh, c.ls);
    return (u >> 16) + (int64_t)((uint64_t)((int64_t)sh * c.hs) << 16);
}

// ---------------------------------------------------------------- 1. scores

// key planes of a step: two tiles of 128 positions x 4 planes x 32 d; two steps where several blocks share them
__host__ __device__ constexpr int tree_a_bytes(int NT) { return 32768 * NT; }
__host__ __device__ constexpr size_t tree_b_bytes(int NT, int hd) { return (size_t)((hd + 127) / 128) * 64 * NT * 128; }
__host__ __device__ constexpr size_t tree_scores_smem(int NT, int hd) { return 1024 + tree_a_bytes(NT) + tree_b_bytes(NT, hd); }

// A CTA takes a.tpc tiles of 128 positions of one (sequence, kv head) and up to
// a.passes blocks of NC = 8 NT columns. With hd <= 64 the key planes of a tile are made
// once for all its blocks, with one block the query planes once for all its tiles.
// Two CTAs an SM (three with 8 columns; four would spill: 92 us for 88 with
// 64 single tokens) overlap one another's loads, products and epilogues; TMEM holds
// 128 NT columns a CTA. Measured: 64 single tokens at 2000 positions (32 heads over 4 of
// 64) 88 us, 260 MB of keys at 3.0 TB/s; 8 drafts of 16-48 nodes 143 us, of which the
// tensor cores need 25: issue (47 %) of the byte planes and the epilogue bounds it; from
// the packed cache 69 us (2 drafts, 32 heads of 128).
template <int NT, bool PK, bool W>
__global__ void __launch_bounds__(256, NT == 1 ? 3 : 2) k_tree_scores(const __grid_constant__ TreeArgs a) {
    extern __shared__ __align__(16) char tree_smem[];
    constexpr int NC = 8 * NT, HC = NC / 2;
    __shared__ int64_t ksum[128];              // sum of a position's key
    __shared__ unsigned long long qsum[NC];    // 2^15 times the sum of a column's query
    __shared__ int64_t *scol[NC];              // a column's row of scores
    __shared__ __align__(8) uint64_t mbar[2];  // the products of a step's key planes are done
    __shared__ uint32_t tmem_s;
    const int tile = blockIdx.x % a.tiles, rest = blockIdx.x / a.tiles;
    const int group = rest % a.groups, g = rest / a.groups % a.c.nkv, b = rest / a.groups / a.c.nkv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int grp = a.nh / a.c.nkv, hd = a.c.hd, KS = (hd + 31) / 32;
    TreeSeq s;
    if (!tree_seq(a, b, s)) return;
    const int cols = s.n * grp, T = s.len + s.n, tb0 = tile * a.tpc * 128, te = min(T, tb0 + a.tpc * 128);
    const int p0 = group * a.passes, p1 = min(p0 + a.passes, (cols + NC - 1) / NC);   // column blocks
    if (tb0 >= te || p0 >= p1) return;
    char *const sA = tree_smem + ((1024 - (smem_u32(tree_smem) & 1023)) & 1023), *const sB = sA + tree_a_bytes(NT);

    // conversion: two threads a position; eight lanes in a row take positions whose
    // swizzles differ, so that their 16-byte stores meet no bank twice
    const int cq = lane >> 1, ch = lane & 1, cp = warp * 16 + ((cq & 8) | ((cq & 3) << 1) | ((cq >> 2) & 1));
    const TreeRows kr = tree_rows<PK>(a, false, (size_t)s.sq * a.c.max_seq * a.c.nkv + g, T);
    TreeKeys<PK, W> kx;
    if (tb0 + cp < te) kx.load(kr, tb0 + cp, 0, ch);
    if (warp == 0) tmem_alloc(&tmem_s, 128 * NT);
    if (tid == 0) {
        mbar_init(&mbar[0], 1);
        mbar_init(&mbar[1], 1);
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // epilogue: TMEM lane quadrant warp & 3, half of the columns warp >> 2
    const uint32_t tmem = tmem_s, tlane = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (warp >> 2) * HC;
    const int ep = (warp & 3) * 32 + lane;
    const TreeScale scale = tree_scale_of(a.scale);
    int batch = 0, made_at = 0;   // steps issued; half of the key planes that a tile's first step went to
    for (int tb = tb0; tb < te; tb += 128) {
    const int Tl = min(128, te - tb);
    unsigned long long sum = 0;
    for (int pass = p0; pass < p1; pass++) {
        // the diagonals that plane 0 does not start
#pragma unroll
        for (int sd = 8; sd < 14; sd++)
#pragma unroll
            for (int c = 0; c < HC; c += 4) tmem_zero4(tlane + sd * NC + c);
        tmem_st_wait();
        const int c0 = pass * NC, nc = min(NC, cols - c0);
        if (p1 - p0 > 1 || tb == tb0) {   // query planes of the block: a thread four d of one 16-byte piece
            if (tid < NC) {
                const int cc = c0 + min(tid, nc - 1), nd = cc / grp;
                scol[tid] = a.sc + ((size_t)(s.row0 + nd) * a.nh + g * grp + cc - nd * grp) * a.Tw;
            }
            for (int e = tid; e < NC * KS * 8; e += 256) {   // (column, step, half, quad): a column's 8 KS threads in a row
                const int w = e & 3, h = (e >> 2) & 1, ks = (e >> 3) % KS, col = (e >> 3) / KS;
                const int cc = c0 + min(col, nc - 1), nd = cc / grp;
                const int64_t *q = a.q + (int64_t)(s.row0 + nd) * a.qs + (int64_t)(g * grp + cc - nd * grp) * hd + ks * 32;
                int64_t x[4];
                if constexpr (W) {
                    const longlong2 u = __ldg(reinterpret_cast<const longlong2 *>(q + tree_d<PK>(h, 4 * w)));
                    const longlong2 v = __ldg(reinterpret_cast<const longlong2 *>(q + tree_d<PK>(h, 4 * w + 2)));
                    x[0] = u.x; x[1] = u.y; x[2] = v.x; x[3] = v.y;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) x[i] = ks * 32 + tree_d<PK>(h, 4 * w + i) < hd ? q[tree_d<PK>(h, 4 * w + i)] : 0;
                }
                uint32_t o[8];
                byte_planes4(x, o);
                o[7] ^= 0x80808080u;
                if (!W)   // beyond hd x_u is 0, not 2^63: nothing meets whatever the keys hold there
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (ks * 32 + tree_d<PK>(h, 4 * w + i) >= hd) o[7] &= ~(0xFFu << (8 * i));
                char *dst = sB + (size_t)(ks >> 2) * 64 * NT * 128 + w * 4;
#pragma unroll
                for (int j = 0; j < 8; j++)
                    *reinterpret_cast<uint32_t *>(dst + tree_sw(j * NC + col, (ks & 3) * 2 + h)) = o[j];
            }
            for (int col = warp; col < NC; col += 8) {   // a warp a column's sum
                const int cc = c0 + min(col, nc - 1), nd = cc / grp;
                const int64_t *q = a.q + (int64_t)(s.row0 + nd) * a.qs + (int64_t)(g * grp + cc - nd * grp) * hd;
                unsigned long long qs = 0;
                for (int d = lane; d < hd; d += 32) qs += (unsigned long long)__ldg(q + d);
                for (int m = 16; m >= 1; m >>= 1) qs += __shfl_xor_sync(0xffffffffu, qs, m);
                if (lane == 0) qsum[col] = qs << 15;
            }
        }
        const bool made = NT == 2 && KS <= 2 && pass > p0;   // the key planes stand
        for (int ks = 0; ks < KS; ks++, batch++) {
            // the half that this step's planes are in: batch & 1, or, when they stand, where they were made
            const int half = NT == 1 ? 0 : made ? (made_at + ks) & 1 : batch & 1;
            if (!made) {
                if (ks == 0) made_at = half;
                if (batch >= NT) mbar_wait(&mbar[(batch - NT) & 1], (uint32_t)((batch - NT) >> 1) & 1u);
                if (cp < Tl) {
                    int64_t x[16];
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        int64_t e[4];
                        kx.get(kr, w, e);
#pragma unroll
                        for (int i = 0; i < 4; i++) x[4 * w + i] = e[i];
                    }
                    if (pass == p0)
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            if (W || ks * 32 + tree_d<PK>(ch, i) < hd) sum += (unsigned long long)x[i];
                    char *const A = sA + (size_t)half * 32768;
#pragma unroll
                    for (int hw = 0; hw < 2; hw++) {   // planes 0-3 from the low words, 4-7 from the high ones
                        uint32_t o[4][4];
#pragma unroll
                        for (int w = 0; w < 4; w++) {
                            tree_bytes4((uint32_t)((uint64_t)x[4 * w] >> (32 * hw)), (uint32_t)((uint64_t)x[4 * w + 1] >> (32 * hw)),
                                        (uint32_t)((uint64_t)x[4 * w + 2] >> (32 * hw)),
                                        (uint32_t)((uint64_t)x[4 * w + 3] >> (32 * hw)), o[w]);
                            if (hw) o[w][3] ^= 0x80808080u;
                        }
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            *reinterpret_cast<uint4 *>(A + hw * 16384 + tree_sw(cp, j * 2 + ch)) =
                                make_uint4(o[0][j], o[1][j], o[2][j], o[3][j]);
                    }
                }
                // the next step's keys are on their way meanwhile
                if (ks + 1 < KS) {
                    if (cp < Tl) kx.load(kr, tb + cp, (ks + 1) * 32, ch);
                } else if (KS > 2 && pass + 1 < p1) {
                    if (cp < Tl) kx.load(kr, tb + cp, 0, ch);
                } else if (tb + 128 + cp < te) {
                    kx.load(kr, tb + 128 + cp, 0, ch);
                }
                if (ks == KS - 1 && pass == p0) {
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    if (ch == 0) ksum[cp] = (int64_t)sum;
                }
            }
            if (!made || ks == 0) {
                fence_async_smem();
                tc_fence_before();
                __syncthreads();
            }
            if (tid == 0) {
                tc_fence_after();
                const char *A = sA + (size_t)half * 32768;
                const uint64_t bd = smem_desc_sw128(sB + (size_t)(ks >> 2) * 64 * NT * 128) + 2 * (ks & 3);
#pragma unroll
                for (int i = 0; i < 8; i++)
                    tc_mma_i8(tmem + i * NC, smem_desc_sw128(A + (i >> 2) * 16384) + 2 * (i & 3), bd,
                              idesc_i8(false, false, 128, 8 * NC), ks > 0 || i > 0);
                tc_commit(&mbar[batch & 1]);
            }
        }
        // (a wait that runs out has recorded IQ_ERR_TIMEOUT; the outputs then mean nothing)
        mbar_wait(&mbar[(batch - 1) & 1], (uint32_t)((batch - 1) >> 1) & 1u);
        tc_fence_after();
        const unsigned long long kp = 0 - ((unsigned long long)ksum[ep] << 15);
#pragma unroll
        for (int c = 0; c < HC; c += 4) {
            uint32_t v[14][4];
#pragma unroll
            for (int sd = 0; sd < 14; sd++) tmem_ld4(tlane + sd * NC + c, v[sd]);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 4; i++) {
                // bits 48 .. 111 of sum_s v_s 2^(8s): below 2^48 a chain of floors leaves the
                // carry; above, 2^32 v_10 and on need their low words only
                uint32_t lo = v[0][i];
#pragma unroll
                for (int k = 1; k < 6; k++) lo = (lo >> 8) + v[k][i];
                const uint32_t hi = v[10][i] + (v[11][i] << 8) + (v[12][i] << 16) + (v[13][i] << 24);
                const int col = (warp >> 2) * HC + c + i;
                uint64_t dot = kp - qsum[col] + ((uint64_t)hi << 32) + (lo >> 8);
                madu(dot, v[6][i], 1);
                madu(dot, v[7][i], 1 << 8);
                madu(dot, v[8][i], 1 << 16);
                madu(dot, v[9][i], 1 << 24);
                if (ep < Tl && col < nc) scol[col][tb + ep] = tree_scale((int64_t)dot, scale);
            }
        }
        tc_fence_before();
        __syncthreads();   // sums, TMEM and the query planes are free
        tc_fence_after();
    }
    }
    if (warp == 0) tmem_dealloc(tmem, 128 * NT);
}

// --------------------------------------------------------------- 2. softmax

#define TREE_M 4503599627370496.0            // 2^52
#define TREE_MB 0x4330000000000000ull        // its bits
#define TREE_A 6755399441055744.0            // 1.5 2^52
#define TREE_AB 0x4338000000000000ull
#define TREE_MASK 0xFFFFFFFFFFFFFull

__device__ __forceinline__ double tree_u52(uint64_t x) {   // exact for x < 2^52
    return __longlong_as_double((long long)(x | TREE_MB)) - TREE_M;
}
// floor(r^2 / 2^48) for r < 2^56, r = h 2^32 + l: h^2 2^16 + (2 h l + (l^2 >> 32) >> 16)
__device__ __forceinline__ uint64_t tree_sqr(uint64_t r) {
    const uint32_t l = (uint32_t)r, h = (uint32_t)(r >> 32);
    uint64_t x = __umulhi(l, l);
    madu(x, 2 * h, l);
    x >>= 16;
    madu(x, h << 8, h << 8);
    return x;
}
// 1 where q r + c < 0 (mod 2^64, as a signed number), else 0
__device__ __forceinline__ uint32_t tree_more(uint64_t q, uint64_t r, uint64_t c) {
    madu(c, (uint32_t)q, (uint32_t)r);
    const uint32_t h = (uint32_t)(c >> 32) + (uint32_t)q * (uint32_t)(r >> 32) + (uint32_t)(q >> 32) * (uint32_t)r;
    return h >> 31;
}
// fp_exp(-d) (fp_math.h:714-732) for 0 <= d <= 10
__device__ __forceinline__ int64_t tree_exp(uint64_t d) {
    double g = __longlong_as_double((long long)(((d >> 14) + IQ_ONE) | TREE_MB));   // M + r
#pragma unroll
    for (int i = 0; i < 12; i++) {
        const double u = __fma_rn(g, 0x1p-24, -TREE_M * 0x1p-24);
        g = __fma_rd(u, u, TREE_M);
    }
    const uint64_t r = tree_sqr(tree_sqr((uint64_t)__double_as_longlong(g) & TREE_MASK));   // 2^48 <= r < 2^62.5
    // floor(2^96 / r), at most 2^48: reciprocal by two Newton steps (relative error
    // below 2^-51), lowered by 2^-50 so that its floor is q or q - 1; the sign of
    // (q + 1) r - 2^96 - 1 (2^96 = 0 mod 2^64) tells which
    const double y = f64_rcp(f64_u64(r));
    const uint64_t q = (uint64_t)__double_as_longlong(__fma_rd(y, 0x1p96 - 0x1p46, TREE_M)) & TREE_MASK;
    return (int64_t)(q + tree_more(q, r, r - 1));
}
// fp_div(e, S) 2^-48 as a double for 0 <= e <= S, 2^48 <= S < 2^63, e <= 2^48,
// inv = f64_rcp(S) 2^48 lowered like the quotient of tree_exp
__device__ __forceinline__ double tree_prob(int64_t e, int64_t S, double inv) {
    const uint64_t q = (uint64_t)__double_as_longlong(__fma_rd(tree_u52((uint64_t)e), inv, TREE_M)) & TREE_MASK;
    return tree_u52(q + tree_more(q, (uint64_t)S, (uint64_t)S - 1 - ((uint64_t)e << 48))) * 0x1p-48;
}

// A row in which a score difference wraps: fp_safe_exp of the wrapped difference, the
// int64 sum, fp_div and fp_mul term by term. p goes through the row of the
// workspace, which is then zero. The scores are made again.
template <bool PK, class Sees>
__device__ __noinline__ void tree_wrapped(const TreeArgs &a, const TreeSeq &s, int r, int h, int T, int64_t m, int64_t *row,
                                          int64_t *out, uint64_t *red, const Sees &sees) {
    const int hd = a.c.hd, g = h / (a.nh / a.c.nkv);
    const size_t vec0 = (size_t)s.sq * a.c.max_seq * a.c.nkv + g;
    const TreeRows kr = tree_rows<PK>(a, false, vec0, T), vr = tree_rows<PK>(a, true, vec0, T);
    const int64_t *q = a.q + (int64_t)r * a.qs + (int64_t)h * hd;
    uint64_t sum = 0;
    for (int t = threadIdx.x; t < T; t += blockDim.x) {
        int64_t e = 0;
        if (sees(t)) {
            i128 dot = 0;
            for (int d = 0; d < hd; d++) dot += d_mul128(q[d], tree_key<PK>(kr, t, d));
            e = d_safe_exp((int64_t)((uint64_t)d_mul((int64_t)(dot >> 48), a.scale) - (uint64_t)m));
        }
        row[t] = e;
        sum += (uint64_t)e;
    }
    const int64_t S = (int64_t)(uint64_t)cta_sum_i128((i128)(u128)sum, red);
    for (int t = threadIdx.x; t < T; t += blockDim.x)
        if (S > 0) row[t] = d_div(row[t], S);
    __syncthreads();
    for (int d = threadIdx.x; d < hd; d += blockDim.x) {
        uint64_t acc = 0;
        for (int t = 0; t < T; t++) acc += (uint64_t)d_mul(row[t], tree_val<PK>(vr, t, d));
        out[d] = (int64_t)acc;
    }
    __syncthreads();
    for (int t = threadIdx.x; t < min(a.Tw, (s.len + s.n + 3) & ~3); t += blockDim.x) row[t] = 0;
}

// A CTA a node row and head (blockIdx.y). The scores stay in shared memory
// (SM), longer rows in the workspace. Positions that the row does not see get a
// score 11 below the maximum, whose exponential is 0, so that one loop serves
// all. A row whose score differences wrap (the reference's int64 then gives other
// numbers, reproduced here) is finished here term by term and leaves zeros to
// k_tree_pv. Measured: 102 us for the 13.6 M (row, head, position) of 8 drafts of 16-48
// nodes, issue 66 %: about 160 instructions each, most of them 12 squarings of two fused
// multiply-adds, 2 in 32-bit pieces and 2 quotients.
#define TREE_SM_T 128
#define TREE_SM_MAX 2560   // positions whose scores are kept in shared memory
template <bool PK, bool SM>
__global__ void __launch_bounds__(TREE_SM_T, 10) k_tree_softmax(const __grid_constant__ TreeArgs a) {
    extern __shared__ __align__(16) char tree_smem[];
    __shared__ uint64_t red[64];
    __shared__ int64_t wmax[TREE_SM_T / 32];
    __shared__ uint64_t wsum[TREE_SM_T / 32];
    __shared__ int up[TREE_MAX_NODES];
    __shared__ uint32_t anc[TREE_MAX_NODES / 32];
    const int b = blockIdx.x / a.max_nodes, node = blockIdx.x - b * a.max_nodes, tid = threadIdx.x;
    TreeSeq s;
    if (!tree_seq(a, b, s) || node >= s.n) return;
    const int r = s.row0 + node, hd = a.c.hd, T = s.len + node + 1;   // no later node is seen
    // ancestors of the node
    for (int i = tid; i <= node; i += TREE_SM_T) up[i] = a.parent[s.row0 + i];
    if (tid < TREE_MAX_NODES / 32) anc[tid] = 0;
    __syncthreads();
    if (tid == 0)
        for (int j = node;;) {
            anc[j >> 5] |= 1u << (j & 31);
            const int p = up[j];
            if (p < 0 || p >= j) break;
            j = p;
        }
    tree_prev_kernel();
    __syncthreads();
    auto sees = [&](int t) {
        const int j = t - s.len;
        return j < 0 || (t < T && (anc[j >> 5] >> (j & 31) & 1));
    };
    const int end = min(a.Tw, (s.len + s.n + 3) & ~3);   // k_tree_pv reads fours up to here
    const int h = blockIdx.y;
    int64_t *row = a.sc + ((size_t)r * a.nh + h) * a.Tw, m = INT64_MIN;
    int64_t *x = SM ? reinterpret_cast<int64_t *>(tree_smem) : row;   // each thread its own positions throughout
#pragma unroll 4
    for (int t = tid; t < s.len; t += TREE_SM_T) {
        const int64_t v = row[t];
        m = max(m, v);
        if (SM) x[t] = v;
    }
    const int t_end = s.len + (tid - s.len % TREE_SM_T + TREE_SM_T) % TREE_SM_T;   // its first position from the draft on
    for (int t = t_end; t < end; t += TREE_SM_T)
        if (sees(t)) {
            m = max(m, row[t]);
            if (SM) x[t] = row[t];
        }
    for (int k = 16; k >= 1; k >>= 1) m = max(m, (int64_t)__shfl_xor_sync(0xffffffffu, m, k));
    if ((tid & 31) == 0) wmax[tid >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < TREE_SM_T / 32; k++) m = max(m, wmax[k]);
    for (int t = t_end; t < end; t += TREE_SM_T)
        if (!sees(t)) x[t] = (int64_t)((uint64_t)m - 11 * (uint64_t)IQ_ONE);
    uint64_t sum = 0;
    int wraps = 0;   // sign: a difference of 2^63 or more
#pragma unroll 4
    for (int t = tid; t < end; t += TREE_SM_T) {
        const uint64_t d = (uint64_t)m - (uint64_t)x[t];
        wraps |= (int)(d >> 32);
        const int64_t e = tree_exp(d);   // (anything where d is beyond 10)
        const int64_t v = d <= 10 * (uint64_t)IQ_ONE ? e : 0;
        x[t] = v;
        sum += (uint64_t)v;
    }
    for (int k = 16; k >= 1; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
    if ((tid & 31) == 0) wsum[tid >> 5] = sum;
    int64_t *out = a.out + ((size_t)r * a.nh + h) * hd;
    if (__syncthreads_or(wraps < 0)) {
        tree_wrapped<PK>(a, s, r, h, T, m, row, out, red, sees);
        return;
    }
    uint64_t S = 0;
#pragma unroll
    for (int k = 0; k < TREE_SM_T / 32; k++) S += wsum[k];
    const double inv = f64_rcp(f64_u64(S)) * (0x1p48 - 0x1p-2);
    double *p = reinterpret_cast<double *>(row);
#pragma unroll 4
    for (int t = tid; t < end; t += TREE_SM_T) p[t] = tree_prob(x[t], (int64_t)S, inv);
    for (int d = tid; d < hd; d += TREE_SM_T) out[d] = 0;   // k_tree_pv adds
}

// ---------------------------------------------------- 3. probabilities x values

// A CTA takes a.chunk positions of CG x 8 CB columns of one (sequence, kv head); a
// warp 32 d of 8 CB columns and every tg_n-th four positions. A lane holds V of
// position lane & 3 at d = 16 k + 2 (lane >> 2) + {0, 1}, k < 2, i.e. column lane >> 2 of
// the 8-wide tiles 2k and 2k + 1, and of each tile's output the columns
// 2 (lane & 3) + {0, 1}.
// W: tiles of a.tp positions come through shared memory in two stages, each row of
// values and of probabilities one bulk copy, so that whole rows are asked of HBM
// at once, far ahead, and read once for all columns. Rows are 32 bytes apart
// from a multiple of 128, which puts the four positions (or columns) of a
// quarter-warp on different banks. Else the lanes read global memory themselves (scores
// and values so: 263 us for 175 with 64 single tokens, 427 for 339 with 8 drafts).
// Measured: 64 single tokens 54 us (292 MB, 5.5 TB/s); 8 drafts 115 us, 42 % of the FP64
// rate of 64 terms a clock and SM; the rest is conversions and waiting for tiles (issue 42 %).
struct TreeTile { int vrow, vpitch, ppitch, bytes; };   // bytes of a stage
template <bool PK>
__host__ __device__ constexpr TreeTile tree_tile(int hd, int nc, int tp) {
    const int vrow = hd * (PK ? 2 : 8);
    return TreeTile{vrow, vrow + 32, tp * 8 + 32, tp * (vrow + 32) + nc * (tp * 8 + 32) + (PK ? tp * 8 : 0)};
}
template <bool PK>
__host__ __device__ constexpr size_t tree_pv_smem(int hd, int nc, int tp, bool w) {
    return (size_t)nc * ((hd + 31) / 32 * 32) * 8 + (w ? 2 * (size_t)tree_tile<PK>(hd, nc, tp).bytes : 0);
}
__device__ __forceinline__ void bulk_row(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void async8(void *dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" :: "r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <int CB, bool PK, bool W>
__global__ void __launch_bounds__(256, 2) k_tree_pv(const __grid_constant__ TreeArgs a) {
    extern __shared__ __align__(16) char tree_smem[];
    __shared__ __align__(8) uint64_t full[2];
    constexpr int CW = 8 * CB;
    const int chunk = blockIdx.x % a.chunks, rest = blockIdx.x / a.chunks;
    const int blk = rest % a.cblocks, g = rest / a.cblocks % a.c.nkv, b = rest / a.cblocks / a.c.nkv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, tq = lane & 3;
    const int grp = a.nh / a.c.nkv, hd = a.c.hd, nd = (hd + 31) >> 5, hdp = nd * 32;
    TreeSeq s;
    if (!tree_seq(a, b, s)) return;
    const int CG = a.cg, NC = CG * CW;   // CG nd <= 8
    const int cols = min(NC, s.n * grp - blk * NC), c0 = blk * NC, tb = chunk * a.chunk;
    const int Tl = min(a.chunk, s.len + s.n - tb);
    if (Tl <= 0 || cols <= 0) return;
    unsigned long long *const red = reinterpret_cast<unsigned long long *>(tree_smem);   // [NC][hdp]
    char *const stage = tree_smem + (size_t)NC * hdp * 8;
    const int units = CG * nd, tg_n = 8 / units;   // warps from units * tg_n on idle
    const int unit = warp % units, tg = warp / units, pc = unit % CG * CW, db = unit / CG * 32;
    const bool on = tg < tg_n && pc < cols;
    for (int e = tid; e < NC * hdp; e += 256) red[e] = 0;
    const TreeRows vr = tree_rows<PK>(a, true, ((size_t)s.sq * a.c.max_seq + tb) * a.c.nkv + g, Tl);
    auto prow = [&](int col) {   // a column's probabilities from tb on (a missing one: the last, not kept)
        const int cc = c0 + min(col, cols - 1), n = cc / grp;
        return reinterpret_cast<const double *>(a.sc) + ((size_t)(s.row0 + n) * a.nh + g * grp + cc - n * grp) * a.Tw + tb;
    };
    double f[CB][4][2];
    uint32_t vm = 0;
    const int step = tg_n * 4;
    // four positions: probabilities p, values u (two pairs); SPLIT: values beyond the chain as
    // n 2^51 + f, 8 p n added in shared memory
    auto four = [&](auto split, const double (&p)[CB], const longlong2 (&u)[2], bool live) {
        constexpr bool SPLIT = decltype(split)::value;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            int64_t w[2] = {u[k].x, u[k].y};
            if (SPLIT) {
                const int64_t n0 = (w[0] >> 51) + (w[0] >> 50 & 1), n1 = (w[1] >> 51) + (w[1] >> 50 & 1);
                // the other lanes' columns of this position too: p from the lane that holds it
                for (int i = 0; i < CW; i++) {
                    const double pi = __shfl_sync(0xffffffffu, CB == 1 || i < 8 ? p[0] : p[CB - 1], (i & 7) * 4 + tq);
                    const uint64_t p8 = (uint64_t)(pi * 0x1p51);
                    unsigned long long *dst = red + (pc + i) * hdp + db + 16 * k + 2 * gq;
                    if (n0 && live) atomicAdd(dst, (unsigned long long)(p8 * (uint64_t)n0));
                    if (n1 && live) atomicAdd(dst + 1, (unsigned long long)(p8 * (uint64_t)n1));
                }
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
                if (!SPLIT) tree_hi(vm, w[j], TREE_V1);
                else w[j] = (int64_t)((uint64_t)w[j] << 13) >> 13;
                const double v = __hiloint2double((int)(w[j] >> 32) + 0x43380000, (int)w[j]) - TREE_A;
#pragma unroll
                for (int cb = 0; cb < CB; cb++) dmma_rd(f[cb][2 * k + j][0], f[cb][2 * k + j][1], p[cb], v);
            }
        }
    };
    auto start = [&]() {
#pragma unroll
        for (int cb = 0; cb < CB; cb++)
#pragma unroll
            for (int k = 0; k < 4; k++) f[cb][k][0] = f[cb][k][1] = TREE_A;
    };
    if constexpr (W) {
        const int tp = a.tp, nst = (Tl + tp - 1) / tp;
        const TreeTile tl = tree_tile<PK>(hd, NC, tp);
        auto nv = [&](int i) { return min(tp, Tl - i * tp); };
        const int own = lane * 8 + warp;   // the row that this thread copies: a warp issues its lanes' copies in turn, so all warps share them
        const double *my_p = prow(own);
        // (p rows are zero up to the next multiple of four positions)
        auto load_v = [&](int i, int sl) {
            char *st = stage + sl * tl.bytes;
            const int n = nv(i);
            if (tid == 0)
                mbar_expect_tx(&full[sl], (uint32_t)(n * tl.vrow + NC * ((n + 3) & ~3) * 8));
            if (own < n) {
                const size_t t = (size_t)(i * tp + own);
                bulk_row(st + own * tl.vpitch, vr.x + t * vr.rs, tl.vrow, &full[sl]);
                if (PK) async8(st + tp * tl.vpitch + NC * tl.ppitch + own * 8, vr.mag + t * vr.ms);
            }
        };
        auto load_p = [&](int i, int sl) {
            char *st = stage + sl * tl.bytes + tp * tl.vpitch;
            if (own < NC) bulk_row(st + own * tl.ppitch, my_p + i * tp, ((nv(i) + 3) & ~3) * 8, &full[sl]);
        };
        if (tid == 0) {
            mbar_init(&full[0], 1);
            mbar_init(&full[1], 1);
            fence_mbar_init();
        }
        __syncthreads();
        int batch = 0;   // tiles loaded: tile number batch of this CTA waits for phase batch >> 1 of its stage
        auto sum = [&](auto split, bool first) {
            start();
            for (int i = 0; i < min(2, nst); i++) load_v(i, (batch + i) & 1);
            if (first) tree_prev_kernel();
            for (int i = 0; i < min(2, nst); i++) load_p(i, (batch + i) & 1);
            async_wait();
            __syncthreads();
            for (int i = 0; i < nst; i++, batch++) {
                const int sl = batch & 1, n = nv(i);
                mbar_wait(&full[sl], (uint32_t)(batch >> 1) & 1u);
                const char *sv = stage + sl * tl.bytes, *sp = sv + tp * tl.vpitch;
                auto at = [&](int t0, int t) {   // positions t0 .. t0 + 3, this lane's values at t
                    const char *row = sv + t * tl.vpitch;
                    double p[CB];
#pragma unroll
                    for (int cb = 0; cb < CB; cb++)
                        p[cb] = *reinterpret_cast<const double *>(sp + (pc + cb * 8 + gq) * tl.ppitch + (t0 + tq) * 8);
                    longlong2 u[2];
                    if (PK) {
                        const int64_t M = *reinterpret_cast<const int64_t *>(sp + NC * tl.ppitch + t * 8);
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const ushort2 q = *reinterpret_cast<const ushort2 *>(row + (db + 16 * k + 2 * gq) * 2);
                            u[k] = make_longlong2(kv_value(q.x, M, vr.bits), kv_value(q.y, M, vr.bits));
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 2; k++)
                            u[k] = *reinterpret_cast<const longlong2 *>(row + (db + 16 * k + 2 * gq) * 8);
                    }
                    four(split, p, u, t0 + tq < n);
                };
                if (on && n == tp) {
#pragma unroll 4
                    for (int t0 = tg * 4; t0 < tp; t0 += step) at(t0, t0 + tq);
                } else if (on) {
                    for (int t0 = tg * 4; t0 < n; t0 += step) at(t0, min(t0 + tq, n - 1));
                }
                async_wait();
                __syncthreads();   // the tile is consumed, the next one's magnitudes are here
                if (i + 2 < nst) {
                    load_v(i + 2, sl);
                    load_p(i + 2, sl);
                }
            }
        };
        sum(std::false_type{}, true);
        if (__syncthreads_or(vm >= 2 * TREE_V1)) sum(std::true_type{}, false);   // a value beyond the chain: once more
    } else {
        const double *pp[CB];
#pragma unroll
        for (int cb = 0; cb < CB; cb++) pp[cb] = prow(pc + cb * 8 + gq) + tq;
        auto sum = [&](auto split) {
            start();
#pragma unroll 1
            for (int t0 = tg * 4; t0 < Tl; t0 += step) {
                double p[CB];
#pragma unroll
                for (int cb = 0; cb < CB; cb++) p[cb] = pp[cb][t0];
                longlong2 u[2];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const int t = min(t0 + tq, Tl - 1), d = db + 16 * k + 2 * gq;
                    u[k].x = tree_val<PK>(vr, t, min(d, hd - 1));
                    u[k].y = tree_val<PK>(vr, t, min(d + 1, hd - 1));
                }
                four(split, p, u, t0 + tq < Tl);
            }
        };
        tree_prev_kernel();
        __syncthreads();
        if (on) {
            sum(std::false_type{});
            if (__any_sync(0xffffffffu, vm >= 2 * TREE_V1)) sum(std::true_type{});
        }
    }
    // partial outputs of the tg_n position groups meet in shared memory, group after group
    const int od = db + 4 * tq;   // tile k, output j: + 16 (k >> 1) + (k & 1) + 2 j
    for (int turn = 0; turn < tg_n; turn++) {
        __syncthreads();
        if (on && tg == turn)
#pragma unroll
            for (int cb = 0; cb < CB; cb++) {
                unsigned long long *dst = red + (pc + cb * 8 + gq) * hdp + od;
#pragma unroll
                for (int k = 0; k < 4; k += 2) {   // tiles k, k + 1: four outputs in a row
                    ulonglong2 *q = reinterpret_cast<ulonglong2 *>(dst + 8 * k);
                    ulonglong2 u = q[0], w = q[1];
                    u.x += (unsigned long long)__double_as_longlong(f[cb][k][0]) - TREE_AB;
                    u.y += (unsigned long long)__double_as_longlong(f[cb][k + 1][0]) - TREE_AB;
                    w.x += (unsigned long long)__double_as_longlong(f[cb][k][1]) - TREE_AB;
                    w.y += (unsigned long long)__double_as_longlong(f[cb][k + 1][1]) - TREE_AB;
                    q[0] = u;
                    q[1] = w;
                }
            }
    }
    __syncthreads();
    for (int e = tid; e < cols * hdp; e += 256) {
        const int col = e / hdp, d = e - col * hdp, cc = c0 + col, n = cc / grp;
        if (d < hd && red[e])
            atomicAdd(reinterpret_cast<unsigned long long *>(a.out) +
                          ((size_t)(s.row0 + n) * a.nh + g * grp + cc - n * grp) * hd + d, red[e]);
    }
}

}  // namespace iq
