// iq_tree.cuh -- attention of drafted tokens over the cache (iq_attn_tree_dev).
// Per node row r and query head h, over the positions t it sees (all before
// the draft, its ancestors, itself), in the reference's order (llama_int.c:1432-1529):
//   s_t = fp_mul((int64)(sum_d (i128)q[d] k_t[d] >> 48), fp_inv_sqrt(hd))
//   m = max s;  e_t = fp_safe_exp(s_t - m);  S = sum e;  p_t = S > 0 ? fp_div(e_t, S) : e_t
//   out[d] = sum_t fp_mul(p_t, v_t[d])   (wrapping int64)
#pragma once
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
    int64_t *sc;   // [rows][nh][max_len]
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

__device__ __forceinline__ int64_t tree_kv(const KVArgs &c, bool val, size_t vec, int d) {
    const size_t e = vec * c.hd + d;
    if (!c.kbits) return (val ? c.v : c.k)[e];
    return val ? kv_value(c.vq[e], c.vmag[vec], c.vbits) : kv_value(c.kq[e], c.kmag[vec], c.kbits);
}

// One CTA a (query head, node), scores in the workspace.
__global__ void __launch_bounds__(256) k_tree_simple(TreeArgs a) {
    __shared__ uint64_t red[64];
    __shared__ int64_t qs[256];
    __shared__ unsigned char anc[TREE_MAX_NODES];
    TreeSeq s;
    const int b = blockIdx.x / a.max_nodes, node = blockIdx.x % a.max_nodes, h = blockIdx.y;
    if (!tree_seq(a, b, s) || node >= s.n) return;
    const int r = s.row0 + node, hd = a.c.hd, T = s.len + node + 1, g = h / (a.nh / a.c.nkv);
    for (int i = threadIdx.x; i <= node; i += blockDim.x) anc[i] = 0;
    for (int d = threadIdx.x; d < hd; d += blockDim.x) qs[d] = a.q[(int64_t)r * a.qs + (int64_t)h * hd + d];
    __syncthreads();
    if (threadIdx.x == 0)
        for (int j = node; ;) {
            anc[j] = 1;
            const int p = a.parent[s.row0 + j];
            if (p < 0 || p >= j) break;
            j = p;
        }
    __syncthreads();
    int64_t *sc = a.sc + ((size_t)r * a.nh + h) * a.max_len;
    const size_t v0 = (size_t)s.sq * a.c.max_seq;
    int64_t mx = INT64_MIN;
    for (int t = threadIdx.x; t < T; t += blockDim.x) {
        if (t >= s.len && !anc[t - s.len]) continue;
        const size_t vec = (v0 + t) * a.c.nkv + g;
        i128 dot = 0;
        for (int d = 0; d < hd; d++) dot += d_mul128(qs[d], tree_kv(a.c, false, vec, d));
        sc[t] = d_mul((int64_t)(dot >> 48), a.scale);
        mx = max(mx, sc[t]);
    }
    mx = cta_max_i64(mx, (int64_t *)red);
    uint64_t sum = 0;
    for (int t = threadIdx.x; t < T; t += blockDim.x) {
        int64_t e = 0;
        if (t < s.len || anc[t - s.len]) e = d_safe_exp((int64_t)((uint64_t)sc[t] - (uint64_t)mx));
        sc[t] = e;
        sum += (uint64_t)e;
    }
    const int64_t S = (int64_t)(uint64_t)cta_sum_i128((i128)(u128)sum, red);
    if (S > 0)
        for (int t = threadIdx.x; t < T; t += blockDim.x) sc[t] = d_div(sc[t], S);
    __syncthreads();
    for (int d = threadIdx.x; d < hd; d += blockDim.x) {
        uint64_t acc = 0;
        for (int t = 0; t < T; t++)
            if (sc[t]) acc += (uint64_t)d_mul(sc[t], tree_kv(a.c, true, (v0 + t) * a.c.nkv + g, d));
        a.out[(size_t)r * a.nh * hd + (size_t)h * hd + d] = (int64_t)acc;
    }
}

}  // namespace iq
