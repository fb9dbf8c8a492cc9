// iq_ops.cu -- C ABI of the operators around drafted tokens: rotary tables and
// rotation, cache rows, tree attention, log probabilities (declared in iq.h).
#include <atomic>
#include <climits>
#include "iq_common.cuh"
#include "iq_ops.cuh"
#include "iq_tree.cuh"
#include "iq_score.cuh"

using namespace iq;

static bool misaligned(const void *p, size_t n) { return ((uintptr_t)p & (n - 1)) != 0; }

// ---- host copies of the fp_math steps that a table's constants need

static int64_t h_mul(int64_t a, int64_t b) { return (int64_t)(((i128)a * b) >> 48); }
static int64_t h_exp(int64_t x) {   // fp_exp (fp_math.h:714-732)
    int64_t r = IQ_ONE + ((x < 0 ? -x : x) >> 14);
    for (int i = 0; i < 14; i++) r = h_mul(r, r);
    return x >= 0 ? r : r ? (int64_t)(((u128)1 << 96) / (u128)(uint64_t)r) : 0;
}
#define IQ_LN2 195103586505167LL
static int64_t h_log(int64_t x) {   // fp_log (fp_math.h:752-771), x > 0
    int64_t y = (int64_t)(63 - __builtin_clzll((uint64_t)x) - 48) * IQ_LN2;
    for (int i = 0; i < 10; i++) {
        const int64_t ey = h_exp(y);
        if (ey == 0) break;
        const int64_t yn = y - IQ_ONE + (int64_t)(((i128)x << 48) / ey);
        const int64_t d = yn < y ? y - yn : yn - y;
        if (d < 2) break;
        y = yn;
    }
    return y;
}
// ln of a whole number: fp_log below 2^14, where its Newton steps stay in the
// range of fp_exp; above, of theta / 2^k, plus k ln 2
static int64_t h_ln_int(int theta) {
    const int bl = 32 - __builtin_clz((unsigned)theta), k = bl > 14 ? bl - 14 : 0;
    return h_log((int64_t)(((uint64_t)theta << 48 - k))) + k * IQ_LN2;
}

// fp_inv_sqrt(fp_from_int(hd)) (fp_math.h:658-707): the score scale (llama_int.c:1433)
static int64_t h_att_scale(int hd) {
    const int64_t x = (int64_t)hd << 48;
    const int k = (63 - __builtin_clzll((uint64_t)x) - 48) >> 1;
    const int64_t n = x >> (2 * k);
    int64_t y = 63 - __builtin_clzll((uint64_t)n) == 48 ? IQ_ONE : IQ_ONE >> 1;
    for (int i = 0; i < 8; i++) y = (int64_t)(((i128)y * (3 * IQ_ONE - h_mul(n, h_mul(y, y)))) >> 49);
    return y >> k;
}

// fp_math_init (fp_math.h:785-858): pi by Machin, atan(2^-i), the CORDIC gain
static int64_t h_atan(int64_t x, int terms) {
    const int64_t x2 = h_mul(x, x);
    int64_t t = x, s = x;
    for (int n = 1; n <= terms; n++) {
        t = -h_mul(t, x2);
        const int64_t c = t / (2 * n + 1);
        if (c == 0) break;
        s += c;
    }
    return s;
}
struct HostCordic {
    int64_t pi, gain, angles[25];
    HostCordic() {
        pi = (h_atan(IQ_ONE / 5, 40) << 4) - (h_atan(IQ_ONE / 239, 15) << 2);
        angles[0] = pi >> 2;
        for (int i = 1; i < 25; i++) angles[i] = h_atan(IQ_ONE >> i, 40);
        int64_t k = IQ_ONE;
        for (int i = 0; i < 48; i++) k = h_mul(k, IQ_ONE + (2 * i < 63 ? IQ_ONE >> (2 * i) : 0));
        // fp_sqrt (fp_math.h:624-650): the largest r with r^2 <= k 2^48, bit by bit
        int64_t r = 0;
        for (int b = 50; b >= 0; b--) {
            const int64_t c = r | (int64_t)1 << b;
            if ((i128)c * c <= (i128)k << 48) r = c;
        }
        gain = (int64_t)(((i128)IQ_ONE << 48) / r);
    }
};

static int rope_check(const iq_rope *r, int hd, RopeArgs *a) {
    if (!r || !r->d_cos || !r->d_sin || !r->d_pos || r->n_pos < 1 || r->rot_dim < 2 || (r->rot_dim & 1) ||
        r->rot_dim > hd || (r->layout != IQ_ROPE_HALF && r->layout != IQ_ROPE_INTERLEAVED))
        return IQ_ERR_ARG;
    if (misaligned(r->d_cos, 8) || misaligned(r->d_sin, 8) || misaligned(r->d_pos, 4)) return IQ_ERR_ARG;
    *a = RopeArgs{r->d_cos, r->d_sin, r->d_pos, r->n_pos, r->rot_dim, r->layout};
    return IQ_OK;
}

// the 16-byte form: whole items of four elements, aligned tables
static bool rope_wide(const RopeArgs &r, int hd) {
    return hd % 4 == 0 && r.rot % 4 == 0 && !misaligned(r.cos, 16) && !misaligned(r.sin, 16);
}

static int cache_check(const iq_kv_cache *c, KVArgs *a) {
    if (!c || c->seqs < 1 || c->max_seq < 1 || c->kv_heads < 1 || c->head_dim < 1 || c->head_dim > 256 ||
        c->kv_heads > 65536)
        return IQ_ERR_ARG;
    const bool packed = c->k_bits || c->v_bits;
    if (packed) {
        if (c->k_bits < 1 || c->k_bits > 8 || c->v_bits < 1 || c->v_bits > 16) return IQ_ERR_ARG;
        if (!c->kq || !c->vq || !c->k_mag || !c->v_mag || misaligned(c->vq, 2) || misaligned(c->k_mag, 8) ||
            misaligned(c->v_mag, 8))
            return IQ_ERR_ARG;
    } else if (!c->k || !c->v || misaligned(c->k, 8) || misaligned(c->v, 8)) {
        return IQ_ERR_ARG;
    }
    *a = KVArgs{c->k, c->v, c->kq, c->vq, c->k_mag, c->v_mag, c->seqs, c->max_seq, c->kv_heads, c->head_dim,
                c->k_bits, c->v_bits};
    return IQ_OK;
}

static int tree_check(const iq_kv_cache *cache, int nh, int n_seq, int rows, int max_nodes, int max_len, KVArgs *c) {
    int rc;
    if ((rc = cache_check(cache, c))) return rc;
    if (nh < 1 || nh > 4096 || nh % c->nkv || n_seq < 1 || n_seq > 65536 || rows < 1 || max_nodes < 1 || max_len < 1) return IQ_ERR_ARG;
    if (max_nodes > TREE_MAX_NODES || max_len > c->max_seq || max_len > 32767)
        return IQ_ERR_RANGE;
    return IQ_OK;
}

// How a call is cut (see k_tree_scores and k_tree_pv).
static void tree_plan(TreeArgs *a) {
    const int grp = a->nh / a->c.nkv, sms = dev_info().sms;
    const int64_t cols = (int64_t)std::min(a->max_nodes, a->rows) * grp;
    // the row stride keeps every row 16-byte aligned
    a->Tw = (a->max_len + 3) / 4 * 4;
    // columns of all sequences, on average over them (rows outside the sequences may be many,
    // a sequence has no more than cols)
    const int64_t avg = std::min(cols, std::max<int64_t>(1, (int64_t)a->rows * grp / a->n_seq));
    // 8 columns a block for single tokens of up to 8 heads a kv head (64 of them at 2000
    // positions: 175 us, with half-empty blocks of 16: 190 us)
    const int nt = cols <= 8 ? 1 : 2, blocks = (int)((cols + 8 * nt - 1) / (8 * nt));
    // up to 8 blocks share the key planes (8 drafts of 16-48 nodes: 339 us; 2 blocks 363, one
    // 414), fewer where that leaves SMs without a CTA; a single block's CTA walks over up to
    // 8 tiles on the same terms (64 single tokens: 175 us; one tile a CTA 179)
    const int tiles = (a->max_len + 127) / 128;
    const int64_t pairs = (int64_t)a->n_seq * a->c.nkv;
    a->passes = 8;
    while (a->passes > 1 && pairs * tiles * ((avg + 8 * nt * a->passes - 1) / (8 * nt * a->passes)) < 4 * sms) a->passes /= 2;
    a->tpc = blocks == 1 ? 8 : 1;
    while (a->tpc > 1 && pairs * ((tiles + a->tpc - 1) / a->tpc) < 6 * sms) a->tpc /= 2;
    a->tiles = (tiles + a->tpc - 1) / a->tpc;
    a->groups = (blocks + a->passes - 1) / a->passes;
    // groups of 16 columns that share a tile of values (cg hd <= 256), once the sequences fill
    // them: 52 columns of 128: 2 groups 344 us, 1 group 360; 32 columns of 64: 139 and 126;
    // 256 columns of 64: 4 groups 339 us, 2 groups 341, 1 group 355
    a->cg = avg >= 96 && a->c.hd <= 64 ? 4 : avg >= 48 && a->c.hd <= 128 ? 2 : 1;
    // positions a tile of values and probabilities: two stages and the outputs of two CTAs
    // an SM (whole sixteens: every row of a tile starts on a 16-byte boundary). Short
    // tiles cost: 16 positions for 64 take 206 us for 175 with single tokens, 352 for 339 with drafts
    const int hdp = (a->c.hd + 31) / 32 * 32;
    a->tp = std::max(16, (cols <= 8 ? std::min(64, 4096 / hdp) : std::min(32, 2048 / hdp)) / 16 * 16);
    const int per = cols <= 8 ? 8 : 16 * a->cg;
    a->cblocks = (int)((cols + per - 1) / per);
    // long chunks (a CTA's start and end cost as much as 100 positions); with 8 columns
    // already when they make one wave (64 single tokens: 512 positions 63 us, 1024 54 us)
    a->chunk = 2048;
    const int64_t pv = pairs * ((avg + per - 1) / per), want = cols <= 8 ? sms * 3 / 2 : 4 * sms;
    while (a->chunk > 128 && pv * ((a->max_len + a->chunk - 1) / a->chunk) < want) a->chunk /= 2;
    a->chunks = (a->max_len + a->chunk - 1) / a->chunk;
}

// One kernel; prev: it waits for the one before itself (tree_prev_kernel), so it may start early.
template <class... P, class... X>
static int tree_launch(void (*k)(P...), int64_t grid_x, int grid_y, int threads, size_t smem, cudaStream_t s, bool prev, X... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)grid_x, (unsigned)grid_y);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = prev ? 1 : 0;
    IQ_CUDA(cudaLaunchKernelEx(&cfg, k, args...));
    return IQ_OK;
}

template <int NT, bool PK, bool W>
static int tree_scores(const TreeArgs &a, cudaStream_t s) {
    static std::atomic<uint64_t> set{0};   // devices whose shared-memory limit is raised
    int dev = 0;
    IQ_CUDA(cudaGetDevice(&dev));
    if (!(set.load() >> dev & 1)) {
        IQ_CUDA(cudaFuncSetAttribute(k_tree_scores<NT, PK, W>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)tree_scores_smem(NT, 256)));
        set.fetch_or(1ull << dev);
    }
    return tree_launch(k_tree_scores<NT, PK, W>, (int64_t)a.n_seq * a.c.nkv * a.groups * a.tiles, 1, 256,
                       tree_scores_smem(NT, a.c.hd), s, false, a);
}
template <int CB, bool PK, bool W>
static int tree_pv(const TreeArgs &a, int64_t ctas, cudaStream_t s) {
    static std::atomic<uint64_t> set{0};
    int dev = 0;
    IQ_CUDA(cudaGetDevice(&dev));
    if (!(set.load() >> dev & 1)) {
        IQ_CUDA(cudaFuncSetAttribute(k_tree_pv<CB, PK, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, 112 * 1024));
        set.fetch_or(1ull << dev);
    }
    return tree_launch(k_tree_pv<CB, PK, W>, ctas, 1, 256, tree_pv_smem<PK>(a.c.hd, a.cg * 8 * CB, a.tp, W), s, true, a);
}
template <bool PK, bool W>
static int launch_tree(const TreeArgs &a, cudaStream_t s) {
    const bool eight = (int64_t)std::min(a.max_nodes, a.rows) * (a.nh / a.c.nkv) <= 8;
    int rc = eight ? tree_scores<1, PK, W>(a, s) : tree_scores<2, PK, W>(a, s);
    if (rc) return rc;
    const int64_t rows = (int64_t)a.n_seq * a.max_nodes;
    // scores in shared memory: 339 us for 343 (drafts)
    rc = a.Tw <= TREE_SM_MAX
             ? tree_launch(k_tree_softmax<PK, true>, rows, a.nh, TREE_SM_T, (size_t)a.Tw * 8, s, true, a)
             : tree_launch(k_tree_softmax<PK, false>, rows, a.nh, TREE_SM_T, 0, s, true, a);
    if (rc) return rc;
    const int64_t pv = (int64_t)a.n_seq * a.c.nkv * a.cblocks * a.chunks;
    return eight ? tree_pv<1, PK, W>(a, pv, s) : tree_pv<2, PK, W>(a, pv, s);
}

// CTAs a row (1, 2, 4 or 8): as many as fill the GPU with the rows at hand, but at least
// 2048 logits a CTA; more where the slices of five CTAs would not fit an SM. A slice beyond
// one CTA's shared memory is read twice, and so are rows that fill the GPU with one CTA
// each (512 rows of 32000: 89 us; in shared memory over a cluster 124 us).
static int lp_launch(LpArgs *a, cudaStream_t s) {
    static std::atomic<uint64_t> set{0};   // devices whose shared-memory limit is raised
    const size_t many = 36 * 1024, one = 200 * 1024;
    int dev = 0;
    IQ_CUDA(cudaGetDevice(&dev));
    auto bytes = [&]() { return (size_t)((a->V + a->cs - 1) / a->cs + 1) * 8; };
    const int sms = dev_info().sms;
    a->cs = 1;
    const bool full = a->rows >= 2 * sms;   // one CTA a row keeps every SM busy
    while (!full && a->cs < 8 && (bytes() > many || ((int64_t)a->rows * a->cs < 4 * sms && a->V / a->cs > 4096))) a->cs *= 2;
    const bool sm = bytes() <= (full ? many : one);
    if (sm && !(set.load() >> dev & 1)) {
        IQ_CUDA(cudaFuncSetAttribute(k_logprobs<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)one));
        set.fetch_or(1ull << dev);
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)a->cs;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)((int64_t)a->rows * a->cs));
    cfg.blockDim = dim3(LP_T);
    cfg.dynamicSmemBytes = sm ? bytes() : 0;
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = a->cs > 1 ? 1 : 0;
    IQ_CUDA(sm ? cudaLaunchKernelEx(&cfg, k_logprobs<true>, *a) : cudaLaunchKernelEx(&cfg, k_logprobs<false>, *a));
    return IQ_OK;
}

extern "C" {

IQ_API int iq_rope_tables_dev(int64_t *d_cos, int64_t *d_sin, int rot_dim, int n_pos, int theta,
                              const iq_rope_scaling *sc, void *stream) {
    if (!d_cos || !d_sin || misaligned(d_cos, 8) || misaligned(d_sin, 8) || rot_dim < 2 || rot_dim > 256 ||
        (rot_dim & 1) || n_pos < 1 || n_pos > (1 << 24) || theta < 1)
        return IQ_ERR_ARG;
    static const HostCordic hc;
    RopeTab t = {rot_dim / 2, rot_dim, n_pos, IQ_ROPE_SCALE_NONE, 0, h_ln_int(theta), IQ_ONE, 0, IQ_ONE, 0, hc.pi, hc.gain, {}};
    std::copy(hc.angles, hc.angles + 25, t.angles);
    if (sc) {
        if (sc->kind < IQ_ROPE_SCALE_NONE || sc->kind > IQ_ROPE_SCALE_PARTS || sc->mscale < 0 ||
            sc->mscale > 1024 * IQ_ONE)
            return IQ_ERR_ARG;
        if (sc->kind != IQ_ROPE_SCALE_NONE && (sc->factor < IQ_ONE || sc->factor > 1024 * IQ_ONE)) return IQ_ERR_ARG;
        t.kind = sc->kind;
        t.mscale = sc->mscale == IQ_ONE ? 0 : sc->mscale;
        if (sc->kind != IQ_ROPE_SCALE_NONE) t.factor = sc->factor;
        if (sc->kind == IQ_ROPE_SCALE_NTK) {
            if (rot_dim < 4) return IQ_ERR_ARG;
            t.ln_theta += h_mul(h_log(sc->factor), (int64_t)(((i128)rot_dim << 48) / (rot_dim - 2)));
        }
        if (sc->kind == IQ_ROPE_SCALE_PARTS) {
            // orig_len <= 2^16 and th <= 1: the turns stay below 2^14
            if (sc->orig_len < 1 || sc->orig_len > (1 << 16) || sc->low < 0 || sc->high <= sc->low) return IQ_ERR_ARG;
            t.orig_len = sc->orig_len;
            t.low = sc->low;
            t.span = sc->high - sc->low;
        }
    }
    if (t.ln_theta > 20 * IQ_ONE) return IQ_ERR_RANGE;
    int dev, rc;
    if ((rc = cur_device(&dev))) return rc;
    const int64_t n = (int64_t)n_pos * t.half, blocks = (n + 255) / 256, cap = (int64_t)dev_info().sms * 8;
    k_rope_tables<<<(int)(blocks < cap ? blocks : cap), 256, 0, pick(stream)>>>(d_cos, d_sin, t);
    IQ_CHECK_LAUNCH();
    return IQ_OK;
}

IQ_API int iq_rope_dev(int64_t *d_out, const int64_t *d_x, const iq_rope *rope, int rows, int heads, int head_dim,
                       int64_t x_stride, int64_t out_stride, void *stream) {
    RopeArgs r;
    if (rows < 0 || heads < 1 || heads > 65536 || head_dim < 1 || head_dim > 256) return IQ_ERR_ARG;
    const int64_t w = (int64_t)heads * head_dim;
    if (x_stride < w || out_stride < w) return IQ_ERR_ARG;
    if (rows == 0) return IQ_OK;   // (an empty tensor's pointer may be NULL)
    if (!d_out || !d_x || misaligned(d_out, 8) || misaligned(d_x, 8) || (d_out == d_x && x_stride != out_stride))
        return IQ_ERR_ARG;
    int dev, rc;
    if ((rc = rope_check(rope, head_dim, &r))) return rc;
    if ((rc = cur_device(&dev))) return rc;
    const bool wide = rope_wide(r, head_dim) && !misaligned(d_x, 16) && !misaligned(d_out, 16) && x_stride % 2 == 0 &&
                      out_stride % 2 == 0;
    const int items = heads * (wide ? head_dim / 4 : (head_dim + 1) / 2);
    int tx = 256;
    while (tx > 32 && tx / 2 >= items) tx /= 2;
    const dim3 block(tx, 256 / tx), grid((rows + block.y - 1) / block.y, std::min(64, (items + tx - 1) / tx));
    if (wide) k_rope<true><<<grid, block, 0, pick(stream)>>>(d_out, d_x, r, rows, heads, head_dim, x_stride, out_stride);
    else k_rope<false><<<grid, block, 0, pick(stream)>>>(d_out, d_x, r, rows, heads, head_dim, x_stride, out_stride);
    IQ_CHECK_LAUNCH();
    return IQ_OK;
}

IQ_API int iq_kv_write_dev(const iq_kv_cache *cache, const int64_t *d_k, const int64_t *d_v, const int *d_seq,
                           const int *d_slot, int rows, int64_t k_stride, int64_t v_stride, const iq_rope *rope,
                           void *stream) {
    KVArgs c;
    RopeArgs r = {};
    int dev, rc;
    if ((rc = cache_check(cache, &c))) return rc;
    const int64_t w = (int64_t)c.nkv * c.hd;
    if (rows < 0 || k_stride < w || v_stride < w || (int64_t)rows * c.nkv > INT_MAX / 2) return IQ_ERR_ARG;
    if (rows == 0) return IQ_OK;
    if (!d_k || !d_v || !d_slot || misaligned(d_k, 8) || misaligned(d_v, 8) || misaligned(d_slot, 4) ||
        misaligned(d_seq, 4))
        return IQ_ERR_ARG;
    if (rope && (rc = rope_check(rope, c.hd, &r))) return rc;
    if ((rc = cur_device(&dev))) return rc;
    const int64_t vecs = (int64_t)rows * c.nkv * 2;
    cudaStream_t st = pick(stream);
    const bool wide = rope_wide(r, c.hd) && !misaligned(d_k, 16) && !misaligned(d_v, 16) && k_stride % 2 == 0 && v_stride % 2 == 0 &&
                      (c.kbits ? !misaligned(c.kq, 2) && !misaligned(c.vq, 4) : !misaligned(c.k, 16) && !misaligned(c.v, 16));
    if (wide) {
        int log_l = 0;   // lanes a vector
        while (log_l < 5 && 1 << log_l < c.hd / 4) log_l++;
        const int blocks = (int)(((vecs << log_l) + 255) / 256);
        auto *kern = c.kbits ? c.hd <= 128 ? k_kv_write_wide<true, 1> : k_kv_write_wide<true, 2>
                             : c.hd <= 128 ? k_kv_write_wide<false, 1> : k_kv_write_wide<false, 2>;
        kern<<<blocks, 256, 0, st>>>(c, d_k, d_v, d_seq, d_slot, rows, k_stride, v_stride, r, log_l);
    } else {
        const int blocks = (int)((vecs + 7) / 8);
        if (c.kbits)
            k_kv_write<true><<<blocks, 256, 0, st>>>(c, d_k, d_v, d_seq, d_slot, rows, k_stride, v_stride, r);
        else
            k_kv_write<false><<<blocks, 256, 0, st>>>(c, d_k, d_v, d_seq, d_slot, rows, k_stride, v_stride, r);
    }
    IQ_CHECK_LAUNCH();
    return IQ_OK;
}

IQ_API int iq_kv_read_dev(int64_t *d_k, int64_t *d_v, const iq_kv_cache *cache, const int *d_seq, const int *d_slot,
                          int rows, void *stream) {
    KVArgs c;
    int dev, rc;
    if ((rc = cache_check(cache, &c))) return rc;
    if (rows < 0 || (int64_t)rows * c.nkv > INT_MAX / 2) return IQ_ERR_ARG;
    if (rows == 0) return IQ_OK;
    if (!d_k || !d_v || !d_slot || misaligned(d_k, 8) || misaligned(d_v, 8) || misaligned(d_slot, 4) ||
        misaligned(d_seq, 4))
        return IQ_ERR_ARG;
    if ((rc = cur_device(&dev))) return rc;
    const bool wide = c.hd % 4 == 0 && !misaligned(d_k, 16) && !misaligned(d_v, 16) &&
                      (c.kbits ? !misaligned(c.kq, 4) && !misaligned(c.vq, 8) : !misaligned(c.k, 16) && !misaligned(c.v, 16));
    const int64_t blocks = ((int64_t)rows * c.nkv * 2 * (wide ? c.hd / 4 : c.hd) + 255) / 256, cap = (int64_t)dev_info().sms * 64;
    cudaStream_t st = pick(stream);
    if (wide) k_kv_read<true><<<(int)std::min(blocks, cap), 256, 0, st>>>(d_k, d_v, c, d_seq, d_slot, rows);
    else k_kv_read<false><<<(int)std::min(blocks, cap), 256, 0, st>>>(d_k, d_v, c, d_seq, d_slot, rows);
    IQ_CHECK_LAUNCH();
    return IQ_OK;
}

IQ_API int iq_attn_tree_work(const iq_kv_cache *cache, int num_heads, int n_seq, int rows, int max_nodes, int max_len,
                             int64_t *bytes) {
    KVArgs c;
    int rc;
    if (!bytes) return IQ_ERR_ARG;
    if ((rc = tree_check(cache, num_heads, n_seq, rows, max_nodes, max_len, &c))) return rc;
    *bytes = (int64_t)rows * num_heads * ((max_len + 3) / 4 * 4) * 8;
    return IQ_OK;
}

IQ_API int iq_attn_tree_dev(int64_t *d_out, const int64_t *d_q, const iq_kv_cache *cache, int num_heads,
                            const int *d_seq, const int *d_len, const int *d_start, const int *d_parent, int n_seq,
                            int rows, int max_nodes, int max_len, int64_t q_stride, void *d_work, int64_t work_bytes,
                            void *stream) {
    TreeArgs a = {};
    int dev, rc;
    if ((rc = tree_check(cache, num_heads, n_seq, rows, max_nodes, max_len, &a.c))) return rc;
    if (!d_out || !d_q || !d_len || !d_start || !d_parent || misaligned(d_out, 8) || misaligned(d_q, 8) ||
        misaligned(d_len, 4) || misaligned(d_start, 4) || misaligned(d_parent, 4) || misaligned(d_seq, 4) ||
        misaligned(d_work, 16) || d_out == d_q || q_stride < (int64_t)num_heads * a.c.hd || !d_work ||
        work_bytes < (int64_t)rows * num_heads * ((max_len + 3) / 4 * 4) * 8)
        return IQ_ERR_ARG;
    if ((rc = cur_device(&dev))) return rc;
    a.out = d_out; a.q = d_q; a.seq = d_seq; a.len = d_len; a.start = d_start; a.parent = d_parent;
    a.n_seq = n_seq; a.rows = rows; a.max_nodes = max_nodes; a.max_len = max_len; a.nh = num_heads;
    a.qs = q_stride;
    a.sc = (int64_t *)d_work;
    a.scale = h_att_scale(a.c.hd);
    tree_plan(&a);
    const int64_t most = std::max({(int64_t)n_seq * a.c.nkv * a.groups * a.tiles,
                                   (int64_t)n_seq * a.c.nkv * a.cblocks * a.chunks, (int64_t)n_seq * max_nodes});
    if (most > INT_MAX) return IQ_ERR_RANGE;
    // whole 32-wide steps in aligned pieces: 16 bytes of queries, vectors and codes
    const bool wide = a.c.hd % 32 == 0 && !misaligned(d_q, 16) && q_stride % 2 == 0 &&
                      (a.c.kbits ? !misaligned(a.c.kq, 16) && !misaligned(a.c.vq, 16)
                                 : !misaligned(a.c.k, 16) && !misaligned(a.c.v, 16));
    cudaStream_t st = pick(stream);
    if (a.c.kbits) return wide ? launch_tree<true, true>(a, st) : launch_tree<true, false>(a, st);
    return wide ? launch_tree<false, true>(a, st) : launch_tree<false, false>(a, st);
}

IQ_API int iq_logprobs_dev(const int64_t *d_logits, int64_t ld, int rows, int vocab, const int *d_tokens,
                           int64_t *d_logp, int64_t *d_entropy, int top, int *d_top_ids, int64_t *d_top_logp,
                           void *stream) {
    if (rows < 0 || vocab < 1 || ld < vocab || top < 0 || top > vocab) return IQ_ERR_ARG;
    if (vocab > (1 << 20) || top > IQ_LP_MAX_TOP || rows > INT_MAX / 8) return IQ_ERR_RANGE;
    if (rows == 0) return IQ_OK;
    if (!d_logits || !d_tokens != !d_logp || (top && (!d_top_ids || !d_top_logp)) || misaligned(d_logits, 8) ||
        misaligned(d_tokens, 4) || misaligned(d_logp, 8) || misaligned(d_entropy, 8) || misaligned(d_top_ids, 4) ||
        misaligned(d_top_logp, 8))
        return IQ_ERR_ARG;
    int dev, rc;
    if ((rc = cur_device(&dev))) return rc;
    LpArgs a = {d_logits, ld, rows, vocab, top, d_tokens, d_logp, d_entropy, d_top_ids, d_top_logp, 1};
    return lp_launch(&a, pick(stream));
}

}  // extern "C"
