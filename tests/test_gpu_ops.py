"""GPU tests of the operators around drafted tokens against whole-number
references (ops_ref): every result is an integer defined exactly, so equality
is the tolerance."""
import ctypes

import numpy as np
import pytest

import configs
import iq
import ops_ref as ref
from helpers import ONE, model_weights

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

RANGE = -6
KEEP = -7777777          # what outputs hold before a call


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t.to(dtype) if dtype else t).cuda()


def i32(a):
    return dev(np.asarray(a, np.int32))


def full(*shape):
    return torch.full(shape, KEEP, dtype=torch.int64, device="cuda")


def rnd(rng, *shape, scale=1.0):
    return ref.q48(rng.standard_normal(shape) * scale)


def wide(rng, *shape):
    """Values over the whole int64 range, the ends among them."""
    a = rng.integers(-(1 << 63), (1 << 63) - 1, shape, dtype=np.int64)
    f = a.reshape(-1)
    f[: min(4, f.size)] = [ref.I64_MIN, ref.I64_MAX, 0, -1][: min(4, f.size)]
    return a


@pytest.fixture(autouse=True)
def clean_status():
    iq.device_status()
    yield
    assert iq.device_status() == 0


# ------------------------------------------------------------------- rotary

SCALES = [dict(), dict(kind="linear", factor=4 * ONE), dict(kind="ntk", factor=ONE * 5 // 2),
          dict(kind="parts", factor=8 * ONE, orig_len=2048, low=ONE, high=32 * ONE),
          dict(kind="parts", factor=3 * ONE, orig_len=100, low=0, high=ONE, mscale=ONE * 9 // 8),
          dict(kind="none", mscale=ONE // 2), dict(kind="linear", factor=ONE)]


@pytest.mark.parametrize("sc", SCALES)
@pytest.mark.parametrize("rot,theta", [(64, 10000), (4, 16383), (256, 1000000), (30, 1)])
def test_rope_tables(rot, theta, sc):
    n = 70000
    cos, sin = full(n, rot // 2), full(n, rot // 2)
    iq.rope_tables_dev(cos, sin, rot, n, theta, sc or None)
    at = [0, 1, 2, 3, 77, 2047, 32767, 32768, 69999]
    c, s = ref.tables(rot, at, theta, **sc)
    assert (cos[at].cpu().numpy() == c).all() and (sin[at].cpu().numpy() == s).all()
    assert int((cos == KEEP).sum()) == 0 and int((sin == KEEP).sum()) == 0


def test_rope_tables_far_and_single():
    n = 1 << 24
    cos, sin = full(n, 1), full(n, 1)
    iq.rope_tables_dev(cos, sin, 2, n, 10000)
    at = [0, n - 1, n // 3]
    c, s = ref.tables(2, at, 10000)
    assert (cos[at].cpu().numpy() == c).all() and (sin[at].cpu().numpy() == s).all()
    one = full(1, 3)
    iq.rope_tables_dev(one, one.clone(), 6, 1, 10000)
    assert (one.cpu().numpy() == ref.tables(6, [0], 10000)[0]).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rows,heads,hd,rot,xs,os", [
    (1, 36, 64, 64, 0, 0), (5, 3, 128, 96, 1, 3), (7, 1, 2, 2, 0, 0), (3, 2, 33, 32, 0, 5), (2, 5, 255, 14, 1, 0),
    (130, 4, 256, 256, 2, 2), (9, 2, 6, 4, 0, 0), (2, 3, 20, 20, 1, 1), (2, 70, 40, 8, 4, 2)])
def test_rope(layout, rows, heads, hd, rot, xs, os):
    rng = np.random.default_rng(rows * 1000 + hd)
    w, n = heads * hd, 50
    x = wide(rng, rows, w + xs) if rows % 2 else rnd(rng, rows, w + xs, scale=3)
    cos, sin = rnd(rng, n, rot // 2), rnd(rng, n, rot // 2)
    pos = rng.integers(0, n, rows)
    pos[rows // 2] = -1 if rows > 2 else pos[rows // 2]
    out = full(rows, w + os)
    r = iq.Rope(dev(cos), dev(sin), i32(pos), n, rot, layout)
    iq.rope_dev(out, dev(x), r, rows, heads, hd, x_stride=w + xs, out_stride=w + os)
    want = np.full((rows, w + os), KEEP, np.int64)
    live = pos >= 0
    want[live, :w] = ref.rotate(x[:, :w].reshape(rows, heads, hd), cos[pos], sin[pos], rot, layout)[live].reshape(-1, w)
    assert (out.cpu().numpy() == want).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_in_place_unaligned_and_bad_position(layout):
    rng = np.random.default_rng(5)
    rows, heads, hd, n = 6, 3, 48, 9
    x, cos, sin = rnd(rng, rows, heads * hd), rnd(rng, n, 12), rnd(rng, n, 12)
    pos = np.array([0, 8, 9, 3, -1, 1 << 30])
    buf = torch.empty(rows * heads * hd + 1, dtype=torch.int64, device="cuda")
    d = buf[1:]                                   # 8-byte aligned only
    d.copy_(dev(x).flatten())
    iq.rope_dev(d, d, iq.Rope(dev(cos), dev(sin), i32(pos), n, 24, layout), rows, heads, hd)
    want = x.copy().reshape(rows, heads, hd)
    live = (pos >= 0) & (pos < n)
    want[live] = ref.rotate(want[live], cos[pos[live]], sin[pos[live]], 24, layout)
    assert (d.cpu().numpy().reshape(want.shape) == want).all()
    assert iq.device_status() == RANGE


# -------------------------------------------------------------------- cache

def new_cache(seqs, max_seq, nkv, hd, kb, vb):
    """(cache, its tensors), all elements KEEP or a small mark."""
    if kb:
        t = dict(kq=torch.full((seqs, max_seq, nkv, hd), 77, dtype=torch.uint8, device="cuda"),
                 vq=torch.full((seqs, max_seq, nkv, hd), 77, dtype=torch.int16, device="cuda"),
                 k_mag=full(seqs, max_seq, nkv), v_mag=full(seqs, max_seq, nkv))
    else:
        t = dict(k=full(seqs, max_seq, nkv, hd), v=full(seqs, max_seq, nkv, hd))
    return iq.KVCache(seqs, max_seq, nkv, hd, k_bits=kb, v_bits=vb, **t), t


def host_cache(t):
    h = {n: x.cpu().numpy().copy() for n, x in t.items()}
    if "vq" in h:
        h["vq"] = h["vq"].view(np.uint16)
    return h


def write_ref(h, k, v, seq, slot, kb, vb):
    for r in range(len(slot)):
        for head in range(k.shape[1]):
            at = (seq[r], slot[r], head)
            if kb:
                h["kq"][at], h["k_mag"][at] = ref.pack(k[r, head], kb)
                h["vq"][at], h["v_mag"][at] = ref.pack(v[r, head], vb)
            else:
                h["k"][at], h["v"][at] = k[r, head], v[r, head]


@pytest.mark.parametrize("kb,vb", [(0, 0), (8, 10), (1, 1), (4, 16), (8, 16)])
@pytest.mark.parametrize("rows,nkv,hd,rot,layout", [
    (1, 4, 64, 64, "half"), (9, 2, 128, 96, "interleaved"), (3, 3, 1, 0, ""), (5, 1, 255, 128, "half"),
    (4, 2, 256, 256, "interleaved"), (33, 1, 40, 0, ""), (6, 2, 65, 2, "half")])
def test_kv_write_and_read(kb, vb, rows, nkv, hd, rot, layout):
    rng = np.random.default_rng(rows * 100 + hd + kb)
    seqs, max_seq, n = 3, 17, 30
    k, v = rnd(rng, rows, nkv, hd), rnd(rng, rows, nkv, hd, scale=40)
    v[0] = 0                                                        # a vector without magnitude
    if rows > 3:
        k[1], v[1] = wide(rng, nkv, hd), wide(rng, nkv, hd)         # wraps as the reference's int64
        v[2] = rng.integers(-(1 << 62), 1 << 62, (nkv, hd))
        v[3] = rng.integers(-2, 3, (nkv, hd))
    at = rng.permutation(seqs * max_seq)[:rows]
    seq, slot = at // max_seq, at % max_seq
    pos = rng.integers(0, n, rows)
    cos, sin = rnd(rng, n, max(1, rot // 2)), rnd(rng, n, max(1, rot // 2))
    if rows > 5:
        slot[4], seq[5], pos[3] = -1, -1, -1                        # padding rows
    w = nkv * hd
    c, t = new_cache(seqs, max_seq, nkv, hd, kb, vb)
    buf = np.zeros((rows, 2 * w + 1), np.int64)
    buf[:, :w], buf[:, w:2 * w] = k.reshape(rows, w), v.reshape(rows, w)
    d = dev(buf)
    want = host_cache(t)
    live = (slot >= 0) & (seq >= 0)
    r = None
    if rot:
        r = iq.Rope(dev(cos), dev(sin), i32(pos), n, rot, layout)
        live &= pos >= 0
        k = ref.rotate(k, cos[pos], sin[pos], rot, layout)
    iq.kv_write_dev(c, d, d[:, w:], i32(slot), rows, seq=i32(seq), rope=r, k_stride=2 * w + 1, v_stride=2 * w + 1)
    write_ref(want, k[live], v[live], seq[live], slot[live], kb, vb)
    got = host_cache(t)
    for name in want:
        assert (got[name] == want[name]).all(), name
    # read back: written and padding rows, the same row twice
    rs, rq = np.r_[slot, slot[:1], -1], np.r_[seq, seq[:1], 0]
    ko, vo = full(rows + 2, nkv, hd), full(rows + 2, nkv, hd)
    iq.kv_read_dev(ko, vo, c, i32(rs), rows + 2, seq=i32(rq))
    for i in range(rows + 2):
        for h in range(nkv):
            if rs[i] < 0 or rq[i] < 0:
                wk = wv = np.full(hd, KEEP)
            elif kb:
                a = (rq[i], rs[i], h)
                wk = ref.unpack(want["kq"][a], want["k_mag"][a], kb)
                wv = ref.unpack(want["vq"][a], want["v_mag"][a], vb)
            else:
                wk, wv = want["k"][rq[i], rs[i], h], want["v"][rq[i], rs[i], h]
            assert (ko[i, h].cpu().numpy() == wk).all() and (vo[i, h].cpu().numpy() == wv).all()


def test_kv_bad_rows_are_left_out_and_recorded():
    c, t = new_cache(2, 8, 1, 4, 0, 0)
    x = dev(np.arange(16).reshape(4, 4))
    iq.kv_write_dev(c, x, x, i32([0, 8, 1, 2]), 4, seq=i32([0, 0, 2, -1]))
    assert iq.device_status() == RANGE
    k = t["k"].cpu().numpy()
    assert (k[0, 0, 0] == [0, 1, 2, 3]).all() and (k.reshape(16, 4)[1:] == KEEP).all()
    o = full(2, 1, 4)
    iq.kv_read_dev(o, o.clone(), c, i32([0, 1 << 20]), 2)
    assert iq.device_status() == RANGE
    assert (o.cpu().numpy()[:, 0] == [[0, 1, 2, 3], [KEEP] * 4]).all()


# --------------------------------------------------------------------- tree

def chain(n):
    return list(range(-1, n - 1))


def bush(rng, n):
    return [-1 if i == 0 or rng.random() < 0.2 else int(rng.integers(max(0, i - 5), i)) for i in range(n)]


def run_tree(q, t, kvb, lens, starts, parents, nh, max_nodes=None, max_len=None, seqs=None, q_stride=None, rows=None,
             stream=None):
    kb, vb = kvb
    shape = t["kq" if kb else "k"].shape
    cache = iq.KVCache(shape[0], shape[1], shape[2], shape[3], k_bits=kb, v_bits=vb, **t)
    rows = q.shape[0] if rows is None else rows
    n = [b - a for a, b in zip(starts, starts[1:])]
    max_nodes = max_nodes or max(n)
    max_len = max_len or max(a + b for a, b in zip(lens, n))
    size = dict(n_seq=len(lens), rows=rows, max_nodes=max_nodes, max_len=max_len)
    need = iq.attn_tree_work(cache, nh, **size)
    work = torch.empty((need + 7) // 8 + 1, dtype=torch.int64, device="cuda")
    out = full(rows, nh * shape[3])
    iq.attn_tree_dev(out, q, cache, nh, i32(lens), i32(starts), i32(parents), work=work,
                     seqs=None if seqs is None else i32(seqs), q_stride=q_stride, **size)
    return out.cpu().numpy()


def check_tree(rng, nh, nkv, hd, lens, trees, kvb=(0, 0), q=None, k=None, v=None, pad=0, **kw):
    """One random case against the reference; trees: parents per sequence."""
    kb, vb = kvb
    S, max_seq = len(lens), max(a + len(p) for a, p in zip(lens, trees)) + pad
    starts = np.r_[0, np.cumsum([len(p) for p in trees])].tolist()
    parents = [x for p in trees for x in p]
    rows = starts[-1]
    q = rnd(rng, rows, nh, hd, scale=1.5) if q is None else q
    if kb:
        t = dict(kq=dev(rng.integers(0, 1 << kb, (S, max_seq, nkv, hd)), torch.uint8),
                 vq=dev(rng.integers(0, 1 << vb, (S, max_seq, nkv, hd)), torch.int16),
                 k_mag=dev(rng.integers(0, 4 * ONE, (S, max_seq, nkv))),
                 v_mag=dev(rng.integers(0, 4 * ONE, (S, max_seq, nkv))))
        h = host_cache(t)
        k = np.array([ref.unpack(c, m, kb) for c, m in zip(h["kq"].reshape(-1, hd), h["k_mag"].reshape(-1))])
        v = np.array([ref.unpack(c, m, vb) for c, m in zip(h["vq"].reshape(-1, hd), h["v_mag"].reshape(-1))])
        k, v = k.reshape(S, max_seq, nkv, hd), v.reshape(S, max_seq, nkv, hd)
    else:
        k = rnd(rng, S, max_seq, nkv, hd) if k is None else k
        v = rnd(rng, S, max_seq, nkv, hd) if v is None else v
        t = dict(k=dev(k), v=dev(v))
    got = run_tree(dev(q.reshape(rows, -1)), t, kvb, lens, starts, parents, nh, **kw)
    want = ref.tree(q, k, v, lens, starts, parents, nh)
    assert (got == want.reshape(rows, -1)).all()


GEOM = [(8, 2, 32), (4, 4, 128), (3, 1, 40), (7, 1, 64), (16, 1, 64), (1, 1, 1), (2, 1, 256), (6, 2, 17), (32, 4, 64),
        (20, 1, 16), (5, 5, 96)]


@pytest.mark.parametrize("kvb", [(0, 0), (8, 10)])
@pytest.mark.parametrize("nh,nkv,hd", GEOM)
def test_tree_geometries(nh, nkv, hd, kvb):
    rng = np.random.default_rng(nh * 100 + hd)
    check_tree(rng, nh, nkv, hd, [0, 37, 70], [bush(rng, 5), bush(rng, 1), bush(rng, 9)], kvb, pad=3)


@pytest.mark.parametrize("ln", [0, 1, 2, 7, 15, 16, 17, 31, 63, 64, 65, 127, 255, 256, 257, 300])
def test_tree_single_token_lengths(ln):
    """A decode step: one node over a context of ln positions."""
    rng = np.random.default_rng(ln)
    check_tree(rng, 4, 2, 32, [ln, max(0, ln - 1)], [[-1], [-1]])


@pytest.mark.parametrize("n", [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 33, 64, 65, 100])
def test_tree_node_counts(n):
    rng = np.random.default_rng(n)
    check_tree(rng, 2, 1, 16, [11, 0], [bush(rng, n), chain(max(1, n // 2))])


def test_tree_most_nodes():
    rng = np.random.default_rng(9)
    check_tree(rng, 1, 1, 8, [3], [bush(rng, 256)])
    check_tree(rng, 1, 1, 8, [0], [chain(256)])


@pytest.mark.parametrize("kvb", [(0, 0), (1, 1), (5, 16)])
@pytest.mark.parametrize("ln", [900, 2050, 5000])
def test_tree_long_contexts(ln, kvb):
    rng = np.random.default_rng(ln)
    check_tree(rng, 4, 2, 16, [ln, ln // 3], [bush(rng, 3), bush(rng, 12)], kvb)


def test_tree_longest_context():
    rng = np.random.default_rng(1)
    check_tree(rng, 2, 1, 4, [32766], [[-1]])
    check_tree(rng, 1, 1, 4, [32700], [bush(rng, 9)])


def test_tree_flat_and_peaked_scores():
    """All scores equal; one far above the rest (every other probability 0); scores a few units apart."""
    rng = np.random.default_rng(2)
    nh, nkv, hd, n, T = 4, 2, 32, 5, 130
    for s in (0.0, 60.0, 0.2):
        q = np.full((n, nh, hd), ref.q48(s), np.int64)
        k = np.full((1, T, nkv, hd), ref.q48(0.01), np.int64)
        k[0, 77] = ref.q48(1.0)
        check_tree(rng, nh, nkv, hd, [T - n], [bush(rng, n)], q=q, k=k)


@pytest.mark.parametrize("vs", [7.9, 8.1, 100.0, 20000.0])
def test_tree_large_values(vs):
    """Values around and beyond the range of the fast sum of products."""
    rng = np.random.default_rng(3)
    v = rnd(rng, 2, 150, 2, 32, scale=0.1)
    v[0, ::7], v[0, 1::7], v[1, 100, 1, 3] = ref.q48(vs), ref.q48(-vs), ref.q48(vs)
    check_tree(rng, 4, 2, 32, [140, 90], [bush(rng, 6), bush(rng, 8)], v=v, pad=4)


def test_tree_whole_int64_range():
    """Scores and values that wrap: the same integers as the reference, whatever they mean."""
    rng = np.random.default_rng(4)
    q, k, v = wide(rng, 7, 4, 32), wide(rng, 2, 60, 2, 32), wide(rng, 2, 60, 2, 32)
    check_tree(rng, 4, 2, 32, [50, 0], [bush(rng, 4), bush(rng, 3)], q=q, k=k, v=v)
    q = rng.integers(-(1 << 56), 1 << 56, (7, 4, 32))
    k = rng.integers(-(1 << 56), 1 << 56, (2, 60, 2, 32))
    check_tree(rng, 4, 2, 32, [50, 0], [bush(rng, 4), bush(rng, 3)], q=q, k=k, v=v)
    q = rng.integers(-(1 << 55), 1 << 55, (7, 4, 32))
    q[0, 0, 0], q[0, 0, 1], k[0, 0, 0, 0], k[0, 1, 0, 0] = -(1 << 55), (1 << 55) - 1, -(1 << 55), (1 << 55) - 1
    check_tree(rng, 4, 2, 32, [50, 0], [bush(rng, 4), bush(rng, 3)], q=q, k=k >> 2, v=v >> 12)


def test_tree_masked_slots_are_not_read_into_results():
    """Extreme values in slots a node does not see change nothing for it."""
    rng = np.random.default_rng(6)
    nh, nkv, hd = 4, 2, 32
    trees = [[-1, -1, 0, 1, 2, -1]]
    q, k, v = rnd(rng, 6, nh, hd), rnd(rng, 1, 80, nkv, hd), rnd(rng, 1, 80, nkv, hd)
    k[0, 41], v[0, 41] = ref.I64_MIN, ref.I64_MAX        # node 1: only nodes 1 and 3 see it
    k[0, 46:], v[0, 46:] = ref.I64_MAX, ref.I64_MIN      # beyond the draft
    check_tree(rng, nh, nkv, hd, [40], trees, q=q, k=k, v=v, max_len=60)


def test_tree_rows_outside_and_bad_sequences():
    """Rows behind the last sequence and of a sequence beyond its bounds stay; bad parents count as -1."""
    rng = np.random.default_rng(7)
    nh, nkv, hd, S, M = 4, 2, 16, 5, 40
    k, v = rnd(rng, S, M, nkv, hd), rnd(rng, S, M, nkv, hd)
    t = dict(k=dev(k), v=dev(v))
    starts, parents = [1, 3, 3, 5, 8, 9], [-1] * 12
    lens = [10, 5, 39, 20, -1]                            # the third: 39 + 2 > 40; the last: negative
    parents[2], parents[6], parents[7] = 0, 5, 0          # node 1 of the fourth names a later node
    q = rnd(rng, 12, nh, hd)
    got = run_tree(dev(q.reshape(12, -1)), t, (0, 0), lens, starts, parents, nh, max_nodes=3, max_len=M)
    assert iq.device_status() == RANGE
    want = np.full((12, nh, hd), KEEP, np.int64)
    good = ref.tree(q[:8], [k[0], k[1], k[2][:0], k[3]], [v[0], v[1], v[2][:0], v[3]], [10, 5, 0, 20], [1, 3, 3, 3, 3], parents, nh)
    want[1:3] = good[1:3]
    want[5:8] = ref.tree(q[5:8], [k[3]], [v[3]], [20], [0, 3], parents[5:8], nh)
    assert (got == want.reshape(12, -1)).all()
    # starts beyond the rows, falling starts, an unknown cache sequence, a padding sequence (-1)
    for st, sq, want_status in (([0, 13], [0], RANGE), ([2, 1], [0], RANGE), ([0, 1], [5], RANGE), ([0, 1], [-1], 0),
                                ([-1, 1], [0], RANGE), ([0, 4], [0], RANGE)):
        got = run_tree(dev(q.reshape(12, -1)), t, (0, 0), [3], st, parents, nh, max_nodes=3, max_len=M, seqs=sq)
        assert (got == KEEP).all() and iq.device_status() == want_status


def test_tree_shared_cache_sequence_and_strided_queries():
    """Two drafts over the same cache sequence (read only), query rows inside a wider buffer."""
    rng = np.random.default_rng(8)
    nh, nkv, hd = 8, 2, 32
    k, v = rnd(rng, 3, 90, nkv, hd), rnd(rng, 3, 90, nkv, hd)
    trees = [bush(rng, 4), bush(rng, 6)]
    starts = [0, 4, 10]
    q = rnd(rng, 10, nh * hd + 5)
    got = run_tree(dev(q), dict(k=dev(k), v=dev(v)), (0, 0), [80, 33], starts, trees[0] + trees[1], nh, seqs=[2, 2],
                   q_stride=nh * hd + 5)
    want = ref.tree(q[:, : nh * hd].reshape(10, nh, hd).copy(), [k[2], k[2]], [v[2], v[2]], [80, 33], starts,
                    trees[0] + trees[1], nh)
    assert (got == want.reshape(10, -1)).all()


def test_tree_chain_equals_one_by_one():
    """A chain of nodes = the same tokens as single-node calls over the growing context."""
    rng = np.random.default_rng(10)
    nh, nkv, hd, ln, n = 8, 2, 64, 333, 19
    t = dict(k=dev(rnd(rng, 1, 400, nkv, hd)), v=dev(rnd(rng, 1, 400, nkv, hd)))
    q = dev(rnd(rng, n, nh * hd))
    whole = run_tree(q, t, (0, 0), [ln], [0, n], chain(n), nh)
    for i in range(n):
        one = run_tree(q[i:i + 1], t, (0, 0), [ln + i], [0, 1], [-1], nh)
        assert (one[0] == whole[i]).all()


def test_tree_many_rows_batch():
    """More work than one wave of blocks, checked on a sample of rows."""
    rng = np.random.default_rng(11)
    S, nh, nkv, hd, M = 40, 8, 2, 64, 700
    lens = [int(x) for x in rng.integers(0, 600, S)]
    trees = [bush(rng, int(x)) for x in rng.integers(1, 64, S)]
    starts = np.r_[0, np.cumsum([len(p) for p in trees])].tolist()
    parents = [x for p in trees for x in p]
    k, v, q = rnd(rng, S, M, nkv, hd), rnd(rng, S, M, nkv, hd), rnd(rng, starts[-1], nh, hd)
    got = run_tree(dev(q.reshape(starts[-1], -1)), dict(k=dev(k), v=dev(v)), (0, 0), lens, starts, parents, nh)
    scale = ref.fp(ref.INV_SQRT, hd << 48)
    for b in range(0, S, 3):
        paths = ref.ancestors(trees[b])
        for i in {0, len(trees[b]) - 1}:
            see = np.r_[np.arange(lens[b]), lens[b] + np.array(paths[i])].astype(int)
            for h in (0, 5):
                want = ref.attend(q[starts[b] + i, h], k[b, see, h // 4], v[b, see, h // 4], scale)
                assert (got[starts[b] + i, h * hd:(h + 1) * hd] == want).all()


# ------------------------------------------------------------------- scores

def check_logprobs(l, tokens, top, ld=None):
    rows, V = l.shape
    ld = ld or V
    buf = np.full((rows, ld), ref.I64_MAX, np.int64)
    buf[:, :V] = l
    logp, ent = full(rows), full(rows)
    ids, tl = torch.full((rows, top), -5, dtype=torch.int32, device="cuda"), full(rows, top)
    iq.logprobs_dev(dev(buf), rows, V, tokens=None if tokens is None else i32(tokens),
                    logp=None if tokens is None else logp, entropy=ent, top=top, top_ids=ids if top else None,
                    top_logp=tl if top else None, ld=ld)
    for r in range(rows):
        bad = tokens is None or not 0 <= tokens[r] < V
        lp, h, best, bl = ref.logprobs(l[r], None if bad else tokens[r], top)
        assert int(logp[r]) == (KEEP if bad else lp)
        assert int(ent[r]) == h
        assert ids[r].tolist() == best and tl[r].tolist() == bl


@pytest.mark.parametrize("V,top", [(1, 0), (1, 1), (2, 2), (31, 31), (32, 32), (33, 5), (255, 8), (1000, 1),
                                   (4097, 32), (32000, 5), (32003, 20), (65537, 3), (131072, 32), (300001, 7)])
def test_logprobs_sizes(V, top):
    rng = np.random.default_rng(V + top)
    l = rnd(rng, 3, V, scale=2.5)
    check_logprobs(l, rng.integers(0, V, 3), top, ld=V + (V % 3))


def test_logprobs_many_rows():
    rng = np.random.default_rng(12)
    check_logprobs(rnd(rng, 333, 700, scale=4), rng.integers(-1, 700, 333), 6)
    check_logprobs(rnd(rng, 20, 9000, scale=4), None, 3)


def test_logprobs_ties_masks_and_extremes():
    rng = np.random.default_rng(13)
    V = 5000
    l = rnd(rng, 12, V)
    l[0] = 0                                               # all equal
    l[1] = ref.I64_MIN                                     # all at the lowest value
    l[2] = ref.I64_MIN
    l[2, 17] = ref.I64_MAX                                 # the widest spread: d passes int64
    l[3, ::2] = ref.I64_MIN                                # half masked
    l[4] = rng.integers(0, 3, V) * ONE                     # many ties
    l[5] = np.sort(l[5])
    l[6] = np.sort(l[6])[::-1]
    l[7, :] = -34 * ONE
    l[7, 4999] = 0                                         # all others exactly at the cut-off
    l[8, :] = -34 * ONE + 1
    l[8, 0] = 0
    l[9] = wide(rng, V)
    l[10] = ref.I64_MAX
    l[11, 100:150] = l[11].max() + 1                       # more equal maxima than alternatives
    tokens = [3, 4, 18, 0, 9, 4999, 4999, 0, 4999, 5, 77, 120]
    for top in (0, 1, 8, 32):
        check_logprobs(l, tokens, top)


def test_logprobs_close_to_real_logarithms():
    """Against a 64-bit float log-softmax: E is within 2^-44 relative plus 2^-48 a
    logit, ln within 2^-46, and the 64-bit reference within 1e-13 or so of itself."""
    rng = np.random.default_rng(14)
    l = rnd(rng, 4, 32000, scale=6)
    logp, ent = full(4), full(4)
    tok = i32([1, 2, 3, 4])
    iq.logprobs_dev(dev(l), 4, 32000, tokens=tok, logp=logp, entropy=ent)
    x = torch.log_softmax(dev(l).double() / ONE, -1)
    tol = 2.0 ** -44 + 32000 * 2.0 ** -48 + 2.0 ** -46 + 1e-12
    assert (logp.double() / ONE - x.gather(1, tok.long()[:, None])[:, 0]).abs().max().item() < tol
    # entropy: the same error on ln S, and d <= 34 times it on each probability
    assert (ent.double() / ONE + (x.exp() * x).sum(-1)).abs().max().item() < 40 * tol


# ------------------------------------------------ streams, graphs, together

def test_other_stream_and_two_at_once():
    rng = np.random.default_rng(15)
    nh, nkv, hd, n = 8, 2, 32, 12
    q = [dev(rnd(rng, n, nh * hd)) for _ in range(2)]
    t = dict(k=dev(rnd(rng, 1, 300, nkv, hd)), v=dev(rnd(rng, 1, 300, nkv, hd)))
    l = [dev(rnd(rng, 40, 6000, scale=3)) for _ in range(2)]
    cache = iq.KVCache(1, 300, nkv, hd, **t)
    size = dict(n_seq=1, rows=n, max_nodes=n, max_len=300)
    ln, st, par = i32([250]), i32([0, n]), i32(chain(n))
    need = iq.attn_tree_work(cache, nh, **size) // 8 + 1

    def calls(i, stream, out, lp, work):
        iq.attn_tree_dev(out, q[i], cache, nh, ln, st, par, work=work, stream=stream, **size)
        iq.logprobs_dev(l[i], 40, 6000, entropy=lp, stream=stream)

    outs = [(full(n, nh * hd), full(40), torch.empty(need, dtype=torch.int64, device="cuda")) for _ in range(4)]
    for i in range(2):
        calls(i, None, *outs[i])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for i in range(2):
            calls(i, streams[i], *outs[2 + i])
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(outs[i][0], outs[2 + i][0]) and torch.equal(outs[i][1], outs[2 + i][1])


def test_captured_and_replayed():
    """All calls in one CUDA graph, replayed on changed inputs; two graphs with their own workspaces at once."""
    rng = np.random.default_rng(16)
    nh, nkv, hd, n, M, npos = 8, 2, 32, 6, 128, 200
    cos, sin = full(npos, hd // 2), full(npos, hd // 2)
    iq.rope_tables_dev(cos, sin, hd, npos, 10000)
    w = (nh + 2 * nkv) * hd

    def make():
        s = dict(qkv=dev(rnd(rng, n, w)), q=full(n, nh * hd), out=full(n, nh * hd), pos=i32(range(50, 50 + n)),
                 slot=i32(range(50, 50 + n)), par=i32(chain(n)), ln=i32([50]), st=i32([0, n]),
                 k=dev(rnd(rng, 1, M, nkv, hd)), v=dev(rnd(rng, 1, M, nkv, hd)), logp=full(n), tok=i32([3] * n))
        s["cache"] = iq.KVCache(1, M, nkv, hd, k=s["k"], v=s["v"])
        s["size"] = dict(n_seq=1, rows=n, max_nodes=n, max_len=M)
        s["work"] = torch.empty(iq.attn_tree_work(s["cache"], nh, **s["size"]) // 8 + 1, dtype=torch.int64, device="cuda")
        return s

    def calls(s):
        rope = iq.Rope(cos, sin, s["pos"], npos, hd)
        iq.rope_dev(s["q"], s["qkv"], rope, n, nh, hd, x_stride=w)
        iq.kv_write_dev(s["cache"], s["qkv"][:, nh * hd:], s["qkv"][:, (nh + nkv) * hd:], s["slot"], n, rope=rope,
                        k_stride=w, v_stride=w)
        iq.attn_tree_dev(s["out"], s["q"], s["cache"], nh, s["ln"], s["st"], s["par"], work=s["work"], **s["size"])
        iq.logprobs_dev(s["out"], n, nh * hd, tokens=s["tok"], logp=s["logp"])

    states = [make(), make()]
    for s in states:
        calls(s)
    torch.cuda.synchronize()
    graphs = []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            calls(s)
        graphs.append(g)
    for s in states:
        s["qkv"].copy_(dev(rnd(rng, n, w)))
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in states]
    for g, st in zip(graphs, side):
        with torch.cuda.stream(st):
            for _ in range(3):
                g.replay()
    torch.cuda.synchronize()
    got = [(s["out"].clone(), s["logp"].clone(), s["k"].clone()) for s in states]
    for s, (o, lp, k) in zip(states, got):
        calls(s)
        torch.cuda.synchronize()
        assert torch.equal(s["out"], o) and torch.equal(s["logp"], lp) and torch.equal(s["k"], k)


def _forward(c, w, toks, pos, slot, parents, ln, kvs, tables, kvb):
    """llama_forward's layers on drafted rows with the library's operators; logits on the device."""
    n, d, hd, nh, nkv = len(toks), c["dim"], c["head_dim"], c["n_heads"], c["n_kv_heads"]
    kvd, ml = nkv * hd, c["max_seq"]
    x = dev(w["embed"][toks])
    nrm, qkv, q, att = full(n, d), full(n, d + 2 * kvd), full(n, d), full(n, d)
    rope = iq.Rope(tables[0], tables[1], i32(pos), ml, hd)
    size = dict(n_seq=1, rows=n, max_nodes=n, max_len=ml)
    for l, lay in enumerate(w["layers"]):
        n1, wq, wk, wv, wo, n2, wg, wu, wd = [dev(a) for a in lay]
        iq.rmsnorm_dev(nrm, x, n1, n, d)
        wqkv = torch.cat([wq, wk, wv])
        iq.gemm_dev(qkv, wqkv, nrm, n, d + 2 * kvd, d)
        iq.rope_dev(q, qkv, rope, n, nh, hd, x_stride=d + 2 * kvd)
        cache = kvs[l]
        iq.kv_write_dev(cache, qkv[:, d:], qkv[:, d + kvd:], i32(slot), n, rope=rope, k_stride=d + 2 * kvd,
                        v_stride=d + 2 * kvd)
        work = torch.empty(iq.attn_tree_work(cache, nh, **size) // 8 + 1, dtype=torch.int64, device="cuda")
        iq.attn_tree_dev(att, q, cache, nh, i32([ln]), i32([0, n]), i32(parents), work=work, **size)
        o = full(n, d)
        iq.gemm_dev(o, wo, att, n, d, d)
        x = x + o
        iq.rmsnorm_dev(nrm, x, n2, n, d)
        it = c["inter"]
        g, u, a = full(n, it), full(n, it), full(n, it)
        iq.gemm_dev(g, wg, nrm, n, it, d)
        iq.gemm_dev(u, wu, nrm, n, it, d)
        iq.fp_dev("silu", g, None, a, n * it)
        iq.fp_dev("mul", a, u, g, n * it)
        iq.gemm_dev(o, wd, g, n, d, it)
        x = x + o
    iq.rmsnorm_dev(nrm, x, dev(w["final_norm"]), n, d)
    logits = full(n, c["vocab"])
    iq.gemm_dev(logits, dev(w["lm_head"]), nrm, n, c["vocab"], d)
    return logits


@pytest.mark.parametrize("kvb", [(0, 0), (8, 10)])
def test_verifying_a_draft_equals_the_model(kvb):
    """Rotate, write the cache, attend, score: every node's logits equal the model's own
    forward along the node's path, and its log probabilities the reference's on those logits."""
    c = configs.TINY_TEST
    w = model_weights(7, c)
    rng = np.random.default_rng(17)
    prompt = [int(x) for x in rng.integers(3, c["vocab"], 9)]
    draft = [int(x) for x in rng.integers(3, c["vocab"], 7)]
    parents = [-1, 0, 0, 1, 2, -1, 5]
    depth = [len(p) - 1 for p in ref.ancestors(parents)]
    tabs = (full(c["max_seq"], c["head_dim"] // 2), full(c["max_seq"], c["head_dim"] // 2))
    iq.rope_tables_dev(*tabs, c["head_dim"], c["max_seq"], c["rope_theta"])
    kvs = [new_cache(1, c["max_seq"], c["n_kv_heads"], c["head_dim"], *kvb)[0] for _ in range(c["n_layers"])]
    n, P = len(draft), len(prompt)
    first = _forward(c, w, prompt, range(P), range(P), chain(P), 0, kvs, tabs, kvb)
    logits = _forward(c, w, draft, [P + x for x in depth], range(P, P + n), parents, P, kvs, tabs, kvb)
    m = iq.Model(c)
    m.load(w)
    if kvb[0]:
        m.set_kv_packed(*kvb)
    for i, t in enumerate(prompt):
        lg = m.forward(t, i)[1]
        assert (first[i].cpu().numpy() == lg).all()
    for i, path in enumerate(ref.ancestors(parents)):
        for j, node in enumerate(path):
            lg = m.forward(draft[node], P + j)[1]
        assert (logits[i].cpu().numpy() == lg).all()
    m.close()
    tok = [int(x) for x in rng.integers(0, c["vocab"], n)]
    logp, ids, tl = full(n), torch.zeros(n, 4, dtype=torch.int32, device="cuda"), full(n, 4)
    iq.logprobs_dev(logits, n, c["vocab"], tokens=i32(tok), logp=logp, top=4, top_ids=ids, top_logp=tl)
    for i in range(n):
        lp, _, best, bl = ref.logprobs(logits[i].tolist(), tok[i], 4)
        assert (int(logp[i]), ids[i].tolist(), tl[i].tolist()) == (lp, best, bl)


# -------------------------------------------- other shapes and paths of the kernels

@pytest.mark.parametrize("nh,nkv,hd,n", [(8, 2, 128, 9), (8, 1, 192, 5), (16, 1, 64, 9), (24, 1, 32, 7), (3, 3, 160, 20)])
@pytest.mark.parametrize("kvb", [(0, 0), (7, 13)])
def test_tree_many_columns_a_kv_head(nh, nkv, hd, n, kvb):
    """Several blocks of columns over one set of keys, narrow and wide heads."""
    rng = np.random.default_rng(hd + n)
    check_tree(rng, nh, nkv, hd, [150, 20], [bush(rng, n), bush(rng, max(1, n // 2))], kvb)


def test_tree_unaligned_cache_and_queries():
    """Cache and query pointers on 8-byte boundaries only give the same results."""
    rng = np.random.default_rng(18)
    nh, nkv, hd, S, M = 8, 2, 64, 2, 75
    q, k, v = rnd(rng, 9, nh, hd), rnd(rng, S, M, nkv, hd), rnd(rng, S, M, nkv, hd)
    trees = [bush(rng, 4), bush(rng, 5)]
    args = ((0, 0), [70, 30], [0, 4, 9], trees[0] + trees[1], nh)
    want = run_tree(dev(q.reshape(9, -1)), dict(k=dev(k), v=dev(v)), *args)

    def shifted(a):
        buf = torch.empty(a.size + 1, dtype=torch.int64, device="cuda")
        buf[1:].copy_(dev(a).flatten())
        return buf[1:].view(a.shape)

    assert (run_tree(shifted(q.reshape(9, -1)), dict(k=shifted(k), v=shifted(v)), *args) == want).all()
    assert (run_tree(dev(q.reshape(9, -1)), dict(k=dev(k), v=shifted(v)), *args) == want).all()
    assert (want == ref.tree(q, list(k), list(v), [70, 30], [0, 4, 9], trees[0] + trees[1], nh).reshape(9, -1)).all()


def test_tree_batched_decode_over_several_tiles():
    """Many single tokens: a block of columns walks over several tiles of positions."""
    rng = np.random.default_rng(19)
    S, nh, nkv, hd, M = 150, 16, 8, 32, 1300
    lens = [int(x) for x in rng.integers(0, M - 1, S)]
    lens[:4] = [0, 127, 128, M - 1]
    k, v, q = rnd(rng, S, M, nkv, hd), rnd(rng, S, M, nkv, hd), rnd(rng, S, nh, hd)
    got = run_tree(dev(q.reshape(S, -1)), dict(k=dev(k), v=dev(v)), (0, 0), lens, list(range(S + 1)), [-1] * S, nh)
    scale = ref.fp(ref.INV_SQRT, hd << 48)
    for b in [0, 1, 2, 3, 77, 149]:
        for h in (0, 7, 15):
            want = ref.attend(q[b, h], k[b, : lens[b] + 1, h // 2], v[b, : lens[b] + 1, h // 2], scale)
            assert (got[b, h * hd:(h + 1) * hd] == want).all()


@pytest.mark.parametrize("vs", [7.99, 8.01, 63.0, 300.0])
def test_tree_large_values_everywhere(vs):
    """Every value near +-vs, wide tiles and several chunks of positions."""
    rng = np.random.default_rng(20)
    v = ref.q48(vs) * rng.choice([-1, 1], (1, 700, 2, 64)) + rng.integers(-1000, 1000, (1, 700, 2, 64))
    k = rnd(rng, 1, 700, 2, 64)
    check_tree(rng, 8, 2, 64, [690], [bush(rng, 3)], k=k, v=v, pad=7)


def test_logprobs_a_block_a_row():
    """Enough rows that each is one block's, rows longer than its shared memory, ties among them."""
    rng = np.random.default_rng(21)
    l = rnd(rng, 300, 6001, scale=3)
    l[7] = 5
    l[8, ::3] = l[8].max() + 1
    l[9] = ref.I64_MIN
    check_logprobs(l, rng.integers(0, 6001, 300), 4, ld=6002)


def test_wide_and_narrow_forms_agree():
    """Rotation and cache rows through 16-byte pieces and element by element (shifted pointers)."""
    rng = np.random.default_rng(22)
    rows, heads, hd, rot, n = 5, 3, 64, 48, 20
    x, cos, sin = rnd(rng, rows, heads * hd, scale=2000), rnd(rng, n, rot // 2), rnd(rng, n, rot // 2)
    x[0, :8] = [ref.I64_MAX, ref.I64_MIN, 1 << 60, -(1 << 60), (1 << 60) - 1, 0, 1, -1]
    cos[0, :3] = [1 << 49, (1 << 49) - 1, -(1 << 49)]
    pos = np.array([0, 1, 0, 19, 7])
    for layout in ("half", "interleaved"):
        r = iq.Rope(dev(cos), dev(sin), i32(pos), n, rot, layout)
        a, b = full(rows, heads * hd), torch.full((rows * heads * hd + 1,), KEEP, dtype=torch.int64, device="cuda")
        iq.rope_dev(a, dev(x), r, rows, heads, hd)
        iq.rope_dev(b[1:], dev(x), r, rows, heads, hd)
        want = ref.rotate(x.reshape(rows, heads, hd), cos[pos], sin[pos], rot, layout).reshape(rows, -1)
        assert (a.cpu().numpy() == want).all() and (b[1:].cpu().numpy().reshape(rows, -1) == want).all()


@pytest.mark.parametrize("nh,nkv,hd,n", [(16, 1, 128, 8), (16, 1, 96, 9), (24, 1, 64, 11), (32, 2, 32, 20), (12, 1, 120, 12)])
@pytest.mark.parametrize("kvb", [(0, 0), (8, 10)])
def test_tree_columns_that_share_values(nh, nkv, hd, n, kvb):
    """Enough columns a sequence that groups of them share a tile of values, ragged at the last group."""
    rng = np.random.default_rng(hd + n)
    check_tree(rng, nh, nkv, hd, [90, 33], [bush(rng, n), bush(rng, n - 3)], kvb, pad=5)


@pytest.mark.parametrize("kvb", [(0, 0), (8, 10)])
def test_cache_offsets_beyond_32_bits(kvb):
    """The last sequence of a cache whose element offsets (exact: byte offsets too) pass 32 bits."""
    rng = np.random.default_rng(23)
    kb, vb = kvb
    nkv, hd, M, nh, n, ln = 2, 256, 32767, 4, 3, 200
    S = (1 << (32 if kb else 31)) // (M * nkv * hd) + 2
    make = lambda dt, *tail: torch.empty((S, M, nkv) + tail, dtype=dt, device="cuda")
    t = (dict(kq=make(torch.uint8, hd), vq=make(torch.int16, hd), k_mag=make(torch.int64), v_mag=make(torch.int64))
         if kb else dict(k=make(torch.int64, hd), v=make(torch.int64, hd)))
    small, ts = new_cache(1, M, nkv, hd, kb, vb)
    big = iq.KVCache(S, M, nkv, hd, k_bits=kb, v_bits=vb, **t)
    rows = ln + n
    k, v = dev(rnd(rng, rows, nkv * hd)), dev(rnd(rng, rows, nkv * hd))
    slot = np.arange(rows)
    slot[-1] = M - 1                                  # the last vector of the cache
    iq.kv_write_dev(big, k, v, i32(slot), rows, seq=i32([S - 1] * rows))
    iq.kv_write_dev(small, k, v, i32(slot), rows)
    at = torch.from_numpy(slot).cuda()
    for name in t:
        assert (t[name][S - 1][at] == ts[name][0][at]).all()
    got, want = [full(rows, nkv * hd) for _ in range(2)], [full(rows, nkv * hd) for _ in range(2)]
    iq.kv_read_dev(*got, big, i32(slot), rows, seq=i32([S - 1] * rows))
    iq.kv_read_dev(*want, small, i32(slot), rows)
    assert all((a == b).all() for a, b in zip(got, want))
    q = dev(rnd(rng, 2, nh * hd, scale=1.5))
    args = (kvb, [ln], [0, 2], [-1, 0], nh)
    assert (run_tree(q, t, *args, seqs=[S - 1]) == run_tree(q, ts, *args)).all()


def test_strides_beyond_32_bits():
    """Rows of queries, of a rotation and of logits more than 2^32 elements apart."""
    rng = np.random.default_rng(24)
    nh, hd, V, st = 4, 64, 500, (1 << 32) + 2
    big = torch.empty(st + V, dtype=torch.int64, device="cuda")
    x = rnd(rng, 2, V, scale=2)
    for r in range(2):
        big[r * st:r * st + V].copy_(dev(x[r]))
    ids, tl, lp = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), full(2, 3), full(2)
    ids1, tl1, lp1 = ids.clone(), tl.clone(), lp.clone()
    iq.logprobs_dev(big, 2, V, i32([3, 499]), lp, None, 3, ids, tl, ld=st)
    iq.logprobs_dev(dev(x), 2, V, i32([3, 499]), lp1, None, 3, ids1, tl1)
    assert (ids == ids1).all() and (tl == tl1).all() and (lp == lp1).all()
    _, t = new_cache(1, 40, 2, hd, 0, 0)
    t["k"].copy_(dev(rnd(rng, 1, 40, 2, hd)))
    t["v"].copy_(dev(rnd(rng, 1, 40, 2, hd)))
    q = dev(np.ascontiguousarray(x[:, :nh * hd]))
    args = (t, (0, 0), [30], [0, 2], [-1, 0], nh)
    assert (run_tree(big, *args, q_stride=st, rows=2) == run_tree(q, *args)).all()
    cos, sin = dev(rnd(rng, 5, hd // 2)), dev(rnd(rng, 5, hd // 2))
    rope, want = iq.Rope(cos, sin, i32([4, 2]), 5, hd), full(2, nh * hd)
    iq.rope_dev(want, q, rope, 2, nh, hd)
    iq.rope_dev(big, big, rope, 2, nh, hd, x_stride=st, out_stride=st)
    assert all((big[r * st:r * st + nh * hd] == want[r]).all() for r in range(2))


@pytest.mark.parametrize("sq", [-1, -7, -(1 << 31)])
def test_tree_negative_cache_sequence_is_padding(sq):
    """Any negative sequence index leaves its rows as they were, silently, as the other operators' do."""
    rng = np.random.default_rng(25)
    t = dict(k=dev(rnd(rng, 1, 8, 1, 16)), v=dev(rnd(rng, 1, 8, 1, 16)))
    q = dev(rnd(rng, 2, 32))
    got = run_tree(q, t, (0, 0), [3, 4], [0, 1, 2], [-1, -1], 2, seqs=[0, sq])
    assert (got[1] == KEEP).all() and (got[0] == run_tree(q[:1], t, (0, 0), [3], [0, 1], [-1], 2)[0]).all()


# table values up to 2.0, where the halves of the fast products are largest; -2.0 and beyond are the general form's
NEAR_TWO = [2 * ONE - 1, 2 * ONE - (1 << 31), 2 * ONE - (1 << 31) - 1, 2 * ONE - (1 << 31) + 1, 2 * ONE - (1 << 32),
            -2 * ONE + 1, -2 * ONE + (1 << 31), -2 * ONE + (1 << 31) - 1, -2 * ONE, 2 * ONE, ONE + 11, 0]
NEAR_X = [1 << 59, (1 << 59) - 1, (1 << 59) - (1 << 31), -(1 << 59), -(1 << 59) - 1, -(1 << 59) + 1, (1 << 60) - 1,
          -(1 << 60), 1 << 60, (1 << 31) - 1, -(1 << 31), 3 * ONE]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("where", ["cos", "sin", "both"])
def test_rotation_by_table_values_near_two(layout, where):
    """Each value alone among ordinary ones, as either pair of its 16-byte piece, in the rotation and in written keys."""
    rng = np.random.default_rng(26)
    heads, hd, half = 2, 64, 32
    rows = n = 2 * len(NEAR_TWO)
    cos, sin = rnd(rng, n, half, scale=0.3), rnd(rng, n, half, scale=0.3)
    for i, c in enumerate(NEAR_TWO * 2):                  # position i: value i, in the first or the second pair
        at = slice(i // len(NEAR_TWO), None, 4)
        if where != "sin":
            cos[i, at] = c
        if where != "cos":
            sin[i, at] = c
    x = rnd(rng, rows, heads, hd, scale=3)
    x[:, 0, :12] = NEAR_X
    x[:, 0, 32:44] = NEAR_X[::-1]
    pos = rng.permutation(n)
    r = iq.Rope(dev(cos), dev(sin), i32(pos), n, hd, layout)
    want = ref.rotate(x, cos[pos], sin[pos], hd, layout)
    out = full(rows, heads * hd)
    iq.rope_dev(out, dev(x), r, rows, heads, hd)
    assert (out.cpu().numpy().reshape(want.shape) == want).all()
    for kb, vb in ((0, 0), (8, 10)):
        c, t = new_cache(1, rows, heads, hd, kb, vb)
        h = host_cache(t)
        iq.kv_write_dev(c, dev(x), dev(x), i32(range(rows)), rows, rope=r)
        write_ref(h, want, x, [0] * rows, range(rows), kb, vb)
        got = host_cache(t)
        for name in h:
            assert (got[name] == h[name]).all(), name


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("mscale", [2 * ONE, 2 * ONE - 1, 1024 * ONE])
def test_rotation_by_scaled_tables(mscale, layout):
    """Tables with a large factor on cos and sin, then rows rotated by them."""
    rng = np.random.default_rng(27)
    n, heads, hd = 4096, 2, 64
    cos, sin = full(n, hd // 2), full(n, hd // 2)
    iq.rope_tables_dev(cos, sin, hd, n, 10000, dict(mscale=mscale))
    pos = np.r_[0:24, rng.integers(0, n, 200)]
    c, s = ref.tables(hd, pos.tolist(), 10000, mscale=mscale)
    assert (cos[dev(pos)].cpu().numpy() == c).all() and (sin[dev(pos)].cpu().numpy() == s).all()
    x, out = rnd(rng, len(pos), heads, hd, scale=3), full(len(pos), heads * hd)
    iq.rope_dev(out, dev(x), iq.Rope(cos, sin, i32(pos), n, hd, layout), len(pos), heads, hd)
    assert (out.cpu().numpy().reshape(x.shape) == ref.rotate(x, c, s, hd, layout)).all()


@pytest.mark.parametrize("kb,vb", [(8, 10), (1, 1), (4, 16)])
@pytest.mark.parametrize("hd", [64, 256, 33])
def test_codes_of_the_lowest_value(hd, kb, vb):
    """INT64_MIN wraps below every magnitude: code 0 beside small elements, zeros and large ones, as K and as V, in
    16-byte pieces and element by element."""
    rng = np.random.default_rng(hd + kb)
    mags = [0, 1, 5, ONE, 3 * ONE, (1 << 61) - 1, 1 << 61, (1 << 62) - 1, ref.I64_MAX]
    rows, nkv = 2 * len(mags), 2
    x = np.zeros((rows, nkv, hd), np.int64)
    for i, m in enumerate(mags):
        x[2 * i:2 * i + 2] = rng.integers(-m, m, (2, nkv, hd), endpoint=True)
        x[2 * i:2 * i + 2, :, 0] = m
    for r in range(rows):                         # one in each lane's place in turn, and a few in one vector
        x[r, 0, 1 + 7 * r % (hd - 1)] = ref.I64_MIN
        x[r, 1, 1::5] = ref.I64_MIN
    for skip in (0, 1):
        buf = torch.empty(x.size + 1, dtype=torch.int64, device="cuda")
        d = buf[skip:x.size + skip]               # 16-byte aligned, and 8-byte aligned only
        d.copy_(dev(x).flatten())
        c, t = new_cache(1, rows, nkv, hd, kb, vb)
        h = host_cache(t)
        iq.kv_write_dev(c, d, d, i32(range(rows)), rows)
        write_ref(h, x, x, [0] * rows, range(rows), kb, vb)
        got = host_cache(t)
        for name in h:
            assert (got[name] == h[name]).all(), name


@pytest.mark.parametrize("kvb", [(0, 0), (8, 10)])
@pytest.mark.parametrize("nh,nkv,hd,S,n,rows", [(32, 4, 64, 4, 1, 64), (32, 4, 64, 1, 1, 1000), (8, 1, 64, 2, 1, 25),
                                                (4, 4, 64, 1, 2, 500), (32, 4, 32, 3, 1, 64), (32, 4, 128, 2, 1, 99),
                                                (16, 2, 64, 2, 3, 400), (8, 1, 256, 1, 1, 300)])
def test_tree_many_padding_rows(nh, nkv, hd, S, n, rows, kvb):
    """Many more rows than the sequences' nodes: a batch padded to a fixed size."""
    rng = np.random.default_rng(rows + hd)
    kb, vb = kvb
    lens, trees, M = [70 + 9 * i for i in range(S)], [bush(rng, n) for _ in range(S)], 120
    starts, parents = list(range(0, S * n + 1, n)), [x for p in trees for x in p]
    q, k, v = rnd(rng, rows, nh * hd), rnd(rng, S * M, nkv * hd), rnd(rng, S * M, nkv * hd)
    c, t = new_cache(S, M, nkv, hd, kb, vb)
    at = np.arange(S * M)
    iq.kv_write_dev(c, dev(k), dev(v), i32(at % M), S * M, seq=i32(at // M))
    kr, vr = full(S * M, nkv * hd), full(S * M, nkv * hd)
    iq.kv_read_dev(kr, vr, c, i32(at % M), S * M, seq=i32(at // M))
    got = run_tree(dev(q), t, kvb, lens, starts, parents + [-1] * (rows - S * n), nh)
    kr, vr = (list(x.cpu().numpy().reshape(S, M, nkv, hd)) for x in (kr, vr))
    want = ref.tree(q[:S * n].reshape(S * n, nh, hd), kr, vr, lens, starts, parents, nh)
    assert (got[:S * n] == want.reshape(S * n, -1)).all() and (got[S * n:] == KEEP).all()


def test_a_failed_call_is_not_reported_again():
    """An allocation that the device refuses fails its own call; the next call is answered for itself."""
    x = dev(np.zeros((1, 8), np.int64))
    rng = np.zeros((8192, 2), np.uint64)
    with pytest.raises(iq.IQError) as e:
        iq.sample_dev(x, 8192, (1 << 31) - 1, ONE, 0, 0, rng)     # 140 TB of work space: nothing is launched
    assert e.value.status == -3
    iq.softmax_dev(x, 1, 8)
    logp = full(1)
    iq.logprobs_dev(x, 1, 8, i32([3]), logp)
    assert int(logp[0]) == ref.logprobs([ONE // 8] * 8, 3, 0)[0]


def test_torch_default_stream_given_explicitly():
    """Calls on torch.cuda.default_stream() follow what torch has queued there, and torch follows them."""
    rng = np.random.default_rng(28)
    x = dev(rnd(rng, 2000, 4096))
    cos, sin, pos = dev(rnd(rng, 5, 32)), dev(rnd(rng, 5, 32)), i32([3] * 2000)
    want, out, y = full(2000, 4096), full(2000, 4096), torch.zeros_like(x)
    rope = iq.Rope(cos, sin, pos, 5, 64)
    iq.rope_dev(want, x, rope, 2000, 64, 64)
    torch.cuda.synchronize()
    s = torch.cuda.default_stream()
    for _ in range(20):
        y.zero_()
        for _ in range(8):
            y.add_(x, alpha=3)
        y.sub_(x, alpha=23)                 # 24 x - 23 x, last of ten passes over y
        iq.rope_dev(out, y, rope, 2000, 64, 64, stream=s)
        assert torch.equal(out, want)
        out.fill_(KEEP)
