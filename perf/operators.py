"""Cases and plain forms of the operators around drafted tokens and scoring.

Everything is Q16.48 (int64, 1.0 = 2^48), and every output is a whole number
that is defined exactly: rotary tables and rotation, cache rows written (exact
or as b-bit codes) and read back, attention of a tree of drafted tokens over
the cache, and log probabilities with entropy and top alternatives.

``run`` computes the plain forms in 64-bit integer torch operations, or, with
``own`` set, calls the library through its Python binding.
"""
import math
import os
import sys
from decimal import Decimal, getcontext

import numpy as np
import torch

own = False

ONE = 1 << 48
M24 = (1 << 24) - 1
_iq = None


def _lib():
    """The repository's binding, imported only for the library's calls."""
    global _iq
    if _iq is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "int-llm_b200"))
        import iq
        _iq = iq
    return _iq


# ------------------------------------------------------------------- cases

# Geometries: 32 heads over 4 kv heads of 64 and 32 over 32 of 128 are the
# repository's two model configurations, 8 over 2 of 32 its small test model.

def listed():
    return [
        # one decode row: rotate the q and k heads of a fused q|k|v row
        dict(name="rope decode row", op="rope", rows=1, heads=36, tail=4, hd=64, rot=64, layout="half", n_pos=2048),
        # a prefill chunk of the 128-wide heads, interleaved pairs, three quarters of the head rotated
        dict(name="rope prefill partial", op="rope", rows=2048, heads=64, tail=32, hd=128, rot=96,
             layout="interleaved", n_pos=8192),
        # tables of a context stretched beyond the trained one, positions past 32767
        dict(name="rope tables stretched", op="tables", n_pos=65536, rot=128, scale="parts", orig=2048),
        # a decode step of 64 sequences written as 8-bit keys and 10-bit values, keys rotated on the way
        dict(name="kv write decode batch", op="kv_write", rows=64, seqs=64, max_seq=512, heads=4, hd=64, rot=64,
             layout="half", k_bits=8, v_bits=10, n_pos=2048),
        # a prefill chunk of the 128-wide heads written as codes
        dict(name="kv write prefill", op="kv_write", rows=2048, seqs=2, max_seq=2112, heads=32, hd=128, rot=128,
             layout="half", k_bits=4, v_bits=16, n_pos=2112),
        # a whole packed sequence read back to int64
        dict(name="kv read sequence", op="kv_read", rows=2048, seqs=8, max_seq=2048, heads=4, hd=64, k_bits=8,
             v_bits=10),
        # one token over a short context: the latency of a single decode step
        dict(name="tree single token", op="tree", seqs=1, len_lo=384, len_hi=384, nodes_lo=1, nodes_hi=1, heads=32,
             kv_heads=4, hd=64, max_seq=2048, k_bits=0, v_bits=0),
        # a batch of single tokens over long contexts (batched decode)
        dict(name="tree decode batch", op="tree", seqs=64, len_lo=1900, len_hi=2047, nodes_lo=1, nodes_hi=1, heads=32,
             kv_heads=4, hd=64, max_seq=2112, k_bits=0, v_bits=0),
        # drafted trees of 16 to 48 tokens over long ragged contexts
        dict(name="tree drafts", op="tree", seqs=8, len_lo=1100, len_hi=2000, nodes_lo=16, nodes_hi=48, heads=32,
             kv_heads=4, hd=64, max_seq=2112, k_bits=0, v_bits=0),
        # drafted trees over the packed cache, 128-wide heads, one kv head a query head
        dict(name="tree drafts packed", op="tree", seqs=2, len_lo=1501, len_hi=2001, nodes_lo=13, nodes_hi=25,
             heads=32, kv_heads=32, hd=128, max_seq=2112, k_bits=8, v_bits=10),
        # the token just decoded, with 5 alternatives
        dict(name="logprobs one row", op="logprobs", rows=1, vocab=32000, top=5),
        # scoring a prompt: every row's given token, entropy and 8 alternatives
        dict(name="logprobs prompt", op="logprobs", rows=512, vocab=32000, top=8),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "tables", "kv_write", "kv_read", "tree", "tree", "logprobs", "logprobs"])
    if op == "rope":
        hd = 2 * _log(rng, 8, 64)
        return dict(op=op, rows=_log(rng, 1, 2048), heads=_log(rng, 1, 48), tail=rng.choice([0, 1, 3, 4]), hd=hd,
                    rot=2 * rng.randint(1, hd // 2), layout=rng.choice(["half", "interleaved"]), n_pos=4096)
    if op == "tables":
        return dict(op=op, n_pos=_log(rng, 64, 65536), rot=2 * rng.randint(2, 64),
                    scale=rng.choice(["none", "linear", "ntk", "parts"]), orig=rng.choice([2048, 4096]))
    if op in ("kv_write", "kv_read"):
        hd = 2 * _log(rng, 8, 64)
        seqs = _log(rng, 1, 32)
        c = dict(op=op, rows=0, seqs=seqs, max_seq=rng.randint(65, 1200), heads=_log(rng, 1, 16), hd=hd,
                 k_bits=rng.randint(1, 8), v_bits=rng.randint(1, 16))
        c["rows"] = min(_log(rng, 1, 2048), seqs * c["max_seq"])
        if op == "kv_write":
            c.update(rot=2 * rng.randint(0, hd // 2), layout=rng.choice(["half", "interleaved"]), n_pos=2048)
        return c
    if op == "tree":
        grp = rng.choice([1, 2, 3, 4, 7, 8])
        kvh = _log(rng, 1, 8)
        seqs = _log(rng, 1, 8)
        hi = _log(rng, 1, 1200)
        nodes = _log(rng, 1, 48)
        packed = rng.random() < 0.4
        c = dict(op=op, seqs=seqs, len_lo=rng.randint(0, hi), len_hi=hi, nodes_lo=rng.randint(1, nodes),
                 nodes_hi=nodes, heads=grp * kvh, kv_heads=kvh, hd=rng.choice([16, 32, 40, 64, 96, 128]),
                 max_seq=hi + nodes + rng.randint(0, 100), k_bits=rng.randint(1, 8) if packed else 0,
                 v_bits=rng.randint(1, 16) if packed else 0)
        # no dearer than the largest listed case (its plain form holds every product)
        most = 600_000_000
        while c["seqs"] * c["nodes_hi"] * c["heads"] * (c["len_hi"] + c["nodes_hi"]) * c["hd"] > most:
            c["nodes_hi"] = max(1, c["nodes_hi"] // 2)
            c["nodes_lo"] = min(c["nodes_lo"], c["nodes_hi"])
            if c["nodes_hi"] == 1 and c["seqs"] > 1:
                c["seqs"] //= 2
            elif c["nodes_hi"] == 1:
                c["len_hi"] //= 2
                c["len_lo"] = min(c["len_lo"], c["len_hi"])
        return c
    vocab = _log(rng, 300, 131072)
    return dict(op=op, rows=min(_log(rng, 1, 512), 16_000_000 // vocab), vocab=vocab, top=rng.randint(0, 32))


def _spread(lo, hi, n):
    """n sizes from lo to hi, the same for every seed."""
    return [lo + (hi - lo) * ((i * 7) % n) // max(1, n - 1) for i in range(n)]


# ------------------------------------------------------------------ inputs

def _q48(t):
    return (t * float(ONE)).to(torch.int64)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dev = dict(device="cuda", generator=g)

    def normal(*shape, std=1.0):
        return _q48(torch.randn(*shape, dtype=torch.float64, **dev) * std)

    def tables(n_pos, half):
        # angles as a model has them: one frequency a pair, theta = 10000
        f = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / max(1, half))
        a = torch.arange(n_pos, dtype=torch.float64, device="cuda")[:, None] * f
        return _q48(torch.cos(a)), _q48(torch.sin(a))

    s = dict(case)
    op = case["op"]
    if op == "rope":
        rows, heads, hd = case["rows"], case["heads"], case["hd"]
        s["x"] = normal(rows, (heads + case["tail"]) * hd)
        s["cos"], s["sin"] = tables(case["n_pos"], case["rot"] // 2)
        s["pos"] = torch.randint(0, case["n_pos"], (rows,), dtype=torch.int32, **dev)
    elif op == "tables":
        r = np.random.RandomState(seed & 0x7fffffff)
        s["theta"] = int(r.randint(5000, 500000))
        s["factor"] = int(r.randint(2 * 256, 16 * 256)) * (ONE // 256)
    elif op in ("kv_write", "kv_read"):
        rows, kvh, hd, seqs, max_seq = (case[k] for k in ("rows", "heads", "hd", "seqs", "max_seq"))
        kq = torch.zeros(seqs, max_seq, kvh, hd, dtype=torch.uint8, device="cuda")
        vq = torch.zeros(seqs, max_seq, kvh, hd, dtype=torch.int16, device="cuda")
        km = torch.zeros(seqs, max_seq, kvh, dtype=torch.int64, device="cuda")
        vm = torch.zeros_like(km)
        at = torch.randperm(seqs * max_seq, **dev)[:rows]
        s["seq"], s["slot"] = (at // max_seq).to(torch.int32), (at % max_seq).to(torch.int32)
        if op == "kv_write":
            s["kv"] = normal(rows, 2 * kvh * hd)
            s["cos"], s["sin"] = tables(case["n_pos"], max(1, case["rot"] // 2))
            s["pos"] = torch.randint(0, case["n_pos"], (rows,), dtype=torch.int32, **dev)
        else:
            kq.random_(0, 1 << case["k_bits"], generator=g)
            vq.copy_(torch.randint(0, 1 << case["v_bits"], vq.shape, **dev))
            km.copy_(_q48(torch.rand(km.shape, dtype=torch.float64, **dev) * 4))
            vm.copy_(_q48(torch.rand(vm.shape, dtype=torch.float64, **dev) * 4))
        s.update(kq=kq, vq=vq, km=km, vm=vm)
    elif op == "tree":
        seqs, heads, kvh, hd, max_seq = (case[k] for k in ("seqs", "heads", "kv_heads", "hd", "max_seq"))
        lens = _spread(case["len_lo"], case["len_hi"], seqs)
        nodes = _spread(case["nodes_lo"], case["nodes_hi"], seqs)
        rows = sum(nodes)
        r = np.random.RandomState(seed & 0x7fffffff)
        parents, starts = [], [0]
        for n in nodes:
            # a drafted tree: each node hangs on one of the last few, some on the root
            parents += [-1 if i == 0 or r.rand() < 0.1 else int(r.randint(max(0, i - 6), i)) for i in range(n)]
            starts.append(starts[-1] + n)
        i32 = dict(dtype=torch.int32, device="cuda")
        s["lens"], s["starts"] = torch.tensor(lens, **i32), torch.tensor(starts, **i32)
        s["parents"] = torch.tensor(parents, **i32)
        s["rows"], s["max_nodes"] = rows, max(nodes)
        s["max_len"] = max(a + b for a, b in zip(lens, nodes))
        s["q"] = normal(rows, heads * hd, std=1.5)
        if case["k_bits"]:
            shape = (seqs, max_seq, kvh, hd)
            s["kq"] = torch.randint(0, 1 << case["k_bits"], shape, dtype=torch.uint8, **dev)
            s["vq"] = torch.randint(0, 1 << case["v_bits"], shape, dtype=torch.int32, **dev).to(torch.int16)
            s["km"] = _q48(2 + torch.rand(shape[:3], dtype=torch.float64, **dev))
            s["vm"] = _q48(2 + torch.rand(shape[:3], dtype=torch.float64, **dev))
        else:
            s["k"] = normal(seqs, max_seq, kvh, hd)
            s["v"] = normal(seqs, max_seq, kvh, hd)
        # the row of each (sequence, node), and `rows` where there is none
        at = np.full((seqs, max(nodes)), rows)
        for i, n in enumerate(nodes):
            at[i, :n] = np.arange(starts[i], starts[i] + n)
        s["row_at"] = torch.tensor(at, device="cuda")
        s["of_row"] = torch.tensor([i * max(nodes) + j for i, n in enumerate(nodes) for j in range(n)], device="cuda")
    else:
        s["logits"] = normal(case["rows"], case["vocab"], std=2.5)
        s["tokens"] = torch.randint(0, case["vocab"], (case["rows"],), dtype=torch.int32, **dev)
    return s


# ------------------------------------------------- arithmetic, in int64 torch

def _mul(a, b):
    """floor(a b / 2^48) mod 2^64, from 24-bit low and 40-bit high parts."""
    a1, a0, b1, b0 = a >> 24, a & M24, b >> 24, b & M24
    m1, m2 = a1 * b0, a0 * b1
    low = (m1 & M24) + (m2 & M24) + (a0 * b0 >> 24)
    return a1 * b1 + (m1 >> 24) + (m2 >> 24) + (low >> 24)


def _div(a, b, bits=48):
    """floor(a 2^bits / b) for 0 <= a, 0 < b < 2^62.5 and quotients below 2^50: a
    64-bit float's estimate, corrected by its exact remainder (mod 2^64)."""
    q = (a.double() * float(1 << bits) / b.double()).to(torch.int64)
    r = (a << bits) - q * b
    return q + (r >= b).to(torch.int64) - (r < 0).to(torch.int64)


def _exp_neg(d):
    """fp_exp(-d) for 0 <= d <= 10: 1 / (1 + d / 2^14)^(2^14) by 14 squarings."""
    r = ONE + (d >> 14)
    for _ in range(14):
        r = _mul(r, r)
    return _div(torch.full_like(r, ONE), r)


def _c(t, dev):
    return torch.tensor(t, dtype=torch.int64, device=dev)


# rotary tables: frequencies fp_exp(-(2 i / rot) ln theta), angles mod 2 pi, CORDIC

def _fmul(a, b):
    return ((a * b >> 48) + (1 << 63)) % (1 << 64) - (1 << 63)


def _fexp(x):
    if x >= 0:
        r = ONE + (x >> 14)
        for _ in range(14):
            r = _fmul(r, r)
        return r
    p = _fexp(-x)
    return ONE * ONE // p if p else 0


LN2 = 195103586505167


def _flog(x):
    y = (x.bit_length() - 49) * LN2
    for _ in range(10):
        e = _fexp(y)
        if e == 0:
            break
        n = y - ONE + (x << 48) // e
        if abs(n - y) < 2:
            break
        y = n
    return y


def _fsqrt(x):
    return math.isqrt(x << 48)


def _atan(x, terms):
    x2, t, s = _fmul(x, x), x, x
    for n in range(1, terms + 1):
        t = -_fmul(t, x2)
        c = abs(t) // (2 * n + 1) * (1 if t >= 0 else -1)
        if c == 0:
            break
        s += c
    return s


PI = (_atan(ONE // 5, 40) << 4) - (_atan(ONE // 239, 15) << 2)
ANGLES = [PI >> 2] + [_atan(ONE >> i, 40) if i < 25 else ONE >> i for i in range(1, 48)]


def _gain():
    k = ONE
    for i in range(48):
        k = _fmul(k, ONE + (ONE >> (2 * i) if 2 * i < 63 else 0))
    return (ONE << 48) // _fsqrt(k)


GAIN = _gain()


def _fln_int(theta):
    """ln of a whole number, shifted into fp_log's range where it leaves it."""
    k = max(0, theta.bit_length() - 14)
    return _flog((theta << 48) >> k) + k * LN2


def _freqs(case, theta, factor):
    """One frequency a pair, scaled for long contexts."""
    rot, kind = case["rot"], case["scale"]
    lt = _fln_int(theta)
    if kind == "ntk":
        lt += _fmul(_flog(factor), (rot << 48) // (rot - 2))
    out = []
    for i in range(rot // 2):
        y = _fmul(-((2 * i << 48) // rot), lt)
        if y < -10 * ONE:
            th = _fexp(y >> 1)
            th = _fmul(th, th)
        else:
            th = _fexp(y)
        if kind == "linear":
            th = (th << 48) // factor
        elif kind == "parts":
            # turns over the trained length: below 1 fully scaled, above 32 as trained
            turns = (case["orig"] * th << 48) // (2 * PI)
            t = min(max(turns - ONE, 0), 31 * ONE)
            w = t // 31
            th = _fmul(th, w) + _fmul((th << 48) // factor, ONE - w)
        out.append(th)
    return out


def _plain_tables(s):
    th = _c(_freqs(s, s["theta"], s["factor"]), "cuda")
    p = torch.arange(s["n_pos"], device="cuda")[:, None]
    w = 2 * PI
    n = (p.double() * th.double() / w).to(torch.int64)
    a = p * th - n * w            # wrapped products: the difference is small and exact
    a = torch.where(a < 0, a + w, torch.where(a >= w, a - w, a))
    a = torch.where(a > PI, a - w, a)
    neg = (a > (PI >> 1)) | (a < -(PI >> 1))
    z = torch.where(a > (PI >> 1), PI - a, torch.where(a < -(PI >> 1), -PI - a, a))
    x, y = torch.full_like(z, GAIN), torch.zeros_like(z)
    for i in range(48):
        up, xs, ys = z >= 0, x >> i, y >> i
        x, y = torch.where(up, x - ys, x + ys), torch.where(up, y + xs, y - xs)
        z = torch.where(up, z - ANGLES[i], z + ANGLES[i])
    return {"cos": torch.where(neg, -x, x), "sin": y}


def _rotate(x, cos, sin, pos, rot, layout):
    """x [rows, heads, hd] with the first `rot` elements of each head rotated."""
    c, n = cos[pos.long()][:, None], sin[pos.long()][:, None]
    r = x[..., :rot]
    a, b = (r[..., : rot // 2], r[..., rot // 2:]) if layout == "half" else (r[..., 0::2], r[..., 1::2])
    u, w = _mul(a, c) - _mul(b, n), _mul(b, c) + _mul(a, n)
    turned = torch.cat([u, w], -1) if layout == "half" else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_rope(s):
    x = s["x"].view(s["rows"], -1, s["hd"])[:, : s["heads"]]
    return {"out": _rotate(x, s["cos"], s["sin"], s["pos"], s["rot"], s["layout"])}


# the cache: magnitude and b-bit codes per (position, head) vector

def _codes(x, bits):
    m = x.abs().amax(-1)
    d = (2 * m)[..., None].clamp(min=1)
    q = _div(x + m[..., None], d.expand_as(x), bits).clamp(0, (1 << bits) - 1)
    return torch.where(m[..., None] == 0, 0, q), m


def _values(q, m, bits):
    """floor((2 q + 1) m / 2^bits) - m"""
    c, m = 2 * q + 1, m[..., None]
    return ((c * (m >> 24)) << (24 - bits)) + (c * (m & M24) >> bits) - m


def _plain_kv_write(s):
    kv = s["kv"].view(s["rows"], 2, s["heads"], s["hd"])
    k, v = kv[:, 0], kv[:, 1]
    if s["rot"]:
        k = _rotate(k, s["cos"], s["sin"], s["pos"], s["rot"], s["layout"])
    at = (s["seq"].long(), s["slot"].long())
    kc, km = _codes(k, s["k_bits"])
    vc, vm = _codes(v, s["v_bits"])
    s["kq"][at], s["km"][at] = kc.to(torch.uint8), km
    s["vq"][at], s["vm"][at] = vc.to(torch.int16), vm
    return {n: s[n] for n in ("kq", "km", "vq", "vm")}


def _plain_kv_read(s):
    at = (s["seq"].long(), s["slot"].long())
    return {"k": _values(s["kq"][at].long(), s["km"][at], s["k_bits"]),
            "v": _values(s["vq"][at].long() & 0xffff, s["vm"][at], s["v_bits"])}


# attention of a tree of drafted tokens

def _finv_sqrt(x):
    """fp_inv_sqrt: 8 Newton steps on the value scaled into [0.5, 2)."""
    k = (x.bit_length() - 49) >> 1
    n = x >> (2 * k) if k >= 0 else x << (-2 * k)
    y = ONE if n.bit_length() == 49 else ONE >> 1
    for _ in range(8):
        y = y * (3 * ONE - _fmul(n, _fmul(y, y))) >> 49
    return y >> k if k >= 0 else y << -k


def _limbs(x):
    """x = l0 + l1 2^22 + l2 2^44 as 64-bit floats (l2 signed)."""
    m = (1 << 22) - 1
    return [t.double() for t in (x & m, (x >> 22) & m, x >> 44)]


def _plain_tree(s):
    S, H, G, hd = s["seqs"], s["heads"], s["kv_heads"], s["hd"]
    N, T, grp = s["max_nodes"], s["max_len"], s["heads"] // s["kv_heads"]
    if s["k_bits"]:
        k = _values(s["kq"][:, :T].long(), s["km"][:, :T], s["k_bits"])
        v = _values(s["vq"][:, :T].long() & 0xffff, s["vm"][:, :T], s["v_bits"])
    else:
        k, v = s["k"][:, :T], s["v"][:, :T]
    k, v = k.transpose(1, 2), v.transpose(1, 2)                                  # [S, G, T, hd]
    q = torch.cat([s["q"], torch.zeros_like(s["q"][:1])])[s["row_at"]]           # [S, N, H hd]
    q = q.view(S, N, G, grp, hd).permute(0, 2, 3, 1, 4).reshape(S, G, grp * N, hd)
    # ancestors of each node, itself among them
    par = torch.cat([s["parents"], s["parents"].new_full((1,), -1)])[s["row_at"]].long()
    node = torch.arange(N, device="cuda")
    anc = ((par[..., None] == node) | (node[:, None] == node)).double()
    for _ in range(max(1, N.bit_length())):
        anc = (anc @ anc > 0).double()
    t = torch.arange(T, device="cuda")
    ln, j = s["lens"].long()[:, None], t - s["lens"].long()[:, None]             # [S, T]
    drafted = torch.gather(anc, 2, j.clamp(0, N - 1)[:, None].expand(S, N, T)) > 0
    see = (t < ln)[:, None] | (drafted & ((j >= 0) & (j < N))[:, None])          # [S, N, T]
    see = see[:, None, None].expand(S, G, grp, N, T).reshape(S, G, grp * N, T)
    # q . k exactly: 22-bit limbs, each product sum below 2^53
    c = [0] * 5
    kl = [x.transpose(2, 3) for x in _limbs(k)]
    for i, x in enumerate(_limbs(q)):
        for n, y in enumerate(kl):
            c[i + n] = c[i + n] + (x @ y).to(torch.int64)
    dot = ((((c[0] >> 22) + c[1]) >> 22) + c[2] >> 4) + (c[3] << 18) + (c[4] << 40)
    sc = _mul(dot, _c(_finv_sqrt(hd << 48), "cuda"))
    top = torch.where(see, sc, -(1 << 63)).amax(-1, keepdim=True)
    d = top - sc
    live = see & (d <= 10 * ONE)
    e = torch.where(live, _exp_neg(torch.where(live, d, 0)), 0)
    p = _div(e, e.sum(-1, keepdim=True).clamp(min=1).expand_as(e))
    o = _mul(p[..., None], v[:, :, None]).sum(-2)                                # [S, G, grp N, hd]
    o = o.view(S, G, grp, N, hd).permute(0, 3, 1, 2, 4).reshape(S * N, H * hd)
    return {"out": o[s["of_row"]]}


# log probabilities

getcontext().prec = 60
_ln2 = Decimal(2).ln()
LOG2E_60 = int((1 / _ln2 * (1 << 60)).to_integral_value())
LN2_60 = int((_ln2 * (1 << 60)).to_integral_value())
POW = [int(((-_ln2 * j / 64).exp() * ONE).to_integral_value()) for j in range(64)]
COEF = [int((_ln2 ** k / math.factorial(k) * ONE).to_integral_value()) for k in range(6)]


def _exp_tail(d):
    """e^-d in Q48 without a cut-off: 2^-k times a table of 64 powers times a
    polynomial of degree 5, each product floored; 0 from d = 34 on."""
    far = (d < 0) | (d >= 34 * ONE)
    d = torch.where(far, 0, d)
    m30 = (1 << 30) - 1
    a1, a0, b1, b0 = d >> 30, d & m30, LOG2E_60 >> 30, LOG2E_60 & m30
    y = a1 * b1 + (a1 * b0 + a0 * b1 + (a0 * b0 >> 30) >> 30)
    f, k = y & (ONE - 1), y >> 48
    r = f & ((1 << 42) - 1)
    h = torch.full_like(r, COEF[5])
    for c in COEF[4::-1]:
        h = c - _mul(h, r)
    e = _mul(_c(POW, d.device)[f >> 42], h) >> k
    return torch.where(far, 0, e)


def _bit_length(x):
    n = torch.zeros_like(x)
    for b in (32, 16, 8, 4, 2, 1):
        up = (x >> b) > 0
        n, x = n + b * up, torch.where(up, x >> b, x)
    return n + (x > 0)


def _wide(x):
    """Sum over the row of non-negative values, as (high, low 24 bits)."""
    hi, lo = (x >> 24).sum(-1), (x & M24).sum(-1)
    return hi + (lo >> 24), lo & M24


def _shift(hi, lo, n):
    """(hi 2^24 + lo) 2^-n, floored, for -38 <= n <= 24."""
    down = n.clamp(min=0)
    both = torch.where(n > 0, (hi << (24 - down)) | (lo >> down), (hi << 24) | lo)
    return both << (-n).clamp(min=0)


def _ln_wide(hi, lo):
    """ln(S / 2^48) in Q48: 50 bits of log2 by repeated squaring, times ln 2."""
    bl = 24 + _bit_length(hi)
    y, z = _shift(hi, lo, bl - 62), torch.zeros_like(hi)
    m31 = (1 << 31) - 1
    for _ in range(50):
        y1, y0 = y >> 31, y & m31
        y = 2 * y1 * y1 + (2 * y1 * y0 + (y0 * y0 >> 31) >> 30)
        bit = y >> 62
        z, y = 2 * z + bit, y >> bit
    a = (bl - 49 << 50) + z
    a1, a0, b1, b0 = a >> 31, a & m31, LN2_60 >> 31, LN2_60 & m31
    return a1 * b1 + (a1 * b0 + a0 * b1 + (a0 * b0 >> 31) >> 31)


def _plain_logprobs(s):
    lg, tok, top = s["logits"], s["tokens"].long(), s["top"]
    m = lg.amax(-1, keepdim=True)
    d = m - lg
    e = _exp_tail(d)
    sh, sl = _wide(e)
    ah, al = _wide(torch.where(e > 0, _mul(e, d), 0))
    z = _ln_wide(sh, sl)
    n = (24 + _bit_length(torch.maximum(sh, ah)) - 61).clamp(min=0)
    a, b = _shift(ah, al, n), _shift(sh, sl, n)
    whole = a // b
    h = z + (whole << 48) + _div(a - whole * b, b)
    low = -(1 << 63)

    def lp(x):
        return torch.where(x < 0, low, torch.where(x > (1 << 63) - 1 - z[:, None], low, -x - z[:, None]))

    v, i = torch.sort(lg, dim=-1, descending=True, stable=True)
    return {"logp": lp(torch.gather(d, 1, tok[:, None]))[:, 0], "entropy": h,
            "top_ids": i[:, :top].to(torch.int32), "top_logp": lp(m - v[:, :top])}


# --------------------------------------------------------------------- run

def _own_run(s):
    iq, op = _lib(), s["op"]
    new = dict(dtype=torch.int64, device="cuda")
    if op == "tables":
        half = s["rot"] // 2
        cos, sin = torch.empty(s["n_pos"], half, **new), torch.empty(s["n_pos"], half, **new)
        sc = dict(kind=s["scale"], factor=s["factor"], orig_len=s["orig"], low=ONE, high=32 * ONE)
        iq.rope_tables_dev(cos, sin, s["rot"], s["n_pos"], s["theta"], sc)
        return {"cos": cos, "sin": sin}
    if op == "rope":
        out = torch.empty(s["rows"], s["heads"], s["hd"], **new)
        rope = iq.Rope(s["cos"], s["sin"], s["pos"], s["n_pos"], s["rot"], s["layout"])
        iq.rope_dev(out, s["x"], rope, s["rows"], s["heads"], s["hd"], x_stride=s["x"].stride(0))
        return {"out": out}
    if op in ("kv_write", "kv_read"):
        w = s["heads"] * s["hd"]
        cache = iq.KVCache(s["seqs"], s["max_seq"], s["heads"], s["hd"], kq=s["kq"], vq=s["vq"], k_mag=s["km"],
                           v_mag=s["vm"], k_bits=s["k_bits"], v_bits=s["v_bits"])
        if op == "kv_write":
            rope = iq.Rope(s["cos"], s["sin"], s["pos"], s["n_pos"], s["rot"], s["layout"]) if s["rot"] else None
            iq.kv_write_dev(cache, s["kv"], s["kv"][:, w:], s["slot"], s["rows"], seq=s["seq"], rope=rope,
                            k_stride=2 * w, v_stride=2 * w)
            return {n: s[n] for n in ("kq", "km", "vq", "vm")}
        k, v = torch.empty(s["rows"], s["heads"], s["hd"], **new), torch.empty(s["rows"], s["heads"], s["hd"], **new)
        iq.kv_read_dev(k, v, cache, s["slot"], s["rows"], seq=s["seq"])
        return {"k": k, "v": v}
    if op == "tree":
        packed = dict(kq=s["kq"], vq=s["vq"], k_mag=s["km"], v_mag=s["vm"], k_bits=s["k_bits"], v_bits=s["v_bits"]) \
            if s["k_bits"] else dict(k=s["k"], v=s["v"])
        cache = iq.KVCache(s["seqs"], s["max_seq"], s["kv_heads"], s["hd"], **packed)
        size = dict(n_seq=s["seqs"], rows=s["rows"], max_nodes=s["max_nodes"], max_len=s["max_len"])
        if "work" not in s:      # a program keeps its workspace
            n = iq.attn_tree_work(cache, s["heads"], **size)
            s["work"] = torch.empty(max(1, n), dtype=torch.uint8, device="cuda")
        out = torch.empty(s["rows"], s["heads"] * s["hd"], **new)
        iq.attn_tree_dev(out, s["q"], cache, s["heads"], s["lens"], s["starts"], s["parents"], work=s["work"], **size)
        return {"out": out}
    rows, top = s["rows"], s["top"]
    i32 = dict(dtype=torch.int32, device="cuda")
    logp, ent = torch.empty(rows, **new), torch.empty(rows, **new)
    ids, tl = torch.empty(rows, top, **i32), torch.empty(rows, top, **new)
    iq.logprobs_dev(s["logits"], rows, s["vocab"], tokens=s["tokens"], logp=logp, entropy=ent, top=top,
                    top_ids=ids, top_logp=tl)
    return {"logp": logp, "entropy": ent, "top_ids": ids, "top_logp": tl}


def run(state):
    if own:
        return _own_run(state)
    return {"rope": _plain_rope, "tables": _plain_tables, "kv_write": _plain_kv_write, "kv_read": _plain_kv_read,
            "tree": _plain_tree, "logprobs": _plain_logprobs}[state["op"]](state)


def work(case):
    op = case["op"]
    if op == "rope":
        n = case["rows"] * case["heads"] * case["hd"]
        pairs = case["rows"] * case["heads"] * case["rot"] // 2
        return {"bytes": 16 * n + 8 * case["rows"] * case["rot"], "flops": 6 * pairs}
    if op == "tables":
        n = case["n_pos"] * case["rot"] // 2
        return {"bytes": 16 * n, "flops": 48 * 5 * n}
    if op in ("kv_write", "kv_read"):
        n = case["rows"] * case["heads"] * case["hd"]
        return {"bytes": 2 * 8 * n + 3 * n + 16 * case["rows"] * case["heads"], "flops": 6 * n}
    if op == "tree":
        lens = _spread(case["len_lo"], case["len_hi"], case["seqs"])
        nodes = _spread(case["nodes_lo"], case["nodes_hi"], case["seqs"])
        ctx = sum(a + b for a, b in zip(lens, nodes))
        cells = sum((a + b) * b for a, b in zip(lens, nodes)) * case["heads"]
        one = 16 if not case["k_bits"] else 3
        return {"bytes": ctx * case["kv_heads"] * case["hd"] * one + 16 * sum(nodes) * case["heads"] * case["hd"],
                "flops": 4 * cells * case["hd"]}
    n = case["rows"] * case["vocab"]
    return {"bytes": 8 * n + case["rows"] * (20 + 12 * case["top"]), "flops": 30 * n}


# ---------------------------------------------------- exact, in Python's whole numbers

def _i64(x):
    return (int(x) + (1 << 63)) % (1 << 64) - (1 << 63)


def _ints(t):
    return np.array(t.cpu().tolist(), dtype=object)


def _wrap(a):
    return np.array([_i64(x) for x in np.ravel(a)], dtype=np.int64).reshape(np.shape(a))


def _x_rotate(x, cos, sin, pos, rot, layout):
    x = x.copy()
    for r in range(x.shape[0]):
        c, n = cos[pos[r]][None], sin[pos[r]][None]
        i, j = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
        a, b = x[r][:, i].copy(), x[r][:, j].copy()
        x[r][:, i], x[r][:, j] = (a * c >> 48) - (b * n >> 48), (b * c >> 48) + (a * n >> 48)
    return x


def _x_exp(d):
    """1 / (1 + d 2^-14)^(2^14), floored at each step, for 0 <= d <= 10."""
    r = ONE + (d >> 14)
    for _ in range(14):
        r = r * r >> 48
    return (1 << 96) // r


def _x_value(q, m, bits):
    return ((2 * q + 1) * m >> bits) - m


def _x_tail(d):
    if d >= 34 << 48:
        return 0
    y = d * LOG2E_60 >> 60
    f, k = y % ONE, y // ONE
    r, h = f % (1 << 42), COEF[5]
    for c in (COEF[4], COEF[3], COEF[2], COEF[1], COEF[0]):
        h = c - (h * r >> 48)
    return (POW[f >> 42] * h >> 48) >> k


def _x_ln(s):
    bl = s.bit_length()
    y, z = (s << 62 - bl if bl <= 62 else s >> bl - 62), 0
    for _ in range(50):
        y = y * y >> 61
        z, y = 2 * z + (y >> 62), y >> (y >> 62)
    return ((bl - 49 << 50) + z) * LN2_60 >> 62


def _size(case):
    op = case["op"]
    if op == "tables":
        return 60 * case["n_pos"] * case["rot"]
    if op == "tree":
        return work(case)["flops"] // 2 + case["seqs"] * case["max_seq"] * case["kv_heads"] * case["hd"]
    return work(case)["flops"] + case.get("seqs", 0) * case.get("max_seq", 0) * case["heads"] * case["hd"] // 4 \
        if op != "logprobs" else work(case)["flops"]


def exact(case, seed):
    if _size(case) > 16_000_000:
        return None
    s, op = prepare(case, seed), case["op"]
    if op == "tables":
        th = _freqs(case, s["theta"], s["factor"])
        cs, sn = np.zeros((case["n_pos"], len(th)), np.int64), np.zeros((case["n_pos"], len(th)), np.int64)
        for p in range(case["n_pos"]):
            for i, f in enumerate(th):
                a = p * f % (2 * PI)
                a -= 2 * PI if a > PI else 0
                far = abs(a) > PI >> 1 if a >= 0 else a < -(PI >> 1)
                z, x, y = (PI - a if a > 0 else -PI - a) if far else a, GAIN, 0
                for n in range(48):
                    x, y, z = (x - (y >> n), y + (x >> n), z - ANGLES[n]) if z >= 0 else \
                        (x + (y >> n), y - (x >> n), z + ANGLES[n])
                cs[p, i], sn[p, i] = -x if far else x, y
        return {"cos": cs, "sin": sn}
    if op == "rope":
        x = _ints(s["x"]).reshape(case["rows"], -1, case["hd"])[:, : case["heads"]]
        return {"out": _wrap(_x_rotate(x, _ints(s["cos"]), _ints(s["sin"]), s["pos"].tolist(), case["rot"],
                                       case["layout"]))}
    if op == "kv_write":
        kv = _ints(s["kv"]).reshape(case["rows"], 2, case["heads"], case["hd"])
        k = _x_rotate(kv[:, 0], _ints(s["cos"]), _ints(s["sin"]), s["pos"].tolist(), case["rot"], case["layout"]) \
            if case["rot"] else kv[:, 0]
        out = {n: s[n].cpu().numpy().copy() for n in ("kq", "km", "vq", "vm")}
        for r, (b, t) in enumerate(zip(s["seq"].tolist(), s["slot"].tolist())):
            for x, q, m, bits in ((k, "kq", "km", case["k_bits"]), (kv[:, 1], "vq", "vm", case["v_bits"])):
                for h in range(case["heads"]):
                    top = max(abs(v) for v in x[r, h])
                    out[m][b, t, h] = top
                    code = [min((1 << bits) - 1, (v + top << bits) // (2 * top)) if top else 0 for v in x[r, h]]
                    out[q][b, t, h] = np.array(code).astype(out[q].dtype)
        return out
    if op == "kv_read":
        out = {}
        at = (s["seq"].long(), s["slot"].long())
        for n, q, m, bits in (("k", "kq", "km", case["k_bits"]), ("v", "vq", "vm", case["v_bits"])):
            out[n] = _wrap(_x_value(_ints(s[q][at].long() & 0xffff), _ints(s[m][at])[..., None], bits))
        return out
    if op == "tree":
        G, hd, grp = case["kv_heads"], case["hd"], case["heads"] // case["kv_heads"]
        scale, starts, par = _finv_sqrt(hd << 48), s["starts"].tolist(), s["parents"].tolist()
        out = np.zeros((s["rows"], case["heads"], hd), np.int64)
        q = _ints(s["q"]).reshape(s["rows"], case["heads"], hd)
        for b, ln in enumerate(s["lens"].tolist()):
            n = starts[b + 1] - starts[b]
            if case["k_bits"]:
                k = _x_value(_ints(s["kq"][b, : ln + n].long()), _ints(s["km"][b, : ln + n])[..., None],
                             case["k_bits"])
                v = _x_value(_ints(s["vq"][b, : ln + n].long() & 0xffff), _ints(s["vm"][b, : ln + n])[..., None],
                             case["v_bits"])
            else:
                k, v = _ints(s["k"][b, : ln + n]), _ints(s["v"][b, : ln + n])
            for i in range(n):
                see, j = list(range(ln)), i
                while j >= 0:
                    see.append(ln + j)
                    j = par[starts[b] + j]
                for h in range(case["heads"]):
                    sc = [_i64(_i64(int(x) >> 48) * scale >> 48) for x in k[see, h // grp].dot(q[starts[b] + i, h])]
                    e = [_x_exp(max(sc) - x) if max(sc) - x <= 10 * ONE else 0 for x in sc]
                    tot = sum(e)
                    p = np.array([(x << 48) // tot for x in e], dtype=object)
                    out[starts[b] + i, h] = [_i64(x) for x in (p[:, None] * v[see, h // grp] >> 48).sum(0)]
        return {"out": out.reshape(s["rows"], -1)}
    logp, ent, ids, tl = [], [], [], []
    for lg, t in zip(s["logits"].tolist(), s["tokens"].tolist()):
        m = max(lg)
        e = [_x_tail(m - x) for x in lg]
        tot, a = sum(e), sum(x * (m - y) >> 48 for x, y in zip(e, lg))
        z, n = _x_ln(tot), max(0, max(tot, a).bit_length() - 61)
        best = sorted(range(len(lg)), key=lambda i: (-lg[i], i))[: case["top"]]
        logp.append(max(-(1 << 63), lg[t] - m - z))
        ent.append(z + ((a >> n) << 48) // (tot >> n))
        ids.append(best)
        tl.append([max(-(1 << 63), lg[i] - m - z) for i in best])
    k = (case["rows"], case["top"])
    return {"logp": np.array(logp, np.int64), "entropy": np.array(ent, np.int64),
            "top_ids": np.array(ids, np.int32).reshape(k), "top_logp": np.array(tl, np.int64).reshape(k)}
