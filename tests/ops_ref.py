"""Whole-number references of the operators around drafted tokens (rotary,
cache rows, tree attention, log probabilities): Python integers, with the
oracle's C restatement for the fp_math functions on arrays."""
import math
from decimal import Decimal, getcontext

import numpy as np

import oracle as orc
from helpers import ONE

MUL, DIV, INV_SQRT, EXP, LOG, COS, SIN, SAFE_EXP = 0, 1, 4, 5, 6, 7, 8, 11
LN2 = 195103586505167
I64_MIN, I64_MAX = -(1 << 63), (1 << 63) - 1


def wrap(x):
    return (int(x) + (1 << 63)) % (1 << 64) - (1 << 63)


def fp(fn, x, y=0):
    return int(orc.O.iqo_fp(fn, wrap(x), wrap(y)))


def mul(a, b):
    a, b = np.broadcast_arrays(np.asarray(a, np.int64), np.asarray(b, np.int64))
    a, b = np.ascontiguousarray(a), np.ascontiguousarray(b)
    return orc.fp_vec(MUL, a, b).reshape(a.shape)


def q48(a):
    return np.round(np.asarray(a) * float(ONE)).astype(np.int64)


# ------------------------------------------------------------------- rotary

def pi():
    """pi of the reference's tables: 4 atan(1), from its CORDIC angles (cos of it is -1 to rounding)."""
    at = lambda x, terms: _atan(x, terms)  # noqa: E731
    return (at(ONE // 5, 40) << 4) - (at(ONE // 239, 15) << 2)


def _atan(x, terms):
    x2 = x * x >> 48
    t = s = x
    for n in range(1, terms + 1):
        t = -(t * x2 >> 48)
        c = abs(t) // (2 * n + 1) * (1 if t >= 0 else -1)
        if c == 0:
            break
        s += c
    return s


def ln_int(theta):
    k = max(0, theta.bit_length() - 14)
    return fp(LOG, (theta << 48) >> k) + k * LN2


def freqs(rot, theta, kind="none", factor=ONE, orig_len=0, low=0, high=ONE, mscale=0):
    lt = ln_int(theta)
    if kind == "ntk":
        lt += fp(MUL, fp(LOG, factor), (rot << 48) // (rot - 2))
    out = []
    for i in range(rot // 2):
        y = fp(MUL, -((2 * i << 48) // rot), lt)
        th = fp(EXP, y) if y >= -10 * ONE else fp(MUL, fp(EXP, y >> 1), fp(EXP, y >> 1))
        if kind == "linear":
            th = (th << 48) // factor
        if kind == "parts":
            turns = (orig_len * th << 48) // (2 * pi())
            w = (min(max(turns - low, 0), high - low) << 48) // (high - low)
            th = fp(MUL, th, w) + fp(MUL, (th << 48) // factor, ONE - w)
        out.append(th)
    return out


def tables(rot, positions, theta, **scaling):
    """cos, sin rows of the given positions."""
    w, ms = 2 * pi(), scaling.get("mscale", 0)
    a = []
    for p in positions:
        for f in freqs(rot, theta, **scaling):
            r = p * f % w
            a.append(r - w if r > w // 2 else r)
    a = np.array(a, np.int64)
    c, s = orc.fp_vec(COS, a), orc.fp_vec(SIN, a)
    if ms:
        c, s = mul(c, ms), mul(s, ms)
    return c.reshape(len(positions), -1), s.reshape(len(positions), -1)


def rotate(x, cos, sin, rot, layout):
    """x [rows, heads, hd]; cos, sin [rows, rot / 2]."""
    out = x.copy()
    i, j = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    a, b, c, s = x[..., i], x[..., j], cos[:, None], sin[:, None]
    with np.errstate(over="ignore"):
        out[..., i] = mul(a, c) - mul(b, s)
        out[..., j] = mul(b, c) + mul(a, s)
    return out


# -------------------------------------------------------------------- cache

def pack(x, bits):
    """kv_pack_vector (llama_int.c:1197-1218) on one vector: codes, magnitude."""
    m = 0
    for v in x:
        a = wrap(-int(v)) if v < 0 else int(v)
        m = max(m, a)
    if m == 0:
        return [0] * len(x), 0
    codes = []
    for v in x:
        num, den = wrap(int(v) + m) << bits, wrap(2 * m)
        t = abs(num) // abs(den) * (1 if (num < 0) == (den < 0) else -1)
        codes.append(min(max(t, 0), (1 << bits) - 1))
    return codes, m


def unpack(codes, m, bits):
    return [wrap(((2 * int(q) + 1) * int(m) >> bits) - int(m)) for q in codes]


# --------------------------------------------------------------------- tree

def ancestors(parents):
    """For each node the nodes it sees, itself last; a parent that is no earlier node counts as none."""
    out = []
    for i in range(len(parents)):
        path, j = [], i
        while True:
            path.append(j)
            p = int(parents[j])
            if p < 0 or p >= j:
                break
            j = p
        out.append(path[::-1])
    return out


def attend(q, k, v, scale):
    """One query [hd] over the rows k, v [T, hd] it sees (llama_int.c:1432-1529)."""
    hd = len(q)
    dots = [wrap(sum(int(a) * int(b) for a, b in zip(q, row)) >> 48) for row in k] if hd * len(k) < 4096 else \
        [wrap(int(x) >> 48) for x in k.astype(object).dot(q.astype(object))]
    s = mul(np.array(dots, np.int64), scale)
    with np.errstate(over="ignore"):
        e = orc.fp_vec(SAFE_EXP, s - s.max())
        tot = int(np.sum(e, dtype=np.int64))
        p = orc.fp_vec(DIV, e, np.full_like(e, tot)) if tot > 0 else e
        return np.sum(mul(p[:, None], v), axis=0, dtype=np.int64)


def tree(q, ks, vs, lens, starts, parents, nh):
    """q [rows, nh, hd]; ks, vs: per sequence [T, nkv, hd]."""
    out = np.zeros_like(q)
    hd = q.shape[2]
    scale = fp(INV_SQRT, hd << 48)
    for b, (k, v) in enumerate(zip(ks, vs)):
        grp, n = nh // k.shape[1], starts[b + 1] - starts[b]
        for i, path in enumerate(ancestors(parents[starts[b]:starts[b + 1]])):
            see = np.r_[np.arange(lens[b]), lens[b] + np.array(path)].astype(int)
            for h in range(nh):
                out[starts[b] + i, h] = attend(q[starts[b] + i, h], k[see, h // grp], v[see, h // grp], scale)
    return out


# ------------------------------------------------------------------- scores

getcontext().prec = 50
_ln2 = Decimal(2).ln()
_L2E, _N2 = [int((x * (1 << 60)).to_integral_value()) for x in (1 / _ln2, _ln2)]
_POW = [int(((-_ln2 * j / 64).exp() * ONE).to_integral_value()) for j in range(64)]
_COEF = [int((_ln2 ** k / math.factorial(k) * ONE).to_integral_value()) for k in range(6)]


def exp_down(d):
    if d >= 34 * ONE:
        return 0
    y = d * _L2E >> 60
    f, r, h = y % ONE, y % (1 << 42), _COEF[5]
    for c in _COEF[4::-1]:
        h = c - (h * r >> 48)
    return (_POW[f >> 42] * h >> 48) >> (y >> 48)


def ln_sum(s):
    bl = s.bit_length()
    y, z = (s << (62 - bl) if bl <= 62 else s >> (bl - 62)), 0
    for _ in range(50):
        y = y * y >> 61
        z, y = 2 * z + (y >> 62), y >> (y >> 62)
    return (((bl - 49) << 50) + z) * _N2 >> 62


def logprobs(row, token, top):
    """(log probability of token, entropy, ids, their log probabilities) of one row of logits."""
    row = [int(x) for x in row]
    m = max(row)
    seen = {}
    tot = acc = 0
    for x in row:
        if x not in seen:
            e = exp_down(m - x)
            seen[x] = e, e * (m - x) >> 48
        tot += seen[x][0]
        acc += seen[x][1]
    z, n = ln_sum(tot), max(0, max(tot, acc).bit_length() - 61)
    best = sorted(range(len(row)), key=lambda i: (-row[i], i))[:top]
    lp = lambda i: max(I64_MIN, row[i] - m - z)  # noqa: E731
    return lp(token) if token is not None else None, z + (((acc >> n) << 48) // (tot >> n)), best, [lp(i) for i in best]
