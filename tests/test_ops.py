"""CPU tests of the operators around drafted tokens: their refusals (checked
before any device work) and the whole-number identities the kernels rest on."""
import ctypes
import math
import random
from fractions import Fraction

import numpy as np
import pytest

import iq
import ops_ref as ref
import oracle as orc
from helpers import ONE

ARG, RANGE = -1, -6
P = 1 << 20          # a non-null address that is never read: every call below is refused


def status(name, *args):
    return getattr(iq.lib(), name)(*args)


def rope(**kw):
    r = iq.Rope.__new__(iq.Rope)
    ctypes.Structure.__init__(r)
    for k, v in dict(dict(d_cos=P, d_sin=P, d_pos=P, n_pos=8, rot_dim=16, layout=0), **kw).items():
        setattr(r, k, v)
    return ctypes.byref(r)


def cache(**kw):
    c = iq.KVCache.__new__(iq.KVCache)
    ctypes.Structure.__init__(c)
    d = dict(seqs=2, max_seq=64, kv_heads=2, head_dim=16, k_bits=0, v_bits=0, k=P, v=P, kq=P, vq=P, k_mag=P, v_mag=P)
    for k, v in dict(d, **kw).items():
        setattr(c, k, v)
    return ctypes.byref(c)


def scaling(**kw):
    return ctypes.byref(iq._RopeScaling(**dict(dict(kind=1, orig_len=64, factor=2 * ONE, low=0, high=ONE), **kw)))


@pytest.mark.parametrize("bad,want", [
    (dict(cos=None), ARG), (dict(sin=P + 4), ARG), (dict(rot=0), ARG), (dict(rot=7), ARG), (dict(rot=258), ARG),
    (dict(n_pos=0), ARG), (dict(n_pos=(1 << 24) + 1), ARG), (dict(theta=0), ARG),
    (dict(sc=dict(kind=4)), ARG), (dict(sc=dict(factor=ONE - 1)), ARG), (dict(sc=dict(factor=1025 * ONE)), ARG),
    (dict(sc=dict(kind=2), rot=2), ARG), (dict(sc=dict(kind=3, orig_len=0)), ARG),
    (dict(sc=dict(kind=3, low=ONE)), ARG), (dict(sc=dict(mscale=-1)), ARG),
    (dict(theta=(1 << 31) - 1), RANGE), (dict(theta=400000000, sc=dict(kind=2, factor=1000 * ONE)), RANGE)])
def test_rope_tables_refusals(bad, want):
    a = dict(dict(cos=P, sin=P, rot=16, n_pos=8, theta=10000, sc=None), **bad)
    sc = scaling(**a["sc"]) if a["sc"] is not None else None
    assert status("iq_rope_tables_dev", a["cos"], a["sin"], a["rot"], a["n_pos"], a["theta"], sc, None) == want


@pytest.mark.parametrize("bad", [
    dict(out=None), dict(x=None), dict(out=P + 4), dict(rows=-1), dict(heads=0), dict(hd=0), dict(hd=257),
    dict(xs=31), dict(os=31), dict(x=P, out=P, os=40), dict(r=dict(rot_dim=18)), dict(r=dict(rot_dim=3)),
    dict(r=dict(rot_dim=0)), dict(r=dict(layout=2)), dict(r=dict(d_pos=None)), dict(r=dict(d_cos=P + 2)),
    dict(r=dict(n_pos=0)), dict(r=None)])
def test_rope_refusals(bad):
    a = dict(dict(out=2 * P, x=P, rows=2, heads=2, hd=16, xs=32, os=32, r={}), **bad)
    r = rope(**a["r"]) if a["r"] is not None else None
    assert status("iq_rope_dev", a["out"], a["x"], r, a["rows"], a["heads"], a["hd"], a["xs"], a["os"], None) == ARG


BAD_CACHE = [dict(seqs=0), dict(max_seq=0), dict(kv_heads=0), dict(head_dim=0), dict(head_dim=257), dict(k=None),
             dict(v=P + 4), dict(k_bits=8), dict(v_bits=3), dict(k_bits=9, v_bits=8), dict(k_bits=8, v_bits=17),
             dict(k_bits=8, v_bits=8, kq=None), dict(k_bits=8, v_bits=8, vq=P + 1),
             dict(k_bits=8, v_bits=8, v_mag=P + 4)]


@pytest.mark.parametrize("bad", BAD_CACHE)
def test_cache_refusals(bad):
    c = cache(**bad)
    assert status("iq_kv_write_dev", c, P, P, None, P, 1, 32, 32, None, None) == ARG
    assert status("iq_kv_read_dev", P, P, c, None, P, 1, None) == ARG
    n = ctypes.c_int64()
    assert status("iq_attn_tree_work", c, 4, 1, 1, 1, 1, ctypes.byref(n)) == ARG
    assert status("iq_attn_tree_dev", P, 2 * P, c, 4, None, P, P, P, 1, 1, 1, 1, 64, P, 1 << 30, None) == ARG


def test_kv_row_refusals():
    c = cache()
    assert status("iq_kv_write_dev", c, None, P, None, P, 1, 32, 32, None, None) == ARG
    assert status("iq_kv_write_dev", c, P, P, None, None, 1, 32, 32, None, None) == ARG
    assert status("iq_kv_write_dev", c, P, P, None, P, -1, 32, 32, None, None) == ARG
    assert status("iq_kv_write_dev", c, P, P, None, P, 1, 31, 32, None, None) == ARG
    assert status("iq_kv_write_dev", c, P, P, None, P, 1, 32, 31, None, None) == ARG
    assert status("iq_kv_write_dev", c, P, P, P + 2, P, 1, 32, 32, None, None) == ARG
    assert status("iq_kv_write_dev", c, P, P, None, P, 1, 32, 32, rope(rot_dim=18), None) == ARG
    assert status("iq_kv_write_dev", c, P, P, None, P, 0, 32, 32, None, None) == 0     # no rows: nothing to do
    assert status("iq_kv_read_dev", None, P, c, None, P, 1, None) == ARG
    assert status("iq_kv_read_dev", P, P, c, None, P + 1, 1, None) == ARG
    assert status("iq_kv_read_dev", P, P, c, None, P, 0, None) == 0


@pytest.mark.parametrize("bad,want", [
    (dict(out=None), ARG), (dict(q=None), ARG), (dict(out=P, q=P), ARG), (dict(lens=None), ARG),
    (dict(starts=None), ARG), (dict(parents=P + 2), ARG), (dict(nh=3), ARG), (dict(nh=0), ARG), (dict(n_seq=0), ARG),
    (dict(rows=0), ARG), (dict(nodes=0), ARG), (dict(ml=0), ARG), (dict(qs=63), ARG), (dict(work=P + 4), ARG),
    (dict(wb=-1), ARG), (dict(nodes=257), RANGE), (dict(ml=65), RANGE)])
def test_tree_refusals(bad, want):
    a = dict(dict(out=P, q=2 * P, nh=4, seqs=None, lens=P, starts=P, parents=P, n_seq=1, rows=2, nodes=2, ml=64,
                  qs=64, work=P, wb=1 << 30), **bad)
    assert status("iq_attn_tree_dev", a["out"], a["q"], cache(), a["nh"], a["seqs"], a["lens"], a["starts"],
                  a["parents"], a["n_seq"], a["rows"], a["nodes"], a["ml"], a["qs"], a["work"], a["wb"], None) == want


def test_tree_context_limit():
    """Beyond 32767 positions the int64 softmax sum could wrap: refused."""
    n = ctypes.c_int64()
    c = cache(max_seq=40000)
    assert status("iq_attn_tree_work", c, 4, 1, 1, 1, 32767, ctypes.byref(n)) == 0
    assert status("iq_attn_tree_work", c, 4, 1, 1, 1, 32768, ctypes.byref(n)) == RANGE


@pytest.mark.parametrize("bad,want", [
    (dict(lg=None), ARG), (dict(lg=P + 4), ARG), (dict(ld=99), ARG), (dict(rows=-1), ARG), (dict(V=0), ARG),
    (dict(tok=None), ARG), (dict(lp=None), ARG), (dict(top=-1), ARG), (dict(top=3, ids=None), ARG),
    (dict(top=3, tl=None), ARG), (dict(V=20, top=21), ARG), (dict(top=33), RANGE),
    (dict(V=(1 << 20) + 1, ld=1 << 21), RANGE), (dict(rows=0), 0)])
def test_logprobs_refusals(bad, want):
    a = dict(dict(lg=P, ld=100, rows=1, V=100, tok=P, lp=P, ent=P, top=1, ids=P, tl=P), **bad)
    assert status("iq_logprobs_dev", a["lg"], a["ld"], a["rows"], a["V"], a["tok"], a["lp"], a["ent"], a["top"],
                  a["ids"], a["tl"], None) == want


def test_binding_refuses_host_and_wrong_types():
    import torch
    x = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError):
        iq.Rope(x, x, x.int(), 4, 2)
    with pytest.raises(ValueError):
        iq.logprobs_dev(x.int(), 1, 4)


def test_binding_refuses_a_cache_of_another_device(monkeypatch):
    cache, rope = iq.KVCache(1, 1, 1, 4), iq.Rope(None, None, None, 1, 2)
    monkeypatch.setattr(iq, "_raw_device", lambda: 1)
    cache.dev = rope.dev = 0
    with pytest.raises(ValueError, match="device 0"):
        iq.kv_read_dev(None, None, cache, None, 1)
    with pytest.raises(ValueError, match="device 0"):
        iq.rope_dev(None, None, rope, 1, 1, 4)


# ------------------------------------------------------------- identities

def test_reference_tables_equal_rope_init():
    """The references of the scaled tables reduce to rope_init where nothing is scaled."""
    for rot, theta in ((32, 10000), (64, 10000), (128, 500)):
        n = 40
        c, s = np.empty((n, rot // 2), np.int64), np.empty((n, rot // 2), np.int64)
        orc.O.iqo_rope_tables(rot, n, theta, orc.p(c), orc.p(s))
        rc, rs = ref.tables(rot, range(n), theta)
        assert (c == rc).all() and (s == rs).all()


def test_angle_reduction_from_a_double_quotient():
    """p th mod 2 pi with the quotient from doubles: off by at most one, wrapped remainder exact."""
    w = 2 * ref.pi()
    rng = random.Random(1)
    for _ in range(20000):
        p = rng.choice([rng.randrange(1 << 24), (1 << 24) - 1 - rng.randrange(9)])
        th = rng.choice([rng.randrange(1, ONE + 1), ONE, w // rng.randrange(7, 99)])
        q = int(float(p) * float(th) / float(w))
        r = ref.wrap(p * th - q * w)
        r = r + w if r < 0 else r - w if r >= w else r
        assert r == p * th % w


def test_code_and_value_of_a_cache_vector():
    """kv_code's estimate and remainder, and kv_value's 32-bit halves."""
    rng = random.Random(2)
    for _ in range(20000):
        M = rng.choice([rng.randrange(1, 1 << 61), rng.randrange(1, 1 << 20), (1 << 61) - 1, 1])
        x = rng.choice([rng.randint(-M, M), M, -M, 0, M - 1])
        b = rng.randint(1, 16)
        u, D = x + M, 2 * M
        q = int(float(u) * (float(1 << b) / float(D)))
        r = ref.wrap((u << b) - q * D)
        q = q - 1 if r < 0 else q + 1 if r >= D else q
        assert q == (u << b) // D
        code = min(q, (1 << b) - 1)
        c = 2 * code + 1
        lo, hi = c * (M & 0xffffffff), c * (M >> 32)
        assert ref.wrap((hi << (32 - b)) + (lo >> b) - M) == ((2 * code + 1) * M >> b) - M


def test_exp_down_and_ln_accuracy():
    """E(d) within 2^-44 relative plus one unit of 2^-48 of e^-d; ln within 2^-46."""
    rng = random.Random(3)
    for _ in range(3000):
        d = rng.choice([rng.randrange(34 * ONE), rng.randrange(ONE), rng.randrange(1 << 30), 34 * ONE - 1])
        e, want = ref.exp_down(d), math.exp(-d / ONE) * ONE
        assert want * (1 - 2.0 ** -44) - 1 <= e <= want * (1 + 2.0 ** -44)
    assert ref.exp_down(0) == ONE and ref.exp_down(34 * ONE) == 0
    for _ in range(500):
        s = rng.randrange(ONE, 1 << rng.randint(49, 68))
        assert abs(ref.ln_sum(s) / ONE - math.log(s / ONE)) < 2.0 ** -46
    assert ref.ln_sum(ONE) == 0


def test_lowered_reciprocals_give_the_quotient_or_one_less():
    # floor(2^96 / r) from a reciprocal off by at most 2^-51, lowered by 2^-50: the floor is q or
    # q - 1, and the sign of (floor + 1) r - 2^96 - 1 in 64 bits tells which
    rng = random.Random(11)
    top = int(2 ** 62.5)
    rs = [1 << 48, (1 << 48) + 1, (1 << 62), top] + [rng.randrange(1 << 48, top) for _ in range(2000)]
    for r in rs:
        q = (1 << 96) // r
        for err in (Fraction(-1, 1 << 51), Fraction(0), Fraction(1, 1 << 51)):
            f = math.floor(Fraction(1, r) * (1 + err) * ((1 << 96) - (1 << 46)))
            assert f in (q - 1, q)
            sign = (((f + 1) * r - (1 << 96) - 1) % (1 << 64)) >> 63
            assert f + sign == q


def test_score_from_shifted_bytes():
    # q.k >> 48 (mod 2^64) from unsigned bytes of x + 2^63: diagonals i + j <= 13 and the sums of q and k
    rng = random.Random(12)
    for hd in (1, 7, 64):
        for _ in range(20):
            q = [rng.choice([rng.getrandbits(64) - (1 << 63), -(1 << 63), (1 << 63) - 1, 0]) for _ in range(hd)]
            k = [rng.choice([rng.getrandbits(64) - (1 << 63), -(1 << 63), (1 << 63) - 1, -1]) for _ in range(hd)]
            diag = [0] * 14
            for a, b in zip(q, k):
                a, b = a + (1 << 63), b + (1 << 63)
                for i in range(8):
                    for j in range(min(8, 14 - i)):
                        diag[i + j] += (a >> 8 * j & 255) * (b >> 8 * i & 255)
            assert max(diag) < 1 << 28
            low = 0
            for v in diag[:6]:
                low = (low >> 8) + v   # floors of floors
            dot = (low >> 8) + sum(v << 8 * (s - 6) for s, v in enumerate(diag) if s >= 6) - ((sum(q) + sum(k)) << 15)
            assert dot % (1 << 64) == (sum(a * b for a, b in zip(q, k)) >> 48) % (1 << 64)


def test_products_of_signed_halves():
    """mul_small: floor(x c / 2^48) for |x| < 2^59 and |c| < 2^49 from 32-bit halves, no intermediate beyond its type."""
    def fits(v, bits):
        assert -(1 << bits - 1) <= v < 1 << bits - 1
        return v

    def halves(x):
        low = (x & 0xffffffff) - ((x & 0x80000000) << 1)
        return fits((x >> 32) + (low < 0), 32), low

    rng = random.Random(13)
    X, C = 1 << 59, 1 << 49
    ends = lambda m: [m - 1, m - (1 << 31), m - (1 << 31) - 1, -m, -m + 1, -m + (1 << 31), 0, -1, 1 << 31]  # noqa: E731
    xs = ends(X) + [rng.randrange(-X, X) for _ in range(400)]
    cs = ends(C) + [ONE + 11, -ONE] + [rng.randrange(-C, C) for _ in range(100)]
    for x in xs:
        xh, xl = halves(x)
        for c in cs:
            ch, cl = halves(c)
            t = fits((xl * cl >> 32) + xh * cl, 64)
            t = fits(t + xl * ch, 64) >> 16
            assert fits(t + fits(8 * xh, 32) * fits(ch << 13, 32), 64) == x * c >> 48


def test_code_from_a_lowered_quotient():
    """kv_code: the estimate u inv rounded down, inv lowered by 2^-50, is q or q - 1 whichever way each rounding before
    it goes, and the sign of (q + 1) D - u 2^b - 1 in 64 bits tells which; an element whose magnitude wraps
    (INT64_MIN) is the one that x + M leaves negative, and its code is 0."""
    rng = random.Random(14)
    half = Fraction(1, 1 << 53)
    for _ in range(1500):
        M = rng.choice([rng.randrange(1, 1 << 61), rng.randrange(1, 1 << 20), (1 << 61) - 1, 1, 2, ONE])
        x = rng.choice([rng.randint(-M, M), M, -M, 0, M - 1, 1 - M])
        b = rng.choice([1, 4, 8, 16])
        u, D = x + M, 2 * M
        q = (u << b) // D
        for e in (-1, 1):
            # D as a double, its reciprocal, the scaled reciprocal and u as a double, each off by its bound
            inv = Fraction(1, D) / (1 + e * half) * (1 + Fraction(e, 1 << 51)) * (1 << b) * (1 - Fraction(1, 1 << 50))
            f = math.floor(u * (1 + e * half) * inv * (1 + e * half))
            assert f in (q - 1, q) or (u == 0 and f == 0)
            sign = ((f + 1) * D - (u << b) - 1) % (1 << 64) >> 63
            assert f + sign == q
    for M in (0, 1, ONE, (1 << 61) - 1):
        assert ref.pack([M, ref.I64_MIN, -M], 8) == ([255 if M else 0, 0, 0], M)
        assert ref.wrap(ref.I64_MIN + M) < 0 <= min(-M + M, M + M)


def test_explicit_streams():
    """torch's default stream (handle 0) is the legacy default stream, not the library's own; numbers go through."""
    class Stream:
        def __init__(self, handle):
            self.cuda_stream = handle

    assert iq._cur(Stream(0)) == 1 and iq._sp(Stream(0)).value == 1
    assert iq._cur(Stream(0x70)) == 0x70 and iq._sp(Stream(0x70)).value == 0x70
    for handle in (0, 1, 0x70):
        assert iq._cur(handle) == handle and (iq._sp(handle).value or 0) == handle


class _Binding:
    """The binding with host memory as its device and its calls recorded, not made."""

    def __init__(self, monkeypatch):
        import torch
        self.t, self.calls = torch, []
        monkeypatch.setattr(iq, "_raw_device", lambda: -1)      # a host tensor's device number
        monkeypatch.setattr(iq, "_call", lambda *a: self.calls.append(a))

    def q(self, *shape):
        return self.t.zeros(*shape, dtype=self.t.int64)

    def i(self, n):
        return self.t.zeros(n, dtype=self.t.int32)


OPERANDS = [(op, name) for op, names in dict(
    tables="cos sin", rope_of="cos sin pos", rope="out x", cache="k v", packed="kq vq k_mag v_mag",
    write="k v seq slot", read="k v seq slot", tree="out q seqs lens starts parents",
    logprobs="logits tokens logp entropy top_ids top_logp").items() for name in names.split()]


def _make(b, op):
    """(operands of a call by name, the call)"""
    q, i, t = b.q, b.i, b.t
    if op == "tables":
        return dict(cos=q(6, 4), sin=q(6, 4)), lambda a: iq.rope_tables_dev(a["cos"], a["sin"], 8, 6, 10000, stream=1)
    if op == "rope_of":
        return dict(cos=q(6, 4), sin=q(6, 4), pos=i(3)), lambda a: iq.rope_dev(
            q(3, 16), q(3, 16), iq.Rope(a["cos"], a["sin"], a["pos"], 6, 8), 3, 2, 8, stream=1)
    if op == "rope":
        r = iq.Rope(q(6, 4), q(6, 4), i(3), 6, 8)
        return dict(out=q(3, 16), x=q(3, 16)), lambda a: iq.rope_dev(a["out"], a["x"], r, 3, 2, 8, stream=1)
    if op == "cache":
        return dict(k=q(2, 5, 2, 8), v=q(2, 5, 2, 8)), lambda a: iq.KVCache(2, 5, 2, 8, **a)
    if op == "packed":
        n = (2, 5, 2, 8)
        return dict(kq=t.zeros(n, dtype=t.uint8), vq=t.zeros(n, dtype=t.int16), k_mag=q(2, 5, 2), v_mag=q(2, 5, 2)), \
            lambda a: iq.KVCache(2, 5, 2, 8, k_bits=8, v_bits=10, **a)
    c = iq.KVCache(2, 5, 2, 8, q(2, 5, 2, 8), q(2, 5, 2, 8))
    if op == "write":
        return dict(k=q(3, 16), v=q(3, 16), slot=i(3), seq=i(3)), \
            lambda a: iq.kv_write_dev(c, a["k"], a["v"], a["slot"], 3, seq=a["seq"], stream=1)
    if op == "read":
        return dict(k=q(3, 16), v=q(3, 16), slot=i(3), seq=i(3)), \
            lambda a: iq.kv_read_dev(a["k"], a["v"], c, a["slot"], 3, seq=a["seq"], stream=1)
    if op == "tree":
        return dict(out=q(3, 32), q=q(3, 32), lens=i(2), starts=i(3), parents=i(3), seqs=i(2)), \
            lambda a: iq.attn_tree_dev(cache=c, num_heads=4, n_seq=2, rows=3, max_nodes=2, max_len=5, work=q(100),
                                       stream=1, **a)
    return dict(logits=q(3, 50), tokens=i(3), logp=q(3), entropy=q(3), top_ids=i(12), top_logp=q(3, 4)), \
        lambda a: iq.logprobs_dev(a["logits"], 3, 50, a["tokens"], a["logp"], a["entropy"], 4, a["top_ids"],
                                  a["top_logp"], stream=1)


@pytest.mark.parametrize("op,name", OPERANDS)
def test_binding_refuses_wrong_operands(op, name, monkeypatch):
    """An operand that is one element short, of real numbers, scattered in memory, repeated or elsewhere is refused
    before the library sees its address; the right one passes."""
    b = _Binding(monkeypatch)
    args, call = _make(b, op)
    call(args)
    x, n = args[name], len(b.calls)
    real = {1: b.t.float8_e4m3fn, 2: b.t.bfloat16, 4: b.t.float32, 8: b.t.float64}[x.element_size()]
    twice = b.t.zeros(2 * x.numel(), dtype=x.dtype)
    for bad, why in ((x.flatten()[1:], "expected|3 rows"), (x.to(real), "one of"), (twice[::2], "strides"),
                     (x.flatten()[:1].expand(x.numel()), "strides")):
        with pytest.raises(ValueError, match=f"{name}.*{why}" if why != "expected|3 rows" else why):
            call(dict(args, **{name: bad}))
    assert len(b.calls) == n
    monkeypatch.setattr(iq, "_raw_device", lambda: 0)
    with pytest.raises(ValueError, match="memory of the device 0|of device"):
        call(args)
    monkeypatch.setattr(iq, "_raw_device", lambda: -1)
    call(dict(args, **{name: twice[1:x.numel() + 1]}))       # a longer or flat one in one piece is right


def test_binding_row_layouts(monkeypatch):
    """Row operands: contiguous by length, views by their strides; a Rope by its rows; a work space in one piece."""
    b = _Binding(monkeypatch)
    q = b.q
    rope = iq.Rope(q(6, 4), q(6, 4), b.i(6), 6, 8)
    out = q(6, 16)

    def x(t, ld, rows=6):
        iq.rope_dev(out, t, rope, rows, 2, 8, x_stride=ld, stream=1)
        assert b.calls.pop()[2] == t.data_ptr()

    x(q(6, 40)[:, 8:24], 40)
    x(q(6, 40)[:, 8:], 40)
    x(q(6, 5, 8)[:, 1:3], 40)                       # heads of a fused row
    x(q(2, 3, 40)[:, :, :16], 40)                   # rows in two dimensions
    x(q(12, 16)[::2], 32)
    x(q(2, 200)[:, :96].view(2, 6, 16), 16)         # rows side by side in the last dimensions
    x(q(5 * 40 + 16), 40)                           # ends with the last row
    x(q(1, 40)[:, 3:19], 16, rows=1)
    x(q(4, 40)[:, :16], 99, rows=1)                 # one row: no distance
    x(q(4, 40)[:, :16], 40, rows=0)
    for t, ld, rows in ((q(5 * 40 + 15), 40, 6), (q(5, 40)[:, :16], 40, 6), (q(6, 40)[:, :15], 40, 6),
                        (q(6, 40)[:, :16], 16, 6), (q(16, 6).t(), 16, 6), (q(16, 16).t(), 16, 6),
                        (q(2, 4, 40)[:, :3, :16], 40, 6), (q(2, 200)[:, :80].view(2, 5, 16), 16, 6),
                        (q(1, 16).expand(6, 16), 16, 6), (q(6, 8, 5)[:, :, :2], 40, 6), (q(32)[::2], 16, 1),
                        (q(7, 16), 16, 7)):
        with pytest.raises(ValueError):
            iq.rope_dev(q(7, 16), t, rope, rows, 2, 8, x_stride=ld, stream=1)
    c = iq.KVCache(1, 5, 2, 8, q(1, 5, 2, 8), q(1, 5, 2, 8))
    call = lambda w: iq.attn_tree_dev(q(32), q(32), c, 4, b.i(1), b.i(2), b.i(1), 1, 1, 1, 5, w, stream=1)  # noqa: E731
    call(q(10))
    assert b.calls.pop()[14:16][-1] == 80
    for w in (q(20)[::2], q(1).expand(100)):
        with pytest.raises(ValueError, match="work"):
            call(w)


def test_calls_without_rows():
    """No rows: nothing to do, whatever the rows' pointers (an empty tensor's is NULL); sizes are checked all the same."""
    c, r = cache(), rope(d_pos=None)
    assert status("iq_rope_dev", None, None, r, 0, 2, 16, 32, 32, None) == 0
    assert status("iq_kv_write_dev", c, None, None, None, None, 0, 32, 32, r, None) == 0
    assert status("iq_kv_read_dev", None, None, c, None, None, 0, None) == 0
    assert status("iq_logprobs_dev", None, 100, 0, 100, None, None, None, 3, None, None, None) == 0
    assert status("iq_rope_dev", None, None, r, 0, 0, 16, 32, 32, None) == ARG
    assert status("iq_kv_write_dev", c, None, None, None, None, 0, 31, 32, r, None) == ARG
    assert status("iq_kv_read_dev", None, None, cache(seqs=0), None, None, 0, None) == ARG
    assert status("iq_logprobs_dev", None, 99, 0, 100, None, None, None, 3, None, None, None) == ARG


def test_binding_calls_without_rows(monkeypatch):
    b = _Binding(monkeypatch)
    q, i = b.q, b.i
    r, c = iq.Rope(q(6, 4), q(6, 4), i(0), 6, 8), iq.KVCache(2, 5, 2, 8, q(2, 5, 2, 8), q(2, 5, 2, 8))
    monkeypatch.undo()
    monkeypatch.setattr(iq, "_raw_device", lambda: -1)
    iq.rope_dev(q(0, 16), q(0, 16), r, 0, 2, 8, stream=1)
    iq.kv_write_dev(c, q(0, 16), q(0, 16), i(0), 0, seq=i(0), rope=r, stream=1)
    iq.kv_read_dev(q(0, 16), q(0, 16), c, i(0), 0, stream=1)
    iq.logprobs_dev(q(0, 50), 0, 50, i(0), q(0), q(0), 3, i(0), q(0, 3), stream=1)
