"""Python host-side binding of libiq.so (the C ABI in include/iq.h) -- TEST AND
BENCH TOOLING, not the product: the product is the C ABI (include/iq.h,
libiq.so), which C hosts such as llama_int.c call directly. This module is how
the tests and bench.py reach that ABI from Python; torch appears here only to
hand over device memory and streams.

This is a thin ctypes mirror of the reference's operator surface: ``matmul_vec``
(llama_int.c:1014) with its argument order ``(out, weight, in, M, N)``, where M
is the number of output rows and N the input length. Host arrays are numpy
int64; device arrays are anything exposing ``data_ptr()`` (torch tensors are
used only as device-memory plumbing). Every call raises ``IQError`` on a
non-zero status; there is no CPU fallback: if libiq.so is missing or no B200
is present, calls fail loudly.
"""
import ctypes
import os

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("IQ_LIB") or os.path.join(HERE, "libiq.so")  # IQ_LIB: another build

IQ_FN = dict(mul=0, div=1, sqrt=2, sqrt_fast=3, inv_sqrt=4, exp=5, log=6, cos=7, sin=8,
             sigmoid=9, silu=10, safe_exp=11, exp_dyadic=12)

# every symbol include/iq.h declares, with (restype, argtypes)
_P = ctypes.c_void_p
_I = ctypes.c_int
_I64 = ctypes.c_int64
SIGNATURES = {
    "iq_status_str": (ctypes.c_char_p, [_I]),
    "iq_last_cuda_error": (_I, []),
    "iq_version": (_I, []),
    "iq_set_device": (_I, [_I]),
    "iq_matmul_vec": (_I, [_P, _P, _P, _I, _I]),
    "iq_weight_register": (_I, [_P, _I, _I]),
    "iq_weight_unregister": (_I, [_P]),
    "iq_weight_cache_clear": (_I, []),
    "iq_weight_check_mode": (_I, [_I]),
    "iq_weight_cache_limit": (_I, [_I64]),
    "iq_weight_cache_stats": (_I, [_P, _P]),
    "iq_matvec_dev": (_I, [_P, _P, _P, _I, _I, _P]),
    "iq_gemm_dev": (_I, [_P, _P, _P, _I, _I, _I, _P]),
    "iq_pack_weights_dev": (_I, [_P, _I, _I, _P, _P]),
    "iq_pack_weights_fmt_dev": (_I, [_P, _I, _I, _I, _P, _P]),
    "iq_packed_free": (_I, [_P]),
    "iq_packed_info": (_I, [_P, _P, _P, _P]),
    "iq_matvec_packed_dev": (_I, [_P, _P, _P, _P]),
    "iq_matvec_packed_noalloc_dev": (_I, [_P, _P, _P, _P]),
    "iq_packed_bytes": (_I, [_P, _P]),
    "iq_packed_format": (_I, [_P, _P]),
    "iq_pack_weights_tc_dev": (_I, [_P, _I, _I, _P, _P]),
    "iq_packed_tc_free": (_I, [_P]),
    "iq_packed_tc_info": (_I, [_P, _P, _P, _P]),
    "iq_gemm_tc_dev": (_I, [_P, _P, _P, _I, _P]),
    "iq_device_status": (_I, []),
    "iq_wait_selftest": (_I, [_I64]),
    "iq_bench_i8_peak": (_I, [_I, _P, _P]),
    "iq_fp_dev": (_I, [_I, _P, _P, _P, _I64, _P]),
    "iq_rmsnorm_dev": (_I, [_P, _P, _P, _I, _I, _P]),
    "iq_softmax_dev": (_I, [_P, _I, _I, _P]),
    "iq_rope_tables_dev": (_I, [_P, _P, _I, _I, _I, _P, _P]),
    "iq_rope_dev": (_I, [_P, _P, _P, _I, _I, _I, _I64, _I64, _P]),
    "iq_kv_write_dev": (_I, [_P, _P, _P, _P, _P, _I, _I64, _I64, _P, _P]),
    "iq_kv_read_dev": (_I, [_P, _P, _P, _P, _P, _I, _P]),
    "iq_attn_tree_work": (_I, [_P, _I, _I, _I, _I, _I, _P]),
    "iq_attn_tree_dev": (_I, [_P, _P, _P, _I, _P, _P, _P, _P, _I, _I, _I, _I, _I64, _P, _I64, _P]),
    "iq_logprobs_dev": (_I, [_P, _I64, _I, _I, _P, _P, _P, _I, _P, _P, _P]),
    "iq_model_create": (_I, [_P, _I, _I, _P]),
    "iq_nccl_unique_id": (_I, [_P]),
    "iq_tp_shard_info": (_I, [_P, _I, _I, _P]),
    "iq_model_create_tp": (_I, [_P, _I, _I, _I, _I, _P, _P]),
    "iq_model_destroy": (_I, [_P]),
    "iq_model_load_globals": (_I, [_P, _P, _P, _P]),
    "iq_model_load_layer": (_I, [_P, _I, _P]),
    "iq_model_synth": (_I, [_P, _I, _I]),
    "iq_model_config": (_I, [_P, _P]),
    "iq_mgw_read_config": (_I, [ctypes.c_char_p, _P, _P]),
    "iq_model_load_mgw": (_I, [_P, ctypes.c_char_p]),
    "iq_model_reset": (_I, [_P]),
    "iq_forward": (_I, [_P, _I, _I, _P, _P]),
    "iq_generate": (_I, [_P, _P, _I, _I, _P, _P, _P]),
    "iq_generate_batch": (_I, [_P, _P, _I, _I, _P, _P, _P]),
    "iq_generate_sampled": (_I, [_P, _P, _I, _I, _I64, _I, _I64, ctypes.c_uint64, _P, _P, _P]),
    "iq_sample_dev": (_I, [_P, _I, _I, _I64, _I, _I64, _P, _P]),
    "iq_rng_seed": (_I, [ctypes.c_uint64, _P]),
    "iq_decode_steps_timed": (_I, [_P, _I, _I, _P]),
    "iq_model_set_attention": (_I, [_P, _I]),
    "iq_model_weight_bytes": (_I, [_P, _P, _P]),
    "iq_model_set_decode": (_I, [_P, _I]),
    "iq_model_set_timeout": (_I, [_P, _I64]),
    "iq_model_set_peer_check": (_I, [_P, _P, _P]),
    "iq_model_set_kv_packed": (_I, [_P, _I, _I]),
    "iq_selftest_watchdog": (_I, [_I, _P, _P]),
    "iq_model_decode_info": (_I, [_P, _P, _P]),
    "iq_bench_grid_sync": (_I, [_I, _I, _I, _P]),
    "iq_model_decode_stamps": (_I, [_P, _P, _I]),
    "iq_tensor_seed": (ctypes.c_uint64, [_I, ctypes.c_char_p]),
    "iq_synth_weights": (_I, [ctypes.c_uint64, _P, _I64]),
    "iq_synth_acts": (_I, [ctypes.c_uint64, _P, _I64]),
    "iq_synth_tokens": (_I, [ctypes.c_uint64, _P, _I, _I]),
    "iq_bf16_to_q1648": (_I64, [ctypes.c_uint16]),
    "iq_q1648_to_bf16": (ctypes.c_uint16, [_I64]),
}


class IQError(RuntimeError):
    def __init__(self, fn, status, lib):
        self.status = status
        msg = lib.iq_status_str(status).decode()
        cuda = lib.iq_last_cuda_error()
        super().__init__(f"{fn} failed: {msg} (status {status}, last cudaError {cuda})")


_lib = None


def lib():
    """Load libiq.so (built in-tree by the package Makefile)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"libiq.so not built at {LIB_PATH}; run __graft_entry__.build()")
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _lib = L
    return _lib


def _call(name, *args):
    rc = getattr(_lib or lib(), name)(*args)
    if rc != 0:
        raise IQError(name, rc, _lib)
    return rc


def _hp(a):
    assert isinstance(a, np.ndarray) and a.flags.c_contiguous
    return a.ctypes.data_as(ctypes.c_void_p)


def _dp(t):
    if t is None:
        return None
    return ctypes.c_void_p(t.data_ptr())


_CUDA_STREAM_LEGACY = 0x1


def _handle(stream):
    """Handle of an explicit stream: a torch stream's, or a number (0: the library's own
    stream). torch's default stream has handle 0, which the library would read as its
    own: name the legacy default stream (cudaStreamLegacy) instead."""
    h = getattr(stream, "cuda_stream", None)
    return stream if h is None else h or _CUDA_STREAM_LEGACY


def _sp(stream):
    """Stream argument: an explicit stream, else torch's current stream when torch
    has initialised CUDA (so device calls order with the tensors' producers),
    else NULL = the library's own stream."""
    if stream is None:
        import sys
        t = sys.modules.get("torch")
        if t is not None and t.cuda.is_initialized():
            return ctypes.c_void_p(_handle(t.cuda.current_stream()))
        return None
    return ctypes.c_void_p(_handle(stream))


# ---------------------------------------------------------------- host API

def matmul_vec(out, weight, inp, M, N):
    """Drop-in for matmul_vec(out, weight, in, M, N) on host int64 arrays."""
    assert out.dtype == weight.dtype == inp.dtype == np.int64
    assert out.size >= M and inp.size >= N and weight.size >= M * N
    _call("iq_matmul_vec", _hp(out), _hp(weight), _hp(inp), M, N)


def weight_register(weight, M, N):
    _call("iq_weight_register", _hp(weight), M, N)


def weight_unregister(weight):
    _call("iq_weight_unregister", _hp(weight))


def weight_cache_clear():
    _call("iq_weight_cache_clear")


WCHECK = dict(none=0, sampled=1, full=2)


def weight_check_mode(mode):
    _call("iq_weight_check_mode", WCHECK[mode] if isinstance(mode, str) else mode)


def weight_cache_limit(nbytes):
    _call("iq_weight_cache_limit", nbytes)


def weight_cache_stats():
    """(entries, device bytes) of the drop-in's weight cache."""
    e, b = ctypes.c_int(), ctypes.c_int64()
    _call("iq_weight_cache_stats", ctypes.byref(e), ctypes.byref(b))
    return e.value, b.value


def nccl_unique_id():
    """128-byte NCCL id for iq_model_create_tp (made on one rank, shared with all)."""
    buf = ctypes.create_string_buffer(128)
    _call("iq_nccl_unique_id", buf)
    return buf.raw


def tp_shard_info(cfg, tp_size, tp_rank):
    """Row ownership of a tensor-parallel rank (see iq_tp_shard_info)."""
    c = cfg if isinstance(cfg, Config) else Config.from_dict(cfg)
    info = (ctypes.c_int * 8)()
    _call("iq_tp_shard_info", ctypes.byref(c), tp_size, tp_rank, info)
    keys = ("q_lo", "nh", "kv_lo", "nkv", "d_lo", "d_n", "it_lo", "it_n")
    return dict(zip(keys, list(info)))


def mgw_config(path):
    """(config dict, lm_head_tied) of an int-llm .mgw file."""
    c = Config()
    tied = ctypes.c_int(0)
    _call("iq_mgw_read_config", os.fsencode(path), ctypes.byref(c), ctypes.byref(tied))
    return dict(dim=c.hidden_dim, n_heads=c.num_heads, n_kv_heads=c.num_kv_heads, head_dim=c.head_dim,
                n_layers=c.num_layers, inter=c.intermediate_dim, vocab=c.vocab_size, max_seq=c.max_seq_len,
                rope_theta=c.rope_theta), bool(tied.value)


def set_device(d):
    _call("iq_set_device", d)


# -------------------------------------------------------------- device API

def matvec_dev(out, w, x, M, N, stream=None):
    _call("iq_matvec_dev", _dp(out), _dp(w), _dp(x), M, N, _sp(stream))


class Packed:
    """Byte-plane packed weights on the device (iq_pack_weights_dev)."""

    def __init__(self, d_w, M, N, stream=None, fmt=None):
        """fmt: None = the library's choice, 'planes' or 'bf16'."""
        self.h = ctypes.c_void_p()
        self.M, self.N = M, N
        f = {None: -1, "planes": 0, "bf16": 1}[fmt]
        _call("iq_pack_weights_fmt_dev", _dp(d_w), M, N, f, _sp(stream), ctypes.byref(self.h))

    def info(self):
        """(np, p0, residual_entries): stored planes p0 .. p0+np-1 and the sparse residual size."""
        a, b, c = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
        _call("iq_packed_info", self.h, ctypes.byref(a), ctypes.byref(b), ctypes.byref(c))
        return a.value, b.value, c.value

    def fmt(self):
        """'planes' (byte-plane window) or 'bf16' (2 bytes per weight)."""
        f = ctypes.c_int()
        _call("iq_packed_format", self.h, ctypes.byref(f))
        return ("planes", "bf16")[f.value]

    def nbytes(self):
        """Bytes of the stored form one matvec launch reads (iq_packed_bytes)."""
        b = ctypes.c_int64()
        _call("iq_packed_bytes", self.h, ctypes.byref(b))
        return b.value

    def free(self):
        if self.h:
            _call("iq_packed_free", self.h)
            self.h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def matvec_packed_dev(out, packed, x, stream=None):
    _call("iq_matvec_packed_dev", _dp(out), packed.h, _dp(x), _sp(stream))


class PackedTC:
    """Weights packed for the tcgen05 GEMM (iq_pack_weights_tc_dev)."""

    def __init__(self, d_w, M, N, stream=None):
        self.h = ctypes.c_void_p()
        _call("iq_pack_weights_tc_dev", _dp(d_w), M, N, _sp(stream), ctypes.byref(self.h))

    def info(self):
        """(np, p0, residual_entries) of the GEMM form."""
        a, b, c = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
        _call("iq_packed_tc_info", self.h, ctypes.byref(a), ctypes.byref(b), ctypes.byref(c))
        return a.value, b.value, c.value

    def free(self):
        if self.h:
            _call("iq_packed_tc_free", self.h)
            self.h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def gemm_tc_dev(out, packed, X, rows, stream=None):
    _call("iq_gemm_tc_dev", _dp(out), packed.h, _dp(X), rows, _sp(stream))


def sample_dev(d_logits, rows, V, temperature, top_k, top_p, rng):
    """sample_token per row on the device; rng: uint64 [rows][2], advanced in place."""
    out = np.zeros(rows, dtype=np.int32)
    assert rng.dtype == np.uint64 and rng.flags.c_contiguous
    _call("iq_sample_dev", _dp(d_logits), rows, V, temperature, top_k, top_p, _hp(rng), _hp(out))
    return out


def device_status():
    """IQ_OK, or the timeout status a kernel's bounded wait recorded (then cleared)."""
    return lib().iq_device_status()


def bench_i8_peak(iters=20000):
    """(int8 TOP/s, ms) of the tcgen05 kind::i8 peak kernel on the current device."""
    t, ms = ctypes.c_double(), ctypes.c_float()
    _call("iq_bench_i8_peak", iters, ctypes.byref(t), ctypes.byref(ms))
    return t.value, ms.value


def gemm_dev(out, w, X, rows, M, N, stream=None):
    _call("iq_gemm_dev", _dp(out), _dp(w), _dp(X), rows, M, N, _sp(stream))


def fp_dev(fn, x, y, out, n, stream=None):
    code = IQ_FN[fn] if isinstance(fn, str) else fn
    _call("iq_fp_dev", code, _dp(x), _dp(y), _dp(out), n, _sp(stream))


def rmsnorm_dev(out, x, w, rows, dim, stream=None):
    _call("iq_rmsnorm_dev", _dp(out), _dp(x), _dp(w), rows, dim, _sp(stream))


def softmax_dev(x, rows, n, stream=None):
    _call("iq_softmax_dev", _dp(x), rows, n, _sp(stream))


# ------------------------- drafted tokens: rotary, cache, tree attention, scores

_raw_device = _raw_stream = None     # torch's current device and stream handle, bound at the first call
_i8 = _i16 = _i32 = _i64 = ()        # types of operands of 1, 2, 4 and 8 bytes


def _bind_torch():
    global _raw_device, _raw_stream, _i8, _i16, _i32, _i64
    import torch
    _raw_device, _raw_stream = _raw_device or torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
    _i8, _i16 = (torch.uint8, torch.int8), (torch.int16, torch.uint16)
    _i32, _i64 = (torch.int32, torch.uint32), (torch.int64, torch.uint64)


def _device():
    """The device that calls go to: torch's current one (None without a GPU)."""
    if _raw_device is None or not _i8:
        _bind_torch()
    try:
        return _raw_device()
    except RuntimeError:
        return None


def _dev_ptr(t, types, dev, name, n, width=0, rows=1, ld=0):
    """Device pointer of t (None: NULL) after checking that it has one of the types, lies on the device `dev`
    and holds what the call takes there: n elements side by side or, in a tensor that is not contiguous,
    `rows` rows of `width` elements ld apart (n = (rows - 1) ld + width)."""
    if t is not None:
        if t.dtype in types and t.get_device() == dev and (
                t.numel() >= n if t.is_contiguous() else _holds(t, width or n, rows, ld)):
            return t.data_ptr()
        raise ValueError(_refusal(t, types, dev, name, n, width or n, rows, ld))


def _refusal(t, types, dev, name, n, width, rows, ld):
    if t.dtype not in types:
        return f"{name}: one of {types} expected, got {t.dtype}"
    if t.is_contiguous() and t.numel() < n:
        return f"{name} holds {t.numel()} elements, {n} expected"
    if not t.is_contiguous() and not _holds(t, width, rows, ld):
        return (f"{name}: {rows} rows of {width} elements, {ld} apart, expected, got shape {tuple(t.shape)} with "
                f"strides {t.stride()}")
    return f"{name} must be in memory of the device {dev}, where calls go to, got {t.device}"


def _holds(t, width, rows, ld):
    """Whether the strided t holds `rows` rows of `width` elements side by side, ld elements apart: its
    last dimensions as one row or several, the ones before as their number."""
    shape, steps, n, r = t.shape, t.stride(), 1, 1
    if len(steps) == 2 and steps[1] == 1 and (steps[0] == ld or rows <= 1):   # columns of a matrix, as of a fused q|k|v
        return shape[0] >= rows and shape[1] >= width
    for size, step in zip(reversed(shape), reversed(steps)):
        if size == 1:
            continue
        if r == 1 and step == n:
            n *= size
        elif step == ld * r:
            r *= size
        else:
            break
    return rows < 1 or n >= (rows - 1) * ld + width or (n >= width and r >= rows)


def _cur(stream, dev=None):
    """Stream argument as _sp's: an explicit one, else torch's current stream on `dev`."""
    return _raw_stream(dev) or _CUDA_STREAM_LEGACY if stream is None else _handle(stream)


def _ref(x, dev, rows=0):
    """x (a Rope or KVCache) by reference, after checking that its tensors lie where calls go to and
    that a Rope has the positions of `rows` rows."""
    if x.dev is not None and x.dev != dev:
        raise ValueError(f"{type(x).__name__} of device {x.dev}, calls go to device {dev}")
    if rows and rows > x.rows:
        raise ValueError(f"Rope of {x.rows} positions, {rows} rows")
    return ctypes.byref(x)


ROPE_LAYOUT = dict(half=0, interleaved=1)
ROPE_SCALE = dict(none=0, linear=1, ntk=2, parts=3)


class _RopeScaling(ctypes.Structure):
    _fields_ = [("kind", _I), ("orig_len", _I), ("factor", _I64), ("low", _I64), ("high", _I64), ("mscale", _I64)]


def rope_tables_dev(cos, sin, rot_dim, n_pos, theta, scaling=None, stream=None):
    """Tables [n_pos][rot_dim / 2]; scaling: dict of kind, factor, orig_len, low, high, mscale (Q16.48 ints)."""
    sc, dev, n = None, _device(), n_pos * (rot_dim // 2)
    if scaling is not None:
        f = dict(scaling)
        f["kind"] = ROPE_SCALE[f.get("kind", "none")]
        sc = ctypes.byref(_RopeScaling(**f))
    _call("iq_rope_tables_dev", _dev_ptr(cos, _i64, dev, "cos", n), _dev_ptr(sin, _i64, dev, "sin", n), rot_dim, n_pos,
          theta, sc, _cur(stream, dev))


class Rope(ctypes.Structure):
    """iq_rope: tables, the rows' positions (int32) and the layout ('half' or 'interleaved')."""
    _fields_ = [("d_cos", _P), ("d_sin", _P), ("d_pos", _P), ("n_pos", _I), ("rot_dim", _I), ("layout", _I)]

    def __init__(self, cos, sin, pos, n_pos, rot_dim, layout="half"):
        dev, n, rows = _device(), n_pos * (rot_dim // 2), 0 if pos is None else pos.numel()
        super().__init__(_dev_ptr(cos, _i64, dev, "cos", n), _dev_ptr(sin, _i64, dev, "sin", n),
                         _dev_ptr(pos, _i32, dev, "pos", rows), n_pos, rot_dim, ROPE_LAYOUT[layout])
        self.keep = (cos, sin, pos)
        self.dev = None if cos is None else dev
        self.rows = rows


def rope_dev(out, x, rope, rows, heads, head_dim, x_stride=None, out_stride=None, stream=None):
    dev, w = _device(), heads * head_dim
    xs, outs = w if x_stride is None else x_stride, w if out_stride is None else out_stride
    _call("iq_rope_dev", _dev_ptr(out, _i64, dev, "out", (rows - 1) * outs + w, w, rows, outs),
          _dev_ptr(x, _i64, dev, "x", (rows - 1) * xs + w, w, rows, xs),
          _ref(rope, dev, rows), rows, heads, head_dim, xs, outs, _cur(stream, dev))


class KVCache(ctypes.Structure):
    """iq_kv_cache over the caller's tensors: k and v (exact), or kq, vq, k_mag, v_mag with k_bits and v_bits."""
    _fields_ = [("seqs", _I), ("max_seq", _I), ("kv_heads", _I), ("head_dim", _I), ("k_bits", _I), ("v_bits", _I),
                ("k", _P), ("v", _P), ("kq", _P), ("vq", _P), ("k_mag", _P), ("v_mag", _P)]

    def __init__(self, seqs, max_seq, kv_heads, head_dim, k=None, v=None, kq=None, vq=None, k_mag=None, v_mag=None,
                 k_bits=0, v_bits=0):
        dev, m = _device(), seqs * max_seq * kv_heads
        n = m * head_dim
        super().__init__(seqs, max_seq, kv_heads, head_dim, k_bits, v_bits, _dev_ptr(k, _i64, dev, "k", n),
                         _dev_ptr(v, _i64, dev, "v", n), _dev_ptr(kq, _i8, dev, "kq", n),
                         _dev_ptr(vq, _i16, dev, "vq", n), _dev_ptr(k_mag, _i64, dev, "k_mag", m),
                         _dev_ptr(v_mag, _i64, dev, "v_mag", m))
        self.keep = (k, v, kq, vq, k_mag, v_mag)
        self.dev = None if k is None and kq is None else dev


def kv_write_dev(cache, k, v, slot, rows, seq=None, rope=None, k_stride=None, v_stride=None, stream=None):
    dev, w = _device(), cache.kv_heads * cache.head_dim
    ks, vs = w if k_stride is None else k_stride, w if v_stride is None else v_stride
    _call("iq_kv_write_dev", _ref(cache, dev), _dev_ptr(k, _i64, dev, "k", (rows - 1) * ks + w, w, rows, ks),
          _dev_ptr(v, _i64, dev, "v", (rows - 1) * vs + w, w, rows, vs), _dev_ptr(seq, _i32, dev, "seq", rows),
          _dev_ptr(slot, _i32, dev, "slot", rows), rows, ks, vs, None if rope is None else _ref(rope, dev, rows),
          _cur(stream, dev))


def kv_read_dev(k, v, cache, slot, rows, seq=None, stream=None):
    dev, n = _device(), rows * cache.kv_heads * cache.head_dim
    _call("iq_kv_read_dev", _dev_ptr(k, _i64, dev, "k", n), _dev_ptr(v, _i64, dev, "v", n), _ref(cache, dev),
          _dev_ptr(seq, _i32, dev, "seq", rows), _dev_ptr(slot, _i32, dev, "slot", rows), rows, _cur(stream, dev))


def attn_tree_work(cache, num_heads, n_seq, rows, max_nodes, max_len):
    """Workspace bytes of attn_tree_dev."""
    n = _I64()
    _call("iq_attn_tree_work", ctypes.byref(cache), num_heads, n_seq, rows, max_nodes, max_len, ctypes.byref(n))
    return n.value


def attn_tree_dev(out, q, cache, num_heads, lens, starts, parents, n_seq, rows, max_nodes, max_len, work=None,
                  seqs=None, q_stride=None, stream=None):
    """Tree attention; work: a contiguous device tensor of at least attn_tree_work(...) bytes."""
    dev, w = _device(), num_heads * cache.head_dim
    qs = w if q_stride is None else q_stride
    n = nbytes = 0
    if work is not None:
        n = work.numel()
        nbytes = n * work.element_size()
    _call("iq_attn_tree_dev", _dev_ptr(out, _i64, dev, "out", rows * w),
          _dev_ptr(q, _i64, dev, "q", (rows - 1) * qs + w, w, rows, qs), _ref(cache, dev), num_heads,
          _dev_ptr(seqs, _i32, dev, "seqs", n_seq), _dev_ptr(lens, _i32, dev, "lens", n_seq),
          _dev_ptr(starts, _i32, dev, "starts", n_seq + 1), _dev_ptr(parents, _i32, dev, "parents", rows), n_seq, rows,
          max_nodes, max_len, qs, None if work is None else _dev_ptr(work, (work.dtype,), dev, "work", n), nbytes,
          _cur(stream, dev))


def logprobs_dev(logits, rows, vocab, tokens=None, logp=None, entropy=None, top=0, top_ids=None, top_logp=None,
                 ld=None, stream=None):
    dev, ld = _device(), vocab if ld is None else ld
    _call("iq_logprobs_dev", _dev_ptr(logits, _i64, dev, "logits", (rows - 1) * ld + vocab, vocab, rows, ld), ld, rows,
          vocab, _dev_ptr(tokens, _i32, dev, "tokens", rows), _dev_ptr(logp, _i64, dev, "logp", rows),
          _dev_ptr(entropy, _i64, dev, "entropy", rows), top, _dev_ptr(top_ids, _i32, dev, "top_ids", rows * top),
          _dev_ptr(top_logp, _i64, dev, "top_logp", rows * top), _cur(stream, dev))


# --------------------------------------------------------- synthetic inputs

def synth_weights(cfg, name, shape):
    a = np.empty(shape, dtype=np.int64)
    _call("iq_synth_weights", lib().iq_tensor_seed(cfg, name.encode()), _hp(a), a.size)
    return a


def synth_acts(cfg, name, shape):
    a = np.empty(shape, dtype=np.int64)
    _call("iq_synth_acts", lib().iq_tensor_seed(cfg, name.encode()), _hp(a), a.size)
    return a


def synth_tokens(cfg, name, n, vocab):
    a = np.empty(n, dtype=np.int32)
    _call("iq_synth_tokens", lib().iq_tensor_seed(cfg, name.encode()), _hp(a), n, vocab)
    return a


# ------------------------------------------------------------------- model

class Config(ctypes.Structure):
    """iq_config (llama_config_t, llama_int.c:788-798)."""
    _fields_ = [(n, ctypes.c_int) for n in ("hidden_dim", "num_heads", "num_kv_heads", "head_dim",
                                             "num_layers", "intermediate_dim", "vocab_size",
                                             "max_seq_len", "rope_theta")]

    @classmethod
    def from_dict(cls, c):
        return cls(c["dim"], c["n_heads"], c["n_kv_heads"], c["head_dim"], c["n_layers"], c["inter"],
                   c["vocab"], c["max_seq"], c["rope_theta"])


class Model:
    """Device-resident integer Llama (iq_model_*): forward / generate with the
    reference's semantics (llama_forward, generate in llama_int.c)."""

    def __init__(self, cfg, max_batch=1, device=0, tp_rank=0, tp_size=1, nccl_id=None):
        self.cfg = cfg if isinstance(cfg, Config) else Config.from_dict(cfg)
        self.max_batch = max_batch
        self.h = ctypes.c_void_p()
        if tp_size == 1:
            _call("iq_model_create", ctypes.byref(self.cfg), max_batch, device, ctypes.byref(self.h))
        else:
            idbuf = ctypes.create_string_buffer(bytes(nccl_id), 128)
            _call("iq_model_create_tp", ctypes.byref(self.cfg), max_batch, device, tp_rank, tp_size,
                  idbuf, ctypes.byref(self.h))

    def close(self):
        if self.h:
            h, self.h = self.h, ctypes.c_void_p()   # the handle is gone even when destroy reports an error
            _call("iq_model_destroy", h)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def load(self, w):
        """w: dict(embed, final_norm, lm_head, layers=[9 arrays per layer])."""
        _call("iq_model_load_globals", self.h, _hp(w["embed"]), _hp(w["final_norm"]), _hp(w["lm_head"]))
        for l, lay in enumerate(w["layers"]):
            arr = (ctypes.c_void_p * 9)(*[a.ctypes.data for a in lay])
            _call("iq_model_load_layer", self.h, l, arr)

    def load_mgw(self, path):
        """Every tensor from an int-llm .mgw file (iq_model_load_mgw)."""
        _call("iq_model_load_mgw", self.h, os.fsencode(path))

    def synth(self, config_index, threads=None):
        _call("iq_model_synth", self.h, config_index, threads or os.cpu_count() or 1)

    def reset(self):
        _call("iq_model_reset", self.h)

    def forward(self, token, pos, want_logits=True):
        lg = np.empty(self.cfg.vocab_size, dtype=np.int64) if want_logits else None
        a = ctypes.c_int(-1)
        _call("iq_forward", self.h, token, pos, _hp(lg) if want_logits else None, ctypes.byref(a))
        return a.value, lg

    def generate(self, prompt, max_new, logit_hash=False):
        pr = np.ascontiguousarray(prompt, dtype=np.int32)
        out = np.zeros(len(pr) + max_new, dtype=np.int32)
        n = ctypes.c_int(0)
        h = ctypes.c_uint64(0)
        _call("iq_generate", self.h, _hp(pr), len(pr), max_new, _hp(out), ctypes.byref(n),
              ctypes.byref(h) if logit_hash else None)
        return out[:n.value].tolist(), (h.value if logit_hash else None)

    def generate_sampled(self, prompt, max_new, temperature, top_k, top_p, seed, logit_hash=False):
        """generate() with sample_token (temperature / top_p in Q16.48)."""
        pr = np.ascontiguousarray(prompt, dtype=np.int32)
        out = np.zeros(len(pr) + max_new, dtype=np.int32)
        n = ctypes.c_int(0)
        h = ctypes.c_uint64(0)
        _call("iq_generate_sampled", self.h, _hp(pr), len(pr), max_new, temperature, top_k, top_p, seed, _hp(out),
              ctypes.byref(n), ctypes.byref(h) if logit_hash else None)
        return out[:n.value].tolist(), (h.value if logit_hash else None)

    def generate_batch(self, prompts, max_new, logit_hash=False):
        """Tokens per sequence; with logit_hash=True also the per-sequence hashes."""
        pr = np.ascontiguousarray(prompts, dtype=np.int32)
        B, L = pr.shape
        assert B == self.max_batch
        out = np.zeros((B, L + max_new), dtype=np.int32)
        n = np.zeros(B, dtype=np.int32)
        hs = np.zeros(B, dtype=np.uint64)
        _call("iq_generate_batch", self.h, _hp(pr), L, max_new, _hp(out), _hp(n), _hp(hs) if logit_hash else None)
        toks = [out[b, :n[b]].tolist() for b in range(B)]
        return (toks, [int(h) for h in hs]) if logit_hash else toks

    def set_attention(self, short_max):
        """Contexts up to short_max use the single-kernel attention (0 = phased only)."""
        _call("iq_model_set_attention", self.h, short_max)

    PEER_CHECK = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p)

    def set_peer_check(self, fn):
        """fn() -> bool, True when another tensor-parallel rank has left; checked
        before every call that launches work (iq_model_set_peer_check)."""
        self._peer_cb = self.PEER_CHECK(lambda _ctx: 1 if fn() else 0) if fn else None
        _call("iq_model_set_peer_check", self.h,
              ctypes.cast(self._peer_cb, ctypes.c_void_p) if fn else None, None)

    def set_timeout(self, ms):
        _call("iq_model_set_timeout", self.h, int(ms))

    def set_kv_packed(self, k_bits, v_bits):
        """The reference's --kv-packed KbVb cache (0, 0 = exact)."""
        _call("iq_model_set_kv_packed", self.h, k_bits, v_bits)

    def set_decode(self, mode):
        """1 = persistent decode kernel where it applies (default), 0 = one kernel per op."""
        _call("iq_model_set_decode", self.h, mode)

    def decode_info(self):
        """(persistent kernel in use, its grid size)."""
        a, b = ctypes.c_int(), ctypes.c_int()
        _call("iq_model_decode_info", self.h, ctypes.byref(a), ctypes.byref(b))
        return bool(a.value), b.value

    def weight_bytes(self):
        """(decode bytes per token, GEMM-form bytes) of this rank's stored weights."""
        d, g = ctypes.c_int64(), ctypes.c_int64()
        _call("iq_model_weight_bytes", self.h, ctypes.byref(d), ctypes.byref(g))
        return d.value, g.value

    def decode_steps_timed(self, pos0, steps):
        ms = ctypes.c_float(0)
        _call("iq_decode_steps_timed", self.h, pos0, steps, ctypes.byref(ms))
        return ms.value
