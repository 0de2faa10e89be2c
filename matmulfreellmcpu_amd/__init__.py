"""MI355X (gfx950) HGRN-Bit engine: Python binding of the C ABI in include/mmfree_hip.h.

The engine itself is libmmfree_hip.so (HIP kernels + C ABI) with the C++17 ``mmfree`` API
above it; this module is the ctypes plumbing that the tests and bench.py use. There is no
fallback: if the library is not built, or no gfx950 device is present, ``Engine()`` raises.

Device buffers for the operator entry points are raw device addresses (ints: the tests
and bench.py allocate them with the library's own ``mmf_malloc`` and fill them with
``mmf_upload``) or any object with a ``data_ptr()`` method on the same device. Nothing here
imports torch: torch's bundled HIP runtime cannot open a device that this library's runtime
already holds in the same process.
"""
from __future__ import annotations

import ctypes as C
import os
from array import array
from struct import Struct

import numpy as np

from .blob import Blob, Config, read_blob, LAYER_PROJS  # noqa: F401

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "_lib", "libmmfree_hip.so")
MKBLOB = os.path.join(HERE, "_lib", "mmfree-mkblob")

FLOAT, FIXED_Q510, INT8_ABSMAX = 0, 1, 2
F32, BF16, F16, I8 = 0, 1, 2, 3  # row types of the layer operators
ACT_NONE, ACT_SIGMOID, ACT_SILU = 0, 1, 2  # of block_norm_q8's gate
MODES = {"float": FLOAT, "fixed": FIXED_Q510, "int8": INT8_ABSMAX}

_vp = C.c_void_p
_sz = C.c_size_t
_i64p = C.POINTER(C.c_int64)
_fp = C.POINTER(C.c_float)


class MmfConfig(C.Structure):
    _fields_ = [("vocab_size", _sz), ("hidden_size", _sz), ("num_hidden_layers", _sz),
                ("intermediate_size", _sz), ("use_lower_bound", C.c_int), ("rms_norm_eps", C.c_float)]


# mmf_scan_args: dtype, softplus; eleven pointers (out ... lens); ten sizes (seqs ... ldz). Packed at once, as a
# ctypes.Structure of as many fields takes longer than the launch.
_SCAN_ARGS = Struct("@2i21Q")

# mmf_decay_args: dtype, scale; eight pointers; thirteen sizes. mmf_block_args: dtype, act; ten pointers; eight sizes; scale,
# eps. mmf_logp_args: dtype, temperature; six pointers; four sizes.
_DECAY_ARGS, _BLOCK_ARGS, _LOGP_ARGS = Struct("@if21Q"), Struct("@2i18Q2f"), Struct("@if10Q")

TOKEN_CB = C.CFUNCTYPE(None, _vp, C.c_int64)

_lib = None


def load_library(path: str = LIB_PATH):
    """Load libmmfree_hip.so (raises if it is not built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise RuntimeError(f"{path} is not built: run `python -c 'import __graft_entry__ as g; g.build()'`")
    L = C.CDLL(path)
    i = C.c_int
    sig = {
        "mmf_create": (i, [C.POINTER(_vp), i]),
        "mmf_destroy": (None, [_vp]),
        "mmf_last_error": (C.c_char_p, [_vp]),
        "mmf_sync": (i, [_vp]),
        "mmf_stream": (_vp, [_vp]),
        "mmf_device_info": (i, [_vp, C.c_char_p, _sz, C.POINTER(i)]),
        "mmf_malloc": (i, [_vp, C.POINTER(_vp), _sz]),
        "mmf_free": (i, [_vp, _vp]),
        "mmf_upload": (i, [_vp, _vp, _vp, _sz]),
        "mmf_download": (i, [_vp, _vp, _vp, _sz]),
        "mmf_proj_register": (i, [_vp, _vp, _sz, _sz, C.c_float, _vp, C.POINTER(i)]),
        "mmf_proj_shape": (i, [_vp, i, C.POINTER(_sz), C.POINTER(_sz)]),
        "mmf_ternary_matmul": (i, [_vp, i, _vp, _vp, _sz]),
        "mmf_ternary_matmul_host": (i, [_vp, i, C.POINTER(i), C.POINTER(_vp), C.POINTER(_vp), _sz]),
        "mmf_proj_release": (i, [_vp, i]),
        "mmf_workspace_bytes": (i, [_vp, C.POINTER(_sz)]),
        "mmf_bitlinear": (i, [_vp, i, i, i, C.c_float, _vp, _vp, _sz, _vp]),
        "mmf_bitlinear_noalloc": (i, [_vp, i, i, i, C.c_float, _vp, _vp, _sz, _vp]),
        "mmf_bitlinear_cluster": (i, [_vp, C.POINTER(i), i, i, i, C.c_float, _vp, C.POINTER(_vp), _sz]),
        "mmf_rmsnorm": (i, [_vp, _vp, _vp, _vp, _sz, _sz, C.c_float]),
        "mmf_swiglu": (i, [_vp, _vp, _vp, _vp, _sz]),
        "mmf_hgrn_scan": (i, [_vp, _vp, _vp, _vp, _sz, _sz, _vp]),
        "mmf_rmsnorm_swishgate": (i, [_vp, _vp, _vp, _vp, _vp, _sz, _sz, C.c_float]),
        "mmf_add_rmsnorm_q8": (i, [_vp, i] + [_vp] * 7 + [_sz] * 7 + [C.c_float]),
        "mmf_w4_register": (i, [_vp, _vp, _vp, _vp, _sz, _sz, _sz, C.POINTER(i)]),
        "mmf_w4_shape": (i, [_vp, i, C.POINTER(_sz), C.POINTER(_sz), C.POINTER(_sz)]),
        "mmf_w4_release": (i, [_vp, i]),
        "mmf_w4_linear": (i, [_vp, i, i, _vp, _vp, i, _vp, _sz, _sz, _sz]),
        "mmf_short_conv": (i, [_vp, i] + [_vp] * 6 + [_sz] * 4 + [i, _sz, _sz]),
        "mmf_selective_scan": (i, [_vp, C.c_char_p]),
        "mmf_w8_register": (i, [_vp, _vp, _vp, _sz, _sz, C.POINTER(i)]),
        "mmf_w8_shape": (i, [_vp, i, C.POINTER(_sz), C.POINTER(_sz)]),
        "mmf_w8_release": (i, [_vp, i]),
        "mmf_w8_linear": (i, [_vp, i, _vp, _vp, _vp, i, _vp, _sz, _sz, _sz]),
        "mmf_decay_attention": (i, [_vp, C.c_char_p]),
        "mmf_block_norm_q8": (i, [_vp, C.c_char_p]),
        "mmf_token_logprobs": (i, [_vp, C.c_char_p]),
        "mmf_model_score": (i, [_vp, _i64p, _sz, _fp, _fp, _sz, _i64p, _fp]),
        "mmf_model_begin": (i, [_vp, C.POINTER(MmfConfig)]),
        "mmf_model_tensor": (i, [_vp, C.c_char_p, i, C.POINTER(_sz), i, _vp]),
        "mmf_model_finalize": (i, [_vp, i, i]),
        "mmf_model_config": (i, [_vp, C.POINTER(MmfConfig)]),
        "mmf_model_generate": (i, [_vp, _i64p, _sz, _sz, C.c_int64, _i64p, _sz, C.POINTER(_sz), TOKEN_CB, _vp]),
        "mmf_model_reset": (i, [_vp, _sz]),
        "mmf_model_prefill": (i, [_vp, _sz, _i64p, _sz, _fp, _i64p]),
        "mmf_model_prefill_streams": (i, [_vp, _sz, _i64p, C.POINTER(C.c_size_t), _fp, _i64p]),
        "mmf_model_step": (i, [_vp, _i64p, _fp, _i64p]),
        "mmf_model_state": (i, [_vp, _fp]),
        "mmf_model_set_scan": (i, [_vp, i]),
        "mmf_model_time_step": (i, [_vp, _i64p, i, i, C.POINTER(C.c_double)]),
        "mmf_model_forward": (i, [_vp, _i64p, _sz, _fp]),
        "mmf_model_trace": (i, [_vp, _i64p, _sz, _fp, _fp, _fp]),
        "mmf_model_time_decode": (i, [_vp, i, i, C.POINTER(C.c_double), C.POINTER(C.c_double)]),
        "mmf_model_time_prefill": (i, [_vp, _i64p, _sz, i, i, C.POINTER(C.c_double), C.POINTER(C.c_double)]),
        "mmf_time_bitlinear": (i, [_vp, i, i, i, C.c_float, _vp, _vp, _sz, i, i, C.POINTER(C.c_double),
                                   C.POINTER(C.c_double), C.POINTER(C.c_double)]),
        "mmf_measure_peaks": (i, [_vp, C.POINTER(C.c_double)]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    _lib = L
    return L


class MmfError(RuntimeError):
    pass


def _ptr(x):
    """Device address of an int, or of an object with data_ptr(), or None."""
    if x is None:
        return None
    if isinstance(x, int):
        return x
    return x.data_ptr()


# Row types of tensors' dtypes by name; -1: of none. Other dtypes (bytes, 16-bit words) are taken as storage.
_ROW_TYPES = {"float32": F32, "bfloat16": BF16, "float16": F16, "int8": I8, "float64": -1}
_row_types = {}  # the same by dtype object, entered as they are met


def _row_type(x):
    """The row type of a tensor, or None of an address or of storage."""
    d = getattr(x, "dtype", None)
    if d not in _row_types:
        _row_types[d] = _ROW_TYPES.get(str(d).rpartition(".")[2])
    return _row_types[d]


def _rows(x, t):
    """As _ptr, of rows of type t: a tensor of another type is refused."""
    if x is None or x.__class__ is int:
        return x
    try:
        if _row_types[x.dtype] == t:
            return x.data_ptr()
    except (AttributeError, KeyError):
        pass
    if _row_type(x) not in (t, None):
        raise ValueError(f"a tensor of {x.dtype} in the place of rows of type {t} (F32, BF16, F16, I8 = 0, 1, 2, 3)")
    return _ptr(x)


def _own_type(x):
    """The row type of a tensor; an address alone is of F32."""
    return F32 if x.__class__ is int else max(_row_type(x) or F32, F32)


_id_types = {}  # whether a dtype object is int64, entered as they are met


def _ids(x):
    """As _ptr, of 64-bit integers: a tensor of another type is refused."""
    if x is None or x.__class__ is int:
        return x
    d = getattr(x, "dtype", None)
    if d not in _id_types:
        _id_types[d] = d is None or str(d).rpartition(".")[2] == "int64"
    if not _id_types[d]:
        raise ValueError(f"a tensor of {d} in the place of int64 ids")
    return _ptr(x)


def _np(a, dtype):
    a = np.ascontiguousarray(a, dtype=dtype)
    return a, a.ctypes.data_as(C.c_void_p)


def _lens(lens, seqs):
    """(sequence lengths as size_t array or None, its address, the number of sequences)."""
    if lens is None:
        return None, None, seqs
    a = array("Q", lens)
    return a, a.buffer_info()[0], len(a)


class Engine:
    """One engine context on one GPU (mmf_create)."""

    def __init__(self, device: int = 0):
        self.lib = load_library()
        h = _vp()
        rc = self.lib.mmf_create(C.byref(h), device)
        if rc != 0:
            raise MmfError(f"mmf_create failed ({rc}): {self.lib.mmf_last_error(None).decode()}")
        self.h = h
        self.cfg = None
        self._cb = None

    def close(self):
        if getattr(self, "h", None):
            self.lib.mmf_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _chk(self, rc):
        if rc != 0:
            raise MmfError(f"mmf error {rc}: {self.lib.mmf_last_error(self.h).decode()}")

    def sync(self):
        self._chk(self.lib.mmf_sync(self.h))

    @property
    def stream(self) -> int:
        return self.lib.mmf_stream(self.h) or 0

    def device_info(self):
        buf = C.create_string_buffer(256)
        cus = C.c_int()
        self._chk(self.lib.mmf_device_info(self.h, buf, 256, C.byref(cus)))
        return buf.value.decode(), cus.value

    # ---- projections / operators ----
    def register_proj(self, wq, scale_w: float, normw=None) -> int:
        wq, wp = _np(wq, np.int8)
        nw = None
        if normw is not None:
            nwa, nw = _np(normw, np.float32)
        pid = C.c_int()
        self._chk(self.lib.mmf_proj_register(self.h, wp, wq.shape[0], wq.shape[1], float(scale_w), nw,
                                             C.byref(pid)))
        return pid.value

    def proj_shape(self, pid):
        n, k = _sz(), _sz()
        self._chk(self.lib.mmf_proj_shape(self.h, pid, C.byref(n), C.byref(k)))
        return n.value, k.value

    def bitlinear(self, pid, x, out, rows, mode=FLOAT, frac_bits=10, eps=1e-6, acc=None):
        self._chk(self.lib.mmf_bitlinear(self.h, pid, mode, frac_bits, eps, _ptr(x), _ptr(out), rows, _ptr(acc)))

    def bitlinear_noalloc(self, pid, x, out, rows, mode=FLOAT, frac_bits=10, eps=1e-6, acc=None):
        """mmf_bitlinear with its scratch in the library's static device array (no allocation)."""
        self._chk(self.lib.mmf_bitlinear_noalloc(self.h, pid, mode, frac_bits, eps, _ptr(x), _ptr(out), rows,
                                                 _ptr(acc)))

    def bitlinear_cluster(self, pids, x, outs, rows, mode=FLOAT, frac_bits=10, eps=1e-6):
        k = len(pids)
        ids = (C.c_int * k)(*pids)
        op = (_vp * k)(*[_ptr(o) for o in outs])
        self._chk(self.lib.mmf_bitlinear_cluster(self.h, ids, k, mode, frac_bits, eps, _ptr(x), op, rows))

    def ternary_matmul(self, pid, x, acc, b):
        self._chk(self.lib.mmf_ternary_matmul(self.h, pid, _ptr(x), _ptr(acc), b))

    def ternary_matmul_host(self, pids, xs):
        """k projections on host arrays in one round trip: xs[z] int32 [b, K_z] -> int32 [b, N_z]."""
        k = len(pids)
        b = xs[0].shape[0]
        xs = [np.ascontiguousarray(x, np.int32) for x in xs]
        accs = [np.zeros((b, self.proj_shape(p)[0]), np.int32) for p in pids]
        ids = (C.c_int * k)(*pids)
        xp = (_vp * k)(*[x.ctypes.data for x in xs])
        ap = (_vp * k)(*[a.ctypes.data for a in accs])
        self._chk(self.lib.mmf_ternary_matmul_host(self.h, k, ids, xp, ap, b))
        return accs

    def proj_release(self, pid):
        self._chk(self.lib.mmf_proj_release(self.h, pid))

    def workspace_bytes(self):
        n = _sz()
        self._chk(self.lib.mmf_workspace_bytes(self.h, C.byref(n)))
        return n.value

    def rmsnorm(self, y, x, w, rows, cols, eps=1e-6):
        self._chk(self.lib.mmf_rmsnorm(self.h, _ptr(y), _ptr(x), _ptr(w), rows, cols, eps))

    def swiglu(self, out, a, b, n):
        self._chk(self.lib.mmf_swiglu(self.h, _ptr(out), _ptr(a), _ptr(b), n))

    def hgrn_scan(self, out, i, f, T, D, state=None):
        self._chk(self.lib.mmf_hgrn_scan(self.h, _ptr(out), _ptr(i), _ptr(f), T, D, _ptr(state)))

    def rmsnorm_swishgate(self, out, g, o, w, rows, cols, eps=1e-6):
        self._chk(self.lib.mmf_rmsnorm_swishgate(self.h, _ptr(out), _ptr(g), _ptr(o), _ptr(w), rows, cols, eps))

    # ---- layer operators: rows of dtype F32, BF16 or F16 (None: the first input's own, F32 for an address; tensors of
    # another type are refused), strides in elements (0: the row's length) ----
    def add_rmsnorm_q8(self, codes, scales, x, w, rows, cols, res=None, h=None, y=None, eps=1e-6, dtype=None, ldx=0,
                       ldres=0, ldh=0, ldy=0, ldcodes=0):
        """h = x + res, its RMS norm as int8 codes with a scale per row (mmf_add_rmsnorm_q8)."""
        t = _own_type(x) if dtype is None else dtype
        rc = self.lib.mmf_add_rmsnorm_q8(self.h, t, _rows(codes, I8), _ptr(scales), _rows(x, t), _rows(res, t), _rows(h, t),
                                         _rows(y, t), _ptr(w), rows, cols, ldx, ldres, ldh, ldy, ldcodes, eps)
        if rc:
            self._chk(rc)

    def register_w4(self, codes, scales, zeros=None, K=None, group=128) -> int:
        """4-bit weights: codes uint8 [N, ceil(K/2)], scales float16 and zeros uint8 (or None: 8) [N, ceil(K/group)]."""
        codes, cp = _np(codes, np.uint8)
        scales, sp = _np(scales, np.float16)
        N, K = codes.shape[0], 2 * codes.shape[1] if K is None else K
        if group < 0:
            raise ValueError(f"group {group} is negative")
        groups = -(-K // group) if group else 1
        if codes.shape != (N, (K + 1) // 2) or scales.shape != (N, groups):
            raise ValueError(f"codes {codes.shape} and scales {scales.shape} are not those of {N} x {K} in groups of {group}")
        zp = None
        if zeros is not None:
            zeros, zp = _np(zeros, np.uint8)
            if zeros.shape != scales.shape:
                raise ValueError(f"zeros {zeros.shape} differ from scales {scales.shape}")
        wid = C.c_int()
        self._chk(self.lib.mmf_w4_register(self.h, cp, sp, zp, N, K, group, C.byref(wid)))
        return wid.value

    def w4_shape(self, wid):
        n, k, g = _sz(), _sz(), _sz()
        self._chk(self.lib.mmf_w4_shape(self.h, wid, C.byref(n), C.byref(k), C.byref(g)))
        return n.value, k.value, g.value

    def w4_release(self, wid):
        self._chk(self.lib.mmf_w4_release(self.h, wid))

    def w4_linear(self, wid, x, out, rows, dtype=None, out_dtype=None, scales=None, ldx=0, ldo=0):
        """out [rows, N] = x [rows, K] times 4-bit weights; dtype I8: codes with their scales [rows]."""
        t = _own_type(x) if dtype is None else dtype
        o = _own_type(out) if out_dtype is None else out_dtype
        rc = self.lib.mmf_w4_linear(self.h, wid, t, _rows(x, t), _ptr(scales), o, _rows(out, o), rows, ldx, ldo)
        if rc:
            self._chk(rc)

    def short_conv(self, out, x, w, rows, D, width, bias=None, state=None, lens=None, seqs=1, silu=True, dtype=None,
                   ldx=0, ldo=0):
        """Short causal convolution of sequences of the lengths lens (None: `seqs` equal ones)."""
        _keep, lp, n = _lens(lens, seqs)
        t = _own_type(x) if dtype is None else dtype
        rc = self.lib.mmf_short_conv(self.h, t, _rows(out, t), _rows(x, t), _ptr(w), _ptr(bias), _ptr(state), lp, n, rows,
                                     D, width, int(silu), ldx, ldo)
        if rc:
            self._chk(rc)

    def selective_scan(self, out, u, dt, A, B, C, rows, D, N, skip=None, z=None, dt_bias=None, state=None, lens=None,
                       seqs=1, softplus=True, dtype=None, ldo=0, ldu=0, lddt=0, ldb=0, ldc=0, ldz=0):
        """Selective state space scan of sequences of the lengths lens (None: `seqs` equal ones)."""
        _keep, lp, n = _lens(lens, seqs)
        t = _own_type(u) if dtype is None else dtype
        up = _rows(u, t) or 0
        d = getattr(u, "dtype", None)
        k = None if d is None else u.__class__  # a tensor like u is of u's type: no call for each
        a = _SCAN_ARGS.pack(t, bool(softplus),
                            out.data_ptr() if out.__class__ is k and out.dtype is d else _rows(out, t) or 0, up,
                            dt.data_ptr() if dt.__class__ is k and dt.dtype is d else _rows(dt, t) or 0,
                            B.data_ptr() if B.__class__ is k and B.dtype is d else _rows(B, t) or 0,
                            C.data_ptr() if C.__class__ is k and C.dtype is d else _rows(C, t) or 0,
                            z.data_ptr() if z.__class__ is k and z.dtype is d else _rows(z, t) or 0,
                            _ptr(A) or 0, _ptr(skip) or 0, _ptr(dt_bias) or 0, _ptr(state) or 0, lp or 0, n, rows, D, N,
                            ldo, ldu, lddt, ldb, ldc, ldz)
        rc = self.lib.mmf_selective_scan(self.h, a)
        if rc:
            self._chk(rc)

    def register_w8(self, codes, scales) -> int:
        """8-bit weights: codes int8 [N, K], scales float32 [N]."""
        given = np.asarray(codes)
        with np.errstate(invalid="ignore"):
            codes, cp = _np(given, np.int8)
        if given.dtype != np.int8 and not np.array_equal(codes, given):
            raise ValueError(f"codes of {given.dtype} that are no int8 numbers")
        scales, sp = _np(scales, np.float32)
        if codes.ndim != 2 or scales.shape != codes.shape[:1]:
            raise ValueError(f"codes {codes.shape} and scales {scales.shape} are not [N, K] and [N]")
        wid = C.c_int()
        self._chk(self.lib.mmf_w8_register(self.h, cp, sp, codes.shape[0], codes.shape[1], C.byref(wid)))
        return wid.value

    def w8_shape(self, wid):
        n, k = _sz(), _sz()
        self._chk(self.lib.mmf_w8_shape(self.h, wid, C.byref(n), C.byref(k)))
        return n.value, k.value

    def w8_release(self, wid):
        self._chk(self.lib.mmf_w8_release(self.h, wid))

    def w8_linear(self, wid, x, scales, out, rows, bias=None, out_dtype=None, ldx=0, ldo=0):
        """out [rows, N] = int8 codes x [rows, K] with scales [rows] times 8-bit weights, plus bias [N] (mmf_w8_linear)."""
        o = _own_type(out) if out_dtype is None else out_dtype
        rc = self.lib.mmf_w8_linear(self.h, wid, _rows(x, I8), _rows(scales, F32), _rows(bias, F32), o, _rows(out, o), rows,
                                    ldx, ldo)
        if rc:
            self._chk(rc)

    def decay_attention(self, out, q, k, v, rows, heads, Dk, Dv, decay=None, gates=None, state=None, lens=None, seqs=1,
                        q_heads=0, k_heads=0, v_heads=0, scale=None, dtype=None, ldo=0, ldq=0, ldk=0, ldv=0, ldg=0):
        """Linear attention with a decay for each head, of sequences of the lengths lens (None: `seqs` equal ones); decay
        [heads] and gates [rows, heads] are log decays, scale None is Dk ** -0.5 (mmf_decay_attention)."""
        _keep, lp, n = _lens(lens, seqs)
        t = _own_type(q) if dtype is None else dtype
        a = _DECAY_ARGS.pack(t, max(Dk, 1) ** -0.5 if scale is None else scale, _rows(out, t) or 0, _rows(q, t) or 0, _rows(k, t) or 0,
                             _rows(v, t) or 0, _rows(decay, F32) or 0, _rows(gates, F32) or 0, _rows(state, F32) or 0, lp or 0,
                             n, rows, heads, q_heads, k_heads, v_heads, Dk, Dv, ldo, ldq, ldk, ldv, ldg)
        rc = self.lib.mmf_decay_attention(self.h, a)
        if rc:
            self._chk(rc)

    def block_norm_q8(self, codes, scales, b, rows, cols, x=None, gate=None, act=ACT_NONE, w_post=None, w_pre=None,
                      channels=None, scale=1.0, h=None, y=None, eps=1e-6, dtype=None, ldb=0, ldx=0, ldgate=0, ldh=0, ldy=0,
                      ldcodes=0):
        """h = x + scale * channels * act(gate) * norm(b) w_post, then norm(h) w_pre as y and as int8 codes with a scale per
        row; codes and scales may both be None (mmf_block_norm_q8)."""
        t = _own_type(b) if dtype is None else dtype
        a = _BLOCK_ARGS.pack(t, act, _rows(b, t) or 0, _rows(x, t) or 0, _rows(gate, t) or 0, _rows(w_post, F32) or 0,
                             _rows(w_pre, F32) or 0, _rows(channels, F32) or 0, _rows(h, t) or 0, _rows(y, t) or 0,
                             _rows(codes, I8) or 0, _rows(scales, F32) or 0, rows, cols, ldb, ldx, ldgate, ldh, ldy, ldcodes,
                             scale, eps)
        rc = self.lib.mmf_block_norm_q8(self.h, a)
        if rc:
            self._chk(rc)

    def token_logprobs(self, logits, rows, V, ids=None, logprobs=None, entropy=None, top=0, top_ids=None, top_logprobs=None,
                       temperature=1.0, dtype=None, ld=0):
        """Log probabilities of ids [rows] (int64), entropies and the `top` most likely tokens of logits [rows, V]
        (mmf_token_logprobs)."""
        t = _own_type(logits) if dtype is None else dtype
        a = _LOGP_ARGS.pack(t, temperature, _rows(logits, t) or 0, _ids(ids) or 0, _rows(logprobs, F32) or 0,
                            _rows(entropy, F32) or 0, _ids(top_ids) or 0, _rows(top_logprobs, F32) or 0, rows, V, top, ld)
        rc = self.lib.mmf_token_logprobs(self.h, a)
        if rc:
            self._chk(rc)

    # ---- model ----
    def load_blob(self, path_or_blob, mode=FLOAT, frac_bits=10):
        """Upload every tensor of an MMFREE1 blob and prepare the engine for `mode`."""
        blob = read_blob(path_or_blob) if isinstance(path_or_blob, str) else path_or_blob
        c = blob.config
        cfg = MmfConfig(c.vocab_size, c.hidden_size, c.num_hidden_layers, c.intermediate_size,
                        int(c.use_lower_bound), c.rms_norm_eps)
        self._chk(self.lib.mmf_model_begin(self.h, C.byref(cfg)))
        for name, arr in blob.tensors.items():
            a = np.ascontiguousarray(arr)
            shape = (_sz * max(a.ndim, 1))(*a.shape)
            dt = 1 if a.dtype == np.int8 else 0
            self._chk(self.lib.mmf_model_tensor(self.h, name.encode(), dt, shape, a.ndim,
                                                a.ctypes.data_as(_vp)))
        self._chk(self.lib.mmf_model_finalize(self.h, mode, frac_bits))
        self.cfg = c
        self.mode = mode
        return self

    def generate(self, ids, new_tokens, eos_id=-1, on_token=None):
        ids, ip = _np(ids, np.int64)
        cap = ids.size + new_tokens
        out = np.zeros(max(cap, 1), np.int64)
        n = _sz()
        cb = TOKEN_CB(lambda _u, t: on_token(int(t))) if on_token else TOKEN_CB()
        self._cb = cb
        self._chk(self.lib.mmf_model_generate(self.h, ids.ctypes.data_as(_i64p), ids.size, new_tokens, eos_id,
                                              out.ctypes.data_as(_i64p), cap, C.byref(n), cb, None))
        return out[:n.value].copy()

    def reset(self, streams=1):
        self._chk(self.lib.mmf_model_reset(self.h, streams))
        self.streams = streams

    def prefill(self, stream, ids, want_logits=False):
        ids = np.ascontiguousarray(ids, np.int64)
        lg = np.empty(self.cfg.vocab_size, np.float32) if want_logits else None
        am = np.zeros(1, np.int64)
        self._chk(self.lib.mmf_model_prefill(self.h, stream, ids.ctypes.data_as(_i64p), ids.size,
                                             lg.ctypes.data_as(_fp) if lg is not None else None,
                                             am.ctypes.data_as(_i64p)))
        return (int(am[0]), lg) if want_logits else int(am[0])

    def prefill_streams(self, prompts, want_logits=False):
        """Prefill streams 0..len(prompts)-1 together (mmf_model_prefill_streams): the same
        first tokens, logits and states as one prefill() per stream in order."""
        ids = np.ascontiguousarray(np.concatenate([np.asarray(p, np.int64).ravel() for p in prompts]), np.int64)
        lens = np.ascontiguousarray([len(p) for p in prompts], np.uint64)
        n = lens.size
        lg = np.empty((n, self.cfg.vocab_size), np.float32) if want_logits else None
        am = np.zeros(n, np.int64)
        self._chk(self.lib.mmf_model_prefill_streams(self.h, n, ids.ctypes.data_as(_i64p),
                                                     lens.ctypes.data_as(C.POINTER(C.c_size_t)),
                                                     lg.ctypes.data_as(_fp) if lg is not None else None,
                                                     am.ctypes.data_as(_i64p)))
        return (am, lg) if want_logits else am

    def step(self, tokens, want_logits=False):
        t = np.ascontiguousarray(tokens, np.int64)
        B = t.size
        lg = np.empty((B, self.cfg.vocab_size), np.float32) if want_logits else None
        am = np.zeros(B, np.int64)
        self._chk(self.lib.mmf_model_step(self.h, t.ctypes.data_as(_i64p),
                                          lg.ctypes.data_as(_fp) if lg is not None else None,
                                          am.ctypes.data_as(_i64p)))
        return (am, lg) if want_logits else am

    def set_scan(self, chunked: bool):
        """Float-mode prefill recurrence: time-ordered (default, bit-exact) or chunked parallel."""
        self._chk(self.lib.mmf_model_set_scan(self.h, 1 if chunked else 0))

    def state(self):
        c = self.cfg
        st = np.empty((c.num_hidden_layers, getattr(self, "streams", 1), c.hidden_size), np.float32)
        self._chk(self.lib.mmf_model_state(self.h, st.ctypes.data_as(_fp)))
        return st

    def forward(self, ids):
        ids = np.ascontiguousarray(ids, np.int64)
        lg = np.empty((ids.size, self.cfg.vocab_size), np.float32)
        self._chk(self.lib.mmf_model_forward(self.h, ids.ctypes.data_as(_i64p), ids.size, lg.ctypes.data_as(_fp)))
        return lg

    def score(self, ids, top=0):
        """(log probability of each token after the first, entropies [T-1]) of a text of T ids, and with top the most likely
        tokens: (..., their ids [T-1, top], their log probabilities). The logits stay on the device (mmf_model_score)."""
        ids = np.ascontiguousarray(ids, np.int64)
        if top < 0:
            raise ValueError(f"top {top} is negative")
        n = max(ids.size - 1, 0)
        lp, ent = np.empty(n, np.float32), np.empty(n, np.float32)
        tid, tlp = np.empty((n, top), np.int64), np.empty((n, top), np.float32)
        self._chk(self.lib.mmf_model_score(self.h, ids.ctypes.data_as(_i64p), ids.size, lp.ctypes.data_as(_fp),
                                           ent.ctypes.data_as(_fp), top, tid.ctypes.data_as(_i64p), tlp.ctypes.data_as(_fp)))
        return (lp, ent, tid, tlp) if top else (lp, ent)

    def trace(self, ids, internals=True):
        c = self.cfg
        ids = np.ascontiguousarray(ids, np.int64)
        T, H, L = ids.size, c.hidden_size, c.num_hidden_layers
        h = np.empty((L, T, H), np.float32)
        st = np.empty((L, H), np.float32)
        it = np.empty((L, 5, T, H), np.float32) if internals else None
        self._chk(self.lib.mmf_model_trace(self.h, ids.ctypes.data_as(_i64p), T, h.ctypes.data_as(_fp),
                                           st.ctypes.data_as(_fp), it.ctypes.data_as(_fp) if internals else None))
        self.streams = 1
        return h, st, it

    def time_decode(self, warmup=3, reps=20):
        step = C.c_double()
        kinds = (C.c_double * 5)()
        self._chk(self.lib.mmf_model_time_decode(self.h, warmup, reps, C.byref(step), kinds))
        return step.value, dict(zip(("ifg", "o", "gate", "down", "lm"), list(kinds)))

    PREFILL_KINDS = ("prologue", "gemm_ifg", "mixer", "gemm_o", "gemm_gate", "gemm_down", "lm", "embed")

    def time_prefill(self, ids, warmup=1, reps=3, kinds=True):
        """Microseconds per prefill (prompt through all layers + final norm/lm_head/argmax of
        the last position) and, with kinds, the microseconds per prefill of each launch kind."""
        ids, _ = _np(ids, np.int64)
        total = C.c_double()
        k = (C.c_double * 8)()
        self._chk(self.lib.mmf_model_time_prefill(self.h, ids.ctypes.data_as(_i64p), ids.size, warmup, reps,
                                                  C.byref(total), k if kinds else None))
        return total.value, (dict(zip(self.PREFILL_KINDS, list(k))) if kinds else None)

    def time_step_kinds(self, tokens, warmup=1, reps=4):
        """Microseconds per serving step in each launch kind (launches timed one by one)."""
        tokens, _ = _np(tokens, np.int64)
        k = (C.c_double * 8)()
        self._chk(self.lib.mmf_model_time_step(self.h, tokens.ctypes.data_as(_i64p), warmup, reps, k))
        return dict(zip(self.PREFILL_KINDS, list(k)))

    def measure_peaks(self):
        """Measured device ceilings: HBM and Infinity Cache read GB/s, int8 MFMA TOP/s, fp32
        FMA TFLOP/s (each from a kernel doing only that work)."""
        v = (C.c_double * 4)()
        self._chk(self.lib.mmf_measure_peaks(self.h, v))
        return {"hbm_read_GBps": round(v[0], 1), "mall_read_GBps": round(v[1], 1),
                "int8_mfma_TOPS": round(v[2], 1), "fp32_fma_TFLOPS": round(v[3], 2)}

    def time_bitlinear(self, proj_id, x, out, rows, mode=FLOAT, frac_bits=10, eps=1e-6, warmup=3, reps=20):
        """(total, prologue, gemm) microseconds per mmf_bitlinear call on device buffers."""
        t, p, g = C.c_double(), C.c_double(), C.c_double()
        self._chk(self.lib.mmf_time_bitlinear(self.h, proj_id, mode, frac_bits, eps, _ptr(x), _ptr(out), rows,
                                              warmup, reps, C.byref(t), C.byref(p), C.byref(g)))
        return t.value, p.value, g.value


def make_blob(path: str, preset: str | None = None, seed: int = 1234, vocab=None, hidden=None, layers=None,
              inter=None, random_norms=False, random_lb=False, lower_bound=True) -> str:
    """Write a seeded synthetic MMFREE1 blob with the in-tree mmfree-mkblob tool."""
    import subprocess
    if not os.path.exists(MKBLOB):
        raise RuntimeError(f"{MKBLOB} is not built")
    cmd = [MKBLOB, "--out", path, "--seed", str(seed)]
    if preset:
        cmd += ["--preset", preset]
    for flag, v in (("--vocab", vocab), ("--hidden", hidden), ("--layers", layers), ("--inter", inter)):
        if v is not None:
            cmd += [flag, str(v)]
    if random_norms:
        cmd.append("--random-norms")
    if random_lb:
        cmd.append("--random-lb")
    if not lower_bound:
        cmd.append("--no-lower-bound")
    subprocess.run(cmd, check=True, stdout=subprocess.DEVNULL)
    return path
