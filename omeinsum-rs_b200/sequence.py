"""Operators of sequence models on the B200 backend: the gated linear
recurrence (om_b200_gated_scan), the softmax cross entropy of a vocabulary's
logits (om_b200_linear_cross_entropy), both with their backward pass, and the
8-bit integer product with its row quantiser (om_b200_matmul_i8,
om_b200_quantize_rows, om_b200_linear_i8).

Every function takes the backend first and tensors that are either

  - torch CUDA tensors on the backend's device (any strides; a view with torch's
    negative bit is refused), or
  - `Strided` views of this backend's `Storage` (see `upload`),

and returns tensors of the kind it was given, row-major.  Shapes are in the
order the text names; nothing waits for the device.  torch's autograd does not
see these calls: results carry no graph, also where an input requires a gradient,
and the gradients come from the *_backward functions.

Torch tensors are ordered with torch's current stream: when the backend runs
on another stream, the call waits for the work queued on torch's stream and
torch's stream for the call (a backend made with `B200(device, stream=...)`
on torch's stream needs neither).  While the backend records a graph no
such waits are made: the tensors must be ready, and stay alive with the graph.
"""
from __future__ import annotations

import ctypes
import functools

import numpy as np

from . import BF16, DTYPES, OmError, Storage, _check, lib

F32, F64, OM_BF16, F16, I8, I32, I64 = 0, 1, 5, 6, 7, 8, 9
_NP = {v: k for k, v in DTYPES.items()}
_NAMES = {"f32": F32, "f64": F64, "bf16": OM_BF16, "f16": F16, "i8": I8, "i32": I32, "i64": I64}
_KINDS = {"linear": 0, "sigmoid": 1}
_torch = None  # the module, from the first torch tensor on
_torch_codes = {}  # torch dtype -> code
_torch_types = {}


_bound = None


def _bind():
    global _bound
    if _bound is None:
        L = lib()
        P, I = ctypes.c_void_p, ctypes.c_int
        L.om_b200_gated_scan.argtypes = [P, I, I] + [P] * 10
        L.om_b200_gated_scan_backward.argtypes = [P, I, I] + [P] * 17
        L.om_b200_linear_cross_entropy.argtypes = [P, I] + [P] * 5 + [I] + [P] * 3
        L.om_b200_linear_cross_entropy_backward.argtypes = [P, I] + [P] * 5 + [I] + [P] * 7
        L.om_b200_quantize_rows.argtypes = [P, I] + [P] * 6
        L.om_b200_matmul_i8.argtypes = [P, I] + [P] * 10
        L.om_b200_linear_i8.argtypes = [P, I] + [P] * 9
        _bound = L
    return _bound


def _invalid(msg):
    return OmError(1, msg)


class Strided:
    """A view of a Storage: shape and strides (in elements) of each axis."""

    def __init__(self, storage: Storage, shape, strides=None, offset: int = 0):
        self.storage = storage
        self.shape = tuple(int(n) for n in shape)
        if strides is None:  # row-major
            strides, s = [], 1
            for n in reversed(self.shape):
                strides.insert(0, s)
                s *= n
        self.strides = tuple(int(s) for s in strides)
        if len(self.strides) != len(self.shape):
            raise _invalid("Strided: a stride for each axis is needed")
        self.offset = int(offset)
        lo = hi = self.offset
        if all(self.shape):
            for n, s in zip(self.shape, self.strides):
                lo, hi = lo + min(0, (n - 1) * s), hi + max(0, (n - 1) * s)
            if lo < 0 or hi >= storage.n:
                raise _invalid(f"Strided: elements {lo}..{hi} of a storage of {storage.n}")

    def to_numpy(self) -> np.ndarray:
        """The values on the host (bf16 as float32)."""
        v = self.storage.to_vec()
        if self.storage.dtype == BF16:
            v = (v["bf16"].astype(np.uint32) << 16).view(np.float32)
        v = v[self.offset:]
        return np.array(np.lib.stride_tricks.as_strided(
            v, self.shape, [s * v.itemsize for s in self.strides]))


def upload(be, array, dtype: str | None = None) -> Strided:
    """A row-major device copy of a numpy array, rounded to `dtype` ("f32",
    "f64", "bf16", "f16", "i8", "i32", "i64"; default: the array's own)."""
    array = np.asarray(array)
    shape = array.shape
    if dtype == "bf16":
        bits = np.ascontiguousarray(array, dtype=np.float32).view(np.uint32).astype(np.uint64)
        nan = (bits & 0x7FFFFFFF) > 0x7F800000
        bits = (bits + 0x7FFF + ((bits >> 16) & 1)) >> 16  # to nearest, ties to even
        data = np.where(nan, 0x7FC0, bits).astype(np.uint16).reshape(-1).view(BF16)
    elif dtype is not None:
        data = array.astype(_NP[_NAMES[dtype]])
    else:
        data = array
        if data.dtype not in DTYPES:
            raise _invalid(f"upload: no device type for {data.dtype}")
    return Strided(be.from_slice(data), shape)


def _learn_torch(dtype, name):
    global _torch
    import torch
    _torch = torch
    for tt, code in ((torch.float32, F32), (torch.float64, F64), (torch.bfloat16, OM_BF16),
                     (torch.float16, F16), (torch.int8, I8), (torch.int32, I32),
                     (torch.int64, I64)):
        _torch_codes[tt] = code
        _torch_types[code] = tt
    if dtype not in _torch_codes:
        raise _invalid(f"{name}: no device type for {dtype}")
    return _torch_codes[dtype]


def _operand(be, t, name):
    """(device pointer, type code, shape, strides) of one argument."""
    if type(t) is Strided:
        s = t.storage
        if s.backend is not be:
            if s.backend.device != be.device:
                raise _invalid(f"{name}: on device {s.backend.device}, the backend on {be.device}")
            if s.backend.home_stream != be.home_stream:
                raise _invalid(f"{name}: belongs to a backend on another stream")
        return (s.ptr or 0) + t.offset * s.dtype.itemsize, DTYPES[s.dtype], t.shape, t.strides
    try:
        if t.get_device() != be.device:  # -1: not on a device at all
            raise _invalid(f"{name}: on {t.device}, the backend on cuda:{be.device}")
        if t.is_neg():
            raise _invalid(f"{name}: a view whose memory holds the negated values; call its resolve_neg()")
        return t.data_ptr(), _torch_codes[t.dtype], t.shape, t.stride()
    except KeyError:
        _learn_torch(t.dtype, name)
        return _operand(be, t, name)
    except AttributeError:
        raise _invalid(f"{name}: a Strided view or a torch CUDA tensor is needed, not {type(t).__name__}") from None


def _typed(be, t, name, ndim, codes):
    o = _operand(be, t, name)
    if len(o[2]) != ndim:
        raise _invalid(f"{name}: must have {ndim} axes")
    if o[1] not in codes:
        raise _invalid(f"{name}: type {_NP[o[1]]} not accepted here")
    return o


def _like(be, t, name, shape, code):
    o = _operand(be, t, name)
    if o[2] != shape:
        raise _invalid(f"{name}: shape {list(o[2])}, expected {list(shape)}")
    if o[1] != code:
        raise _invalid(f"{name}: type {_NP[o[1]]}, expected {_NP[code]}")
    return o


def _vector(be, t, name, shape, code):
    """Pointer of an optional contiguous operand (None: a null pointer)."""
    if t is None:
        return None
    ptr, _, shape, strides = _like(be, t, name, shape, code)
    if type(t) is not Strided:
        if not t.is_contiguous():
            raise _invalid(f"{name}: must be contiguous")
        return ptr
    s = 1
    for n, st in zip(reversed(shape), reversed(strides)):
        if n != 1 and st != s:
            raise _invalid(f"{name}: must be contiguous")
        s *= n
    return ptr


class _Call:
    """One call's outputs and its order with torch's current stream."""
    __slots__ = ("be", "like", "cur", "mine")

    def __init__(self, be, like, *others):
        self.be = be
        self.cur = None
        own = type(like) is Strided
        for t in others:
            if t is not None and (type(t) is Strided) != own:
                raise _invalid("Strided views and torch tensors cannot be mixed in one call")
        if own:
            self.like = None
            return
        self.like = like
        if not be.recording and _torch._C._cuda_getCurrentRawStream(be.device) != be.home_stream:
            self.cur = _torch.cuda.current_stream(like.device)
            self.mine = be.torch_stream()
            self.mine.wait_stream(self.cur)

    def empty(self, code, shape, same=None):
        """(a new row-major tensor, its pointer); `same`: a tensor of that shape
        and type, if there is one, whose layout can be taken over when it is
        row-major too."""
        like = self.like
        if like is not None:
            if same is not None and same.is_contiguous():
                t = _torch.empty_like(same)
            elif like.dtype is _torch_types[code]:
                t = like.new_empty(shape)
            else:
                t = _torch.empty(shape, dtype=_torch_types[code], device=like.device)
            return t, t.data_ptr()
        n = 1
        for s in shape:
            n *= s
        t = Strided(self.be.alloc(n, _NP[code]), shape)
        return t, t.storage.ptr

    def rows(self, code, m, k, row):
        """The same of m rows of k elements, `row` apart."""
        if self.like is not None:
            t = _torch.empty_strided((m, k), (row, 1), dtype=_torch_types[code], device=self.like.device)
            return t, t.data_ptr()
        t = Strided(self.be.alloc(m * row, _NP[code]), (m, k), (row, 1))
        return t, t.storage.ptr

    def done(self, rc):
        if self.cur is not None:
            self.cur.wait_stream(self.mine)
        if rc:
            _check(rc)


@functools.lru_cache(maxsize=512)
def _i64s(*values):
    """An int64 array for the ABI (which only reads it)."""
    return (ctypes.c_int64 * len(values))(*values)


_REALS = (F32, F64, OM_BF16, F16)


def _dtb(strides):
    """Strides of a [batch, time, channel] operand in the ABI's order."""
    return _i64s(strides[2], strides[1], strides[0])


def _cr(strides):
    """Strides of a [row, column] operand in the ABI's order."""
    return _i64s(strides[1], strides[0])


def _kind(kind, who):
    k = _KINDS.get(kind)
    if k is None:
        raise _invalid(f"{who}: kind must be 'linear' or 'sigmoid', not {kind!r}")
    return k


def gated_scan(be, gate, x, h0=None, lengths=None, kind="linear", h_last=None):
    """h_t = a_t h_{t-1} + b_t over [batch, time, channels] (om_b200_gated_scan).

    kind "linear": a = gate, b = x; "sigmoid": a = sigmoid(gate),
    b = (1 - a) x.  h0 [batch, channels] (f32; f64 for f64 inputs) starts the
    state, `lengths` [batch] (int32) ends sequences early.  Returns (h, h_last);
    h_last, when given, receives the last state and may be h0 itself (a decoding
    step updates its state in place)."""
    L = _bind()
    k = _kind(kind, "gated_scan")
    gp, code, shape, gs = _typed(be, gate, "gate", 3, _REALS)
    if x is None:
        raise _invalid("gated_scan: x is needed")
    xp, _, _, xs = _like(be, x, "x", shape, code)
    b, t, d = shape
    st = F64 if code == F64 else F32
    h0p = _vector(be, h0, "h0", (b, d), st)
    lp = _vector(be, lengths, "lengths", (b,), I32)
    call = _Call(be, gate, x, h0, lengths, h_last)
    h, hp = call.empty(code, shape, gate)
    if h_last is None:
        h_last, lastp = call.empty(st, (b, d), h0)
    else:
        lastp = _vector(be, h_last, "h_last", (b, d), st)
    call.done(L.om_b200_gated_scan(be.h, k, code, _i64s(d, t, b), gp, _dtb(gs), xp, _dtb(xs), h0p, lp, hp,
                                   _i64s(1, d, t * d), lastp))
    return h, h_last


def gated_scan_backward(be, gate, x, h, dh, h0=None, dh_last=None, lengths=None, kind="linear"):
    """Gradients (dgate, dx, dh0) of gated_scan, given its output h and the
    gradients reaching h and (optionally) h_last.  x may be None for "linear"."""
    L = _bind()
    k = _kind(kind, "gated_scan_backward")
    gp, code, shape, gs = _typed(be, gate, "gate", 3, _REALS)
    xp = xs = None
    if x is not None:
        xp, _, _, xs = _like(be, x, "x", shape, code)
        xs = _dtb(xs)
    elif kind != "linear":
        raise _invalid("gated_scan_backward: x is needed")
    hp, _, _, hs = _like(be, h, "h", shape, code)
    ep, _, _, es = _like(be, dh, "dh", shape, code)
    b, t, d = shape
    st = F64 if code == F64 else F32
    h0p = _vector(be, h0, "h0", (b, d), st)
    lp = _vector(be, lengths, "lengths", (b,), I32)
    elp = _vector(be, dh_last, "dh_last", (b, d), st)
    call = _Call(be, gate, x, h, dh, h0, dh_last, lengths)
    (dgate, pp), (dx, qp), (dh0, d0p) = call.empty(code, shape, gate), call.empty(code, shape, dh), call.empty(st, (b, d), h0)
    rows = _i64s(1, d, t * d)
    call.done(L.om_b200_gated_scan_backward(be.h, k, code, _i64s(d, t, b), gp, _dtb(gs), xp, xs, hp, _dtb(hs), h0p, lp,
                                            ep, _dtb(es), elp, pp, rows, qp, rows, d0p))
    return dgate, dx, dh0


def _loss_args(be, x, w, targets, who):
    xp, code, (n, d), xs = _typed(be, x, "x", 2, _REALS)
    wp, _, (v, wd), ws = _typed(be, w, "w", 2, (code,))
    if wd != d:
        raise _invalid(f"{who}: x has width {d}, w {wd}")
    tc = _typed(be, targets, "targets", 1, (I32, I64))[1]
    tp = _vector(be, targets, "targets", (n,), tc)
    return code, n, d, v, (_i64s(d, n, v), xp, _cr(xs), wp, _cr(ws), tc, tp), F64 if code == F64 else F32


def linear_cross_entropy(be, x, w, targets):
    """(loss, lse) of the logits x w^T, per token (om_b200_linear_cross_entropy).

    x [tokens, width], w [vocabulary, width], targets [tokens] (i32 or i64;
    one outside the vocabulary carries no loss).  The logits are never kept; they
    may be -inf (a masked vocabulary)."""
    L = _bind()
    code, n, _, _, args, st = _loss_args(be, x, w, targets, "linear_cross_entropy")
    call = _Call(be, x, w, targets)
    loss, lp = call.empty(st, (n,))
    lse, sp = call.empty(st, (n,), loss)
    call.done(L.om_b200_linear_cross_entropy(be.h, code, *args, lp, sp))
    return loss, lse


def linear_cross_entropy_backward(be, x, w, targets, lse, dloss):
    """Gradients (dx, dw) of linear_cross_entropy, given its lse and the
    gradient dloss [tokens] of each token's loss."""
    L = _bind()
    code, n, d, v, args, st = _loss_args(be, x, w, targets, "linear_cross_entropy_backward")
    sp, gp = _vector(be, lse, "lse", (n,), st), _vector(be, dloss, "dloss", (n,), st)
    call = _Call(be, x, w, targets, lse, dloss)
    (dx, dp), (dw, ep) = call.empty(code, (n, d), x), call.empty(code, (v, d), w)
    rows = _i64s(1, d)
    call.done(L.om_b200_linear_cross_entropy_backward(be.h, code, *args, sp, gp, dp, rows, ep, rows))
    return dx, dw


_QUANTISED = (F32, OM_BF16, F16)


def quantize_rows(be, x):
    """(q, scale) of a matrix in 8 bits: scale = max |row| / 127 and
    q = row / scale, rounded (om_b200_quantize_rows).  x is f32, bf16 or f16;
    q's rows start 16 bytes apart or a multiple of that, which matmul_i8 reads
    in place."""
    L = _bind()
    xp, code, (m, k), xs = _typed(be, x, "x", 2, _QUANTISED)
    call = _Call(be, x)
    row = (k + 15) // 16 * 16
    (q, qp), (scale, sp) = call.rows(I8, m, k, row), call.empty(F32, (m,))
    call.done(L.om_b200_quantize_rows(be.h, code, _i64s(k, m), xp, _cr(xs), qp, _i64s(1, row), sp))
    return q, scale


def _code_of(dtype):
    code = _NAMES.get(dtype) if isinstance(dtype, str) else _torch_codes.get(dtype)
    if code not in _QUANTISED:
        raise _invalid(f"a result type of f32, bf16 or f16 is needed, not {dtype!r}")
    return code


def _weights(be, w, w_scale, bias, k):
    wp, _, (n, wk), ws = _typed(be, w, "w", 2, (I8,))
    if wk != k:
        raise _invalid(f"w has {wk} columns, the other matrix {k}")
    tp = _vector(be, w_scale, "w_scale", (n,), F32)
    if tp is None:
        raise _invalid("w_scale is needed")
    return n, wp, _cr(ws), tp, _vector(be, bias, "bias", (n,), F32)


def matmul_i8(be, q, q_scale, w, w_scale, bias=None, dtype="f32"):
    """(q w^T) q_scale[:, None] w_scale + bias of 8-bit matrices
    (om_b200_matmul_i8), as `dtype` ("f32", "bf16", "f16" or the torch type).

    q [rows, inner], w [columns, inner], one scale per row of each."""
    L = _bind()
    qp, _, (m, k), qs = _typed(be, q, "q", 2, (I8,))
    n, wp, ws, tp, bp = _weights(be, w, w_scale, bias, k)
    sp = _vector(be, q_scale, "q_scale", (m,), F32)
    if sp is None:
        raise _invalid("q_scale is needed")
    code = _code_of(dtype)
    call = _Call(be, q, q_scale, w, w_scale, bias)
    y, yp = call.empty(code, (m, n))
    call.done(L.om_b200_matmul_i8(be.h, code, _i64s(k, m, n), qp, _cr(qs), sp, wp, ws, tp, bp, yp, _i64s(1, n)))
    return y


def linear_i8(be, x, w, w_scale, bias=None):
    """matmul_i8 of x's rows, quantised by quantize_rows within the call; the
    result has x's type."""
    L = _bind()
    xp, code, (m, k), xs = _typed(be, x, "x", 2, _QUANTISED)
    n, wp, ws, tp, bp = _weights(be, w, w_scale, bias, k)
    call = _Call(be, x, w, w_scale, bias)
    y, yp = call.empty(code, (m, n))
    call.done(L.om_b200_linear_i8(be.h, code, _i64s(k, m, n), xp, _cr(xs), wp, ws, tp, bp, yp, _i64s(1, n)))
    return y
