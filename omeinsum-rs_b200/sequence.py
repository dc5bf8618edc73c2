"""Operators of sequence models on the B200 backend: the gated linear
recurrence (om_b200_gated_scan), the softmax cross entropy of a vocabulary's
logits (om_b200_linear_cross_entropy), both with their backward pass, and the
8-bit integer product with its row quantiser (om_b200_matmul_i8,
om_b200_quantize_rows, om_b200_linear_i8).

Every function takes the backend first and tensors that are either

  - torch CUDA tensors on the backend's device (any strides), or
  - `Strided` views of a backend's `Storage` (see `upload`),

and returns tensors of the kind it was given, row-major.  Shapes are in the
order the text names; nothing waits for the device.

Torch tensors are ordered with torch's current stream: when the backend runs
on another stream, the call waits for the work queued on torch's stream and
torch's stream for the call (a backend made with `B200(device, stream=...)`
on torch's stream needs neither).  While the backend records a graph no
such waits are made: the tensors must be ready, and stay alive with the graph.
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import BF16, DTYPES, OmError, Storage, _check, lib

F32, F64, OM_BF16, F16, I8, I32, I64 = 0, 1, 5, 6, 7, 8, 9
_NP = {v: k for k, v in DTYPES.items()}
_NAMES = {"f32": F32, "f64": F64, "bf16": OM_BF16, "f16": F16, "i8": I8, "i32": I32, "i64": I64}
_KINDS = {"linear": 0, "sigmoid": 1}
_torch_codes = {}  # torch dtype -> code, filled on the first torch tensor
_torch_types = {}


def _bind():
    L = lib()
    if not getattr(L, "_sequence_bound", False):
        P, I = ctypes.c_void_p, ctypes.c_int
        L.om_b200_gated_scan.argtypes = [P, I, I] + [P] * 10
        L.om_b200_gated_scan_backward.argtypes = [P, I, I] + [P] * 17
        L.om_b200_linear_cross_entropy.argtypes = [P, I] + [P] * 5 + [I] + [P] * 3
        L.om_b200_linear_cross_entropy_backward.argtypes = [P, I] + [P] * 5 + [I] + [P] * 7
        L.om_b200_quantize_rows.argtypes = [P, I] + [P] * 6
        L.om_b200_matmul_i8.argtypes = [P, I] + [P] * 10
        L.om_b200_linear_i8.argtypes = [P, I] + [P] * 9
        L._sequence_bound = True
    return L


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


class _Operand:
    """Device pointer, dtype code, shape and strides of one argument."""
    __slots__ = ("ptr", "code", "shape", "strides", "keep")

    def __init__(self, be, t, name):
        if isinstance(t, Strided):
            if t.storage.backend.device != be.device:
                raise _invalid(f"{name}: on device {t.storage.backend.device}, the backend on {be.device}")
            self.code = DTYPES[t.storage.dtype]
            self.ptr = (t.storage.ptr or 0) + t.offset * t.storage.dtype.itemsize
            self.shape, self.strides = t.shape, t.strides
        elif hasattr(t, "data_ptr"):
            if not t.is_cuda or t.device.index != be.device:
                raise _invalid(f"{name}: on {t.device}, the backend on cuda:{be.device}")
            code = _torch_codes.get(t.dtype)
            if code is None:
                code = _learn_torch(t.dtype, name)
            self.code, self.ptr = code, t.data_ptr()
            self.shape, self.strides = tuple(t.shape), t.stride()
        else:
            raise _invalid(f"{name}: a Strided view or a torch CUDA tensor is needed, not {type(t).__name__}")
        self.keep = t


def _learn_torch(dtype, name):
    import torch
    for tt, code in ((torch.float32, F32), (torch.float64, F64), (torch.bfloat16, OM_BF16),
                     (torch.float16, F16), (torch.int8, I8), (torch.int32, I32),
                     (torch.int64, I64)):
        _torch_codes[tt] = code
        _torch_types[code] = tt
    if dtype not in _torch_codes:
        raise _invalid(f"{name}: no device type for {dtype}")
    return _torch_codes[dtype]


class _Call:
    """One call's outputs and its order with torch's current stream."""

    def __init__(self, be, like, *others):
        self.be = be
        self.torch = self.cur = None
        own = isinstance(like, Strided)
        for t in others:
            if t is not None and isinstance(t, Strided) != own:
                raise _invalid("Strided views and torch tensors cannot be mixed in one call")
        if not own:
            import torch
            self.torch = torch
            self.device = like.device
            if not be.recording:
                cur = torch.cuda.current_stream(like.device)
                if cur.cuda_stream != be.home_stream:
                    self.cur = cur
                    self.mine = torch.cuda.ExternalStream(be.home_stream, device=like.device)
                    self.mine.wait_stream(cur)

    def empty(self, code, *shape):
        if self.torch is not None:
            return self.torch.empty(shape, dtype=_torch_types[code], device=self.device)
        n = 1
        for s in shape:
            n *= s
        return Strided(self.be.alloc(n, _NP[code]), shape)

    def done(self, rc):
        if self.cur is not None:
            self.cur.wait_stream(self.mine)
        _check(rc)


_A3 = ctypes.c_int64 * 3


def _dtb(o: _Operand):
    """Strides of a [batch, time, channel] operand in the ABI's order."""
    s = o.strides
    return _A3(s[2], s[1], s[0])


def _want(o: _Operand, name, shape, *codes):
    if o.shape != tuple(shape):
        raise _invalid(f"{name}: shape {list(o.shape)}, expected {list(shape)}")
    if o.code not in codes:
        raise _invalid(f"{name}: type {_NP[o.code]} not accepted here")


def _vector(be, t, name, shape, code):
    """Pointer of an optional contiguous operand (None: a null pointer)."""
    if t is None:
        return None
    o = _Operand(be, t, name)
    _want(o, name, shape, code)
    s = 1
    for n, st in zip(reversed(o.shape), reversed(o.strides)):
        if n != 1 and st != s:
            raise _invalid(f"{name}: must be contiguous")
        s *= n
    return o.ptr


def _scan_args(be, gate, x, kind, who):
    g = _Operand(be, gate, "gate")
    if kind not in _KINDS:
        raise _invalid(f"{who}: kind must be 'linear' or 'sigmoid', not {kind!r}")
    if len(g.shape) != 3:
        raise _invalid(f"{who}: gate must be [batch, time, channels]")
    if g.code not in (F32, F64, OM_BF16, F16):
        raise _invalid(f"{who}: gate must be f32, f64, bf16 or f16")
    v = None
    if x is not None:
        v = _Operand(be, x, "x")
        _want(v, "x", g.shape, g.code)
    b, t, d = g.shape
    return g, v, _A3(d, t, b), (b, d), F64 if g.code == F64 else F32


def gated_scan(be, gate, x, h0=None, lengths=None, kind="linear", h_last=None):
    """h_t = a_t h_{t-1} + b_t over [batch, time, channels] (om_b200_gated_scan).

    kind "linear": a = gate, b = x; "sigmoid": a = sigmoid(gate),
    b = (1 - a) x.  h0 [batch, channels] (f32; f64 for f64 inputs) starts the
    state, `lengths` [batch] (int32) ends sequences early.  Returns (h, h_last);
    h_last, when given, receives the last state and may be h0 itself (a decoding
    step updates its state in place)."""
    L = _bind()
    g, v, shape, bd, st = _scan_args(be, gate, x, kind, "gated_scan")
    if v is None:
        raise _invalid("gated_scan: x is needed")
    h0p = _vector(be, h0, "h0", bd, st)
    lp = _vector(be, lengths, "lengths", bd[:1], I32)
    call = _Call(be, gate, x, h0, lengths, h_last)
    h = call.empty(g.code, *g.shape)
    if h_last is None:
        h_last = call.empty(st, *bd)
    lastp = _vector(be, h_last, "h_last", bd, st)
    o = _Operand(be, h, "h")
    call.done(L.om_b200_gated_scan(be.h, _KINDS[kind], g.code, shape, g.ptr, _dtb(g), v.ptr, _dtb(v),
                                   h0p, lp, o.ptr, _dtb(o), lastp))
    return h, h_last


def gated_scan_backward(be, gate, x, h, dh, h0=None, dh_last=None, lengths=None, kind="linear"):
    """Gradients (dgate, dx, dh0) of gated_scan, given its output h and the
    gradients reaching h and (optionally) h_last.  x may be None for "linear"."""
    L = _bind()
    g, v, shape, bd, st = _scan_args(be, gate, x, kind, "gated_scan_backward")
    if v is None and kind != "linear":
        raise _invalid("gated_scan_backward: x is needed")
    ho, eo = _Operand(be, h, "h"), _Operand(be, dh, "dh")
    _want(ho, "h", g.shape, g.code)
    _want(eo, "dh", g.shape, g.code)
    h0p = _vector(be, h0, "h0", bd, st)
    lp = _vector(be, lengths, "lengths", bd[:1], I32)
    ep = _vector(be, dh_last, "dh_last", bd, st)
    call = _Call(be, gate, x, h, dh, h0, dh_last, lengths)
    dgate, dx = call.empty(g.code, *g.shape), call.empty(g.code, *g.shape)
    dh0 = call.empty(st, *bd)
    po, qo = _Operand(be, dgate, "dgate"), _Operand(be, dx, "dx")
    call.done(L.om_b200_gated_scan_backward(
        be.h, _KINDS[kind], g.code, shape, g.ptr, _dtb(g), v.ptr if v else None,
        _dtb(v) if v else None, ho.ptr, _dtb(ho), h0p, lp, eo.ptr, _dtb(eo), ep, po.ptr, _dtb(po),
        qo.ptr, _dtb(qo), _vector(be, dh0, "dh0", bd, st)))
    return dgate, dx, dh0


_A2 = ctypes.c_int64 * 2


def _matrix(be, t, name, *codes):
    o = _Operand(be, t, name)
    if len(o.shape) != 2:
        raise _invalid(f"{name}: must have two axes")
    if codes and o.code not in codes:
        raise _invalid(f"{name}: type {_NP[o.code]} not accepted here")
    return o


def _cr(o: _Operand):
    """Strides of a [row, column] operand in the ABI's order."""
    return _A2(o.strides[1], o.strides[0])


def _loss_args(be, x, w, targets, who):
    xo = _matrix(be, x, "x", F32, F64, OM_BF16, F16)
    wo = _matrix(be, w, "w", xo.code)
    to = _Operand(be, targets, "targets")
    n, d = xo.shape
    if wo.shape[1] != d:
        raise _invalid(f"{who}: x has width {d}, w {wo.shape[1]}")
    if to.code not in (I32, I64):
        raise _invalid(f"{who}: targets must be i32 or i64")
    tp = _vector(be, targets, "targets", (n,), to.code)
    return xo, wo, to.code, tp, _A3(d, n, wo.shape[0]), F64 if xo.code == F64 else F32


def linear_cross_entropy(be, x, w, targets):
    """(loss, lse) of the logits x w^T, per token (om_b200_linear_cross_entropy).

    x [tokens, width], w [vocabulary, width], targets [tokens] (i32 or i64;
    one outside the vocabulary carries no loss).  The logits are never kept."""
    L = _bind()
    xo, wo, tc, tp, shape, st = _loss_args(be, x, w, targets, "linear_cross_entropy")
    n = xo.shape[0]
    call = _Call(be, x, w, targets)
    loss, lse = call.empty(st, n), call.empty(st, n)
    call.done(L.om_b200_linear_cross_entropy(be.h, xo.code, shape, xo.ptr, _cr(xo), wo.ptr, _cr(wo), tc, tp,
                                             _vector(be, loss, "loss", (n,), st), _vector(be, lse, "lse", (n,), st)))
    return loss, lse


def linear_cross_entropy_backward(be, x, w, targets, lse, dloss):
    """Gradients (dx, dw) of linear_cross_entropy, given its lse and the
    gradient dloss [tokens] of each token's loss."""
    L = _bind()
    xo, wo, tc, tp, shape, st = _loss_args(be, x, w, targets, "linear_cross_entropy_backward")
    n = xo.shape[0]
    lp, gp = _vector(be, lse, "lse", (n,), st), _vector(be, dloss, "dloss", (n,), st)
    call = _Call(be, x, w, targets, lse, dloss)
    dx, dw = call.empty(xo.code, *xo.shape), call.empty(xo.code, *wo.shape)
    do, eo = _Operand(be, dx, "dx"), _Operand(be, dw, "dw")
    call.done(L.om_b200_linear_cross_entropy_backward(
        be.h, xo.code, shape, xo.ptr, _cr(xo), wo.ptr, _cr(wo), tc, tp, lp, gp, do.ptr, _cr(do),
        eo.ptr, _cr(eo)))
    return dx, dw


def quantize_rows(be, x):
    """(q, scale) of a matrix in 8 bits: scale = max |row| / 127 and
    q = row / scale, rounded (om_b200_quantize_rows).  x is f32, bf16 or f16."""
    L = _bind()
    xo = _matrix(be, x, "x", F32, OM_BF16, F16)
    m, k = xo.shape
    call = _Call(be, x)
    q, scale = call.empty(I8, m, k), call.empty(F32, m)
    qo = _Operand(be, q, "q")
    call.done(L.om_b200_quantize_rows(be.h, xo.code, _A2(k, m), xo.ptr, _cr(xo), qo.ptr, _cr(qo),
                                      _vector(be, scale, "scale", (m,), F32)))
    return q, scale


def _code_of(dtype):
    if isinstance(dtype, str) and dtype in _NAMES:
        return _NAMES[dtype]
    code = _torch_codes.get(dtype)
    if code is None:
        raise _invalid(f"no device type for {dtype!r}")
    return code


def matmul_i8(be, q, q_scale, w, w_scale, bias=None, dtype="f32"):
    """(q w^T) q_scale[:, None] w_scale + bias of 8-bit matrices
    (om_b200_matmul_i8), as `dtype` ("f32", "bf16", "f16" or the torch type).

    q [rows, inner], w [columns, inner], one scale per row of each."""
    L = _bind()
    qo, wo = _matrix(be, q, "q", I8), _matrix(be, w, "w", I8)
    (m, k), n = qo.shape, wo.shape[0]
    if wo.shape[1] != k:
        raise _invalid(f"matmul_i8: q has {k} columns, w {wo.shape[1]}")
    sp, tp = _vector(be, q_scale, "q_scale", (m,), F32), _vector(be, w_scale, "w_scale", (n,), F32)
    bp = _vector(be, bias, "bias", (n,), F32)
    if sp is None or tp is None:
        raise _invalid("matmul_i8: both scales are needed")
    code = _code_of(dtype)
    if code not in (F32, OM_BF16, F16):
        raise _invalid("matmul_i8: dtype must be f32, bf16 or f16")
    call = _Call(be, q, q_scale, w, w_scale, bias)
    y = call.empty(code, m, n)
    yo = _Operand(be, y, "y")
    call.done(L.om_b200_matmul_i8(be.h, code, _A3(k, m, n), qo.ptr, _cr(qo), sp, wo.ptr, _cr(wo), tp, bp,
                                  yo.ptr, _cr(yo)))
    return y


def linear_i8(be, x, w, w_scale, bias=None):
    """matmul_i8 of x's rows, quantised by quantize_rows within the call; the
    result has x's type."""
    L = _bind()
    xo, wo = _matrix(be, x, "x", F32, OM_BF16, F16), _matrix(be, w, "w", I8)
    (m, k), n = xo.shape, wo.shape[0]
    if wo.shape[1] != k:
        raise _invalid(f"linear_i8: x has {k} columns, w {wo.shape[1]}")
    tp, bp = _vector(be, w_scale, "w_scale", (n,), F32), _vector(be, bias, "bias", (n,), F32)
    if tp is None:
        raise _invalid("linear_i8: w_scale is needed")
    call = _Call(be, x, w, w_scale, bias)
    y = call.empty(xo.code, m, n)
    yo = _Operand(be, y, "y")
    call.done(L.om_b200_linear_i8(be.h, xo.code, _A3(k, m, n), xo.ptr, _cr(xo), wo.ptr, _cr(wo), tp, bp,
                                  yo.ptr, _cr(yo)))
    return y
