"""Plain 64-bit forms of the sequence-model operators, and bounds on how far
results in fewer bits may be from them.

U = 2^-24 is half a step of f32 relative to the value; `half(t)` the same for
the type a result is rounded to."""
import numpy as np

U = 2.0 ** -24
HALF = {"f64": 2.0 ** -53, "f32": U, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f64": 0.0, "f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}  # half a step at zero


def state_unit(dtype):
    """Half a step of the type sums and states are held in."""
    return 2.0 ** -53 if dtype == "f64" else U


def rounded(x, dtype):
    """x at the values `dtype` can hold, as f64."""
    x = np.asarray(x, np.float64)
    if dtype == "f64":
        return x
    f = x.astype(np.float32)
    if dtype == "f32":
        return f.astype(np.float64)
    if dtype == "f16":
        return f.astype(np.float16).astype(np.float64)
    bits = f.view(np.uint32).astype(np.uint64)
    bits = (bits + 0x7FFF + ((bits >> 16) & 1)) >> 16 << 16
    out = bits.astype(np.uint32).view(np.float32)
    return np.where(np.isnan(f), np.nan, out).astype(np.float64)


def _factors(gate, x, kind):
    if kind == "linear":
        return gate, x, np.ones_like(gate)
    with np.errstate(over="ignore"):
        a = np.where(gate >= 0, 1 / (1 + np.exp(-gate)), np.exp(gate) / (1 + np.exp(gate)))
        keep = np.where(gate >= 0, np.exp(-gate) / (1 + np.exp(-gate)), 1 / (1 + np.exp(gate)))
    return a, keep * x, keep


# Relative error of sigmoid(g) and 1 - sigmoid(g) in units of U: the f32
# exponential (a step or two, and |g| <= 16 steps of its argument where it is
# formed as a power of two), one addition, one division, one product.
SIGMOID = 32.0


def scan(gate, x, h0, lengths, kind, dtype):
    """(h, h_last, bound of h before its rounding, bound of h_last).

    The term b_s of h_t passes t - s products and at most as many additions
    (any grouping of the chain included, with 8 more for joining groups), each
    off by U relative to it; every factor a of kind "sigmoid" by SIGMOID U. In
    f32 a step's result below 2^-126, the smallest normal number, may be lost
    whole: up to 2^-126 per step, which the later factors carry on."""
    nb, nt, nd = gate.shape
    unit = state_unit(dtype)
    tiny = 0.0 if dtype == "f64" else 2.0 ** -126 / unit
    per = 2.0 + (SIGMOID if kind == "sigmoid" else 0.0)
    a, b, _ = _factors(gate, x, kind)
    h = np.zeros_like(gate)
    bound = np.zeros_like(gate)
    s = np.zeros((nb, nd)) if h0 is None else np.array(h0, np.float64)
    mass, err = np.abs(s), np.zeros_like(s)
    ends = np.full(nb, nt) if lengths is None else np.clip(lengths, 0, nt)
    for t in range(nt):
        on = (t < ends)[:, None]
        ra = np.where(on, a[:, t], 1.0)
        rb = np.where(on, b[:, t], 0.0)
        err = np.where(on, np.abs(ra) * (err + per * mass) + tiny, err)
        s = ra * s + rb
        mass = np.abs(ra) * mass + np.abs(rb)
        h[:, t] = np.where(on, s, 0.0)
        bound[:, t] = np.where(on, unit * (err + (8 + per) * mass), 0.0)
    return h, s, bound, unit * (err + (8 + per) * mass)


def scan_backward(gate, x, h, dh, h0, dh_last, lengths, kind, dtype):
    """(dgate, dx, dh0) from the h that the forward stored, and their bounds."""
    nb, nt, nd = gate.shape
    unit = state_unit(dtype)
    per = 2.0 + (SIGMOID if kind == "sigmoid" else 0.0)
    a, _, keep = _factors(gate, np.zeros_like(gate) if x is None else x, kind)
    carry = np.zeros((nb, nd)) if dh_last is None else np.array(dh_last, np.float64)
    start = np.zeros((nb, nd)) if h0 is None else np.asarray(h0, np.float64)
    mass, err = np.abs(carry), np.zeros_like(carry)
    ends = np.full(nb, nt) if lengths is None else np.clip(lengths, 0, nt)
    out = [np.zeros_like(gate) for _ in range(4)]  # dgate, dx and their bounds
    for t in range(nt - 1, -1, -1):
        on = (t < ends)[:, None]
        total = carry + dh[:, t]
        tm = mass + np.abs(dh[:, t])
        te = err + (8 + per) * tm
        before = h[:, t - 1] if t else start
        if kind == "sigmoid":
            diff, wide = before - x[:, t], np.abs(before) + np.abs(x[:, t])
            slope, sx = a[:, t] * keep[:, t], keep[:, t]
        else:
            diff, wide, slope, sx = before, np.abs(before), 1.0, 1.0
        more = 4 + 2 * (per - 2)
        for k, v in enumerate((total * diff * slope, total * sx,
                               unit * (te + more * tm) * wide * slope, unit * (te + more * tm) * sx)):
            out[k][:, t] = np.where(on, v, 0.0)
        err = np.where(on, np.abs(a[:, t]) * (err + per * tm), err)
        carry = np.where(on, total * a[:, t], carry)
        mass = np.where(on, tm * np.abs(a[:, t]), mass)
    return out[0], out[1], carry, out[2], out[3], unit * (err + (8 + per) * mass)


def loss(x, w, targets, dtype):
    """(loss, lse, z, bound of a logit, bounds of loss and lse).

    A logit is a sum of D products.  16-bit: exact products summed in f32 by
    the tensor cores, 16 (or any number) at a time, without rounding to
    nearest, so up to 2 U of the running sum for each step and each product of
    a step: 2 (D / 8 + 16) U; f32: three TF32 products, 2^-20 of the terms'
    sum; f64: D + 8 roundings."""
    z = x @ w.T
    terms = np.abs(x) @ np.abs(w).T
    d = x.shape[1]
    ez = terms * logit_error(d, dtype)
    top = z.max(1, keepdims=True)
    lse = (top + np.log(np.exp(z - top).sum(1, keepdims=True)))[:, 0]
    ok = (targets >= 0) & (targets < w.shape[0])
    hit = z[np.arange(len(z)), np.where(ok, targets, 0)]
    unit = state_unit(dtype)
    # sum of exponentials: each off by the shift of its logit, its own few
    # steps, |z - top| steps of its argument and the joining of partial sums
    p = np.exp(z - lse[:, None])
    spread = (p * (ez + unit * (16 + 2 * np.abs(z - top)))).sum(1) + 64 * unit
    elae = spread + 4 * unit * np.abs(lse)
    eloss = elae + ez[np.arange(len(z)), np.where(ok, targets, 0)] + 4 * unit * (np.abs(lse) + np.abs(hit))
    return np.where(ok, lse - hit, 0.0), lse, z, ez, np.where(ok, eloss, 0.0), elae


def logit_error(d, dtype):
    if dtype == "f64":
        return (d + 8) * 2.0 ** -53
    if dtype == "f32":
        return 2.0 ** -20 + (d + 8) * U / 8
    return 2 * (d / 8 + 16) * U


def loss_backward(x, w, targets, lse, dloss, dtype):
    """(dx, dw) and their bounds, from the lse that the forward stored."""
    z = x @ w.T
    n, d = x.shape
    v = w.shape[0]
    unit = state_unit(dtype)
    ez = np.abs(x) @ np.abs(w).T * logit_error(d, dtype)
    ok = (targets >= 0) & (targets < v)
    p = np.exp(z - lse[:, None])
    one = np.zeros_like(z)
    one[np.arange(n)[ok], targets[ok]] = 1.0
    g = np.where(ok, dloss, 0.0)[:, None]
    dz = np.where(ok[:, None], g * (p - one), 0.0)
    ep = np.where(ok[:, None], np.abs(g) * (p * (ez + unit * (16 + 2 * np.abs(z - lse[:, None]))) + 2 * unit * (p + one)), 0.0)
    if dtype in ("bf16", "f16"):  # dz in 16 bits; f16 holds it scaled so that the largest is below 2^15
        ep = ep + np.abs(dz) * HALF[dtype] * (1 + HALF[dtype])
        if dtype == "f16":
            ep = ep + np.where(ok[:, None], np.abs(g).max() * 2.0 ** -25 / 2.0 ** 13, 0.0)
    x0 = np.where(ok[:, None], x, 0.0)
    out = []
    for a, b, ea in ((dz, w, ep), (dz.T, x0, ep.T)):
        terms = np.abs(a) @ np.abs(b)
        ref = a @ b
        e = ea @ np.abs(b) + (terms + ea @ np.abs(b)) * logit_error(a.shape[1], dtype)
        # f32 / f64: pieces are added up in the same type
        e = e + np.abs(ref) * HALF[dtype] * 2 + TINY[dtype] + terms * 16 * unit
        if dtype != "f64":
            # below 2^-126 a value of dz and each of the (at most four) partial
            # products of a term may be flushed to zero: 2^-126 |b| and
            # 4 * 2^-126 for every term
            e = e + 2.0 ** -126 * (np.ones_like(a) @ (np.abs(b) + 4))
        out.append((ref, e))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def quantize(x32):
    """q (int8) and scale (f32) by the definition, in f32 arithmetic."""
    x32 = np.asarray(x32, np.float32)
    with np.errstate(all="ignore"):
        top = np.abs(x32).max(1) if x32.shape[1] else np.zeros(len(x32), np.float32)
        scale = (top / np.float32(127)).astype(np.float32)
        r = np.rint(x32 / scale[:, None])
        q = np.where((scale[:, None] > 0) & ~np.isnan(r), np.clip(r, -127, 127), 0)
    return q.astype(np.int8), scale


def matmul_i8(q, q_scale, w, w_scale, bias, dtype):
    """The defined value, step by step in f32, rounded to dtype (as f64)."""
    acc = q.astype(np.float64) @ w.astype(np.float64).T
    y = acc.astype(np.float32) * q_scale[:, None].astype(np.float32) * w_scale[None].astype(np.float32)
    if bias is not None:
        y = y + bias[None].astype(np.float32)
    return rounded(y, dtype)
