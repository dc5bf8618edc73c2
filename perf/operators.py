"""Measured cases of the sequence-model operators, with their plain forms.

Three operators, each a contraction of the kind the library is built around:

scan   h_t = a_t h_{t-1} + b_t along time, a contraction chain per channel.  With kind "linear",
       a = gate and b = x; with kind "sigmoid", a = sigmoid(gate) and b = (1 - a) x.  Backward
       pass included; one time step is the form that serves single tokens.
loss   softmax cross entropy of logits x w^T over a vocabulary, the logits never kept:
       loss_n = log sum_v exp(z_nv) - z_{n, target}, with the gradients of x and w.
i8     y = (q w^T) * row scale * channel scale + bias in 8-bit integers, q the rows of x rounded
       to 127 steps of their largest magnitude.

`own` False computes the plain forms (elementary torch operations in 32 bits), `own` True calls
the library through its Python front end.
"""
import importlib
import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one decoding step of a recurrent layer for a batch of 64 requests: latency alone
        dict(name="scan_step", op="scan", kind="sigmoid", dtype="bf16", batch=64, time=1, dim=2048, ragged=False, train=False),
        # a layer of an ordinary training batch, forward and backward
        dict(name="scan_train", op="scan", kind="sigmoid", dtype="bf16", batch=4, time=4096, dim=2048, ragged=False, train=True),
        # the prefill of one long document: few channels, a long chain, an odd length
        dict(name="scan_long", op="scan", kind="linear", dtype="bf16", batch=1, time=65537, dim=1032, ragged=False, train=False),
        # a padded batch in 32 bits with an odd width, forward and backward
        dict(name="scan_ragged", op="scan", kind="linear", dtype="f32", batch=7, time=1531, dim=1001, ragged=True, train=True),
        # the head of a small language model: a training step of 4096 tokens, odd vocabulary
        dict(name="loss_train", op="loss", dtype="bf16", tokens=4096, dim=1024, vocab=50001, train=True),
        # the largest: a large vocabulary and width, 8192 tokens
        dict(name="loss_large", op="loss", dtype="bf16", tokens=8192, dim=4096, vocab=128000, train=True),
        # scoring a few candidate tokens: the weights are read once, nothing else counts
        dict(name="loss_score", op="loss", dtype="f16", tokens=24, dim=2048, vocab=32000, train=False),
        # a short fine-tuning batch in 32 bits, odd sizes
        dict(name="loss_f32", op="loss", dtype="f32", tokens=509, dim=771, vocab=8191, train=True),
        # one decoded token through a projection: the 8-bit weights are all that is read
        dict(name="i8_token", op="i8", dtype="bf16", rows=1, inner=4096, cols=4096, bias=False, dynamic=True),
        # a decoding batch, odd row count, through a wide projection with a bias
        dict(name="i8_batch", op="i8", dtype="f16", rows=37, inner=2048, cols=8200, bias=True, dynamic=True),
        # a prefill: activations quantised once, then one large product
        dict(name="i8_prefill", op="i8", dtype="bf16", rows=8192, inner=4096, cols=12288, bias=False, dynamic=False),
        # odd everything, results kept in 32 bits
        dict(name="i8_odd", op="i8", dtype="f32", rows=333, inner=1037, cols=1999, bias=True, dynamic=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["scan", "loss", "i8"])
    if op == "scan":
        while True:
            c = dict(op=op, kind=rng.choice(["linear", "sigmoid"]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), batch=_log(rng, 1, 256),
                     time=rng.choice([1, _log(rng, 2, 65536), _log(rng, 2, 65536)]), dim=_log(rng, 16, 8192), ragged=rng.random() < 0.3, train=rng.random() < 0.5)
            if c["batch"] * c["time"] * c["dim"] <= 1 << 26:
                return c
    if op == "loss":
        while True:
            c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), tokens=_log(rng, 1, 8192), dim=_log(rng, 64, 4096), vocab=_log(rng, 100, 128000), train=rng.random() < 0.7)
            if rng.random() < 0.5:  # most models' widths are multiples of 64
                c["dim"] = (c["dim"] + 63) // 64 * 64
            return c
    c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), rows=rng.choice([_log(rng, 1, 64), _log(rng, 1, 8192)]), inner=_log(rng, 32, 4096), cols=_log(rng, 32, 12288),
             bias=rng.random() < 0.5, dynamic=rng.random() < 0.5)
    if rng.random() < 0.5:
        c["inner"] = (c["inner"] + 63) // 64 * 64
    return c


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(dev).manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0, dtype=dt):
        return torch.randn(*shape, generator=g, device=dev).mul_(scale).add_(mean).to(dtype)

    if case["op"] == "scan":
        b, t, d = case["batch"], case["time"], case["dim"]
        gate = normal(b, t, d, scale=1.5, mean=3.0, dtype=torch.float32)  # most gates remember, some forget
        if case["kind"] == "linear":
            gate = gate.sigmoid_()
            gate.masked_fill_(torch.rand(b, t, 1, generator=g, device=dev) < 0.005, 0.0)  # a new document begins
        s = dict(case=case, gate=gate.to(dt), x=normal(b, t, d), h0=normal(b, d, dtype=torch.float32), lengths=None)
        if case["ragged"]:
            s["lengths"] = torch.randint(0, t + 1, (b,), generator=g, device=dev, dtype=torch.int32)
        if case["train"]:
            s |= dict(dh=normal(b, t, d), dh_last=normal(b, d, dtype=torch.float32))
        return s
    if case["op"] == "loss":
        n, d, v = case["tokens"], case["dim"], case["vocab"]
        targets = torch.randint(0, v, (n,), generator=g, device=dev)
        skip = torch.rand(n, generator=g, device=dev) < 0.1  # prompts and padding carry no loss
        s = dict(case=case, x=normal(n, d), w=normal(v, d, scale=1.5 / math.sqrt(d)), targets=targets.masked_fill_(skip, -100))
        if case["train"]:  # of the mean over the tokens that count
            s["dloss"] = (~skip).float() / (~skip).sum().clamp(min=1).float()
        return s
    m, k, n = case["rows"], case["inner"], case["cols"]
    x = normal(m, k, dtype=torch.float32) * torch.exp(normal(k, dtype=torch.float32))  # a few loud channels
    s = dict(case=case, x=x.to(dt), w=torch.randint(-127, 128, (n, k), generator=g, device=dev, dtype=torch.int8),
             w_scale=torch.rand(n, generator=g, device=dev).add_(0.5).mul_(1 / (127 * math.sqrt(k))), bias=None)
    if case["bias"]:
        s["bias"] = normal(n, dtype=torch.float32)
    return s


# ---- the library ---------------------------------------------------------------------------

_library = None


def _lib():
    """The package and a backend on torch's stream, which a program opens once."""
    global _library
    if _library is None:
        om = sys.modules.get("omeinsum_b200")
        if om is None:
            d = os.path.join(ROOT, "omeinsum-rs_b200")
            spec = importlib.util.spec_from_file_location("omeinsum_b200", os.path.join(d, "__init__.py"), submodule_search_locations=[d])
            om = importlib.util.module_from_spec(spec)
            sys.modules["omeinsum_b200"] = om
            spec.loader.exec_module(om)
        dev = torch.cuda.current_device()
        _library = importlib.import_module("omeinsum_b200.sequence"), om.B200(dev, stream=torch.cuda.current_stream(dev).cuda_stream)
    return _library


def _run_own(s):
    seq, be = _lib()
    c = s["case"]
    if c["op"] == "scan":
        h, last = seq.gated_scan(be, s["gate"], s["x"], h0=s["h0"], lengths=s["lengths"], kind=c["kind"])
        if not c["train"]:
            return dict(h=h, last=last)
        dgate, dx, dh0 = seq.gated_scan_backward(be, s["gate"], s["x"], h, s["dh"], h0=s["h0"], dh_last=s["dh_last"], lengths=s["lengths"], kind=c["kind"])
        return dict(h=h, last=last, dgate=dgate, dx=dx, dh0=dh0)
    if c["op"] == "loss":
        loss, lse = seq.linear_cross_entropy(be, s["x"], s["w"], s["targets"])
        if not c["train"]:
            return dict(loss=loss, lse=lse)
        dx, dw = seq.linear_cross_entropy_backward(be, s["x"], s["w"], s["targets"], lse, s["dloss"])
        return dict(loss=loss, lse=lse, dx=dx, dw=dw)
    if c["dynamic"]:
        return dict(y=seq.linear_i8(be, s["x"], s["w"], s["w_scale"], bias=s["bias"]))
    q, scale = seq.quantize_rows(be, s["x"])
    return dict(q=q, scale=scale, y=seq.matmul_i8(be, q, scale, s["w"], s["w_scale"], bias=s["bias"], dtype=s["x"].dtype))


# ---- the plain forms -----------------------------------------------------------------------


def _chain(a, b):
    """All h_t = a_t h_{t-1} + b_t along dimension 1 from h = 0, by doubling; overwrites both."""
    step = 1
    while step < a.shape[1]:
        b[:, step:] += a[:, step:] * b[:, :-step]
        a[:, step:] = a[:, step:] * a[:, :-step]
        step *= 2
    return b


def _plain_scan(s):
    c = s["case"]
    gate, x = s["gate"].float(), s["x"].float()
    dt = s["gate"].dtype
    if c["kind"] == "sigmoid":
        keep = 1 / (1 + torch.exp(gate))  # 1 - a
        a, b = 1 / (1 + torch.exp(-gate)), keep * x
    else:
        keep, a, b = None, gate, x
    live = None
    if s["lengths"] is not None:
        live = torch.arange(a.shape[1], device=a.device)[None, :, None] < s["lengths"][:, None, None]
        a, b = torch.where(live, a, 1.0), torch.where(live, b, 0.0)  # past the end the state stays
    b = b.clone()
    b[:, 0] += a[:, 0] * s["h0"]
    h = _chain(a.clone(), b)
    last = h[:, -1].clone()
    out = dict(h=(h if live is None else h * live).to(dt), last=last)
    if not c["train"]:
        return out
    dh = s["dh"].float()
    dh = (dh if live is None else dh * live).clone()
    dh[:, -1] += s["dh_last"]
    after = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)  # the factor from t + 1 back to t
    total = _chain(after.flip(1), dh.flip(1)).flip(1)
    before = torch.cat([s["h0"][:, None], h[:, :-1]], 1)
    if keep is None:
        dgate, dx = total * before, total
    else:
        dgate, dx = total * (before - x) * a * keep, total * keep
    if live is not None:
        dgate, dx = dgate * live, dx * live
    return dict(out, dgate=dgate.to(dt), dx=dx.to(dt), dh0=total[:, 0] * a[:, 0])


def _plain_loss(s):
    x, w, targets = s["x"].float(), s["w"].float(), s["targets"]
    counts = (targets >= 0) & (targets < w.shape[0])
    at = torch.where(counts, targets, 0)[:, None]
    z = x @ w.t()
    top = z.amax(1, keepdim=True)
    hit = z.gather(1, at)[:, 0]
    z.sub_(top).exp_()
    total = z.sum(1, keepdim=True)
    lse = (top + total.log())[:, 0]
    loss = torch.where(counts, lse - hit, 0.0)
    if not s["case"]["train"]:
        return dict(loss=loss, lse=lse)
    z.div_(total)
    z.scatter_add_(1, at, torch.full_like(at, -1, dtype=z.dtype))
    z.mul_(torch.where(counts, s["dloss"], 0.0)[:, None])
    return dict(loss=loss, lse=lse, dx=(z @ w).to(s["x"].dtype), dw=(z.t() @ x).to(s["w"].dtype))


def _plain_i8(s):
    x = s["x"].float()
    scale = x.abs().amax(1) / torch.full((), 127.0, device=x.device)
    q = torch.where(scale[:, None] > 0, x / scale[:, None], 0.0).round().clamp(-127, 127)
    y = (q @ s["w"].float().t()) * scale[:, None] * s["w_scale"]  # whole numbers, exact below 2^24
    if s["bias"] is not None:
        y = y + s["bias"]
    y = y.to(s["x"].dtype)
    return dict(y=y) if s["case"]["dynamic"] else dict(q=q.to(torch.int8), scale=scale, y=y)


def run(state):
    if own:
        return _run_own(state)
    return {"scan": _plain_scan, "loss": _plain_loss, "i8": _plain_i8}[state["case"]["op"]](state)


# ---- 64 bits -------------------------------------------------------------------------------


def _exact_scan(s):
    c = s["case"]
    kind, train = c["kind"], c["train"]
    nb, nt, _ = s["gate"].shape
    h = s["h0"].double()
    end = s["lengths"].long() if s["lengths"] is not None else torch.full((nb,), nt, device=h.device)
    hs = torch.zeros(s["gate"].shape, dtype=torch.float64, device=h.device)

    def factors(t):
        g = s["gate"][:, t].double()
        return (torch.sigmoid(g), torch.sigmoid(-g)) if kind == "sigmoid" else (g, torch.ones_like(g))

    ragged = s["lengths"] is not None
    for t in range(nt):
        a, k = factors(t)
        new = a * h + k * s["x"][:, t].double()
        if ragged:
            on = (t < end)[:, None]
            h = torch.where(on, new, h)
            hs[:, t] = torch.where(on, new, 0.0)
        else:
            h = hs[:, t] = new
    out = dict(h=hs, last=h)
    if not train:
        return out
    carry = s["dh_last"].double()
    dgate, dx = torch.zeros_like(hs), torch.zeros_like(hs)
    for t in range(nt - 1, -1, -1):
        a, k = factors(t)
        on = (t < end)[:, None]
        total = torch.where(on, carry + s["dh"][:, t].double(), 0.0)
        prev = hs[:, t - 1] if t else s["h0"].double()
        slope = total * (prev - s["x"][:, t].double()) * a * k if kind == "sigmoid" else total * prev
        dgate[:, t], dx[:, t] = slope, total * k
        carry = torch.where(on, total * a, carry)
    return dict(out, dgate=dgate, dx=dx, dh0=carry)


def _exact_loss(s):
    train = s["case"]["train"]
    x, w = s["x"].double(), s["w"].double()
    x.requires_grad_(train)
    w.requires_grad_(train)
    counts = (s["targets"] >= 0) & (s["targets"] < w.shape[0])
    z = torch.mm(x, w.t())
    lse = torch.logsumexp(z, 1)
    loss = torch.where(counts, lse - z[torch.arange(z.shape[0], device=z.device), s["targets"].clamp(min=0)], 0.0)
    if not train:
        return dict(loss=loss, lse=lse)
    loss.backward(s["dloss"].double())
    return dict(loss=loss.detach(), lse=lse.detach(), dx=x.grad, dw=w.grad)


def _exact_i8(s):
    x = s["x"].double()
    scale = (x.abs().max(1).values / 127).float().double()  # the scale is a 32-bit number by definition
    q = torch.zeros_like(x)
    on = scale > 0
    q[on] = torch.round((x[on] / scale[on, None]).float().double()).clamp_(-127, 127)
    y = torch.einsum("mk,nk->mn", q, s["w"].double()) * (scale[:, None] * s["w_scale"].double())
    y = y if s["bias"] is None else y + s["bias"].double()
    return dict(y=y) if s["case"]["dynamic"] else dict(q=None, scale=scale, y=y)


def exact(case, seed):
    if case["op"] == "scan" and case["time"] * (2 if case["train"] else 1) > 100000:
        return None  # one step at a time takes too long
    s = prepare(case, seed)
    return {"scan": _exact_scan, "loss": _exact_loss, "i8": _exact_i8}[case["op"]](s)


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "scan":
        n, states = case["batch"] * case["time"] * case["dim"], case["batch"] * case["dim"]
        arrays = 3 + (0 if not case["train"] else 6 if case["kind"] == "sigmoid" else 5)
        return dict(bytes=n * e * arrays + states * 4 * (5 if case["train"] else 2), flops=n * (10 if case["train"] else 3))
    if case["op"] == "loss":
        n, d, v = case["tokens"], case["dim"], case["vocab"]
        return dict(bytes=(n * d + v * d) * e * (2 if case["train"] else 1) + n * 20, flops=2.0 * n * d * v * (3 if case["train"] else 1))
    m, k, n = case["rows"], case["inner"], case["cols"]
    return dict(bytes=m * k * (e + (0 if case["dynamic"] else 1)) + n * k + m * n * e + 4 * n * (2 if case["bias"] else 1) + 4 * m, flops=2.0 * m * n * k)
