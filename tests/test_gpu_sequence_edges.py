"""The sequence-model operators on the device where values leave the ordinary
range: infinite logits and weights, products of gates that overflow, sizes next
to a limit of the launch, more than one piece of the vocabulary."""
import numpy as np
import pytest

import sequence_parts as parts
import sequence_ref as ref
from conftest import load_pkg
from test_gpu_sequence import be, check_loss, check_scan, i8_inputs, loss_inputs, near, run_scan, scan_inputs, seq, torch_backend  # noqa: F401

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f64", "bf16", "f16"]


# ---- sizes next to a limit of the launch ---------------------------------------

# rows x (inner rounded up to 16) up to and from 40 KiB and 48 KiB, the kernels'
# static shared memory (1 KiB) below 48 KiB among them, and up to 160 KiB, for each
# number of rows that the few-row kernel is compiled for; smaller ones first
I8_SHARED = [(8, 5120, 40), (8, 5136, 40), (7, 6880, 40), (8, 6016, 64), (8, 6032, 64), (8, 6144, 64), (8, 6160, 64), (6, 8192, 64), (5, 9820, 33),
             (7, 7008, 64), (4, 12032, 40), (4, 12288, 64), (3, 16384, 40), (2, 24064, 24), (2, 24576, 24), (1, 40960, 16), (1, 48128, 16),
             (1, 48144, 16), (1, 49152, 16), (1, 49168, 16), (8, 20480, 24), (5, 32768, 24), (8, 20496, 24)]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("shape", I8_SHARED, ids=str)
def test_i8_rows_next_to_48_kib(be, seq, shape, dtype):
    x, w, ws, _ = i8_inputs(sum(shape), *shape, dtype)
    X, W, WS = seq.upload(be, x, dtype), seq.upload(be, w), seq.upload(be, ws)
    rq, rs = ref.quantize(x)
    want = ref.matmul_i8(rq, rs, w, ws, None, dtype)
    assert np.array_equal(seq.linear_i8(be, X, W, WS).to_numpy().astype(np.float64), want)
    q, scale = seq.quantize_rows(be, X)
    assert np.array_equal(seq.matmul_i8(be, q, scale, W, WS, dtype=dtype).to_numpy().astype(np.float64), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(8, 6136, 9), (5, 6136, 9), (5, 6137, 9), (4, 12280, 9), (1, 10230, 9), (1, 10232, 40), (8, 1278, 9), (8, 1280, 9)], ids=str)
def test_loss_rows_next_to_a_limit(be, seq, shape, dtype):
    """x at the sizes where f32 asks for more shared memory, or for another kernel."""
    x, w, targets, g = loss_inputs(sum(shape), *shape, dtype)
    up = lambda v: seq.upload(be, v, dtype)  # noqa: E731
    check_loss(be, seq, up(x), up(w), seq.upload(be, targets, "i64"), seq.upload(be, g), x, w, targets, g, dtype)


# ---- infinite logits ---------------------------------------------------------


def masked_vocabulary(n, v, masked, dtype, seed=21, d=40):
    """x, w, targets, dloss with a column of ones in x and -inf in w's column for
    the masked entries; targets are never masked.  `live`: the other entries."""
    x, w, _, g = loss_inputs(seed, n, d, v, dtype)
    live = np.setdiff1d(np.arange(v), masked)
    r = np.random.default_rng(seed)
    targets = r.choice(live, n)
    x[:, -1], w[:, -1] = 1, 0
    w[masked, -1] = -np.inf
    return x, w, targets, g, live


MASKS = {"end": (32128, np.arange(32000, 32128)), "start": (1000, np.arange(300)), "tiles": (2100, np.r_[256:768, 1024:1280, 2000:2100]),
         "short": (64, np.arange(32, 64))}


def check_masked_forward(be, seq, n, mask, dtype):
    v, masked = MASKS[mask]
    x, w, targets, _, live = masked_vocabulary(n, v, masked, dtype)
    loss, lse = seq.linear_cross_entropy(be, seq.upload(be, x, dtype), seq.upload(be, w, dtype), seq.upload(be, targets, "i64"))
    # masked entries add exactly nothing: the bounds are those of the others
    rl, rs, _, _, el, es = ref.loss(x, w[live], np.searchsorted(live, targets), dtype)
    near(loss.to_numpy(), rl, el)
    near(lse.to_numpy(), rs, es)


@pytest.mark.parametrize("mask", sorted(MASKS))
@pytest.mark.parametrize("n", [1, 8, 9, 200])
@pytest.mark.parametrize("dtype", ["f64", "bf16", "f16"])
def test_loss_of_a_masked_vocabulary(be, seq, dtype, n, mask):
    check_masked_forward(be, seq, n, mask, dtype)


@pytest.mark.parametrize("mask", sorted(MASKS))
@pytest.mark.parametrize("n", [1, 8])
def test_loss_of_a_masked_vocabulary_few_tokens_f32(be, seq, n, mask):
    check_masked_forward(be, seq, n, mask, "f32")


def check_infinite_logits(be, seq, n, dtype):
    """lse by its definition: -inf where every logit is, inf where one is, NaN
    where one is NaN; a masked target's loss is inf."""
    d, v = 24, 600
    x, w, _, _ = loss_inputs(22, n, d, v, dtype)
    x[:, -1], w[:, -1] = 1, 0
    T = seq.upload(be, np.full(n, 5), "i64")

    def run(w):
        loss, lse = seq.linear_cross_entropy(be, seq.upload(be, x, dtype), seq.upload(be, w, dtype), T)
        return loss.to_numpy(), lse.to_numpy()

    gone = w.copy()
    gone[:, -1] = -np.inf
    assert (run(gone)[1] == -np.inf).all()
    one = w.copy()
    one[300, -1] = np.inf
    loss, lse = run(one)
    assert (lse == np.inf).all() and (loss == np.inf).all()
    both = gone.copy()
    both[300:302, -1] = np.inf
    assert (run(both)[1] == np.inf).all()
    for base in (w, gone, one):
        bad = base.copy()
        bad[17, -1] = np.nan
        assert np.isnan(run(bad)[1]).all()
    target = w.copy()
    target[5, -1] = -np.inf
    loss, lse = run(target)
    assert (loss == np.inf).all() and np.isfinite(lse).all()


@pytest.mark.parametrize("n", [1, 8, 9, 200])
@pytest.mark.parametrize("dtype", ["f64", "bf16", "f16"])
def test_loss_of_infinite_logits(be, seq, dtype, n):
    check_infinite_logits(be, seq, n, dtype)


@pytest.mark.parametrize("n", [1, 8])
def test_loss_of_infinite_logits_few_tokens_f32(be, seq, n):
    check_infinite_logits(be, seq, n, "f32")


def check_masked_backward(be, seq, n, mask, dtype):
    """Tokens without a loss get exact zeros and reach nothing, although their
    logits are NaN (0 * -inf); the masked column of dx is 0 * -inf = NaN for the
    others, as the formula has it, and nothing else is touched."""
    v, masked = MASKS[mask]
    x, w, targets, g, live = masked_vocabulary(n, v, masked, dtype)
    x[::3], targets[::3] = np.nan, -100
    if n > 3:
        targets[3] = v
    ignored = (targets < 0) | (targets >= v)
    clean = np.where(ignored[:, None], 0.0, x)
    where = np.where(ignored, -100, np.searchsorted(live, targets))
    lse = np.where(ignored, 0.0, ref.loss(clean, w[live], where, dtype)[1]).astype(g.dtype)
    dx, dw = seq.linear_cross_entropy_backward(be, seq.upload(be, x, dtype), seq.upload(be, w, dtype), seq.upload(be, targets, "i64"),
                                               seq.upload(be, np.where(ignored, np.nan, lse).astype(g.dtype)), seq.upload(be, g))
    dx, dw = (np.asarray(a.to_numpy(), np.float64) for a in (dx, dw))
    ax, aw, ex, ew = ref.loss_backward(clean, w[live], where, lse.astype(np.float64), g, dtype)
    near(dw[live], aw, ew)
    assert not dw[masked].any()  # (NaN counts as any)
    near(dx[:, :-1], ax[:, :-1], ex[:, :-1])
    assert not dx[ignored].any() and np.isnan(dx[~ignored, -1]).all()


@pytest.mark.parametrize("mask", sorted(MASKS))
@pytest.mark.parametrize("n", [1, 2, 8, 9, 200])
@pytest.mark.parametrize("dtype", ["f64", "bf16", "f16"])
def test_loss_gradients_of_a_masked_vocabulary(be, seq, dtype, n, mask):
    check_masked_backward(be, seq, n, mask, dtype)


@pytest.mark.parametrize("mask", sorted(MASKS))
@pytest.mark.parametrize("n", [1, 2, 8])
def test_loss_gradients_of_a_masked_vocabulary_few_tokens_f32(be, seq, n, mask):
    check_masked_backward(be, seq, n, mask, "f32")


@pytest.mark.parametrize("mask", sorted(MASKS))
@pytest.mark.parametrize("n", [9, 200])
def test_loss_of_a_masked_vocabulary_f32(be, seq, n, mask):
    check_masked_forward(be, seq, n, mask, "f32")
    check_masked_backward(be, seq, n, mask, "f32")


@pytest.mark.parametrize("n", [9, 200])
def test_loss_of_infinite_logits_f32(be, seq, n):
    check_infinite_logits(be, seq, n, "f32")


@pytest.mark.parametrize("n", [8, 9, 200])
def test_loss_of_an_infinite_activation_f32(be, seq, n):
    """One token's row holds an infinity: its logits alone are infinite."""
    x, w, _, g = loss_inputs(23, n, 40, 300, "f32")
    w[:, 7] = np.abs(w[:, 7]) + 0.5
    targets = np.random.default_rng(1).integers(0, 300, n)
    clean = x.copy()
    x[4, 7] = np.inf
    loss, lse = seq.linear_cross_entropy(be, seq.upload(be, x, "f32"), seq.upload(be, w, "f32"), seq.upload(be, targets, "i64"))
    rl, rs, _, _, el, es = ref.loss(clean, w, targets, "f32")
    others = np.arange(n) != 4
    near(loss.to_numpy()[others], rl[others], el[others])
    near(lse.to_numpy()[others], rs[others], es[others])
    assert lse.to_numpy()[4] == np.inf


@pytest.mark.parametrize("n", [8, 9, 200])
def test_loss_of_the_largest_f32(be, seq, n):
    """Numbers within half a bf16 step of f32's largest, which round to infinity
    in bf16, times ones of 2^-100 and 2^-110."""
    top = float(np.finfo(np.float32).max)
    for huge, size in (("x", 2.0 ** -100), ("w", 2.0 ** -100), ("w", 2.0 ** -110)):
        x, w, targets, g = loss_inputs(24, n, 24, 200, "f32")
        a, b = (x, w) if huge == "x" else (w, x)
        a[:, 3] = top * np.sign(a[:, 3])
        a[1, 3] = top * (1 - 2.0 ** -9)
        b[:, 3] *= size
        x, w = ref.rounded(x, "f32"), ref.rounded(w, "f32")
        loss, lse = seq.linear_cross_entropy(be, seq.upload(be, x, "f32"), seq.upload(be, w, "f32"), seq.upload(be, targets, "i64"))
        rl, rs, _, _, el, es = ref.loss(x, w, targets, "f32")
        # A number's third bf16 part is rounded to bf16's smallest step, 2^-133, where
        # the number is below 2^-109: up to 2^-134 of it are lost, times the other
        # factor, for each term of a logit; a loss has two logits.  (Here: 2^-134 *
        # 2^128 = 2^-6 for x of 2^-116 beside w of 2^128.)
        lost = 2.0 ** -134 * (np.abs(x).sum(1) + np.abs(w).sum(1).max())
        near(loss.to_numpy(), rl, el + 2 * lost)
        near(lse.to_numpy(), rs, es + lost)


@pytest.mark.parametrize("n", [8, 9, 200])
def test_loss_gradients_of_infinite_dloss_f32(be, seq, n):
    """A token's dloss of infinity makes its own row of dx infinite or NaN and
    leaves the other rows alone."""
    x, w, targets, g = loss_inputs(25, n, 40, 300, "f32")
    targets = np.abs(targets) % 300
    g[2] = np.inf
    X, W, T = seq.upload(be, x, "f32"), seq.upload(be, w, "f32"), seq.upload(be, targets, "i64")
    _, lse = seq.linear_cross_entropy(be, X, W, T)
    dx, _ = seq.linear_cross_entropy_backward(be, X, W, T, lse, seq.upload(be, g))
    g[2] = 0
    ax, _, ex, _ = ref.loss_backward(x, w, targets, lse.to_numpy().astype(np.float64), g, "f32")
    others = np.arange(n) != 2
    near(dx.to_numpy()[others], ax[others], ex[others])
    assert not np.isfinite(dx.to_numpy()[2]).any()


# ---- gates whose products leave the type -----------------------------------------


def growing_inputs(t, d, dtype):
    """A tiny state that grows by more than the type's range of factors and
    shrinks again, is set back by a gate of zero, and the same for the gradient
    from the other end.  Every state and gradient is finite."""
    up = 256.0 if dtype == "f64" else 2.0
    tiny = 2.0 ** -1000 if dtype == "f64" else 2.0 ** -120
    r = np.random.default_rng(t + d)
    gate = 0.5 + 0.5 * r.random((1, t, d))
    x, dh = r.normal(size=(1, t, d)), r.normal(size=(1, t, d))
    gate[:, :140], gate[:, 140:240], gate[:, 240:1000] = up, 1 / up, 1
    x[:, :1000], dh[:, :1000] = 0, 0
    gate[:, 1000], x[:, 1000] = 0, 3
    e = t - 500
    gate[:, e], x[:, e:], dh[:, e:] = 0, 0, 0
    gate[:, e + 1:t - 240], gate[:, t - 240:t - 140], gate[:, t - 140:] = 1, 1 / up, up
    st = np.float64 if dtype == "f64" else np.float32
    ends = [(tiny * (1 + np.arange(d) % 3)).astype(st)[None] for _ in range(2)]
    return [ref.rounded(v, dtype) for v in (gate, x, dh)] + ends


@pytest.mark.parametrize("dtype", ["f32", "f64", "bf16"])
@pytest.mark.parametrize("t,d", [(1700, 9), (6000, 24), (20000, 7), (6000, 2048), (3000, 4100)])
def test_scan_gates_that_grow_past_the_type(be, seq, t, d, dtype):
    """A product of gates outside the state's type, over states inside it."""
    args = growing_inputs(t, d, dtype)
    check_scan(run_scan(be, seq, *args, None, "linear", dtype), *args, None, "linear", dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scan_growing_gates_and_lengths(be, seq, dtype):
    t, d = 5000, 40
    args = growing_inputs(t, d, dtype)
    lengths = np.array([t, 0, 200, 1001, t - 1, 3000], np.int32)
    args = [np.repeat(a, len(lengths), 0) for a in args]
    args[4] *= np.float32(2.0 ** 60)  # the gradient of the last state, where a sequence ends early
    # a gradient that enters before the state has shrunk again grows out of the
    # type as the definition has it; those sequences get none
    args[4][[2]] = 0
    args[4][[0, 4]] *= np.float32(2.0 ** -60)
    check_scan(run_scan(be, seq, *args, lengths, "linear", dtype), *args, lengths, "linear", dtype)


@pytest.mark.parametrize("kind", ["linear", "sigmoid"])
def test_scan_infinite_state(be, seq, kind):
    """An infinite x leaves the state infinite for as long as gates are not
    zero, however many steps that is, and 0 * inf = NaN from a zero gate on."""
    t, d = 9000, 12
    r = np.random.default_rng(3)
    gate = r.normal(size=(1, t, d)) + 1
    if kind == "linear":
        gate = 1 / (1 + np.exp(-gate))
    x = r.normal(size=(1, t, d))
    x[0, 100, 2], x[0, 4000, 5], x[0, 7, 8] = np.inf, -np.inf, np.inf
    if kind == "linear":
        gate[0, 6000, 8] = 0
    gate, x = ref.rounded(gate, "f32"), ref.rounded(x, "f32")
    h, last = seq.gated_scan(be, seq.upload(be, gate, "f32"), seq.upload(be, x, "f32"), kind=kind)
    h = h.to_numpy()[0]
    assert (h[100:, 2] == np.inf).all() and (h[4000:, 5] == -np.inf).all() and (h[7:6000, 8] == np.inf).all()
    assert np.isnan(h[6000:, 8]).all() if kind == "linear" else (h[6000:, 8] == np.inf).all()
    ok = np.setdiff1d(np.arange(d), [2, 5, 8])
    want, wl, e, el = ref.scan(gate[:, :, ok], x[:, :, ok], None, None, kind, "f32")
    near(h[None][:, :, ok], want, e, "f32")
    near(last.to_numpy()[:, ok], wl, el)


# ---- f32 in three parts --------------------------------------------------------


@pytest.mark.parametrize("n", [9, 12, 130, 700])
def test_f32_logits_keep_24_bits(be, seq, n):
    """Logits found back from lse - loss, one target after another."""
    v = 300
    x, w = parts.logit_inputs(n, v, 31)
    z = x @ w.T
    X, W = seq.upload(be, x, "f32"), seq.upload(be, w, "f32")
    for shift in range(0, v, 37):
        targets = (np.arange(n) + shift) % v
        loss, lse = (a.to_numpy().astype(np.float64) for a in seq.linear_cross_entropy(be, X, W, seq.upload(be, targets, "i64")))
        want = z[np.arange(n), targets]
        # the loss is rounded once, of a difference below 70
        assert (np.abs(lse - loss - want) <= parts.LOGIT * want + parts.U * 70).all()


@pytest.mark.parametrize("n,d", [(9, 40), (200, 40), (200, 328), (700, 40)])
def test_f32_gradients_keep_24_bits(be, seq, n, d):
    x, w, targets, g = parts.gradient_inputs(n, d, 32)
    X, W, T = seq.upload(be, x, "f32"), seq.upload(be, w, "f32"), seq.upload(be, targets, "i64")
    _, lse = seq.linear_cross_entropy(be, X, W, T)
    s = lse.to_numpy().astype(np.float64)
    dx, _ = seq.linear_cross_entropy_backward(be, X, W, T, lse, seq.upload(be, g))
    want, _, bound, _ = ref.loss_backward(x, w, targets, s, g, "f32")
    near(dx.to_numpy(), want, bound)
    for k in list(range(0, n, max(1, n // 30))):
        only = np.zeros_like(g)
        only[k] = g[k]
        _, dw = seq.linear_cross_entropy_backward(be, X, W, T, lse, seq.upload(be, only))
        _, want, _, bound = ref.loss_backward(x, w, targets, s, only, "f32")
        near(dw.to_numpy(), want, bound)


# ---- more than one piece of the vocabulary ---------------------------------------


def check_in_blocks(seq, be, n, d, v, dtype):
    """The loss and its gradients against 64 bits in blocks of the vocabulary on the
    device, by the bounds of ref.loss and ref.loss_backward (twice those in f64,
    where the other side rounds as much)."""
    import torch
    tt = dict(f32=torch.float32, f64=torch.float64, bf16=torch.bfloat16, f16=torch.float16)[dtype]
    st = torch.float64 if dtype == "f64" else torch.float32
    unit, half, twice = ref.state_unit(dtype), ref.HALF[dtype], 2.0 if dtype == "f64" else 1.0
    r = torch.Generator("cuda").manual_seed(n + d + v)
    x = torch.randn(n, d, generator=r, device="cuda").to(tt)
    w = torch.empty(v, d, device="cuda", dtype=tt)
    step = max(1, (1 << 25) // max(n, d))
    for i in range(0, v, step):
        w[i:i + step] = torch.randn(min(step, v - i), d, generator=r, device="cuda").mul_(1.5 / d ** 0.5)
    targets = torch.randint(0, v, (n,), generator=r, device="cuda")
    targets[::7] = -100
    targets[1], targets[2] = v - 1, 0
    dloss = torch.rand(n, generator=r, device="cuda", dtype=st) / n
    loss, lse = seq.linear_cross_entropy(be, x, w, targets)
    dx, dw = seq.linear_cross_entropy_backward(be, x, w, targets, lse, dloss)

    ok = targets >= 0
    x64 = x.double()
    x0 = torch.where(ok[:, None], x64, 0.0)
    g = torch.where(ok, dloss.double(), 0.0)[:, None]
    given = lse.double()[:, None]
    true = torch.full((n,), -torch.inf, device="cuda", dtype=torch.double)
    for i in range(0, v, step):
        true = torch.logaddexp(true, torch.logsumexp(x64 @ w[i:i + step].double().t(), 1))
    hit, ehit = torch.zeros(n, device="cuda", dtype=torch.double), torch.zeros(n, device="cuda", dtype=torch.double)
    spread = torch.zeros(n, device="cuda", dtype=torch.double)
    rx, tx, ax = (torch.zeros(n, d, device="cuda", dtype=torch.double) for _ in range(3))

    def inside(got, want, bound):
        off = (got.double() - want).abs()
        bad = ~(off <= bound)
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist(), off[bad][:3].tolist(), bound[bad][:3].tolist())

    def result_bound(ref_value, terms, carried, length, wide):
        e = carried + (terms + carried) * ref.logit_error(length, dtype) + ref_value.abs() * half * 2 + ref.TINY[dtype] + terms * 16 * unit
        return (e if dtype == "f64" else e + 2.0 ** -126 * wide) * twice

    for i in range(0, v, step):
        wb = w[i:i + step].double()
        z = x64 @ wb.t()
        ez = (x64.abs() @ wb.abs().t()) * ref.logit_error(d, dtype)
        here = (targets >= i) & (targets < i + wb.shape[0])
        rows = here.nonzero()[:, 0]
        at = targets[rows] - i
        hit[rows], ehit[rows] = z[rows, at], ez[rows, at]
        p = torch.exp(z - true[:, None])
        spread += (p * (ez + unit * (16 + 2 * (z - true[:, None]).abs()))).sum(1)
        p = torch.exp(z - given)
        one = torch.zeros_like(p)
        one[rows, at] = 1
        dz = g * (p - one)
        ep = g * (p * (ez + unit * (16 + 2 * (z - given).abs())) + 2 * unit * (p + one))
        if dtype in ("bf16", "f16"):
            ep += dz.abs() * half * (1 + half)
            if dtype == "f16":
                ep += torch.where(ok, g.max() * 2.0 ** -38, 0.0)[:, None]
        rx += dz @ wb
        tx += dz.abs() @ wb.abs()
        ax += ep @ wb.abs()
        want = dz.t() @ x0
        inside(dw[i:i + step], want, result_bound(want, dz.abs().t() @ x0.abs(), ep.t() @ x0.abs(), n, (x0.abs() + 4).sum(0)[None]))
    wide = torch.zeros(d, device="cuda", dtype=torch.double)
    for i in range(0, v, step):
        wide += (w[i:i + step].double().abs() + 4).sum(0)
    inside(dx, rx, result_bound(rx, tx, ax, v, wide[None]))
    assert not dx[~ok].any() and not loss[~ok].any()
    elae = spread + 64 * unit + 4 * unit * true.abs()
    inside(lse, true, elae * twice)
    inside(loss[ok], (true - hit)[ok], ((elae + ehit + 4 * unit * (true.abs() + hit.abs())) * twice)[ok])


# 16 bits and f32: pieces of 2^28 / tokens entries in whole 256s; f32 weights in
# pieces of 2^30 / (6 width); f64 and exact f32: pieces of 256 MiB in whole 128s.
# (tokens, width, vocabulary): a last piece of 40 entries beside sums in 4 splits,
# shorter than a split; pairs of SMs with an odd vocabulary; one whole piece more
PIECES = [(4200, 64, 2 * 63744 + 40), (8200, 264, 2 * 32512 + 3), (8200, 72, 2 * 32512 + 256)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", PIECES, ids=str)
def test_loss_in_pieces(seq, shape, dtype):
    be = torch_backend()
    check_in_blocks(seq, be, *shape, dtype)
    be.close()


@pytest.mark.parametrize("shape", [(9, 16384, 2 * 10752 + 40), (9, 16384, 3 * 10752), (130, 20000, 8704 + 1)], ids=str)
def test_loss_f32_weights_in_pieces(seq, shape):
    be = torch_backend()
    check_in_blocks(seq, be, *shape, "f32")
    be.close()


@pytest.mark.parametrize("shape", [(4000, 16, 2 * 8320 + 40), (4000, 33, 3 * 8320)], ids=str)
def test_loss_f64_in_pieces(seq, shape):
    be = torch_backend()
    check_in_blocks(seq, be, *shape, "f64")
    be.close()


@pytest.mark.parametrize("shape", [(4000, 16, 2 * 16768 + 40), (4000, 33, 3 * 16768)], ids=str)
def test_loss_exact_f32_in_pieces(seq, shape):
    be = torch_backend()
    be.set_f32_mode("exact")
    check_in_blocks(seq, be, *shape, "f32")
    be.close()


# ---- next to the engine, and on another device -------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "f64"])
def test_an_einsum_feeds_the_operators_and_takes_their_result(be, seq, dtype):
    """Projections by the engine, the recurrence and the loss on its column-major
    results, and the engine again on a gradient, all on one storage."""
    import importlib
    E = importlib.import_module("omeinsum_b200.einsum")
    b, t, d, e, v = 2, 130, 24, 40, 300
    r = np.random.default_rng(41)
    nt = np.float32 if dtype == "f32" else np.float64
    tol = 1e-5 if dtype == "f32" else 1e-12  # of the terms' sum: the engine's own
    u, wg, wx = (r.normal(size=s).astype(nt) for s in ((b, t, d), (d, e), (d, e)))
    table, targets = (r.normal(size=(v, e)) / e ** 0.5).astype(nt), r.integers(-20, v, b * t)
    sizes = {0: b, 1: t, 2: d, 3: e}
    col = lambda a: be.from_slice(a.reshape(-1, order="F"))  # noqa: E731
    project = E.Einsum([[0, 1, 2], [2, 3]], [0, 1, 3], sizes)
    U = col(u)
    G, X = (seq.Strided(project.execute(be, "standard", [U, col(m)]), (b, t, e), (1, b, b * t)) for m in (wg, wx))
    for got, m in ((G, wg), (X, wx)):
        assert (np.abs(got.to_numpy() - u.astype(float) @ m) <= tol * (np.abs(u) @ np.abs(m))).all()
    gate, x = (a.to_numpy().astype(np.float64) for a in (G, X))
    h, last = seq.gated_scan(be, G, X, kind="sigmoid")
    flat = seq.Strided(h.storage, (b * t, e))
    W, T = seq.upload(be, table), seq.upload(be, targets, "i64")
    g = (r.random(b * t) / (b * t)).astype(nt)
    check_loss(be, seq, flat, W, T, seq.upload(be, g), flat.to_numpy().astype(np.float64), table.astype(np.float64), targets, g, dtype)
    _, lse = seq.linear_cross_entropy(be, flat, W, T)
    dflat, _ = seq.linear_cross_entropy_backward(be, flat, W, T, lse, seq.upload(be, g))
    dh = seq.Strided(dflat.storage, (b, t, e))
    grads = seq.gated_scan_backward(be, G, X, h, dh, kind="sigmoid")
    check_scan([a.to_numpy() for a in (h, last, *grads)], gate, x, dh.to_numpy().astype(np.float64), None, None, None, "sigmoid", dtype)
    # d loss / d wx = sum over b, t of u dx: dx is row-major, so [e, t, b] to the engine
    back = E.Einsum([[0, 1, 2], [3, 1, 0]], [2, 3], sizes).execute(be, "standard", [U, grads[1].storage])
    got = back.to_vec().reshape(d, e, order="F")
    dx = grads[1].to_numpy().astype(np.float64)
    assert (np.abs(got - np.einsum("btd,bte->de", u, dx)) <= tol * np.einsum("btd,bte->de", np.abs(u), np.abs(dx))).all()


def test_the_current_device_is_left_as_it_was(seq):
    """Calls on device 0's backend while another device is current."""
    import torch
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    om = load_pkg()
    be = om.B200(0, stream=torch.cuda.default_stream(0).cuda_stream)
    x = torch.randn(4, 20, 64, device="cuda:0")
    w = torch.randn(30, 64, device="cuda:0")
    t = torch.zeros(80, device="cuda:0", dtype=torch.int64)
    torch.cuda.synchronize(0)
    with torch.cuda.device(1):
        calls = [lambda: seq.gated_scan(be, x, x, kind="sigmoid"),
                 lambda: seq.gated_scan_backward(be, x, x, x, x, kind="sigmoid"),
                 lambda: seq.linear_cross_entropy(be, x.view(80, 64), w, t),
                 lambda: seq.linear_cross_entropy_backward(be, x.view(80, 64), w, t, t.float(), t.float()),
                 lambda: seq.linear_i8(be, w, *seq.quantize_rows(be, w)),
                 lambda: seq.matmul_i8(be, *seq.quantize_rows(be, x[0]), *seq.quantize_rows(be, w))]
        for call in calls:
            call()
            assert torch.cuda.current_device() == 1
    torch.cuda.synchronize(0)
    be.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(2, 4096, 4096), (2, 4096, 4097), (4, 4096, 4096), (4, 4096, 4100), (8, 2048, 4096), (8, 2064, 4096), (3, 1037, 11000),
                                   (8, 1031, 4100), (1, 4096, 16500), (5, 32, 300000), (8, 20480, 300)], ids=str)
def test_i8_few_rows_on_both_sides_of_the_rule(be, seq, shape, dtype):
    """Where few rows change from the CUDA cores to the tensor cores."""
    x, w, ws, bias = i8_inputs(sum(shape), *shape, dtype)
    X, W, WS, B = seq.upload(be, x, dtype), seq.upload(be, w), seq.upload(be, ws), seq.upload(be, bias)
    rq, rs = ref.quantize(x)
    want = ref.matmul_i8(rq, rs, w, ws, bias, dtype)
    assert np.array_equal(seq.linear_i8(be, X, W, WS, bias=B).to_numpy().astype(np.float64), want)
    q, scale = seq.quantize_rows(be, X)
    assert np.array_equal(seq.matmul_i8(be, q, scale, W, WS, bias=B, dtype=dtype).to_numpy().astype(np.float64), want)


def test_loss_exact_f32_of_few_tokens_and_a_vocabulary_past_2_to_22(seq):
    """16 tokens: a piece's columns would be more than the products' grid holds."""
    be = torch_backend()
    be.set_f32_mode("exact")
    check_in_blocks(seq, be, 16, 9, (1 << 22) + 70, "f32")
    be.close()


# ---- strides of zero and below ---------------------------------------------------


def strided(seq, be, m, layout, dtype):
    """(a view with the layout's strides, the matrix that it shows)."""
    r, c = m.shape
    up = lambda v: seq.upload(be, np.ascontiguousarray(v), dtype).storage  # noqa: E731
    if layout == "rows_backwards":
        return seq.Strided(up(m[::-1]), (r, c), (-c, 1), offset=(r - 1) * c), m
    if layout == "columns_backwards":
        return seq.Strided(up(m[:, ::-1]), (r, c), (c, -1), offset=c - 1), m
    if layout == "both_backwards_transposed":
        return seq.Strided(up(m[::-1, ::-1].T), (r, c), (-1, -r), offset=r * c - 1), m
    if layout == "one_row":
        return seq.Strided(up(m[:1]), (r, c), (0, 1)), np.repeat(m[:1], r, 0)
    if layout == "one_column":
        return seq.Strided(up(m[:, :1]), (r, c), (1, 0)), np.repeat(m[:, :1], c, 1)
    return seq.Strided(up(m[:1, :1]), (r, c), (0, 0)), np.full_like(m, m[0, 0])


LAYOUTS = ["rows_backwards", "columns_backwards", "both_backwards_transposed", "one_row", "one_column", "one_value"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,v", [(5, 72, 130), (70, 104, 333), (150, 33, 400)])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_loss_strides_of_zero_and_below(be, seq, layout, n, d, v, dtype):
    x, w, targets, g = loss_inputs(51, n, d, v, dtype)
    (X, xs), (W, ws) = strided(seq, be, x, layout, dtype), strided(seq, be, w, layout, dtype)
    check_loss(be, seq, X, W, seq.upload(be, targets, "i64"), seq.upload(be, g), xs, ws, targets, g, dtype)


def test_loss_exact_f32_strides_of_zero_and_below(seq):
    om = load_pkg()
    be = om.B200(0)
    be.set_f32_mode("exact")
    for layout in LAYOUTS:
        for n, d, v in ((70, 104, 333), (150, 33, 400)):
            x, w, targets, g = loss_inputs(52, n, d, v, "f32")
            (X, xs), (W, ws) = strided(seq, be, x, layout, "f32"), strided(seq, be, w, layout, "f32")
            check_loss(be, seq, X, W, seq.upload(be, targets, "i64"), seq.upload(be, g), xs, ws, targets, g, "f32")
    be.close()


@pytest.mark.parametrize("m,k,n", [(1, 96, 70), (6, 113, 70), (30, 192, 150), (200, 65, 150)])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_i8_strides_of_zero_and_below(be, seq, layout, m, k, n):
    x, w, ws, bias = i8_inputs(53, m, k, n, "bf16")
    WS, B = seq.upload(be, ws), seq.upload(be, bias)
    (X, xs), (W, shown) = strided(seq, be, x, layout, "bf16"), strided(seq, be, w, layout, None)
    rq, rs = ref.quantize(xs)
    want = ref.matmul_i8(rq, rs, shown, ws, bias, "bf16")
    assert np.array_equal(seq.linear_i8(be, X, W, WS, bias=B).to_numpy().astype(np.float64), want)
    q, scale = seq.quantize_rows(be, X)
    assert np.array_equal(q.to_numpy(), rq) and np.array_equal(scale.to_numpy(), rs)
    Q, shown_q = strided(seq, be, rq, layout, None)
    S = np.linspace(0.5, 1.5, m).astype(np.float32)
    want = ref.matmul_i8(shown_q, S, shown, ws, bias, "bf16")
    assert np.array_equal(seq.matmul_i8(be, Q, seq.upload(be, S), W, WS, bias=B, dtype="bf16").to_numpy().astype(np.float64), want)


@pytest.mark.parametrize("kind", ["linear", "sigmoid"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("axes", [(0,), (2,), (0, 1, 2)], ids=str)
def test_scan_strides_below_zero(be, seq, axes, dtype, kind):
    b, t, d = 3, 700, 40
    gate, x, dh, h0, dl = scan_inputs(54, b, t, d, dtype, kind)

    def place(v):
        strides, at = [t * d, d, 1], 0
        for a in axes:
            at += (v.shape[a] - 1) * strides[a]
            strides[a] = -strides[a]
        return seq.Strided(seq.upload(be, np.ascontiguousarray(np.flip(v, axes)), dtype).storage, (b, t, d), strides, offset=at)

    G, X, E, H0, DL = place(gate), place(x), place(dh), seq.upload(be, h0), seq.upload(be, dl)
    h, last = seq.gated_scan(be, G, X, h0=H0, kind=kind)
    grads = seq.gated_scan_backward(be, G, X, place(h.to_numpy()), E, h0=H0, dh_last=DL, kind=kind)
    check_scan([v.to_numpy() for v in (h, last, *grads)], gate, x, dh, h0, dl, None, kind, dtype)


# ---- long in one extent ------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1200000, 9, 600), (300, 1, 5000), (9, 70001, 300), (300000, 24, 1), (40, 16, 2200000)], ids=str)
def test_loss_long_in_one_extent(seq, shape, dtype):
    be = torch_backend()
    check_in_blocks(seq, be, *shape, dtype)
    be.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 100000, 1), (1, 60000, 3), (70000, 3, 8), (200, 2, 9001), (1, 1, 1 << 20), (3, 17, 200003)], ids=str)
def test_scan_long_in_one_extent(be, seq, shape, dtype):
    args = scan_inputs(61, *shape, dtype, "sigmoid")
    check_scan(run_scan(be, seq, *args, None, "sigmoid", dtype), *args, None, "sigmoid", dtype)


@pytest.mark.parametrize("shape", [(1000003, 5, 3), (70001, 33, 1), (1, 7, 1000001), (9, 1, 300007), (3, 131071, 50), (2000, 131071, 30)], ids=str)
def test_i8_long_in_one_extent(be, seq, shape):
    x, w, ws, _ = i8_inputs(62, *shape, "f32")
    X, W, WS = seq.upload(be, x, "f32"), seq.upload(be, w), seq.upload(be, ws)
    rq, rs = ref.quantize(x)
    want = ref.matmul_i8(rq, rs, w, ws, None, "f32")
    q, scale = seq.quantize_rows(be, X)
    assert np.array_equal(q.to_numpy(), rq) and np.array_equal(scale.to_numpy(), rs)
    assert np.array_equal(seq.linear_i8(be, X, W, WS).to_numpy().astype(np.float64), want)
    assert np.array_equal(seq.matmul_i8(be, q, scale, W, WS).to_numpy().astype(np.float64), want)


def test_views_recorded_and_replayed(seq):
    """A recording whose results are views of storages that it allocates itself."""
    om = load_pkg()
    be = om.B200(0)
    gate, x, dh, h0, _ = scan_inputs(71, 2, 300, 40, "bf16", "sigmoid")
    _, w, targets, g = loss_inputs(72, 600, 40, 500, "bf16")
    G, X, E, H0, W, T, D = (seq.upload(be, *a) for a in ((gate, "bf16"), (x, "bf16"), (dh, "bf16"), (h0,), (w, "bf16"), (targets, "i64"), (g,)))

    def run():
        h, last = seq.gated_scan(be, G, X, h0=H0, kind="sigmoid")
        flat = seq.Strided(h.storage, (600, 40))
        loss, lse = seq.linear_cross_entropy(be, flat, W, T)
        grads = seq.linear_cross_entropy_backward(be, flat, W, T, lse, D)
        back = seq.gated_scan_backward(be, G, X, h, E, h0=H0, kind="sigmoid")
        q, scale = seq.quantize_rows(be, W)
        return [h, last, loss, lse, *grads, *back, seq.linear_i8(be, flat, q, scale)]

    want = [v.to_numpy() for v in run()]
    be.graph_begin()
    out = run()
    graph = be.graph_end()
    for _ in range(3):
        graph.launch()
        be.synchronize()
        assert all(np.array_equal(a.to_numpy(), b) for a, b in zip(out, want))
    # other inputs, in place
    be.upload_into(X.storage, seq.upload(be, -x, "bf16").storage.to_vec())
    want = [v.to_numpy() for v in run()]
    graph.launch()
    be.synchronize()
    assert all(np.array_equal(a.to_numpy(), b) for a, b in zip(out, want))
    del out, graph
    be.close()


@pytest.mark.parametrize("n", [8, 200])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f64"])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_loss_gradients_beside_a_dloss_that_is_no_number(be, seq, value, dtype, n):
    """The other tokens' rows of dx keep their accuracy, however small their dloss."""
    x, w, targets, g = loss_inputs(81, n, 40, 3000, dtype)
    targets[:4] = 7
    g *= 2.0 ** -20
    g[2] = value
    X, W, T = seq.upload(be, x, dtype), seq.upload(be, w, dtype), seq.upload(be, targets, "i64")
    _, lse = seq.linear_cross_entropy(be, X, W, T)
    dx, _ = seq.linear_cross_entropy_backward(be, X, W, T, lse, seq.upload(be, g))
    g[2] = 0
    ax, _, ex, _ = ref.loss_backward(x, w, targets, lse.to_numpy().astype(np.float64), g, dtype)
    others = np.arange(n) != 2
    near(dx.to_numpy()[others], ax[others], ex[others])
    assert not np.isfinite(np.asarray(dx.to_numpy(), np.float64)[2]).any()
