"""The sequence-model operators on the device against their plain 64-bit forms
(tests/sequence_ref.py), at the sizes, strides, lengths and values where they
can go wrong."""
import numpy as np
import pytest

import sequence_ref as ref
from conftest import load_pkg

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f64", "bf16", "f16"]


@pytest.fixture(scope="module")
def be():
    om = load_pkg()
    b = om.B200(0)
    yield b
    b.close()


@pytest.fixture(scope="module")
def seq():
    load_pkg()
    import omeinsum_b200.sequence as s
    return s


def near(got, want, bound, dtype=None):
    """|got - want| <= bound, plus one rounding to dtype."""
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    b = bound
    if dtype is not None:
        b = bound * (1 + 2 * ref.HALF[dtype]) + np.abs(want) * ref.HALF[dtype] + ref.TINY[dtype]
    off = np.abs(got - want)
    bad = ~(off <= b) & ~np.isnan(want)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3].tolist(), off[bad][:3], np.broadcast_to(b, off.shape)[bad][:3])


# ---- recurrence ------------------------------------------------------------


def scan_inputs(seed, b, t, d, dtype, kind):
    r = np.random.default_rng(seed)
    gate = r.normal(size=(b, t, d)) * 1.5 + 2
    if kind == "linear":
        gate = 1 / (1 + np.exp(-gate))
        gate[r.random((b, t, d)) < 0.02] = 0
        gate[r.random((b, t, d)) < 0.02] *= -1
    x, dh = r.normal(size=(b, t, d)), r.normal(size=(b, t, d))
    st = np.float64 if dtype == "f64" else np.float32
    h0, dl = r.normal(size=(b, d)).astype(st), r.normal(size=(b, d)).astype(st)
    return [ref.rounded(v, dtype) for v in (gate, x, dh)] + [h0, dl]


def run_scan(be, seq, gate, x, dh, h0, dl, lengths, kind, dtype):
    up = lambda v, t=dtype: None if v is None else seq.upload(be, v, t)  # noqa: E731
    G, X, E, H0, DL, L = up(gate), up(x), up(dh), up(h0, None), up(dl, None), up(lengths, "i32")
    h, last = seq.gated_scan(be, G, X, h0=H0, lengths=L, kind=kind)
    grads = seq.gated_scan_backward(be, G, X, h, E, h0=H0, dh_last=DL, lengths=L, kind=kind)
    return [v.to_numpy() for v in (h, last, *grads)]


def check_scan(got, gate, x, dh, h0, dl, lengths, kind, dtype):
    h, last, eh, el = ref.scan(gate, x, h0, lengths, kind, dtype)
    near(got[0], h, eh, dtype)
    near(got[1], last, el)
    stored = np.asarray(got[0], np.float64)
    dg, dx, d0, eg, ex, e0 = ref.scan_backward(gate, x, stored, dh, h0, dl, lengths, kind, dtype)
    near(got[2], dg, eg, dtype)
    near(got[3], dx, ex, dtype)
    near(got[4], d0, e0)


SCAN_SHAPES = [(1, 1, 1), (3, 1, 64), (64, 1, 2048), (2, 2, 7), (1, 15, 33), (2, 16, 64), (1, 17, 128), (3, 63, 100), (2, 129, 257),
               (1, 513, 40), (2, 1025, 72), (1, 4097, 24), (1, 2050, 264), (5, 300, 1001), (1, 9000, 8), (300, 3, 5)]


@pytest.mark.parametrize("kind", ["linear", "sigmoid"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SCAN_SHAPES, ids=str)
def test_scan(be, seq, shape, dtype, kind):
    args = scan_inputs(sum(shape), *shape, dtype, kind)
    got = run_scan(be, seq, *args, None, kind, dtype)
    check_scan(got, *args, None, kind, dtype)


@pytest.mark.parametrize("kind", ["linear", "sigmoid"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("t,d", [(1, 16), (40, 16), (700, 9), (1500, 130), (4500, 8)])
def test_scan_lengths_hide_what_lies_behind(be, seq, t, d, dtype, kind):
    """NaN and infinity behind a sequence's end reach nothing; lengths of zero,
    one, all, more than all and less than zero."""
    lengths = np.array([0, 1, t, t + 5, -3, t // 2, (t + 1) // 2 + 1], np.int32)
    args = scan_inputs(5, len(lengths), t, d, dtype, kind)
    dirty = [a.copy() for a in args]
    for b, n in enumerate(np.clip(lengths, 0, t)):
        dirty[0][b, n:], dirty[1][b, n:], dirty[2][b, n:] = np.nan, np.inf, np.nan
    got = run_scan(be, seq, *dirty, lengths, kind, dtype)
    check_scan(got, *args, lengths, kind, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scan_without_start_or_last_gradient(be, seq, dtype):
    gate, x, dh, _, _ = scan_inputs(6, 2, 150, 24, dtype, "linear")
    got = run_scan(be, seq, gate, x, dh, None, None, None, "linear", dtype)
    check_scan(got, gate, x, dh, None, None, None, "linear", dtype)
    G, E = seq.upload(be, gate, dtype), seq.upload(be, dh, dtype)
    h, _ = seq.gated_scan(be, G, seq.upload(be, x, dtype))
    without_x = seq.gated_scan_backward(be, G, None, h, E)
    assert np.array_equal(without_x[0].to_numpy(), got[2]) and np.array_equal(without_x[1].to_numpy(), got[3])


def test_scan_empty(be, seq):
    h0 = seq.upload(be, np.arange(6, dtype=np.float32).reshape(2, 3))
    e = seq.upload(be, np.zeros((2, 0, 3), np.float32))
    h, last = seq.gated_scan(be, e, e, h0=h0)
    assert h.shape == (2, 0, 3) and np.array_equal(last.to_numpy(), h0.to_numpy())
    dg, dx, d0 = seq.gated_scan_backward(be, e, e, h, e, h0=h0, dh_last=h0)
    assert np.array_equal(d0.to_numpy(), h0.to_numpy())
    n = seq.upload(be, np.zeros((0, 4, 3), np.float32))
    assert seq.gated_scan(be, n, n)[0].shape == (0, 4, 3)


@pytest.mark.parametrize("kind", ["linear", "sigmoid"])
def test_scan_extreme_gates(be, seq, kind):
    """Gates of +-inf, zero and one; a NaN stays in its channel from its step on."""
    gate, x, dh, h0, dl = scan_inputs(7, 1, 600, 16, "f32", kind)
    if kind == "sigmoid":
        gate[0, 10, 0], gate[0, 20, 1], gate[0, 30, 2], gate[0, 40, 3] = np.inf, -np.inf, 200, -200
    else:
        gate[0, :, 0], gate[0, :, 1] = 0, 1
    gate[0, 300, 5] = np.nan
    got = run_scan(be, seq, gate, x, dh, h0, dl, None, kind, "f32")
    with np.errstate(invalid="ignore"):
        check_scan(got, gate, x, dh, h0, dl, None, kind, "f32")
    assert np.isnan(got[0][0, 300:, 5]).all() and not np.isnan(got[0][0, :300, 5]).any()


@pytest.mark.parametrize("dtype", ["f32", "f64", "bf16"])
def test_scan_growing_gates(be, seq, dtype):
    """Gates above one over a state of zero, long enough for their product to
    overflow: the state stays zero until something enters it, in both directions."""
    t = 3000
    gate, x, dh = np.full((1, t, 24), 8.0), np.zeros((1, t, 24)), np.zeros((1, t, 24))
    gate[:, 2500:] = 0.5
    x[:, 2600] = 3.0
    dh[:, 2700] = 2.0
    gate[:, :2500, 1], x[:, 1000, 1] = -8.0, 0.0
    got = run_scan(be, seq, gate, x, dh, None, None, None, "linear", dtype)
    h = ref.scan(gate[:, 2500:], x[:, 2500:], None, None, "linear", dtype)
    assert not got[0][:, :2500].any()
    near(got[0][:, 2500:], h[0], h[2], dtype)
    near(got[1], h[1], h[3])
    assert not got[3][:, 2701:].any() and np.isfinite(got[3][:, 2500:]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["time_major", "channel_major", "offset", "broadcast", "reversed", "wide_rows"])
def test_scan_strides(be, seq, layout, dtype):
    b, t, d = 3, 260, 72
    gate, x, dh, h0, dl = scan_inputs(8, b, t, d, dtype, "sigmoid")
    if layout == "broadcast":  # one gate for every sequence and channel
        gate = np.broadcast_to(gate[:1, :, :1], gate.shape).copy()

    def place(v):
        if layout == "time_major":
            s = seq.upload(be, v.transpose(1, 0, 2), dtype).storage
            return seq.Strided(s, (b, t, d), (d, b * d, 1))
        if layout == "channel_major":
            s = seq.upload(be, v.transpose(2, 0, 1), dtype).storage
            return seq.Strided(s, (b, t, d), (t, 1, b * t))
        if layout == "offset":
            s = seq.upload(be, np.concatenate([[7.0] * 3, v.reshape(-1)]), dtype).storage
            return seq.Strided(s, (b, t, d), (t * d, d, 1), offset=3)
        if layout == "reversed":
            s = seq.upload(be, v[:, ::-1], dtype).storage
            return seq.Strided(s, (b, t, d), (t * d, -d, 1), offset=(t - 1) * d)
        if layout == "wide_rows":  # a slice of a wider tensor
            wide = np.full((b, t, 3 * d), 9.0)
            wide[:, :, d:2 * d] = v
            s = seq.upload(be, wide, dtype).storage
            return seq.Strided(s, (b, t, d), (t * 3 * d, 3 * d, 1), offset=d)
        return seq.upload(be, v, dtype)

    G = place(gate)
    if layout == "broadcast":
        G = seq.Strided(seq.upload(be, gate[0, :, 0], dtype).storage, (b, t, d), (0, 1, 0))
    X, E, H0, DL = place(x), place(dh), seq.upload(be, h0), seq.upload(be, dl)
    h, last = seq.gated_scan(be, G, X, h0=H0, kind="sigmoid")
    grads = seq.gated_scan_backward(be, G, X, h, E, h0=H0, dh_last=DL, kind="sigmoid")
    check_scan([v.to_numpy() for v in (h, last, *grads)], gate, x, dh, h0, dl, None, "sigmoid", dtype)


def test_scan_step_by_step_is_the_scan(be, seq):
    """Decoding one token at a time, the state updated in place."""
    gate, x, dh, h0, dl = scan_inputs(9, 3, 20, 40, "bf16", "sigmoid")
    H, last = seq.gated_scan(be, seq.upload(be, gate, "bf16"), seq.upload(be, x, "bf16"), h0=seq.upload(be, h0), kind="sigmoid")
    state = seq.upload(be, h0)
    h, _, eh, el = ref.scan(gate, x, h0, None, "sigmoid", "bf16")
    for t in range(20):
        out, same = seq.gated_scan(be, seq.upload(be, gate[:, t:t + 1], "bf16"), seq.upload(be, x[:, t:t + 1], "bf16"), h0=state, kind="sigmoid", h_last=state)
        assert same is state
        near(out.to_numpy()[:, 0], h[:, t], eh[:, t], "bf16")
    near(state.to_numpy(), last.to_numpy().astype(np.float64), 2 * el)


@pytest.mark.parametrize("t", [1, 40, 300, 5000])
def test_scan_state_in_place(be, seq, t):
    """h_last may be h0, however the sequence is cut."""
    gate, x, _, h0, _ = scan_inputs(16, 2, t, 40, "f32", "sigmoid")
    G, X, state = seq.upload(be, gate, "f32"), seq.upload(be, x, "f32"), seq.upload(be, h0)
    want, last = seq.gated_scan(be, G, X, h0=seq.upload(be, h0), kind="sigmoid")
    got, _ = seq.gated_scan(be, G, X, h0=state, kind="sigmoid", h_last=state)
    assert np.array_equal(got.to_numpy(), want.to_numpy()) and np.array_equal(state.to_numpy(), last.to_numpy())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scan_repeats_bit_for_bit(be, seq, dtype):
    args = scan_inputs(10, 1, 20000, 64, dtype, "sigmoid")
    first = run_scan(be, seq, *args, None, "sigmoid", dtype)
    for _ in range(3):
        again = run_scan(be, seq, *args, None, "sigmoid", dtype)
        assert all(np.array_equal(a, b) for a, b in zip(first, again))


# ---- cross entropy ---------------------------------------------------------


def loss_inputs(seed, n, d, v, dtype, scale=1.5):
    r = np.random.default_rng(seed)
    x, w = r.normal(size=(n, d)), r.normal(size=(v, d)) * scale / np.sqrt(d)
    targets = r.integers(0, v, n)
    if n > 2:
        targets[r.random(n) < 0.15] = -100
        targets[1], targets[2] = v - 1, 0
    g = r.random(n) / max(n, 1)
    st = np.float64 if dtype == "f64" else np.float32
    return ref.rounded(x, dtype), ref.rounded(w, dtype), targets, g.astype(st)


def check_loss(be, seq, X, W, T, G, x, w, targets, g, dtype):
    loss, lse = seq.linear_cross_entropy(be, X, W, T)
    rl, rs, _, _, el, es = ref.loss(x, w, targets, dtype)
    near(loss.to_numpy(), rl, el)
    near(lse.to_numpy(), rs, es)
    dx, dw = seq.linear_cross_entropy_backward(be, X, W, T, lse, G)
    ax, aw, ex, ew = ref.loss_backward(x, w, targets, lse.to_numpy().astype(np.float64), g, dtype)
    near(dx.to_numpy(), ax, ex)
    near(dw.to_numpy(), aw, ew)
    ignored = (targets < 0) | (targets >= w.shape[0])
    assert not dx.to_numpy()[ignored].any() and not loss.to_numpy()[ignored].any()


LOSS_SHAPES = [(1, 64, 100), (1, 1, 1), (3, 5, 2), (24, 2048, 1000), (7, 33, 129), (128, 64, 256), (129, 65, 257), (130, 136, 1030), (300, 200, 4111),
               (64, 512, 20000), (513, 96, 777), (257, 1000, 384), (8, 1000, 5003), (5, 2304, 130), (4, 72, 9001), (2, 9001, 40), (2, 16380, 33), (5, 6540, 33), (8, 8000, 70)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", LOSS_SHAPES, ids=str)
def test_loss(be, seq, shape, dtype):
    x, w, targets, g = loss_inputs(sum(shape), *shape, dtype)
    up = lambda v: seq.upload(be, v, dtype)  # noqa: E731
    check_loss(be, seq, up(x), up(w), seq.upload(be, targets, "i64"), seq.upload(be, g), x, w, targets, g, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", [(600, 72, 6500), (2300, 2100, 2305), (130, 264, 9700), (1500, 1025, 7000)], ids=str)
def test_loss_in_pairs_of_sms(be, seq, shape, dtype):
    """Results large enough for two SMs to share a tile, with ragged ends."""
    x, w, targets, g = loss_inputs(sum(shape), *shape, dtype)
    up = lambda v: seq.upload(be, v, dtype)  # noqa: E731
    check_loss(be, seq, up(x), up(w), seq.upload(be, targets, "i64"), seq.upload(be, g), x, w, targets, g, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["transposed", "offset", "wide_rows"])
def test_loss_strides(be, seq, layout, dtype):
    n, d, v = 70, 104, 333
    x, w, targets, g = loss_inputs(11, n, d, v, dtype)

    def place(m):
        r, c = m.shape
        if layout == "transposed":
            return seq.Strided(seq.upload(be, m.T, dtype).storage, (r, c), (1, r))
        if layout == "offset":
            return seq.Strided(seq.upload(be, np.concatenate([[5.0], m.reshape(-1)]), dtype).storage, (r, c), (c, 1), offset=1)
        wide = np.full((r, 2 * c), 3.0)
        wide[:, 8:8 + c] = m
        return seq.Strided(seq.upload(be, wide, dtype).storage, (r, c), (2 * c, 1), offset=8)

    check_loss(be, seq, place(x), place(w), seq.upload(be, targets, "i32"), seq.upload(be, g), x, w, targets, g, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_loss_padding_holds_anything(be, seq, dtype):
    """Rows without a loss may hold NaN and infinity; every row without one."""
    x, w, targets, g = loss_inputs(12, 140, 72, 300, dtype)
    dirty = x.copy()
    ignored = targets < 0
    dirty[ignored] = np.nan
    dirty[np.argmax(ignored), 3] = np.inf
    gd = np.where(ignored, np.nan, g).astype(g.dtype)
    T = seq.upload(be, targets, "i64")
    X, W, G = seq.upload(be, dirty, dtype), seq.upload(be, w, dtype), seq.upload(be, gd)
    loss, lse = seq.linear_cross_entropy(be, X, W, T)
    rl, _, _, _, el, _ = ref.loss(x, w, targets, dtype)
    near(loss.to_numpy(), rl, el)
    dx, dw = seq.linear_cross_entropy_backward(be, X, W, T, lse, G)
    s = np.where(ignored, 0.0, lse.to_numpy().astype(np.float64))
    ax, aw, ex, ew = ref.loss_backward(x, w, targets, s, g, dtype)
    near(dx.to_numpy(), ax, ex)
    near(dw.to_numpy(), aw, ew)
    T = seq.upload(be, np.full(140, 300), "i64")
    loss, lse = seq.linear_cross_entropy(be, X, W, T)
    dx, dw = seq.linear_cross_entropy_backward(be, X, W, T, lse, G)
    assert not loss.to_numpy().any() and not dx.to_numpy().any() and not dw.to_numpy().any()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_loss_sharp_and_flat(be, seq, dtype):
    """Logits far apart (most exponentials vanish) and all alike."""
    for scale in (60.0, 0.0):
        x, w, targets, g = loss_inputs(13, 40, 64, 500, dtype, scale)
        up = lambda v: seq.upload(be, v, dtype)  # noqa: E731
        check_loss(be, seq, up(x), up(w), seq.upload(be, targets, "i64"), seq.upload(be, g), x, w, targets, g, dtype)


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e4])
def test_loss_gradient_of_any_size(be, seq, size):
    """dloss far from one: 16-bit pieces of dz neither vanish nor overflow.
    f16 gradients hold what f16 can: below its smallest step they are zero."""
    for dtype in ("bf16", "f16"):
        x, w, targets, g = loss_inputs(14, 50, 64, 3000, dtype)
        g = (g * size).astype(np.float32)
        X, W, T, G = seq.upload(be, x, dtype), seq.upload(be, w, dtype), seq.upload(be, targets, "i64"), seq.upload(be, g)
        _, lse = seq.linear_cross_entropy(be, X, W, T)
        dx, dw = seq.linear_cross_entropy_backward(be, X, W, T, lse, G)
        ax, aw, ex, ew = ref.loss_backward(x, w, targets, lse.to_numpy().astype(np.float64), g, dtype)
        near(dx.to_numpy(), ax, ex)
        near(dw.to_numpy(), aw, ew)


def test_loss_exact_f32(seq):
    """f32 without the tensor cores (the mode of the library's products)."""
    om = load_pkg()
    be = om.B200(0)
    be.set_f32_mode("exact")
    for shape in [(70, 104, 333), (3, 5, 2), (130, 64, 20000)]:
        x, w, targets, g = loss_inputs(17, *shape, "f32")
        check_loss(be, seq, seq.upload(be, x, "f32"), seq.upload(be, w, "f32"), seq.upload(be, targets, "i64"), seq.upload(be, g), x, w, targets, g, "f32")
    be.close()


def test_loss_no_tokens(be, seq):
    for dtype in TYPES:
        st = np.float64 if dtype == "f64" else np.float32
        X, W = seq.upload(be, np.zeros((0, 8)), dtype), seq.upload(be, np.ones((5, 8)), dtype)
        T, G = seq.upload(be, np.zeros(0), "i64"), seq.upload(be, np.zeros(0, st))
        loss, lse = seq.linear_cross_entropy(be, X, W, T)
        assert loss.shape == lse.shape == (0,)
        dx, dw = seq.linear_cross_entropy_backward(be, X, W, T, lse, G)
        assert dx.shape == (0, 8) and dw.shape == (5, 8) and not dw.to_numpy().any()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_loss_repeats_bit_for_bit(be, seq, dtype):
    x, w, targets, g = loss_inputs(15, 64, 128, 30000, dtype)
    X, W, T, G = seq.upload(be, x, dtype), seq.upload(be, w, dtype), seq.upload(be, targets, "i64"), seq.upload(be, g)
    runs = []
    for _ in range(3):
        loss, lse = seq.linear_cross_entropy(be, X, W, T)
        runs.append([v.to_numpy() for v in (loss, lse, *seq.linear_cross_entropy_backward(be, X, W, T, lse, G))])
    assert all(np.array_equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


# ---- 8-bit product ---------------------------------------------------------


def i8_inputs(seed, m, k, n, dtype):
    r = np.random.default_rng(seed)
    x = ref.rounded(r.normal(size=(m, k)) * np.exp(r.normal(size=k)), dtype)
    w = r.integers(-128, 128, (n, k)).astype(np.int8)
    return x, w, (r.random(n) + 0.5).astype(np.float32) / 127, r.normal(size=n).astype(np.float32)


I8_SHAPES = [(1, 64, 64), (1, 4096, 512), (1, 1, 1), (2, 31, 17), (3, 16, 100), (8, 1000, 130), (9, 256, 64), (16, 48, 257), (17, 128, 256), (37, 2048, 520),
             (64, 515, 129), (127, 96, 33), (128, 128, 128), (129, 160, 300), (300, 1037, 211), (513, 272, 1000), (5, 9000, 40), (260, 64, 2050), (2100, 520, 2400), (1300, 2100, 7000)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", I8_SHAPES, ids=str)
def test_i8(be, seq, shape, dtype):
    """Whole numbers are equal; results are the definition's to the last bit."""
    x, w, ws, bias = i8_inputs(sum(shape), *shape, dtype)
    X, W, WS, Bi = seq.upload(be, x, dtype), seq.upload(be, w), seq.upload(be, ws), seq.upload(be, bias)
    q, scale = seq.quantize_rows(be, X)
    rq, rs = ref.quantize(x)
    assert np.array_equal(q.to_numpy(), rq) and np.array_equal(scale.to_numpy(), rs)
    for b, B in ((None, None), (bias, Bi)):
        want = ref.matmul_i8(rq, rs, w, ws, b, dtype)
        assert np.array_equal(seq.matmul_i8(be, q, scale, W, WS, bias=B, dtype=dtype).to_numpy().astype(np.float64), want)
        assert np.array_equal(seq.linear_i8(be, X, W, WS, bias=B).to_numpy().astype(np.float64), want)


def test_i8_quantiser_values(be, seq):
    """Ties, zeros, the smallest and largest numbers, NaN and infinity."""
    x = np.zeros((9, 40), np.float32)
    x[1, :5] = [127, 0.5, 1.5, -2.5, -0.5]
    x[2, 3] = -1e-45
    x[3, :2] = [3e38, -3.4e38]
    x[4, :3] = [1, np.inf, -5]
    x[5, :3] = [1, np.nan, -5]
    x[6, :4] = [np.nan, np.inf, 1, -np.inf]
    x[7, :] = np.linspace(-1, 1, 40)
    x[8, :3] = [1e-44, 3e-44, -7e-44]
    q, scale = seq.quantize_rows(be, seq.upload(be, x))
    rq, rs = ref.quantize(x)
    assert np.array_equal(scale.to_numpy(), rs, equal_nan=True)
    assert np.array_equal(q.to_numpy(), rq)
    assert list(rq[1, :5]) == [127, 0, 2, -2, 0] and not rq[4:7].any()
    w = np.ones((3, 40), np.int8)
    y = seq.matmul_i8(be, q, scale, seq.upload(be, w), seq.upload(be, np.ones(3, np.float32))).to_numpy()
    assert np.isnan(y[4:7]).all() and not np.isnan(y[[0, 1, 2, 3, 7, 8]]).any()


def test_i8_largest_sums(be, seq):
    """The largest sums that the integers may reach, in every kernel."""
    for m in (1, 20, 200):
        k = 131071
        q, w = np.full((m, k), -128, np.int8), np.full((3, k), -128, np.int8)
        one, s = seq.upload(be, np.ones(m, np.float32)), seq.upload(be, np.ones(3, np.float32))
        y = seq.matmul_i8(be, seq.upload(be, q), one, seq.upload(be, w), s).to_numpy()
        assert (y == np.float32(128 * 128 * 131071)).all()


@pytest.mark.parametrize("m", [1, 5, 30, 200])
@pytest.mark.parametrize("layout", ["transposed", "offset", "wide_rows"])
def test_i8_strides(be, seq, layout, m):
    k, n = 192, 150
    x, w, ws, _ = i8_inputs(3, m, k, n, "f16")
    rq, rs = ref.quantize(x)

    def place(v, dtype=None):
        r, c = v.shape
        if layout == "transposed":
            return seq.Strided(seq.upload(be, np.ascontiguousarray(v.T), dtype).storage, (r, c), (1, r))
        if layout == "offset":
            return seq.Strided(seq.upload(be, np.concatenate([v.reshape(-1)[:1], v.reshape(-1)]), dtype).storage, (r, c), (c, 1), offset=1)
        wide = np.full((r, 2 * c), 3, v.dtype)
        wide[:, 16:16 + c] = v
        return seq.Strided(seq.upload(be, wide, dtype).storage, (r, c), (2 * c, 1), offset=16)

    want = ref.matmul_i8(rq, rs, w, ws, None, "f16")
    W, WS = place(w), seq.upload(be, ws)
    got = seq.matmul_i8(be, place(rq), seq.upload(be, rs), W, WS, dtype="f16").to_numpy()
    assert np.array_equal(got.astype(np.float64), want)
    assert np.array_equal(seq.linear_i8(be, place(x, "f16"), W, WS).to_numpy().astype(np.float64), want)
    q, scale = seq.quantize_rows(be, place(x, "f16"))
    assert np.array_equal(q.to_numpy(), rq) and np.array_equal(scale.to_numpy(), rs)


def test_i8_empty(be, seq):
    q, s = seq.quantize_rows(be, seq.upload(be, np.zeros((0, 8), np.float32)))
    assert q.shape == (0, 8) and s.shape == (0,)
    q, s = seq.quantize_rows(be, seq.upload(be, np.zeros((2, 0), np.float32)))
    assert not s.to_numpy().any()
    w, ws, b = seq.upload(be, np.zeros((3, 0), np.int8)), seq.upload(be, np.ones(3, np.float32)), np.array([1, 2, 3], np.float32)
    y = seq.matmul_i8(be, q, s, w, ws, bias=seq.upload(be, b))
    assert np.array_equal(y.to_numpy(), np.stack([b, b]))
    # more rows than one launch of the few-row kernel takes
    q, s = seq.upload(be, np.zeros((20, 0), np.int8)), seq.upload(be, np.ones(20, np.float32))
    assert np.array_equal(seq.matmul_i8(be, q, s, w, ws, bias=seq.upload(be, b)).to_numpy(), np.tile(b, (20, 1)))
    assert not seq.linear_i8(be, seq.upload(be, np.zeros((20, 0), np.float32)), w, ws).to_numpy().any()
    with pytest.raises(load_pkg().OmError):
        big = seq.Strided(be.alloc(131072, np.int8), (1, 131072))
        seq.matmul_i8(be, big, seq.upload(be, np.ones(1, np.float32)), big, seq.upload(be, np.ones(1, np.float32)))


# ---- more than 2^31 elements -----------------------------------------------


def torch_backend():
    import torch
    return load_pkg().B200(0, stream=torch.cuda.current_stream().cuda_stream)


def test_scan_past_32_bits(seq):
    """2.29e9 elements; a gate of 1/2 and inputs of 1 lead to whole numbers."""
    import torch
    be, t, d = torch_backend(), 70000, 32768
    x = torch.ones(1, t, d, device="cuda", dtype=torch.bfloat16)
    x[0, -1, -1] = 5
    gate = torch.full((1, 1, 1), 0.5, device="cuda", dtype=torch.bfloat16).expand(1, t, d)
    h, last = seq.gated_scan(be, gate, x)
    assert (h[0, 64::997] == 2)[:, :-1].all() and h[0, -1, -1] == 6 and (h[0, -1, :-1] == 2).all() and last[0, -1] == 6
    dgate, dx, dh0 = seq.gated_scan_backward(be, gate, x, h, torch.ones(1, 1, 1, device="cuda", dtype=torch.bfloat16).expand(1, t, d))
    assert (dx[0, -1] == 1).all() and (dx[0, -2] == 1.5).all() and (dx[0, :-64:997] == 2).all()
    assert (dgate[0, -1] == 2).all() and (dgate[0, 64:-64:997] == 4).all() and (dh0 == 1).all()
    be.close()


def test_loss_past_32_bits(seq):
    """600000 x 4096 weights, against 64-bit values of the last entries."""
    import torch
    be, n, d, v = torch_backend(), 64, 4096, 600000
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(n, d, generator=g, device="cuda").bfloat16()
    w = torch.empty(v, d, device="cuda", dtype=torch.bfloat16)
    for i in range(0, v, 100000):
        w[i:i + 100000] = torch.randn(100000, d, generator=g, device="cuda").mul_(1 / 64)
    targets = torch.arange(v - n, v, device="cuda")
    loss, lse = seq.linear_cross_entropy(be, x, w, targets)
    z = torch.cat([x.double() @ w[i:i + 50000].double().t() for i in range(0, v, 50000)], 1)
    want = torch.logsumexp(z, 1)
    hit = z[torch.arange(n), targets]
    # a logit is off by 2 (D / 8 + 16) half steps of its terms' sum, below 40 here
    bound = 2 * (d / 8 + 16) * 2.0 ** -24 * 40
    assert (lse.double() - want).abs().max() < bound and (loss.double() - (want - hit)).abs().max() < 2 * bound
    dloss = torch.full((n,), 1 / 64, device="cuda")
    dx, dw = seq.linear_cross_entropy_backward(be, x, w, targets, lse, dloss)
    tail = 1000
    dz = torch.exp(z[:, -tail:] - lse.double()[:, None])
    dz[torch.arange(n), targets - (v - tail)] -= 1
    dz /= 64
    ref_dw = dz.t() @ x.double()
    # dz to half a step of bf16, the result too, and dz's own error from its logit
    ok = (dw[-tail:].double() - ref_dw).abs() <= (dz.abs().t() @ x.double().abs()) * (2.0 ** -8 + bound) + ref_dw.abs() * 2.0 ** -8 + 2.0 ** -30
    assert ok.all()
    p = torch.exp(z - lse.double()[:, None])
    p[torch.arange(n), targets] -= 1
    ref_dx, mass = torch.zeros(n, d, device="cuda", dtype=torch.double), torch.zeros(n, d, device="cuda", dtype=torch.double)
    for i in range(0, v, 50000):
        part = w[i:i + 50000].double()
        ref_dx += p[:, i:i + 50000] @ part / 64
        mass += p[:, i:i + 50000].abs() @ part.abs() / 64
    assert ((dx.double() - ref_dx).abs() <= mass * (2.0 ** -8 + bound + 2 * (v / 8 + 16) * 2.0 ** -24) + ref_dx.abs() * 2.0 ** -8).all()
    be.close()


def test_i8_past_32_bits(seq):
    """2.5e9 results, the last rows and columns checked."""
    import torch
    be, m, k = torch_backend(), 50000, 64
    g = torch.Generator("cuda").manual_seed(2)
    q, w = (torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8) for _ in range(2))
    one = torch.ones(m, device="cuda")
    y = seq.matmul_i8(be, q, one, w, one, dtype=torch.bfloat16)
    for rows, cols in ((slice(m - 300, m), slice(0, m)), (slice(0, m), slice(m - 300, m))):
        want = (q[rows].double() @ w[cols].double().t()).float().bfloat16()
        assert torch.equal(y[rows, cols], want)
    be.close()


# ---- together, streams, graphs ---------------------------------------------


def test_refusals_at_the_abi(be, seq):
    """What the front end cannot send: the C entries answer with a status."""
    L = seq._bind()
    s3, s2 = seq._i64s(4, 4, 4), seq._i64s(4, 4)
    neg = seq._i64s(4, -1, 4)
    assert L.om_b200_gated_scan(be.h, 2, 0, s3, *[None] * 9) == 1
    assert L.om_b200_gated_scan(be.h, 0, 3, s3, *[None] * 9) == 2
    assert L.om_b200_gated_scan(be.h, 0, 0, neg, *[None] * 9) == 5
    assert L.om_b200_gated_scan(be.h, 0, 0, s3, *[None] * 9) == 1
    assert L.om_b200_gated_scan_backward(be.h, 0, 0, s3, *[None] * 16) == 1
    assert L.om_b200_linear_cross_entropy(be.h, 7, s3, *[None] * 4, 9, *[None] * 3) == 2
    assert L.om_b200_linear_cross_entropy(be.h, 0, s3, *[None] * 4, 0, *[None] * 3) == 2
    assert L.om_b200_linear_cross_entropy(be.h, 0, seq._i64s(0, 4, 4), *[None] * 4, 9, *[None] * 3) == 5
    assert L.om_b200_linear_cross_entropy_backward(be.h, 0, s3, *[None] * 4, 9, *[None] * 7) == 1
    assert L.om_b200_quantize_rows(be.h, 1, s2, *[None] * 5) == 2
    assert L.om_b200_quantize_rows(be.h, 0, s2, *[None] * 5) == 1
    assert L.om_b200_matmul_i8(be.h, 7, s3, *[None] * 9) == 2
    assert L.om_b200_matmul_i8(be.h, 0, s3, *[None] * 9) == 1
    assert L.om_b200_linear_i8(be.h, 0, neg, *[None] * 8) == 5
    a = be.alloc(16, np.float32)
    one = seq._i64s(16, 1)
    assert L.om_b200_copy_strided(be.h, 5, a.ptr, 1, one, one, 0, a.ptr) == 2  # 16-bit types are not the engine's


def layer(seq, be, t):
    """A training step of a one-layer model and a served token after it."""
    h, last = seq.gated_scan(be, t["gate"], t["x"], h0=t["h0"], kind="sigmoid")
    flat = h.reshape(-1, h.shape[-1])
    loss, lse = seq.linear_cross_entropy(be, flat, t["w"], t["targets"])
    dflat, dw = seq.linear_cross_entropy_backward(be, flat, t["w"], t["targets"], lse, t["dloss"])
    grads = seq.gated_scan_backward(be, t["gate"], t["x"], h, dflat.reshape(h.shape), h0=t["h0"], kind="sigmoid")
    step, state = seq.gated_scan(be, t["gate"][:, :1], t["x"][:, :1], h0=last, kind="sigmoid")
    wq, ws = seq.quantize_rows(be, t["w"])
    logits = seq.linear_i8(be, step[:, 0], wq, ws)
    return dict(h=h, last=last, loss=loss, lse=lse, dw=dw, dgate=grads[0], dx=grads[1], dh0=grads[2], logits=logits, state=state)


def layer_inputs(seed, b=2, t=150, d=72, v=1000):
    import torch
    g = torch.Generator("cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    targets = torch.randint(-50, v, (b * t,), generator=g, device="cuda")
    return dict(gate=(n(b, t, d) + 2).bfloat16(), x=n(b, t, d).bfloat16(), h0=n(b, d), w=(n(v, d) / d ** 0.5).bfloat16(), targets=targets,
                dloss=torch.full((b * t,), 1 / (b * t), device="cuda"))


def test_layer_loss_and_served_token_together(be, seq):
    import torch
    t = layer_inputs(1)
    got = {k: v.double().cpu().numpy() for k, v in layer(seq, be, t).items()}
    a = {k: v.double().cpu().numpy() for k, v in t.items()}
    targets = t["targets"].cpu().numpy()
    h, last, eh, el = ref.scan(a["gate"], a["x"], a["h0"], None, "sigmoid", "bf16")
    near(got["h"], h, eh, "bf16")
    near(got["last"], last, el)
    flat = got["h"].reshape(-1, h.shape[-1])
    rl, rs, _, _, bl, bs = ref.loss(flat, a["w"], targets, "bf16")
    near(got["loss"], rl, bl)
    dx, dw, ex, ew = ref.loss_backward(flat, a["w"], targets, got["lse"], a["dloss"], "bf16")
    near(got["dw"], dw, ew)
    # dflat itself is not returned: its bound, carried through the recurrence
    dg, gx, d0, eg, exx, e0 = ref.scan_backward(a["gate"], a["x"], got["h"], dx.reshape(h.shape), a["h0"], None, None, "sigmoid", "bf16")
    _, wide, wide0, _, _, _ = ref.scan_backward(a["gate"], a["x"], got["h"], ex.reshape(h.shape), a["h0"], None, None, "sigmoid", "bf16")
    near(got["dx"], gx, exx + np.abs(wide), "bf16")
    near(got["dh0"], d0, e0 + np.abs(wide0))
    step, _, es, _ = ref.scan(a["gate"][:, :1], a["x"][:, :1], got["last"], None, "sigmoid", "bf16")
    wq, ws = ref.quantize(a["w"])
    srow = torch.from_numpy(step[:, 0]).bfloat16().double().numpy()
    q, qs = ref.quantize(srow)
    want = ref.matmul_i8(q, qs, wq, ws, None, "bf16")
    # a step value one bf16 step off changes a few q by one and the scale by a step
    one = (np.abs(wq.astype(np.float64)) * ws[:, None]).sum(1)[None] * qs[:, None]
    near(got["logits"], want, one + 2 ** -7 * np.abs(want))


def test_other_stream_than_torchs(seq):
    """A backend on its own stream waits for torch's and torch for it."""
    import torch
    om = load_pkg()
    be = om.B200(0)
    want = layer(seq, om.B200(0, stream=torch.cuda.current_stream().cuda_stream), layer_inputs(2))
    want = {k: v.clone() for k, v in want.items()}
    for _ in range(3):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            torch.cuda._sleep(2_000_000)  # the inputs come late
            t = layer_inputs(2)
            got = {k: v + 0 for k, v in layer(seq, be, t).items()}
        side.synchronize()
        assert all(torch.equal(got[k], want[k]) for k in want)
    be.close()


def test_default_stream_backend_called_from_a_side_stream(seq):
    import torch
    om = load_pkg()
    be = om.B200(0, stream=0)
    want = {k: v.clone() for k, v in layer(seq, be, layer_inputs(2)).items()}
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            torch.cuda._sleep(2_000_000)
            t = layer_inputs(2)
            got = {k: v + 0 for k, v in layer(seq, be, t).items()}
        side.synchronize()
        assert all(torch.equal(got[k], want[k]) for k in want)
    be.close()


def test_views_of_another_backend_are_refused(be, seq):
    om = load_pkg()
    other = om.B200(0)
    x = seq.upload(other, np.zeros((2, 16), np.float32))
    with pytest.raises(om.OmError, match="another stream"):
        seq.quantize_rows(be, x)
    other.close()


def test_current_device_and_profiling_are_left_alone(be, seq):
    """Kernel classes are timed like the library's others."""
    be.profile(True)
    x, w = seq.upload(be, np.ones((4, 64)), "bf16"), seq.upload(be, np.ones((300, 64)), "bf16")
    T = seq.upload(be, np.zeros(4), "i64")
    loss, lse = seq.linear_cross_entropy(be, x, w, T)
    seq.linear_cross_entropy_backward(be, x, w, T, lse, seq.upload(be, np.ones(4, np.float32)))
    report = be.profile_report()
    be.profile(False)
    assert {"loss_logits", "loss_dlogits", "loss_dx", "loss_dw"} <= set(report)
    # all logits alike: 300 equal parts
    assert np.allclose(lse.to_numpy(), 64 + np.log(300), rtol=1e-6)


def test_calls_without_waiting_between_them(seq):
    """Two backends on two streams at once, sharing nothing."""
    import torch
    om = load_pkg()
    streams = [torch.cuda.Stream() for _ in range(2)]
    bes = [om.B200(0, stream=s.cuda_stream) for s in streams]
    ins = [layer_inputs(3 + k) for k in range(2)]
    torch.cuda.synchronize()
    want = []
    for b, s, t in zip(bes, streams, ins):
        with torch.cuda.stream(s):
            want.append({k: v.clone() for k, v in layer(seq, b, t).items()})
        torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for b, s, t in zip(bes, streams, ins):
            with torch.cuda.stream(s):
                got.append(layer(seq, b, t))
        torch.cuda.synchronize()
        assert all(torch.equal(g[k], w[k]) for g, w in zip(got, want) for k in w)


def test_recorded_and_replayed(seq):
    """Two recordings of one backend replayed in turn with new inputs, an
    eager call between them."""
    import torch
    om = load_pkg()
    be = om.B200(0)
    ins = [layer_inputs(5), layer_inputs(6, t=700)]
    fresh = [layer_inputs(7), layer_inputs(8, t=700)]
    want = [{k: v.clone() for k, v in layer(seq, be, t).items()} for t in fresh]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for t in ins:
        be.graph_begin()
        outs.append(layer(seq, be, t))
        graphs.append(be.graph_end())
    for t, f in zip(ins, fresh):
        for k in t:
            t[k].copy_(f[k])
    torch.cuda.synchronize()
    for _ in range(3):
        graphs[0].launch()
        layer(seq, be, ins[0])
        graphs[1].launch()
        be.synchronize()
        torch.cuda.synchronize()
        assert all(torch.equal(o[k], w[k]) for o, w in zip(outs, want) for k in w)
    del graphs
    be.close()


def test_torch_graph(seq):
    """Captured by torch's own graphs on the stream the backend shares."""
    import torch
    om = load_pkg()
    side = torch.cuda.Stream()
    be = om.B200(0, stream=side.cuda_stream)
    t, f = layer_inputs(9), layer_inputs(10)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        want = {k: v.clone() for k, v in layer(seq, be, f).items()}
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = layer(seq, be, t)
    for k in t:
        t[k].copy_(f[k])
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out[k], want[k]) for k in want)


def test_borrowed_stream_outlives_the_backend(seq):
    import torch
    om = load_pkg()
    s = torch.cuda.Stream()
    be = om.B200(0, stream=s.cuda_stream)
    with torch.cuda.stream(s):
        x = torch.randn(4, 64, device="cuda")
        q, scale = seq.quantize_rows(be, x)
    be.close()
    with torch.cuda.stream(s):
        y = x * 2
    s.synchronize()
    assert torch.equal(y, x * 2) and q.abs().amax(1).eq(127).all()
