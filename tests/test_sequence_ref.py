"""CPU checks of the sequence-model operators: their plain forms against
differences and against each other, and the refusals that need no GPU."""
import ctypes

import numpy as np
import pytest

import sequence_ref as ref
from conftest import load_pkg


@pytest.mark.parametrize("kind", ["linear", "sigmoid"])
def test_scan_gradient_by_differences(kind):
    r = np.random.default_rng(1)
    shape = (2, 5, 3)
    gate, x, dh = r.normal(size=shape), r.normal(size=shape), r.normal(size=shape)
    h0, dl = r.normal(size=(2, 3)), r.normal(size=(2, 3))
    lengths = np.array([5, 3])

    def value(gate, x, h0):
        h, last, _, _ = ref.scan(gate, x, h0, lengths, kind, "f64")
        return (h * dh).sum() + (last * dl).sum()

    h = ref.scan(gate, x, h0, lengths, kind, "f64")[0]
    got = ref.scan_backward(gate, x, h, dh, h0, dl, lengths, kind, "f64")[:3]
    args = [gate, x, h0]
    for k, g in enumerate(got):
        for i in np.ndindex(*args[k].shape):
            step = 1e-6
            up, down = [a.copy() for a in args], [a.copy() for a in args]
            up[k][i] += step
            down[k][i] -= step
            # central difference: step^2 times a third derivative (below 10
            # here) and the values' rounding over the step
            assert abs((value(*up) - value(*down)) / (2 * step) - g[i]) < 1e-8


def test_loss_gradient_by_differences():
    r = np.random.default_rng(2)
    x, w = r.normal(size=(4, 3)), r.normal(size=(5, 3))
    targets, g = np.array([0, 4, -100, 2]), r.normal(size=4)

    def value(x, w):
        return (ref.loss(x, w, targets, "f64")[0] * g).sum()

    lse = ref.loss(x, w, targets, "f64")[1]
    got = ref.loss_backward(x, w, targets, lse, g, "f64")[:2]
    args = [x, w]
    for k, d in enumerate(got):
        for i in np.ndindex(*args[k].shape):
            step = 1e-6
            up, down = [a.copy() for a in args], [a.copy() for a in args]
            up[k][i] += step
            down[k][i] -= step
            assert abs((value(*up) - value(*down)) / (2 * step) - d[i]) < 1e-8


def test_rounding_helper_matches_torch():
    import torch
    x = np.random.default_rng(3).normal(size=1000) * 10.0 ** np.arange(-5, 5).repeat(100)
    t = torch.from_numpy(x.astype(np.float32))
    assert np.array_equal(ref.rounded(x, "bf16"), t.to(torch.bfloat16).double().numpy())
    assert np.array_equal(ref.rounded(x, "f16"), t.to(torch.float16).double().numpy())


NULL_CALLS = {
    "om_b200_gated_scan": [0, 0] + [None] * 10,
    "om_b200_gated_scan_backward": [0, 0] + [None] * 17,
    "om_b200_linear_cross_entropy": [0] + [None] * 5 + [9] + [None] * 3,
    "om_b200_linear_cross_entropy_backward": [0] + [None] * 5 + [9] + [None] * 7,
    "om_b200_quantize_rows": [0] + [None] * 6,
    "om_b200_matmul_i8": [0] + [None] * 10,
    "om_b200_linear_i8": [0] + [None] * 9,
}


@pytest.mark.parametrize("name", sorted(NULL_CALLS))
def test_null_backend_is_refused(name):
    om = load_pkg()
    import omeinsum_b200.sequence as seq
    fn = getattr(seq._bind(), name)
    assert fn(None, *NULL_CALLS[name]) == 1
    buf = ctypes.create_string_buffer(256)
    om.lib().om_b200_last_error(buf, 256)
    assert b"null" in buf.value and name.encode() in buf.value


def test_create_on_stream_refuses_null():
    om = load_pkg()
    assert om.lib().om_b200_create_on_stream(0, None, None) == 1


class _NoDevice:
    """A storage that is never touched, for refusals before any device call."""

    def __init__(self, n, dtype):
        self.backend, self.device = self, 0
        self.home_stream, self.recording, self.h = 0, False, None
        self.ptr, self.n, self.dtype = 4096, n, np.dtype(dtype)


def _view(shape, dtype=np.float32, strides=None):
    import omeinsum_b200.sequence as seq
    return seq.Strided(_NoDevice(10000, dtype), shape, strides)


def test_python_refusals():
    om = load_pkg()
    import omeinsum_b200.sequence as seq
    be = _NoDevice(0, np.float32)
    f = _view
    bad = [
        lambda: seq.gated_scan(be, f((2, 3)), f((2, 3))),
        lambda: seq.gated_scan(be, f((2, 3, 4)), f((2, 3, 5))),
        lambda: seq.gated_scan(be, f((2, 3, 4)), f((2, 3, 4), np.float64)),
        lambda: seq.gated_scan(be, f((2, 3, 4)), None),
        lambda: seq.gated_scan(be, f((2, 3, 4)), f((2, 3, 4)), kind="other"),
        lambda: seq.gated_scan(be, f((2, 3, 4), np.int32), f((2, 3, 4), np.int32)),
        lambda: seq.gated_scan(be, f((2, 3, 4)), f((2, 3, 4)), h0=f((2, 4), np.float64)),
        lambda: seq.gated_scan(be, f((2, 3, 4)), f((2, 3, 4)), h0=f((2, 4), strides=(1, 2))),
        lambda: seq.gated_scan(be, f((2, 3, 4)), f((2, 3, 4)), lengths=f((2,), np.int64)),
        lambda: seq.gated_scan(be, np.zeros((2, 3, 4)), f((2, 3, 4))),
        lambda: seq.gated_scan_backward(be, f((2, 3, 4)), None, f((2, 3, 4)), f((2, 3, 4)), kind="sigmoid"),
        lambda: seq.gated_scan_backward(be, f((2, 3, 4)), None, f((2, 3, 4)), f((2, 3, 3))),
        lambda: seq.linear_cross_entropy(be, f((4, 8)), f((10, 7)), f((4,), np.int64)),
        lambda: seq.linear_cross_entropy(be, f((4, 8)), f((10, 8), np.float64), f((4,), np.int64)),
        lambda: seq.linear_cross_entropy(be, f((4, 8)), f((10, 8)), f((4,), np.float32)),
        lambda: seq.linear_cross_entropy(be, f((4, 8)), f((10, 8)), f((5,), np.int64)),
        lambda: seq.linear_cross_entropy_backward(be, f((4, 8)), f((10, 8)), f((4,), np.int64), f((4,), np.float64), f((4,))),
        lambda: seq.quantize_rows(be, f((4, 8), np.float64)),
        lambda: seq.quantize_rows(be, f((4, 8, 2))),
        lambda: seq.matmul_i8(be, f((4, 8), np.int8), f((4,)), f((6, 9), np.int8), f((6,))),
        lambda: seq.matmul_i8(be, f((4, 8), np.int8), f((4,)), f((6, 8), np.int8), None),
        lambda: seq.matmul_i8(be, f((4, 8), np.int8), f((4,)), f((6, 8), np.int8), f((6,)), dtype="f64"),
        lambda: seq.matmul_i8(be, f((4, 8), np.int8), f((4,)), f((6, 8), np.int8), f((6,)), dtype="int"),
        lambda: seq.linear_i8(be, f((4, 8)), f((6, 8), np.int8), None),
        lambda: seq.linear_i8(be, f((4, 8)), f((6, 8)), f((6,))),
        lambda: f((200, 200)),
        lambda: f((2, 3), strides=(1,)),
        lambda: f((2, 3), strides=(-5, 1)),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(om.OmError):
            call()
            pytest.fail(f"refusal {k} did not happen")


def test_torch_cpu_tensor_is_refused():
    om = load_pkg()
    import torch
    import omeinsum_b200.sequence as seq
    t = torch.zeros(2, 3, 4)
    with pytest.raises(om.OmError):
        seq.gated_scan(_NoDevice(0, np.float32), t, t)
