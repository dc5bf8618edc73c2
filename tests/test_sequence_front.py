"""CPU checks of the sequence front end: torch tensors whose memory does not hold
their values."""
import pytest

from conftest import load_pkg
from test_sequence_ref import _NoDevice


def _cpu_backend():
    """A backend that takes CPU tensors for its own device's (which torch numbers
    -1), for refusals before any device call."""
    import numpy as np
    be = _NoDevice(0, np.float32)
    be.device = -1
    return be


def test_negated_views_are_refused():
    """The imaginary part of a conjugate is kept as its negative, with a mark."""
    om = load_pkg()
    import torch
    import omeinsum_b200.sequence as seq
    be = _cpu_backend()
    marked = torch.ones(2, 3, 4, dtype=torch.complex64).conj().imag
    assert marked.is_neg()
    plain = torch.ones(2, 3, 4)
    q, w, s = torch.ones(2, 4, dtype=torch.int8), torch.ones(3, 4, dtype=torch.int8), torch.ones(3)
    calls = [
        lambda: seq.gated_scan(be, marked, plain),
        lambda: seq.gated_scan(be, plain, marked),
        lambda: seq.gated_scan(be, plain, plain, h0=marked[:, 0]),
        lambda: seq.gated_scan_backward(be, plain, plain, plain, marked),
        lambda: seq.linear_cross_entropy(be, marked[0], plain[0], torch.zeros(3, dtype=torch.int64)),
        lambda: seq.quantize_rows(be, marked[0]),
        lambda: seq.linear_i8(be, plain[0], w, marked[0, :, 0]),
        lambda: seq.matmul_i8(be, q, marked[:, 0, 0], w, s),
    ]
    for k, call in enumerate(calls):
        with pytest.raises(om.OmError, match="resolve_neg"):
            call()
            pytest.fail(f"refusal {k} did not happen")
