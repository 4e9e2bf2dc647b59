"""selective_scan of states that grow (a above 0), in segments of the time whose growth alone is beyond fp32's range.
The tolerances are those of test_gpu_selective: the exponent of a segment is one product more, of |a sum dt| below
8 T."""

import pytest
import torch

import prlstm_amd
import test_gpu_selective as sel

pytestmark = pytest.mark.gpu
T = 400  # in segments of 80 steps, of 40 above 32 states


def _inputs(dev, N):
    s, dout, dh_n = sel.scan_inputs(dev, torch.float32, T, 1, 5, N, gate=False)
    s["a"] = 0.9 + 0.1 * s["a"].abs() / 8
    s["delta_bias"], s["h0"] = None, torch.zeros_like(s["h0"])
    return s, dout, dh_n


@pytest.mark.parametrize("N", [3, 16, 40])
def test_a_state_of_zero_stays(dev, N):
    """Growth of e^108 and more over a segment: a state that is still 0, and a gradient of it that is 0, stay so."""
    s, dout, _ = _inputs(dev, N)
    s["delta"] = torch.full_like(s["delta"], 3.0)
    s["x"][:T - 20] = 0.0
    dout[15:] = 0.0
    grads = sel.check_scan(s, dout, None, softplus=False)
    assert not bool(grads["x"][15:].any()) and bool(grads["h0"].all())


@pytest.mark.parametrize("N", [3, 16, 40])
def test_a_small_state_grows(dev, N):
    """From 1e-30 by e^108 to e^120 over one segment, and its gradient the other way."""
    s, dout, dh_n = _inputs(dev, N)
    s["delta"] = torch.zeros_like(s["delta"])
    s["delta"][80:120 if N > 32 else 160] = 3.0 if N > 32 else 1.5
    s["x"] = torch.zeros_like(s["x"])
    s["h0"] += 1e-30
    dout[:] = 0.0
    sel.check_scan(s, dout, 1e-30 * dh_n, softplus=False)


@pytest.mark.parametrize("N", [3, 16])
def test_an_infinite_state_stays(dev, N):
    """However far it fades, as it does step by step."""
    s, _, _ = _inputs(dev, N)
    s["a"] = -s["a"]
    s["delta"] = torch.full_like(s["delta"], 2.0)
    s["h0"][0, 2] = float("inf")
    _, h = prlstm_amd.selective_scan(**s, softplus=False)
    assert bool(torch.isposinf(h[0, 2]).all()) and bool(torch.isfinite(h[0, :2]).all())
