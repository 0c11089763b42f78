"""flashrnn_linear element by element within the bounds of tests/_linear_error.py: states that are large against what comes in, forget
gates that are nearly shut, inputs near zero, gates at the ends of their functions."""

import pytest
import torch

from tests import _linear_error as E
from tests.test_linear_error import inputs

pytestmark = pytest.mark.gpu

# tiles of four channels a thread, of one; walks of up to 16 steps; walks of many channels, even and odd
LEAKY = [(3, 300, 1, 72), (2, 170, 1, 31), (5, 16, 2, 34), (16, 40, 32, 128), (33, 21, 1, 999)]
LSTM = [(3, 300, 1, 72), (2, 170, 1, 31), (5, 16, 2, 34), (32, 24, 32, 128), (33, 21, 1, 999)]


def run(function, wx, b, s, n, dh, dl, device, dtype):
    from flashrnn_b200 import flashrnn_linear

    leaves = [t.to(device).requires_grad_(True) for t in (wx.to(dtype), b, s)]
    hidden, last = flashrnn_linear(*leaves, function, None if n is None else n.to(device))
    d = torch.autograd.grad([hidden, last], leaves, [dh.to(device, dtype), dl.to(device)])
    return {"hidden": hidden, "last": last, **dict(zip(("d_wx", "d_b", "d_states"), d))}


def case(function, kind, shape, dtype):
    wx, b, s, n, dh, dl = inputs(function, kind, *shape, seed=sum(shape))
    return wx.to(dtype), b, s, n, dh.to(dtype), dl


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["plain", "resets", "small"])
@pytest.mark.parametrize("shape", LEAKY)
def test_leaky(shape, kind, dtype, cuda_device):
    args = case("leaky", kind, shape, dtype)
    E.check(run("leaky", *args, cuda_device, dtype), E.evaluate(*args[:3], "leaky", *args[3:]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", LSTM)
def test_forget_gate_of_the_lstm(shape, dtype, cuda_device):
    """The state, its gradient and the forget gate's, from the last state alone."""
    wx, b, s, n, dh, dl = case("lstm", "resets", shape, dtype)
    wx[:, :, 2] = torch.where(wx[:, :, 2] < 0, -1, 1) * (0.5 + wx[:, :, 2].abs())
    args = wx, b, s, n, torch.zeros_like(dh), dl
    got, ref = run("lstm", *args, cuda_device, dtype), E.evaluate(*args[:3], "lstm", *args[3:])
    got["d_wx"] = got["d_wx"][:, :, 1]
    ref["d_wx"] = tuple(t[:, :, 1] for t in ref["d_wx"])
    E.check(got, ref, ["last", "d_states", "d_wx"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["plain", "resets", "small", "saturated"])
@pytest.mark.parametrize("shape", LSTM)
def test_lstm(shape, kind, dtype, cuda_device):
    args = case("lstm", kind, shape, dtype)
    E.check(run("lstm", *args, cuda_device, dtype), E.evaluate(*args[:3], "lstm", *args[3:]))
