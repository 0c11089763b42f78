"""The recurrence's last state written over its first: through the C entry, wherever one thread has a channel's whole sequence."""

import pytest
import torch

from tests.test_source_order import CSRC, _body


def test_the_first_state_is_not_loaded_as_constant_data():
    """What a kernel writes must not pass through the read-only path: `first` is read by an ordinary load."""
    ask = _body((CSRC / "linear_scan.cu").read_text(), "void ask(")
    assert "first[" in ask and "__ldg(first" not in ask


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 16, 17, 50])      # walks, one tile
@pytest.mark.parametrize("function", ["leaky", "lstm"])
def test_last_is_initial(function, T, cuda_device):
    from flashrnn_b200 import _lib, flashrnn_linear
    from tests.test_linear_error import inputs

    B, N, D = 5, 3, 44
    wx, b, s, _, _, _ = inputs(function, "plain", B, T, N, D, seed=T)
    wx, b, s = wx.to(cuda_device), b.to(cuda_device), s.to(cuda_device)
    assert _lib.linear_plan(function, B, T, N, D).tiles == 1
    hidden, last = flashrnn_linear(wx, b, s, function)
    state, out = s.clone(), torch.empty_like(hidden)
    rc = _lib.load().frnn_b200_linear_forward(
        _lib.LINEAR_CELLS[function], wx.data_ptr(), 0, b.data_ptr(), state.data_ptr(), None, out.data_ptr(), state.data_ptr(), None, None,
        B, T, N, D, 0, None, torch.cuda.current_stream(cuda_device).cuda_stream)
    assert rc == 0 and torch.equal(out, hidden) and torch.equal(state, last)
