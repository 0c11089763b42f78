"""The recurrence's last state written over its first: through the C entry, wherever one thread has a channel's whole
sequence; ``last_out`` over other inputs."""

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


def overlapping(case, B, N, D, T, device):
    """Arguments of a call without gradients whose last_out lies over one of its inputs, in one buffer of fp32."""
    g = torch.Generator().manual_seed(1)
    n = B * N * D
    flat = torch.randn(2 * n * T + n, generator=g).to(device)
    wx, b, s = torch.randn((B, T, 2, N, D), generator=g).to(device), torch.randn((2, N, D), generator=g).to(device), torch.randn((1, B, 1, N, D), generator=g).to(device)
    lengths = torch.randint(T + 1, (B,), generator=g, dtype=torch.int32).to(device)
    out = flat[:n].view(1, B, 1, N, D)
    if case == "b":
        b = flat[:2 * N * D].view(2, N, D)
    elif case == "wx":
        wx = flat[:2 * n * T].view(B, T, 2, N, D)
    elif case == "lengths":
        flat[:B].view(torch.int32).copy_(lengths)
        lengths = flat[:B].view(torch.int32)
    elif case == "states, shifted":
        s = flat[4:4 + n].view(1, B, 1, N, D)
    elif case == "states":
        s = out
    return wx, b, s, lengths, out


CASES = ["b", "wx", "lengths", "states, shifted", "states", "none"]


@pytest.mark.parametrize("T", [1, 3])
@pytest.mark.parametrize("case", CASES)
def test_a_kernel_writes_over_no_input_but_the_same_state(case, T, monkeypatch):
    from flashrnn_b200 import linear

    wx, b, s, lengths, out = overlapping(case, 6, 1, 8, T, "cpu")
    written = []

    def forward(wx, b, initial, lengths, function, keep, last=None):
        written.append(last)
        return wx[:, :, 0], torch.ones_like(out) if last is None else last.fill_(1), None

    monkeypatch.setattr(linear, "_forward", forward)
    _, last = linear._run(wx, b, s, "leaky", lengths, out, False)
    direct = case == "none" or (case == "states" and T == 1)
    assert written == [out if direct else None] and last is out and (out == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 40])
@pytest.mark.parametrize("case", CASES)
def test_last_out_over_inputs(case, T, cuda_device):
    from flashrnn_b200 import flashrnn_linear

    wx, b, s, lengths, out = overlapping(case, 3000, 1, 24, T, cuda_device)
    with torch.no_grad():
        want = flashrnn_linear(wx.clone(), b.clone(), s.clone(), "leaky", lengths.clone())
        got = flashrnn_linear(wx, b, s, "leaky", lengths, last_out=out)
    assert got[1] is out and all(torch.equal(a, c) for a, c in zip(got, want))
