"""flashrnn_linear on the host: what it refuses, and its plan."""

import pytest
import torch

from flashrnn_b200 import _lib, flashrnn_linear


def args(B=2, T=3, G=2, N=2, D=8):
    return torch.zeros((B, T, G, N, D)), torch.zeros((G, N, D)), torch.zeros((1, B, 1, N, D))


def test_refusals():
    wx, b, s = args()
    n = torch.zeros(2, dtype=torch.int32)
    bad = [
        ("Unknown function", dict(function="gru")),
        ("shape mismatch", dict(function="lstm")),
        ("nonempty Wx", dict(Wx=wx[0])),
        ("nonempty Wx", dict(Wx=wx[:, :0])),
        ("shape mismatch", dict(b=b[:1])),
        ("shape mismatch", dict(b=b.flatten())),
        ("bfloat16 or float32", dict(Wx=wx.double())),
        ("bfloat16 or float32", dict(Wx=wx.half())),
        (r"\[1,B,1,N,D\]", dict(states=s[:, :1])),
        (r"\[1,B,1,N,D\]", dict(states=torch.cat((s, s)))),
        ("floating-point", dict(b=b.int())),
        ("floating-point", dict(states=s.int())),
        ("lengths must be", dict(lengths=n[:1])),
        ("lengths must be", dict(lengths=n.float())),
        ("strided", dict(Wx=wx.to_sparse())),
        ("strided", dict(b=b.to_sparse())),
        ("last_out takes no gradients", dict(Wx=wx.clone().requires_grad_(True), last_out=s.clone())),
        ("last_out must be", dict(last_out=s[:, :1])),
        ("last_out must be", dict(last_out=s.bfloat16())),
        ("last_out must be", dict(last_out=torch.zeros((1, 2, 1, 8, 2)).transpose(3, 4))),
        ("same device", dict(states=s.to("meta"))),
    ]
    for message, change in bad:
        with pytest.raises(ValueError, match=message):
            flashrnn_linear(**{"Wx": wx, "b": b, "states": s, "function": "leaky", "lengths": n, **change})
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        flashrnn_linear(wx, b, s, lengths=n)


def test_plan():
    p = _lib.linear_plan("leaky", 8, 1024, 3, 256)
    assert (p.gates, p.tiles, p.tile_steps * p.tiles) == (2, 8, 1024)
    assert p.starts_bytes == 4 * 8 * 7 * 768 and p.dbpart_bytes == 4 * 8 * 8 * 2 * 768
    assert p.exchange_bytes >= 8 * 8 * 768 * 8
    one = _lib.linear_plan("lstm", 1, _lib.linear_plan("lstm", 1, 1, 1, 1).tile_steps, 1, 7)
    assert (one.gates, one.tiles, one.exchange_bytes, one.starts_bytes, one.dbpart_bytes) == (4, 1, 0, 0, 0)
    many = _lib.linear_plan("leaky", 4096, 2 ** 20, 8, 128)        # sizes past 32 bits
    assert many.starts_bytes == 4 * 4096 * (2 ** 17 - 1) * 1024 and many.dbpart_bytes == 4 * 4096 * 2 * 1024
    lib = _lib.load()
    for a, rc in (((2, 1, 1, 1, 1), -1), ((0, 0, 1, 1, 1), -5), ((0, 1, 1, 1, 0), -5), ((0, 1, 1, 2 ** 16, 2 ** 16), -2), ((1, 2 ** 30, 2 ** 10, 1, 1), -2), ((1, 1, 2 ** 31 - 1, 1, 1), -2)):
        assert lib.frnn_b200_linear_plan(*a, one) == rc, a


@pytest.mark.skipif(torch.cuda.is_available(), reason="calls with pointers to nothing")
def test_c_entries_refuse_before_any_launch():
    lib = _lib.load()
    f = lambda wx=16, bias=16, hidden=16, last=16, exchange=16, err=16, T=300, first=None: lib.frnn_b200_linear_forward(  # noqa: E731
        0, wx, 1, bias, first, None, hidden, last, None, exchange, 1, T, 1, 8, 0, err, None)
    assert f(bias=4) == f(last=8) == f(first=20) == -5 and f(T=2 ** 31 - 1) == -2
    assert f(wx=None) == f(bias=None) == f(hidden=None) == f(last=None) == f(wx=24) == f(hidden=8) == -5
    assert f(exchange=None) == f(err=None) == f(exchange=24) == f(T=0) == -5
    g = lambda starts=16, part=16, dwx=16, dh=16: lib.frnn_b200_linear_backward(  # noqa: E731
        0, 16, 1, 16, None, None, starts, dh, None, dwx, 16, None, part, 16, 1, 300, 1, 8, 0, 16, None)
    assert g(dwx=None) == g(dh=None) == g(dwx=8) == g(dh=8) == g(starts=None) == g(part=None) == -5
    assert lib.frnn_b200_linear_forward(7, 16, 1, 16, None, None, 16, 16, None, 16, 1, 3, 1, 8, 0, 16, None) == -1
