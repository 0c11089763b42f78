"""The bounds of tests/_linear_error.py on the host: the values are those of autograd, 32 bits stay inside, planted mistakes do not."""

import pytest
import torch

from tests import _linear_error as E
from tests import _linear_reference as L


def inputs(function, kind, B=3, T=40, N=2, D=5, seed=0):
    """kind "plain": ordinary gates; "resets": forget gates that are nearly shut every few steps, states large against what comes in;
    "small": inputs and states down to 1e-6; "saturated": gates and states at the ends of their functions, in the LSTM"""
    g = torch.Generator().manual_seed(seed)
    G, fg = L.GATES[function], 0 if function == "leaky" else 1
    wx, b = torch.randn((B, T, G, N, D), generator=g), torch.randn((G, N, D), generator=g) * 0.1
    s = torch.randn((1, B, 1, N, D), generator=g) * 0.5
    b[fg] = torch.rand((N, D), generator=g) * 6
    if kind == "resets":
        b[fg] = 0
        shut = torch.tensor([-8.0, -12.0, -14.0, -16.0, -20.0, -40.0])[torch.randint(6, (B, T, N, D), generator=g)]
        wx[:, :, fg] = torch.where(torch.rand((B, T, N, D), generator=g) < 0.2, shut, 3 + 3 * torch.rand((B, T, N, D), generator=g))
        wx[:, :, -1 if function == "leaky" else 2] *= 0.01
        s *= 10.0 ** (6 * torch.rand((1, B, 1, N, D), generator=g))
    if kind == "small":
        size = 10.0 ** (-1 - 5 * torch.rand((1, N, D), generator=g))
        wx[:, :, -1 if function == "leaky" else 2] *= size
        b[-1 if function == "leaky" else 2] *= size[0]
        s *= size
    if kind == "saturated" and function == "lstm":
        for k, low, high in ((0, 8, 14), (2, 3, 8), (3, 8, 14)):
            wx[:, :, k] = wx[:, :, k].sign() * (low + (high - low) * torch.rand((B, T, N, D), generator=g))
        s = s.sign() * (2 + 6 * torch.rand((1, B, 1, N, D), generator=g))
    dh, dl = torch.randn((B, T, N, D), generator=g), torch.randn((1, B, 1, N, D), generator=g)
    n = torch.tensor([T, 0, 17][:B]) if B == 3 else None
    return wx, b, s, n, dh, dl


def in_32_bits(function, wx, b, s, n, dh, dl, subtract=None):
    """Step by step in 32 bits. subtract, the planted mistakes: "decay", known only as 1 - u; "tanh", from 1 - exp; "slopes", 1 - s and
    1 - t^2."""
    def tanh(y):
        return (1 - torch.exp(-2 * y)) / (1 + torch.exp(-2 * y)) if subtract == "tanh" else torch.tanh(y)

    def slope(y):
        return 1 - torch.tanh(y) ** 2 if subtract == "slopes" else 1 / torch.cosh(y) ** 2

    def rest(y):
        return 1 - torch.sigmoid(y) if subtract == "slopes" else torch.sigmoid(-y)

    x = wx + b
    B, T, _, N, D = wx.shape
    n = torch.full((B,), T) if n is None else n
    on = (torch.arange(T) < n[:, None])[:, :, None, None]
    fg = 0 if function == "leaky" else 1
    f, u = torch.sigmoid(x[:, :, fg]), torch.sigmoid(-x[:, :, fg])
    if subtract == "decay":
        f, fu = 1 - u, u - u * u
    else:
        fu = f * u
    if function == "leaky":
        z = x[:, :, 1]
        v = u * z
    else:
        i, z, o = torch.sigmoid(x[:, :, 0]), tanh(x[:, :, 2]), torch.sigmoid(x[:, :, 3])
        v = i * z
    c, before, after = s[0, :, 0], [], []
    for t in range(T):
        before.append(c)
        new = (c + v[:, t]) - u[:, t] * c if subtract == "decay" else f[:, t] * c + v[:, t]
        c = torch.where(on[:, t], new, c)
        after.append(c)
    before, after = torch.stack(before, 1), torch.stack(after, 1)
    tc = tanh(after)
    hidden, dc = (after, dh) if function == "leaky" else (o * tc, dh * o * slope(after))
    g, d_wx = dl[0, :, 0], torch.zeros_like(wx)
    for t in range(T - 1, -1, -1):
        at = g + dc[:, t]
        if function == "leaky":
            d = [at * (before[:, t] - z[:, t]) * fu[:, t], at * u[:, t]]
        else:
            d = [at * z[:, t] * i[:, t] * rest(x[:, t, 0]), at * before[:, t] * fu[:, t], at * i[:, t] * slope(x[:, t, 2]),
                 dh[:, t] * tc[:, t] * o[:, t] * rest(x[:, t, 3])]
        d_wx[:, t] = torch.where(on[:, t, None], torch.stack(d, 1), torch.zeros(()))
        g = torch.where(on[:, t], f[:, t] * at, g)
    return {"hidden": torch.where(on, hidden, 0.0), "last": c[None, :, None], "d_wx": d_wx, "d_b": d_wx.sum((0, 1)), "d_states": g[None, :, None]}


@pytest.mark.parametrize("function", ["leaky", "lstm"])
@pytest.mark.parametrize("kind", ["plain", "resets", "small", "saturated"])
def test_values_are_those_of_autograd(function, kind):
    args = inputs(function, kind)
    ref, mine = L.run_reference(args[0], args[1], args[2], function, *args[3:]), E.evaluate(*args[:3], function, *args[3:])
    assert set(ref) == set(mine)
    for k in ref:
        torch.testing.assert_close(mine[k][0], ref[k], rtol=1e-9, atol=1e-12)


@pytest.mark.parametrize("function", ["leaky", "lstm"])
@pytest.mark.parametrize("kind", ["plain", "resets", "small", "saturated"])
def test_32_bits_stay_inside(function, kind):
    for seed in range(4):
        args = inputs(function, kind, seed=seed)
        E.check(in_32_bits(function, *args), E.evaluate(*args[:3], function, *args[3:]))


@pytest.mark.parametrize("function", ["leaky", "lstm"])
def test_a_decay_by_subtraction_is_seen(function):
    args = inputs(function, "resets")
    got, ref = in_32_bits(function, *args, subtract="decay"), E.evaluate(*args[:3], function, *args[3:])
    for name in ("last", "d_wx", "d_states"):
        with pytest.raises(AssertionError):
            E.check(got, ref, [name])


def test_a_tanh_that_cancels_is_seen():
    args = inputs("lstm", "small")
    got, ref = in_32_bits("lstm", *args, subtract="tanh"), E.evaluate(*args[:3], "lstm", *args[3:])
    for name in ("hidden", "last", "d_wx"):
        with pytest.raises(AssertionError):
            E.check(got, ref, [name])


def test_slopes_by_subtraction_are_seen():
    args = inputs("lstm", "saturated")
    with pytest.raises(AssertionError):
        E.check(in_32_bits("lstm", *args, subtract="slopes"), E.evaluate(*args[:3], "lstm", *args[3:]), ["d_wx"])
