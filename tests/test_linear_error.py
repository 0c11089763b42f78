"""The bounds of tests/_linear_error.py on the host: the values are those of autograd, 32 bits stay inside, planted mistakes do not."""

import pytest
import torch

from tests import _linear_error as E
from tests import _linear_reference as L


def inputs(function, kind, B=3, T=40, N=2, D=5, seed=0):
    """kind "plain": ordinary gates; "resets": forget gates that are nearly shut every few steps, states large against what comes in"""
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
    dh, dl = torch.randn((B, T, N, D), generator=g), torch.randn((1, B, 1, N, D), generator=g)
    n = torch.tensor([T, 0, 17][:B]) if B == 3 else None
    return wx, b, s, n, dh, dl


def in_32_bits(function, wx, b, s, n, dh, dl, subtract=False):
    """Step by step in 32 bits. subtract: the planted mistake, a decay known only as 1 - u."""
    x = wx + b
    B, T, _, N, D = wx.shape
    n = torch.full((B,), T) if n is None else n
    on = (torch.arange(T) < n[:, None])[:, :, None, None]
    fg = 0 if function == "leaky" else 1
    f, u = torch.sigmoid(x[:, :, fg]), torch.sigmoid(-x[:, :, fg])
    if subtract:
        f, fu = 1 - u, u - u * u
    else:
        fu = f * u
    if function == "leaky":
        z = x[:, :, 1]
        v = u * z
    else:
        i, z, o = torch.sigmoid(x[:, :, 0]), torch.tanh(x[:, :, 2]), torch.sigmoid(x[:, :, 3])
        v = i * z
    c, before, after = s[0, :, 0], [], []
    for t in range(T):
        before.append(c)
        new = (c + v[:, t]) - u[:, t] * c if subtract else f[:, t] * c + v[:, t]
        c = torch.where(on[:, t], new, c)
        after.append(c)
    before, after = torch.stack(before, 1), torch.stack(after, 1)
    tc = torch.tanh(after)
    hidden, dc = (after, dh) if function == "leaky" else (o * tc, dh * o / torch.cosh(after) ** 2)
    g, d_wx = dl[0, :, 0], torch.zeros_like(wx)
    for t in range(T - 1, -1, -1):
        at = g + dc[:, t]
        if function == "leaky":
            d = [at * (before[:, t] - z[:, t]) * fu[:, t], at * u[:, t]]
        else:
            d = [at * z[:, t] * i[:, t] * torch.sigmoid(-x[:, t, 0]), at * before[:, t] * fu[:, t], at * i[:, t] / torch.cosh(x[:, t, 2]) ** 2,
                 dh[:, t] * tc[:, t] * o[:, t] * torch.sigmoid(-x[:, t, 3])]
        d_wx[:, t] = torch.where(on[:, t, None], torch.stack(d, 1), torch.zeros(()))
        g = torch.where(on[:, t], f[:, t] * at, g)
    return {"hidden": torch.where(on, hidden, 0.0), "last": c[None, :, None], "d_wx": d_wx, "d_b": d_wx.sum((0, 1)), "d_states": g[None, :, None]}


@pytest.mark.parametrize("function", ["leaky", "lstm"])
@pytest.mark.parametrize("kind", ["plain", "resets"])
def test_values_are_those_of_autograd(function, kind):
    args = inputs(function, kind)
    ref, mine = L.run_reference(args[0], args[1], args[2], function, *args[3:]), E.evaluate(*args[:3], function, *args[3:])
    assert set(ref) == set(mine)
    for k in ref:
        torch.testing.assert_close(mine[k][0], ref[k], rtol=1e-9, atol=1e-12)


@pytest.mark.parametrize("function", ["leaky", "lstm"])
@pytest.mark.parametrize("kind", ["plain", "resets"])
def test_32_bits_stay_inside(function, kind):
    for seed in range(4):
        args = inputs(function, kind, seed=seed)
        E.check(in_32_bits(function, *args), E.evaluate(*args[:3], function, *args[3:]))


@pytest.mark.parametrize("function", ["leaky", "lstm"])
def test_a_decay_by_subtraction_is_seen(function):
    args = inputs(function, "resets")
    got, ref = in_32_bits(function, *args, subtract=True), E.evaluate(*args[:3], function, *args[3:])
    for name in ("last", "d_wx", "d_states"):
        with pytest.raises(AssertionError):
            E.check(got, ref, [name])
