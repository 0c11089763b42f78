"""The gated linear recurrence in 64 bits with, beside each value, how far an evaluation in 32 bits may be from it.

First order in the rounding errors, element by element, so a bound follows a state through a reset instead of keeping the size of the
largest one. With C_t = f C_{t-1} + |v| and G_t = |dc_t| + f G_{t+1} the recurrences over magnitudes, which bound every partial sum in
any order of the scan, and u = 1 - f:

* an argument x = Wx + b is scaled, added and rounded: off by dx = 2^-22 (|Wx| + |b|);
* a sigmoid, its complement and their product, held by the smaller of f and u: relative error e = 2^-20 + dx (two approximate
  instructions of 2^-22 each, an addition and a product of 2^-24, doubled);
* tanh of y: e |tanh y| + dy (1 - tanh^2 y), relative to its own size however small y is; 1 - tanh^2 y likewise, e + 2 |tanh y| dy;
* a step: E_t = f E_{t-1} + e min(f, u) C_{t-1} + dv + 2^-22 C_t, its roundings being two of 2^-24 and those of the map beside it;
* joining spans, warps, tiles and groups adds at most 32 roundings of 2^-24 of what is joined: 2^-19 C_t;
* the reverse scan the same with G.

Products of k such factors add their relative errors up. SLACK covers what is of second order."""

import torch

SLACK = 1.25
STEP, JOIN, FUNCTION, ARGUMENT = 2.0 ** -22, 2.0 ** -19, 2.0 ** -20, 2.0 ** -22
TINY = 1e-37      # results near the end of the range of 32 bits are flushed


def _sigmoid(x):
    """sigmoid and its complement, neither by subtraction"""
    return 1 / (1 + torch.exp(-x)), 1 / (1 + torch.exp(x))


def evaluate(wx, b, states, function, lengths, dh, dlast):
    """-> {name: (value, bound)} in float64 on the CPU, bound before the last rounding"""
    d = lambda t: None if t is None else t.detach().cpu().double()  # noqa: E731
    wx, b, states, dh, dlast = d(wx), d(b), d(states), d(dh), d(dlast)
    B, T, G, N, D = wx.shape
    lengths = torch.full((B,), T) if lengths is None else lengths.cpu().long().clamp(0, T)
    x, dx = wx + b, ARGUMENT * (wx.abs() + b.abs())
    inside = (torch.arange(T) < lengths[:, None])[:, :, None, None].expand(B, T, N, D)
    zero = torch.zeros(B, N, D, dtype=torch.float64)
    # padding may hold anything
    x = torch.where(inside[:, :, None], x, 0.0)
    dx = torch.where(inside[:, :, None], dx, 0.0)
    dh = torch.where(inside, dh, 0.0)
    fg = 0 if function == "leaky" else 1
    f, u = _sigmoid(x[:, :, fg])
    ef = FUNCTION + dx[:, :, fg]
    if function == "leaky":
        z, dz = x[:, :, 1], dx[:, :, 1]
        v, dv = u * z, u * z.abs() * (ef + STEP) + u * dz
    else:
        (i, ci), (o, co), z = _sigmoid(x[:, :, 0]), _sigmoid(x[:, :, 3]), torch.tanh(x[:, :, 2])
        ei, eo, dy = FUNCTION + dx[:, :, 0], FUNCTION + dx[:, :, 3], dx[:, :, 2]
        sz = 1 / torch.cosh(x[:, :, 2]) ** 2
        dz = FUNCTION * z.abs() + dy * sz
        v, dv = i * z, i * z.abs() * (ei + STEP) + i * dz
    least = torch.minimum(f, u)
    c, C, E = (zero if states is None else states[0, :, 0]), None, zero
    C = c.abs()
    before, Eb, after, Ea = [], [], [], []
    for t in range(T):
        on = inside[:, t]
        before.append(c), Eb.append(E + JOIN * C)
        Cn = f[:, t] * C + v[:, t].abs()
        En = f[:, t] * E + ef[:, t] * least[:, t] * C + dv[:, t] + STEP * Cn
        c = torch.where(on, f[:, t] * c + v[:, t], c)
        C, E = torch.where(on, Cn, C), torch.where(on, En, E)
        after.append(c), Ea.append(E + JOIN * C)
    before, Eb, after, Ea = (torch.stack(q, 1) for q in (before, Eb, after, Ea))
    out = {"last": (c[None, :, None], (E + JOIN * C)[None, :, None])}
    if function == "leaky":
        hidden, eh = after, Ea
        dc, ddc = dh, torch.zeros_like(dh)
    else:
        tc, sc = torch.tanh(after), 1 / torch.cosh(after) ** 2
        ts = sc * torch.minimum(Ea, torch.ones_like(Ea))
        hidden, eh = o * tc, (o * tc).abs() * (eo + 2 * FUNCTION) + o * ts
        dc = dh * o * sc
        ddc = dc.abs() * (eo + 3 * FUNCTION) + 2 * (dh * o).abs() * tc.abs() * ts
    out["hidden"] = (torch.where(inside, hidden, 0.0), torch.where(inside, eh, 0.0))
    g, E = (zero if dlast is None else dlast[0, :, 0]), zero
    Gm = g.abs()
    d_wx, e_wx = torch.zeros_like(wx), torch.zeros_like(wx)
    for t in range(T - 1, -1, -1):
        on = inside[:, t]
        g, E, Gm = g + dc[:, t], E + ddc[:, t], Gm + dc[:, t].abs()
        Eg, ft, ut = E + JOIN * Gm + STEP * Gm, f[:, t], u[:, t]
        df = g * ft * ut
        if function == "leaky":
            diff = before[:, t] - z[:, t]
            terms = [(df * diff, Eg * (ft * ut * diff).abs() + df.abs() * (Eb[:, t] + dz[:, t] + STEP * (before[:, t].abs() + z[:, t].abs()))
                      + 4 * (df * diff).abs() * ef[:, t]),
                     (g * ut, Eg * ut + (g * ut).abs() * (ef[:, t] + STEP))]
        else:
            it, ct, zt, ot, kt = i[:, t], ci[:, t], z[:, t], o[:, t], co[:, t]
            di, do = g * it * ct * zt, dh[:, t] * tc[:, t] * ot * kt
            dzt = g * it * sz[:, t]
            terms = [(di, Eg * (it * ct * zt).abs() + 4 * di.abs() * ei[:, t] + (g * it * ct).abs() * dz[:, t]),
                     (df * before[:, t], Eg * (ft * ut * before[:, t]).abs() + df.abs() * Eb[:, t] + 4 * (df * before[:, t]).abs() * ef[:, t]),
                     (dzt, Eg * it * sz[:, t] + 4 * dzt.abs() * ei[:, t] + 2 * dzt.abs() * (zt.abs() * dy[:, t] + FUNCTION)),
                     (do, 4 * do.abs() * (eo[:, t] + FUNCTION) + (dh[:, t] * ot * kt).abs() * ts[:, t])]
        for k, (val, err) in enumerate(terms):
            d_wx[:, t, k], e_wx[:, t, k] = torch.where(on, val, 0.0), torch.where(on, err, 0.0)
        Gn = ft * Gm
        En = ft * E + ef[:, t] * least[:, t] * Gm + STEP * Gm * ft
        g, E, Gm = torch.where(on, ft * g, g), torch.where(on, En, E), torch.where(on, Gn, Gm)
    out["d_wx"] = (d_wx, e_wx)
    out["d_states"] = (g[None, :, None], (E + JOIN * Gm)[None, :, None])
    # a sum over rows and steps: what each term may be off by, and its own roundings (in two levels, each in turn)
    depth = 2.0 ** -24 * (T + B + 64)
    out["d_b"] = (d_wx.sum((0, 1)), (e_wx + depth * d_wx.abs()).sum((0, 1)))
    return {k: (val, SLACK * err + TINY) for k, (val, err) in out.items()}


def check(got, ref, names=None):
    """Every element within its bound and the last rounding, half a step of its type."""
    for name in names or ref:
        if name not in got:
            continue
        value, bound = ref[name]
        t = got[name].detach().cpu()
        assert torch.isfinite(t).all(), name
        off = (t.double() - value).abs() - bound - torch.finfo(t.dtype).eps / 2 * (value.abs() + bound)
        worst = off.argmax()
        assert off.max() <= 0, (name, off.flatten()[worst].item(), value.flatten()[worst].item(), bound.flatten()[worst].item(), t.flatten()[worst].item())
