"""The gated linear recurrence in 64 bits, one step at a time, with autograd; and what the kernels may be off by."""

import torch

GATES = {"leaky": 2, "lstm": 4}


def reference(wx, b, states, function, lengths=None):
    """wx [B,T,G,N,D] etc. as float64 leaves or constants -> hidden [B,T,N,D], last [1,B,1,N,D]"""
    B, T, G, N, D = wx.shape
    c = torch.zeros((B, N, D), dtype=torch.float64) if states is None else states[0, :, 0]
    out = []
    for t in range(T):
        x = wx[:, t] + b
        if function == "leaky":
            f = torch.sigmoid(x[:, 0])
            new = f * c + (1 - f) * x[:, 1]
            h = new
        else:
            i, f, z, o = torch.sigmoid(x[:, 0]), torch.sigmoid(x[:, 1]), torch.tanh(x[:, 2]), torch.sigmoid(x[:, 3])
            new = f * c + i * z
            h = o * torch.tanh(new)
        if lengths is not None:
            on = (t < lengths)[:, None, None]
            new, h = torch.where(on, new, c), torch.where(on, h, torch.zeros_like(h))
        c = new
        out.append(h)
    return torch.stack(out, 1), c[None, :, None]


def run_reference(wx, b, states, function, lengths, dh, dlast):
    """Values and gradients in float64 on the CPU of the given (already rounded) inputs."""
    leaf = [None if t is None else t.detach().cpu().double().requires_grad_(True) for t in (wx, b, states)]
    hidden, last = reference(*leaf, function, None if lengths is None else lengths.cpu())
    loss = (hidden * dh.cpu().double()).sum()
    if dlast is not None:
        loss = loss + (last * dlast.cpu().double()).sum()
    grads = torch.autograd.grad(loss, [t for t in leaf if t is not None])
    out = {"hidden": hidden.detach(), "last": last.detach(), "d_wx": grads[0], "d_b": grads[1]}
    if states is not None:
        out["d_states"] = grads[2]
    return out


def bounds(ref, wx, b, states, T, dh, dlast):
    """Largest absolute error of each output before its final rounding.

    A step c + v - u c rounds twice in 24 bits: 2^-23 of the larger of |c| and |v|, and at most all T steps add up. Gates come
    from ex2 and rcp approximations of 2 ulp and an argument of up to 2^4 rounded in 24 bits: 2^-19 relative, and what scales a
    state by 1 + e moves it by no more than e of its largest value. So states are off by at most (T 2^-23 + 2^-19) of the largest
    state or input, gradients of the state by the same of the largest such gradient, and a gate's gradient, a product of both with
    a gate, by the sum of the two. A sum of n such terms is off by n times a term's error."""
    e = T * 2.0 ** -23 + 2.0 ** -19
    c = max(1.0, (wx.detach().float().abs().max() + b.detach().float().abs().max()).item(),
            0.0 if states is None else states.detach().float().abs().max().item())
    # |g_t| <= sum over later steps of |dc| f...: bounded by what arrives times the steps that it can add up over
    g = max(dh.abs().float().max().item(), 0.0 if dlast is None else dlast.abs().max().item())
    reach = max(1.0, ref["d_wx"].abs().max().item() / max(g * c, 1e-30), ref["d_states"].abs().max().item() / g if "d_states" in ref else 1.0)
    g = g * reach
    n = wx.shape[0] * T
    return {"hidden": e * c, "last": e * c, "d_wx": 4 * e * g * c, "d_b": 4 * e * g * c * n, "d_states": 2 * e * g}


def check(got, ref, limits):
    for key, want in ref.items():
        t = got[key].detach().cpu()
        half_step = torch.finfo(t.dtype).eps / 2
        off = (t.double() - want).abs() - half_step * want.abs()
        assert torch.isfinite(t.double()).all(), key
        assert off.max().item() <= limits[key], (key, off.max().item(), limits[key])
