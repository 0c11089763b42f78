"""Operators around a recurrent layer whose speed this repository watches: the gated linear recurrence, which has no
recurrent matrix and is scanned in parallel over time, and the matrix product that feeds it and takes its hidden states
back into the residual stream, with bias, activation and residual in its epilogue.

``own`` False computes them in plain form, in 32 bits, rounded once at the end; ``own`` True makes the calls a user makes.
"""

from __future__ import annotations

import math

import torch

own = False

# function -> gates of Wx, in order.  leaky: (f, z); lstm: (i, f, z, o), the LSTM's gates without its recurrent matrix
GATES = {"leaky": 2, "lstm": 4}

# A case of the recurrence: op "linear", kind "infer" or "train", function, B, T, N, D, dtype (of Wx and of the hidden states),
#   states  True: starts from a given state (training hands its gradient back), False: from zeros
#   carry   True: the loss also depends on the last state
#   lengths True: a padded batch, every sequence with a length of its own, an empty one among them
# A case of the product: op "product", kind, rows B x T, I input and J output features, bf16,
#   bias, residual True / False, activation "none", "relu", "silu" or "gelu_tanh"


def _linear(name, kind, function, B, T, N, D, dtype="bfloat16", states=True, carry=False, lengths=False):
    out = {"op": "linear", "kind": kind, "function": function, "B": B, "T": T, "N": N, "D": D, "dtype": dtype,
           "states": states, "carry": carry, "lengths": lengths}
    return {"name": name, **out} if name else out


def _product(name, kind, B, T, I, J, bias=True, activation="none", residual=False):
    out = {"op": "product", "kind": kind, "B": B, "T": T, "I": I, "J": J, "bias": bias, "activation": activation,
           "residual": residual}
    return {"name": name, **out} if name else out


def listed():
    return [
        # serving: one token for four streams, from the state that the last call left
        _linear("linear_decode_lstm_B4_T1_N3_D256", "infer", "lstm", 4, 1, 3, 256),
        # serving: a short piece of a stream, one wide head
        _linear("linear_stream_leaky_B4_T16_N1_D768", "infer", "leaky", 4, 16, 1, 768),
        # a long document read in one go: few channels, all of the parallelism is in time
        _linear("linear_infer_leaky_B1_T65536_N3_D256", "infer", "leaky", 1, 65536, 3, 256, states=False),
        # the headline training shape
        _linear("linear_train_leaky_B8_T1024_N3_D256", "train", "leaky", 8, 1024, 3, 256),
        # narrow heads, four gates, truncated back-propagation over pieces (gradient through the carry)
        _linear("linear_train_lstm_B16_T1024_N12_D64", "train", "lstm", 16, 1024, 12, 64, carry=True),
        # ragged everywhere: padded batch, odd batch and length, fp32
        _linear("linear_train_leaky_fp32_B13_T333_N2_D200_padded", "train", "leaky", 13, 333, 2, 200, "float32", carry=True,
                lengths=True),
        # the largest: one GPU's share of a 32-head layer
        _linear("linear_train_leaky_B32_T2048_N32_D128", "train", "leaky", 32, 2048, 32, 128, states=False),
        # serving: the gate projection of one token for four streams
        _product("product_decode_B4_I768_J1536", "infer", 4, 1, 768, 1536, activation="silu"),
        # a layer's way back into the residual stream
        _product("product_infer_B16_T1024_I768_J768_residual", "infer", 16, 1024, 768, 768, residual=True),
        # the widening product of a feed-forward part, training
        _product("product_train_B8_T1024_I768_J2048_gelu", "train", 8, 1024, 768, 2048, activation="gelu_tanh"),
        # ragged rows and features, everything in the epilogue
        _product("product_train_B13_T333_I200_J600_silu_residual", "train", 13, 333, 200, 600, activation="silu", residual=True),
        # the largest: a wide layer's projection over a whole batch
        _product("product_train_B32_T1024_I2048_J4096_silu", "train", 32, 1024, 2048, 4096, activation="silu"),
    ]


_ITEMS_MAX = 32 * 2048 * 32 * 128              # (batch, step, channel) triples of the largest listed recurrence
_MACS_MAX = 32 * 1024 * 2048 * 4096            # multiply-adds of the largest listed product


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("infer", "train"))
    if rng.random() < 0.5:
        function, dtype = rng.choice(("leaky", "lstm")), rng.choice(("bfloat16", "bfloat16", "float32"))
        B, T, N = _log_int(rng, 1, 64), _log_int(rng, 1, 65536), _log_int(rng, 1, 32)
        D = rng.choice((16, 32, 64, 128, 256, 8 * _log_int(rng, 2, 32), _log_int(rng, 16, 256)))
        cap = _ITEMS_MAX // (4 if function == "lstm" or dtype == "float32" else 1)
        B = max(1, min(B, cap // (T * N * D)))
        states = rng.random() < 0.6
        return _linear(None, kind, function, B, T, N, D, dtype, states, rng.random() < 0.4, rng.random() < 0.4)
    B, T = _log_int(rng, 1, 32), (1 if rng.random() < 0.3 else _log_int(rng, 1, 1024))
    I, J = (8 * _log_int(rng, 8, 512) for _ in range(2))
    if rng.random() < 0.125:
        I, J = I + rng.randrange(1, 8), J + rng.randrange(1, 8)
    B = max(1, min(B, _MACS_MAX // (T * I * J)))
    return _product(None, kind, B, T, I, J, rng.random() < 0.7, rng.choice(("none", "relu", "silu", "gelu_tanh")),
                    rng.random() < 0.5)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape, dtype=torch.float32, scale=1.0):
        return torch.randn(shape, generator=g, device=dev).mul_(scale).to(dtype)

    def rand(*shape):
        return torch.rand(shape, generator=g, device=dev)

    st = {"case": dict(case)}
    train = case["kind"] == "train"
    if case["op"] == "linear":
        B, T, N, D, G = (*(case[k] for k in ("B", "T", "N", "D")), GATES[case["function"]])
        dtype = getattr(torch, case["dtype"])
        st["wx"] = randn(B, T, G, N, D, dtype=dtype)
        st["b"] = randn(G, N, D, scale=0.1)
        st["b"][1 if case["function"] == "lstm" else 0] = rand(N, D) * 6.0    # channels that forget at once to hundreds of steps
        st["states"] = randn(1, B, 1, N, D, scale=0.5) if case["states"] else None
        st["lengths"] = None
        if case["lengths"]:
            st["lengths"] = (rand(B) * (T + 1)).to(torch.int32)
            st["lengths"][B // 2] = 0
            st["lengths"][0] = T
        if train:
            st["dh"] = randn(B, T, N, D, dtype=dtype)
            st["dlast"] = randn(1, B, 1, N, D) if case["carry"] else None
            st["leaves"] = [t.requires_grad_(True) for t in (st["wx"], st["b"], st["states"]) if t is not None]
    else:
        B, T, I, J = (case[k] for k in ("B", "T", "I", "J"))
        bf16 = torch.bfloat16
        st["x"] = randn(B, T, I, dtype=bf16)
        st["weight"] = randn(J, I, dtype=bf16, scale=I ** -0.5)
        st["bias"] = randn(J, dtype=bf16, scale=0.1) if case["bias"] else None
        st["residual"] = randn(B, T, J, dtype=bf16) if case["residual"] else None
        if train:
            st["dy"] = randn(B, T, J, dtype=bf16)
            names = ("x", "weight", "bias", "residual")
            st["leaves"] = [st[k].requires_grad_(True) for k in names if st[k] is not None]
    return st


# ---------------------------------------------------------------------------------------------------- plain forms


def _scan(a, v):
    """y_t = a_t y_{t-1} + v_t along dimension 1, from y_{-1} = 0: spans double until they cover the sequence."""
    s, T = 1, v.shape[1]
    while s < T:
        v = torch.cat((v[:, :s], v[:, s:] + a[:, s:] * v[:, :-s]), 1)
        a = torch.cat((a[:, :s], a[:, s:] * a[:, :-s]), 1)
        s *= 2
    return v


def _linear_plain(st):
    case = st["case"]
    lstm, train = case["function"] == "lstm", case["kind"] == "train"
    dtype = st["wx"].dtype
    x = st["wx"].detach().float() + st["b"].detach()
    init = torch.zeros_like(x[:, 0, 0]) if st["states"] is None else st["states"].detach()[0, :, 0]
    T = x.shape[1]
    valid = None
    if st["lengths"] is not None:
        valid = (torch.arange(T, device=x.device) < st["lengths"][:, None])[:, :, None, None]
    if lstm:
        i, f, z, o = torch.sigmoid(x[:, :, 0]), torch.sigmoid(x[:, :, 1]), torch.tanh(x[:, :, 2]), torch.sigmoid(x[:, :, 3])
        v = i * z
    else:
        f, z = torch.sigmoid(x[:, :, 0]), x[:, :, 1]
        v = (1 - f) * z
    a = f
    if valid is not None:
        a, v = torch.where(valid, a, 1.0), torch.where(valid, v, 0.0)
    c = _scan(a, torch.cat((v[:, :1] + a[:, :1] * init[:, None], v[:, 1:]), 1))
    hidden = o * torch.tanh(c) if lstm else c
    if valid is not None:
        hidden = torch.where(valid, hidden, 0.0)
    out = {"hidden": hidden.to(dtype), "last": c[:, -1:].unsqueeze(0).clone()}
    if not train:
        return out
    dh = st["dh"].float()
    if valid is not None:
        dh = torch.where(valid, dh, 0.0)
    tc = torch.tanh(c) if lstm else None
    dc = dh * o * (1 - tc * tc) if lstm else dh
    if st["dlast"] is not None:
        dc = torch.cat((dc[:, :-1], dc[:, -1:] + st["dlast"][0]), 1)
    after = torch.cat((a[:, 1:], torch.zeros_like(a[:, :1])), 1)           # the decay that a state meets in the next step
    g = _scan(after.flip(1), dc.flip(1)).flip(1)
    before = torch.cat((init[:, None], c[:, :-1]), 1)
    if lstm:
        d = (g * z * i * (1 - i), g * before * f * (1 - f), g * i * (1 - z * z), dh * tc * o * (1 - o))
    else:
        d = (g * (before - z) * f * (1 - f), g * (1 - f))
    d = torch.stack(d, 2)
    if valid is not None:
        d = torch.where(valid[:, :, None], d, 0.0)
    out["d_wx"], out["d_b"] = d.to(dtype), d.sum((0, 1))
    if st["states"] is not None:
        out["d_states"] = (a[:, :1] * g[:, :1]).unsqueeze(0)
    return out


def _act(z, activation):
    """The activation of z and its derivative."""
    if activation == "none":
        return z, torch.ones_like(z)
    if activation == "relu":
        return torch.where(z > 0, z, 0.0), (z > 0).to(z.dtype)
    # silu and the tanh form of gelu are both z * sigmoid(w(z))
    k = 2 * math.sqrt(2 / math.pi)
    w, dw = (z, 1.0) if activation == "silu" else (k * (z + 0.044715 * z * z * z), k * (1 + 3 * 0.044715 * z * z))
    s = torch.sigmoid(w)
    return z * s, s + z * s * (1 - s) * dw


def _product_plain(st):
    case = st["case"]
    x, w = st["x"].detach().float().flatten(0, 1), st["weight"].detach().float()
    z = x @ w.t()
    if st["bias"] is not None:
        z = z + st["bias"].detach().float()
    y, slope = _act(z, case["activation"])
    if st["residual"] is not None:
        y = y + st["residual"].detach().float().flatten(0, 1)
    bf16, rows = torch.bfloat16, st["x"].shape[:2]
    out = {"y": y.to(bf16).unflatten(0, rows)}
    if case["kind"] == "train":
        dz = st["dy"].float().flatten(0, 1) * slope
        out["d_x"], out["d_weight"] = (dz @ w).to(bf16).unflatten(0, rows), (dz.t() @ x).to(bf16)
        if st["bias"] is not None:
            out["d_bias"] = dz.sum(0).to(bf16)
        if st["residual"] is not None:
            out["d_residual"] = st["dy"]
    return out


# ------------------------------------------------------------------------------------------------ the user's calls


def _linear_own(st):
    from flashrnn_b200 import flashrnn_linear

    case = st["case"]
    if case["kind"] == "infer":
        with torch.no_grad():
            hidden, last = flashrnn_linear(st["wx"], st["b"], st["states"], function=case["function"], lengths=st["lengths"])
        return {"hidden": hidden, "last": last}
    hidden, last = flashrnn_linear(st["wx"], st["b"], st["states"], function=case["function"], lengths=st["lengths"])
    outs, grads = ([hidden], [st["dh"]]) if st["dlast"] is None else ([hidden, last], [st["dh"], st["dlast"]])
    d = torch.autograd.grad(outs, st["leaves"], grads)
    return {"hidden": hidden.detach(), "last": last.detach(), **dict(zip(("d_wx", "d_b", "d_states"), d))}


def _product_own(st):
    from flashrnn_b200 import fused_projection

    case = st["case"]
    activation = None if case["activation"] == "none" else case["activation"]
    if case["kind"] == "infer":
        with torch.no_grad():
            return {"y": fused_projection(st["x"], st["weight"], st["bias"], activation=activation, residual=st["residual"])}
    y = fused_projection(st["x"], st["weight"], st["bias"], activation=activation, residual=st["residual"])
    d = torch.autograd.grad(y, st["leaves"], st["dy"])
    names = [k for k in ("x", "weight", "bias", "residual") if st[k] is not None]
    return {"y": y.detach(), **{"d_" + k: t for k, t in zip(names, d)}}


def run(state):
    if state["case"]["op"] == "linear":
        return _linear_own(state) if own else _linear_plain(state)
    return _product_own(state) if own else _product_plain(state)


def work(case):
    train = case["kind"] == "train"
    if case["op"] == "linear":
        B, T, N, D, G = (*(case[k] for k in ("B", "T", "N", "D")), GATES[case["function"]])
        es = 2 if case["dtype"] == "bfloat16" else 4
        items, channels = B * T * N * D, N * D
        # gates in, hidden states out, bias, first and last states; training: gates and dh in, dWx out, their gradients out
        total = items * (G + 1) * es + 4 * (G * channels + (2 if case["states"] else 1) * B * channels)
        if train:
            total += items * (2 * G + 1) * es + 4 * (2 * G * channels + (case["states"] + case["carry"]) * B * channels)
        return {"bytes": float(total), "flops": float(items * (40 if train else 15))}
    M, I, J = case["B"] * case["T"], case["I"], case["J"]
    total = 2 * (M * I + I * J + M * J * (2 if case["residual"] else 1) + (J if case["bias"] else 0))
    if train:   # dy, x and W in, dx, dW and dbias out
        total += 2 * (M * J + 2 * M * I + 2 * I * J + (J if case["bias"] else 0))
        if case["activation"] != "none":
            total += 2 * 2 * M * J           # what the activation's derivative is taken at, out and in again
    return {"bytes": float(total), "flops": float(2 * M * I * J * (3 if train else 1))}


# --------------------------------------------------------------------------------------- in 64 bits, from the definition


def _linear_exact(st):
    case = st["case"]
    lstm = case["function"] == "lstm"
    wx, b = st["wx"].detach(), st["b"].detach().double()
    B, T, G, N, D = wx.shape
    first = torch.zeros((B, N, D), dtype=torch.float64, device=wx.device)
    if st["states"] is not None:
        first = st["states"].detach()[0, :, 0].double()
    lengths = st["lengths"] if st["lengths"] is not None else torch.full((B,), T, device=wx.device)
    inside = lengths[None, :] > torch.arange(T, device=wx.device)[:, None]      # [T, B]

    def gates(t):
        p = wx[:, t].double() + b
        if lstm:
            return 1 / (1 + torch.exp(-p[:, 1])), torch.tanh(p[:, 2]), 1 / (1 + torch.exp(-p[:, 0])), 1 / (1 + torch.exp(-p[:, 3]))
        s = 1 / (1 + torch.exp(-p[:, 0]))
        return s, p[:, 1], 1 / (1 + torch.exp(p[:, 0])), None

    c, cs = first, torch.empty((T, B, N, D), dtype=torch.float64, device=wx.device)
    hidden = torch.zeros((B, T, N, D), dtype=torch.float64, device=wx.device)
    for t in range(T):
        f, z, i, o = gates(t)
        on = inside[t][:, None, None]
        c = torch.where(on, f * c + i * z, c)
        cs[t] = c
        hidden[:, t] = torch.where(on, o * torch.tanh(c) if lstm else c, torch.zeros_like(c))
    out = {"hidden": hidden, "last": c[None, :, None].clone()}
    if case["kind"] != "train":
        return out
    g = torch.zeros_like(first) if st["dlast"] is None else st["dlast"][0, :, 0].double()
    d_wx, d_b = torch.zeros((B, T, G, N, D), dtype=torch.float64, device=wx.device), torch.zeros_like(b)
    for t in range(T - 1, -1, -1):
        f, z, i, o = gates(t)
        on = inside[t][:, None, None]
        dh = st["dh"][:, t].double()
        prev = cs[t - 1] if t else first
        if lstm:
            th = torch.tanh(cs[t])
            s = g + dh * o * (1 - th ** 2)
            d = torch.stack((s * z * i * (1 - i), s * prev * f * (1 - f), s * i * (1 - z ** 2), dh * th * o * (1 - o)), 1)
        else:
            s = g + dh
            d = torch.stack((s * (prev - z) * f * i, s * i), 1)
        d = torch.where(on[:, None], d, torch.zeros_like(d))
        d_wx[:, t] = d
        d_b += d.sum(0)
        g = torch.where(on, s * f, g)
    out.update(d_wx=d_wx, d_b=d_b)
    if st["states"] is not None:
        out["d_states"] = g[None, :, None]
    return out


def _product_exact(st):
    case = st["case"]
    leaf = {k: st[k].detach().double().requires_grad_(True) for k in ("x", "weight", "bias", "residual") if st[k] is not None}
    z = torch.einsum("bti,ji->btj", leaf["x"], leaf["weight"])
    if "bias" in leaf:
        z = z + leaf["bias"]
    if case["activation"] == "relu":
        y = z.clamp(min=0)
    elif case["activation"] == "silu":
        y = z / (1 + torch.exp(-z))
    elif case["activation"] == "gelu_tanh":
        y = z / 2 * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)))
    else:
        y = z
    if "residual" in leaf:
        y = y + leaf["residual"]
    out = {"y": y.detach()}
    if case["kind"] == "train":
        out.update({"d_" + k: d for k, d in zip(leaf, torch.autograd.grad(y, list(leaf.values()), st["dy"].double()))})
        if "d_residual" in out:
            out["d_residual"] = None         # dy itself
    return out


def exact(case, seed):
    if case["op"] == "linear" and case["T"] > (24000 if case["kind"] == "train" else 70000):
        return None                              # step by step in 64 bits: too slow
    st = prepare(case, seed)
    return _linear_exact(st) if case["op"] == "linear" else _product_exact(st)
