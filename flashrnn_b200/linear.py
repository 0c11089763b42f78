"""Gated linear recurrences: cells without a recurrent matrix, scanned in parallel over time.

``flashrnn_linear(Wx, b, states, function, lengths)`` takes gate pre-activations in the layout of ``flashrnn`` and returns the
hidden states, in the type of ``Wx``, and the last state, in fp32, which is a valid ``states`` of the next call and stays
connected to autograd. With ``x = Wx + b``:

* ``"leaky"``, gates (f, z):        ``c_t = sigmoid(f) c_{t-1} + (1 - sigmoid(f)) z``, hidden = c
* ``"lstm"``, gates (i, f, z, o):   ``c_t = sigmoid(f) c_{t-1} + sigmoid(i) tanh(z)``, hidden = sigmoid(o) tanh(c): the LSTM of
  ``flashrnn`` with R = 0 (its state here is c alone, since h is fed back nowhere)

States, sums and gradients are computed in fp32 and rounded once, where they are stored.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .functional import _dense, _error_word, _ptr, _stream, _track, poll_errors

# function -> gates of Wx and b
LINEAR_GATES = {"leaky": 2, "lstm": 4}


def _scratch(plan, device):
    """(exchange buffer, error word) of a launch whose tiles wait for one another, (None, None) of one that has nothing to wait for."""
    if not plan.exchange_bytes:
        return None, None
    return torch.empty(plan.exchange_bytes, dtype=torch.uint8, device=device), _error_word(device)


def _forward(wx, bias, initial, lengths, function: str, keep: bool, last: Optional[torch.Tensor] = None):
    """-> hidden, last, starts (None where nothing has to be kept for the backward pass)"""
    lib = _lib.load()
    poll_errors()
    B, T, _, N, D = wx.shape
    dev = wx.device
    plan = _lib.linear_plan(function, B, T, N, D)
    hidden = torch.empty((B, T, N, D), dtype=wx.dtype, device=dev)
    if last is None:
        last = torch.empty((1, B, 1, N, D), dtype=torch.float32, device=dev)
    starts = None
    if keep and plan.starts_bytes:
        starts = torch.empty(plan.starts_bytes // 4, dtype=torch.float32, device=dev)
    exchange, err = _scratch(plan, dev)
    rc = lib.frnn_b200_linear_forward(
        _lib.LINEAR_CELLS[function], wx.data_ptr(), int(wx.dtype == torch.bfloat16), bias.data_ptr(), _ptr(initial), _ptr(lengths),
        hidden.data_ptr(), last.data_ptr(), _ptr(starts), _ptr(exchange), B, T, N, D, 0, _ptr(err), _stream(dev))
    _lib.check(rc, "frnn_b200_linear_forward")
    if err is not None:
        _track(err, "frnn_b200_linear_forward")
    return hidden, last, starts


class _LinearRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, wx, bias, initial, lengths, function: str):
        hidden, last, starts = _forward(wx, bias, initial, lengths, function, True)
        ctx.save_for_backward(wx, bias, initial, lengths, starts)
        ctx.function = function
        ctx.set_materialize_grads(False)
        return hidden, last

    @staticmethod
    @once_differentiable
    def backward(ctx, d_hidden, d_last):
        wx = ctx.saved_tensors[0]
        if d_hidden is None and d_last is None:
            return (None,) * 5
        with torch.cuda.device(wx.device):
            return _LinearRecurrence._backward(ctx, d_hidden, d_last)

    @staticmethod
    def _backward(ctx, d_hidden, d_last):
        lib = _lib.load()
        poll_errors()
        wx, bias, initial, lengths, starts = ctx.saved_tensors
        B, T, G, N, D = wx.shape
        dev = wx.device
        plan = _lib.linear_plan(ctx.function, B, T, N, D)
        d_hidden = torch.zeros((B, T, N, D), dtype=wx.dtype, device=dev) if d_hidden is None else _dense(d_hidden.to(wx.dtype))
        if d_last is not None:
            d_last = d_last.to(torch.float32).contiguous()
        d_wx, db = torch.empty_like(wx), torch.empty_like(bias)
        d_initial = torch.empty_like(initial) if initial is not None and ctx.needs_input_grad[2] else None
        db_part = torch.empty(plan.dbpart_bytes // 4, dtype=torch.float32, device=dev) if plan.dbpart_bytes else None
        exchange, err = _scratch(plan, dev)
        rc = lib.frnn_b200_linear_backward(
            _lib.LINEAR_CELLS[ctx.function], wx.data_ptr(), int(wx.dtype == torch.bfloat16), bias.data_ptr(), _ptr(initial), _ptr(lengths),
            _ptr(starts), d_hidden.data_ptr(), _ptr(d_last), d_wx.data_ptr(), db.data_ptr(), _ptr(d_initial), _ptr(db_part),
            _ptr(exchange), B, T, N, D, 0, _ptr(err), _stream(dev))
        if err is not None:
            _track(err, "frnn_b200_linear_backward")   # the scan has the word, whether the sum of db behind it was accepted or not
        _lib.check(rc, "frnn_b200_linear_backward")
        need = ctx.needs_input_grad
        return d_wx if need[0] else None, db if need[1] else None, d_initial, None, None


def flashrnn_linear(Wx: torch.Tensor, b: torch.Tensor, states: Optional[torch.Tensor] = None, function: str = "leaky",
                    lengths: Optional[torch.Tensor] = None, last_out: Optional[torch.Tensor] = None):
    """``Wx[B,T,G,N,D], b[G,N,D], states[1,B,1,N,D]`` -> ``(hidden[B,T,N,D], last[1,B,1,N,D])``; ``states=None`` means zeros.

    ``Wx`` is bf16 or fp32, and so are the hidden states; ``b``, ``states`` and ``last`` are fp32 (others are cast). Any sizes;
    a single step (T = 1) is the call of a decoding loop. Differentiable in Wx, b and states (once).

    ``lengths[B]`` (int32 or int64, on the same device; values are clamped to ``[0, T]``) makes it a padded batch: steps at or
    behind a row's length leave its state alone, so ``last`` is the state at its end, and their hidden states and gradients are
    zeros, whatever Wx holds there.

    ``last_out`` (without gradients only) is written and returned as ``last``; it may be ``states`` itself, which a captured
    decoding step then updates in place.
    """
    if function not in LINEAR_GATES:
        raise ValueError(f"Unknown function {function}: flashrnn_linear has {', '.join(LINEAR_GATES)}")
    tensors = [t for t in (Wx, b, states, lengths, last_out) if t is not None]
    if any(t.layout != torch.strided for t in tensors):
        raise ValueError("inputs must have strided tensor layout")
    if Wx.ndim != 5 or min(Wx.shape) < 1:
        raise ValueError("expected a nonempty Wx [B,T,G,N,D]")
    B, T, G, N, D = Wx.shape
    if G != LINEAR_GATES[function] or tuple(b.shape) != (G, N, D):
        raise ValueError(f"shape mismatch for {function}: Wx {tuple(Wx.shape)}, b {tuple(b.shape)}")
    if Wx.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("Wx must be bfloat16 or float32")
    if states is not None and tuple(states.shape) != (1, B, 1, N, D):
        raise ValueError("states must have layout [1,B,1,N,D]")
    if not b.is_floating_point() or (states is not None and not states.is_floating_point()):
        raise ValueError("b and states must be floating-point tensors")
    if lengths is not None and (tuple(lengths.shape) != (B,) or lengths.dtype not in (torch.int32, torch.int64)):
        raise ValueError("lengths must be an int32 or int64 tensor [B]")
    if any(t.device != Wx.device for t in tensors):
        raise ValueError("all inputs must be on the same device")
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (Wx, b, states))
    if last_out is not None:
        if grad or last_out.requires_grad:
            raise ValueError("last_out takes no gradients: call under torch.no_grad()")
        if tuple(last_out.shape) != (1, B, 1, N, D) or last_out.dtype != torch.float32 or not last_out.is_contiguous():
            raise ValueError("last_out must be a contiguous float32 tensor [1,B,1,N,D]")
    if not Wx.is_cuda:
        raise RuntimeError("flashrnn_b200 runs on CUDA devices only (sm_100a); there is no CPU path")
    if torch.cuda.current_device() != Wx.device.index:
        with torch.cuda.device(Wx.device):
            return _run(Wx, b, states, function, lengths, last_out, grad)
    return _run(Wx, b, states, function, lengths, last_out, grad)


def _run(wx, b, states, function, lengths, last_out, grad):
    wx, b = _dense(wx), b.to(torch.float32).contiguous()
    if states is not None:
        states = states.to(torch.float32).contiguous()
    if lengths is not None:
        if lengths.dtype == torch.int64:
            lengths = lengths.clamp(0, wx.shape[1]).to(torch.int32)
        lengths = lengths.contiguous()
    if grad:
        return _LinearRecurrence.apply(wx, b, states, lengths, function)
    out = last_out
    if out is not None and wx.shape[1] > 1:
        # a longer call may read `states` after other parts of `last` are written: a buffer in between, where they can share memory
        if states is not None and states.untyped_storage().data_ptr() == out.untyped_storage().data_ptr():
            out = None
    elif out is not None and states is not None and states.data_ptr() != out.data_ptr() and \
            states.untyped_storage().data_ptr() == out.untyped_storage().data_ptr():
        out = None
    hidden, last, _ = _forward(wx, b, states, lengths, function, False, out)
    if last_out is not None and last is not last_out:
        last = last_out.copy_(last)
    return hidden, last
