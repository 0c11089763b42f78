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

from . import _lib
from .functional import _dense, _launch_word, _launched, _note_stream, _ptr, _refuse_capture, _stream, poll_errors

# function -> gates of Wx and b
LINEAR_GATES = {"leaky": 2, "lstm": 4}


def _forward(wx, bias, initial, lengths, function: str, keep: bool, last: Optional[torch.Tensor] = None):
    """-> hidden, last, starts (None where nothing has to be kept for the backward pass)"""
    lib = _lib.load()
    poll_errors()
    B, T, _, N, D = wx.shape
    dev = wx.device
    plan = _lib.linear_plan(function, B, T, N, D)
    hidden = wx.new_empty((B, T, N, D))
    if last is None:
        last = bias.new_empty((1, B, 1, N, D))
    starts = exchange = err = word = None
    if keep and plan.starts_bytes:
        # with the exchange buffer behind it: an allocation costs a short call more than 2 % of Wx cost a long one's memory
        behind = (plan.starts_bytes + 15) // 16 * 16
        starts = bias.new_empty((behind + plan.exchange_bytes) // 4)
    if plan.exchange_bytes:   # several tiles, which wait for one another
        if starts is None:
            scratch = bias.new_empty(plan.exchange_bytes // 4)
            exchange = scratch.data_ptr()
        else:
            exchange = starts.data_ptr() + behind
        err, word = _launch_word(dev)
    rc = lib.frnn_b200_linear_forward(
        _lib.LINEAR_CELLS[function], wx.data_ptr(), wx.dtype == torch.bfloat16, bias.data_ptr(), _ptr(initial), _ptr(lengths),
        hidden.data_ptr(), last.data_ptr(), _ptr(starts), exchange, B, T, N, D, 0, err, _stream(dev))
    if rc:
        _lib.check(rc, "frnn_b200_linear_forward")
    if err is not None:
        _launched(word, "frnn_b200_linear_forward")
    return hidden, last, starts


class _LinearRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, wx, bias, initial, lengths, function: str):
        _note_stream(ctx, wx.device)
        hidden, last, starts = _forward(wx, bias, initial, lengths, function, True)
        ctx.save_for_backward(wx, bias, initial, lengths, starts)
        ctx.function = function
        ctx.set_materialize_grads(False)
        return hidden, last

    @staticmethod
    def backward(ctx, d_hidden, d_last):
        _refuse_second_derivative(d_hidden, d_last)
        if d_hidden is None and d_last is None:
            return None, None, None, None, None
        wx, bias, initial, lengths, starts = ctx.saved_tensors
        dev = wx.device
        if _current_device() != dev.index:
            with torch.cuda.device(dev):
                return _LinearRecurrence._backward(ctx, d_hidden, d_last, wx, bias, initial, lengths, starts, dev)
        return _LinearRecurrence._backward(ctx, d_hidden, d_last, wx, bias, initial, lengths, starts, dev)

    @staticmethod
    def _backward(ctx, d_hidden, d_last, wx, bias, initial, lengths, starts, dev):
        _refuse_capture(ctx)
        lib = _lib.load()
        poll_errors()
        B, T, _, N, D = wx.shape
        plan = _lib.linear_plan(ctx.function, B, T, N, D)
        d_hidden = wx.new_zeros((B, T, N, D)) if d_hidden is None else _dense(d_hidden)
        if d_last is not None:
            d_last = _dense(d_last)
        d_wx, db = torch.empty_like(wx), torch.empty_like(bias)
        need = ctx.needs_input_grad
        d_initial = torch.empty_like(initial) if need[2] else None
        part = exchange = err = word = None
        if plan.dbpart_bytes:   # and the exchange buffer, whose size is 0 where there is nothing to wait for, in one allocation
            room = plan.exchange_bytes
            scratch = bias.new_empty((room + plan.dbpart_bytes) // 4)
            part = scratch.data_ptr() + room
            if room:
                exchange = scratch.data_ptr()
                err, word = _launch_word(dev)
        rc = lib.frnn_b200_linear_backward(
            _lib.LINEAR_CELLS[ctx.function], wx.data_ptr(), wx.dtype == torch.bfloat16, bias.data_ptr(), _ptr(initial), _ptr(lengths),
            _ptr(starts), d_hidden.data_ptr(), _ptr(d_last), d_wx.data_ptr(), db.data_ptr(), _ptr(d_initial), part, exchange,
            B, T, N, D, 0, err, _stream(dev))
        if err is not None:
            _launched(word, "frnn_b200_linear_backward")   # the scan has the word, whether the sum of db behind it was accepted or not
        if rc:
            _lib.check(rc, "frnn_b200_linear_backward")
        return d_wx if need[0] else None, db if need[1] else None, d_initial, None, None


def _refuse_second_derivative(*grads) -> None:
    if torch.is_grad_enabled() and any(g is not None and g.requires_grad for g in grads):
        raise RuntimeError("this operator's gradients are not differentiable themselves")


def _current_device() -> int:
    return torch._C._cuda_getDevice()


def flashrnn_linear(Wx: torch.Tensor, b: torch.Tensor, states: Optional[torch.Tensor] = None, function: str = "leaky",
                    lengths: Optional[torch.Tensor] = None, last_out: Optional[torch.Tensor] = None):
    """``Wx[B,T,G,N,D], b[G,N,D], states[1,B,1,N,D]`` -> ``(hidden[B,T,N,D], last[1,B,1,N,D])``; ``states=None`` means zeros.

    ``Wx`` is bf16 or fp32, and so are the hidden states; ``b``, ``states`` and ``last`` are fp32 (others are cast). Any sizes;
    a single step (T = 1) is the call of a decoding loop. Differentiable in Wx, b and states (once).

    ``lengths[B]`` (int32 or int64, on the same device; values are clamped to ``[0, T]``) makes it a padded batch: steps at or
    behind a row's length leave its state alone, so ``last`` is the state at its end, and their hidden states and gradients are
    zeros, whatever Wx holds there.

    A state that becomes infinite may turn into a NaN later, in its channel only: a decay of 1/2 or more takes a part of it away, infinity
    from infinity, and over many steps it is multiplied by a decay that has become zero. Sums of a state and its input beyond the range of
    fp32 count as infinite.

    ``last_out`` (without gradients only) is written and returned as ``last``; it may be ``states`` itself, which a captured
    decoding step then updates in place. Where it shares memory with another input, that is written once the call has read it.
    """
    if function not in LINEAR_GATES:
        raise ValueError(f"Unknown function {function}: flashrnn_linear has {', '.join(LINEAR_GATES)}")
    dev, shape = Wx.device, Wx.shape
    if len(shape) != 5 or Wx.layout != torch.strided or Wx.numel() < 1:
        raise ValueError("expected a nonempty Wx [B,T,G,N,D] of strided layout")
    B, T, G, N, D = shape
    if G != LINEAR_GATES[function] or b.shape != shape[2:]:
        raise ValueError(f"shape mismatch for {function}: Wx {tuple(shape)}, b {tuple(b.shape)}")
    if Wx.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("Wx must be bfloat16 or float32")
    if b.layout != torch.strided or not b.is_floating_point():
        raise ValueError("b must be a floating-point tensor of strided layout")
    same = b.device == dev
    requires = Wx.requires_grad or b.requires_grad
    if states is not None:
        if states.shape != (1, B, 1, N, D):
            raise ValueError("states must have layout [1,B,1,N,D]")
        if states.layout != torch.strided or not states.is_floating_point():
            raise ValueError("states must be a floating-point tensor of strided layout")
        same = same and states.device == dev
        requires = requires or states.requires_grad
    if lengths is not None:
        if lengths.shape != (B,) or lengths.layout != torch.strided or lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError("lengths must be an int32 or int64 tensor [B]")
        same = same and lengths.device == dev
    requires = requires and torch.is_grad_enabled()
    if last_out is not None:
        if requires or last_out.requires_grad:
            raise ValueError("last_out takes no gradients: call under torch.no_grad()")
        if last_out.shape != (1, B, 1, N, D) or last_out.dtype != torch.float32 or not last_out.is_contiguous():
            raise ValueError("last_out must be a contiguous float32 tensor [1,B,1,N,D]")
        same = same and last_out.device == dev
    if not same:
        raise ValueError("all inputs must be on the same device")
    if not Wx.is_cuda:
        raise RuntimeError("flashrnn_b200 runs on CUDA devices only (sm_100a); there is no CPU path")
    if _current_device() != dev.index:
        with torch.cuda.device(dev):
            return _run(Wx, b, states, function, lengths, last_out, requires)
    return _run(Wx, b, states, function, lengths, last_out, requires)


def _run(wx, b, states, function, lengths, last_out, grad):
    wx, b = _dense(wx), _state(b)
    if states is not None:
        states = _state(states)
    if lengths is not None:
        if lengths.dtype == torch.int64:
            lengths = lengths.clamp(0, wx.shape[1]).to(torch.int32)
        lengths = lengths.contiguous()
    if grad:
        return _LinearRecurrence.apply(wx, b, states, lengths, function)
    out = last_out
    if out is not None and out.data_ptr() % 16:
        out = None
    if out is not None:
        # a call of several steps may read `states` after other parts of `last` are written, and so may a step where the two overlap without
        # being the same, or where `last_out` lies over another input: a buffer in between
        if _overlap(wx, out) or _overlap(b, out) or (lengths is not None and _overlap(lengths, out)):
            out = None
        elif states is not None and _overlap(states, out) and (wx.shape[1] > 1 or states.data_ptr() != out.data_ptr()):
            out = None
    hidden, last, _ = _forward(wx, b, states, lengths, function, False, out)
    if last_out is not None and out is None:
        last = last_out.copy_(last)
    return hidden, last


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two contiguous tensors share memory."""
    first, second = a.data_ptr(), b.data_ptr()
    return first < second + b.nbytes and second < first + a.nbytes


def _state(t: torch.Tensor) -> torch.Tensor:
    return _dense(t if t.dtype == torch.float32 else t.to(torch.float32))
