"""The input projection in front of the recurrence, fused into this library's data path.

``flashrnn_projected(x, W, R, b, states, ...)`` computes ``Wx = x @ W.T (+ bias_w)`` with a hand-written tcgen05 GEMM
that writes the gate pre-activations directly in the layout and dtype the recurrent kernels stream by TMA
(``[B,T,GW,N,D]``, bf16 by default), then runs the recurrence. The reference leaves this step to the caller
(README.md:16) and benchmarks it as the "-withlinear" variant: a ``torch.nn.Linear(N*D, G*N*D)`` in front of the
kernel (flashrnn/speed_experiments/kernel_speed_benchmark.py:388-408); ``W`` / ``bias_w`` have that layer's layout.

Backward of the projection (``dx = dWx @ W``, ``dW = dWx.T @ x``, ``dbias_w = sum dWx``) uses torch's library GEMMs: they
are plain GEMMs with no recurrence-specific fusion to gain.

``fused_projection(x, weight, bias, activation, residual)`` is the product around a recurrent layer with what surrounds it in the
kernel's epilogue: the way into the gates, the way of the hidden states back into the residual stream, a feed-forward part. Its
gradients run on this library's kernels.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .functional import (SIZES, FlashRNNConfig, _dense, _error_word, _launch_word, _launched, _note_stream, _ptr, _refuse_capture, _stream,
                         _track, flashrnn, poll_errors)
from .linear import _current_device, _refuse_second_derivative


class _Projection(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, out_dtype):
        lib = _lib.load()
        poll_errors()
        B, T, I = x.shape
        J = weight.shape[0]
        dev = x.device
        with torch.cuda.device(dev):
            x16 = x.detach().to(torch.bfloat16).contiguous()
            w16 = weight.detach().to(torch.bfloat16).contiguous()
            b32 = None if bias is None else bias.detach().to(torch.float32).contiguous()
            out = torch.empty((B, T, J), dtype=out_dtype, device=dev)
            err = _error_word(dev)
            rc = lib.frnn_b200_input_projection(
                x16.data_ptr(), w16.data_ptr(), None if b32 is None else b32.data_ptr(), out.data_ptr(),
                int(out_dtype == torch.bfloat16), B, T, J, I, err.data_ptr(), torch.cuda.current_stream(dev).cuda_stream)
            _lib.check(rc, "frnn_b200_input_projection")
            _track(err, "frnn_b200_input_projection")
        ctx.save_for_backward(x16, w16)
        ctx.dtypes = (x.dtype, weight.dtype, None if bias is None else bias.dtype)
        return out

    @staticmethod
    def backward(ctx, d_out):
        x16, w16 = ctx.saved_tensors
        B, T, I = x16.shape
        g = d_out.reshape(B * T, -1).to(torch.bfloat16)
        need = ctx.needs_input_grad
        dx = (g @ w16).reshape(B, T, I).to(ctx.dtypes[0]) if need[0] else None
        dw = (g.t() @ x16.reshape(B * T, I)).to(ctx.dtypes[1]) if need[1] else None
        db = d_out.reshape(B * T, -1).float().sum(0).to(ctx.dtypes[2]) if (need[2] and ctx.dtypes[2] is not None) else None
        return dx, dw, db, None


def input_projection(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                     out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``x[B,T,I] @ weight[J,I].T (+ bias[J]) -> [B,T,J]`` on the tensor cores (bf16 operands, fp32 accumulation)."""
    if x.ndim != 3 or weight.ndim != 2 or weight.shape[1] != x.shape[2]:
        raise ValueError("expected x [B,T,I] and weight [J,I]")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError("expected bias [J]")
    if not x.is_cuda:
        raise RuntimeError("flashrnn_b200 runs on CUDA devices only (sm_100a); there is no CPU path")
    if x.shape[2] % 8 or weight.shape[0] % 64:
        raise ValueError("the projection kernel needs I % 8 == 0 and G*N*D % 64 == 0")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("out_dtype must be bfloat16 or float32")
    if not torch.is_autocast_enabled("cuda"):
        return _Projection.apply(x, weight, bias, out_dtype)
    with torch.autocast("cuda", enabled=False):
        return _Projection.apply(x, weight, bias, out_dtype)


def flashrnn_projected(x, W, R, b, states=None, bias_w=None, function: str = "lstm",
                       config: Optional[FlashRNNConfig] = None, dtype: str = "bfloat16"):
    """``x[B,T,I], W[GW*N*D, I], R[G,N,D,D], b[G,N,D], states[S,B,1,N,D]`` -> ``(states[S,B,T,N,D], last[S,B,1,N,D])``.

    The same as ``flashrnn(x @ W.T ... )`` with the projection done by this library; differentiable in x, W, bias_w,
    R, b and states."""
    if config is not None:
        function, dtype = config.function, config.dtype
    if function not in SIZES:
        raise ValueError(f"Unknown function {function}")
    gw = SIZES[function][1]
    N, D = R.shape[1], R.shape[2]
    if W.shape[0] != gw * N * D:
        raise ValueError(f"W must have {gw} * {N} * {D} rows")
    out_dtype = torch.bfloat16 if dtype == "bfloat16" else torch.float32
    wx = input_projection(x, W, bias_w, out_dtype).view(x.shape[0], x.shape[1], gw, N, D)
    return flashrnn(wx, R, b, states, function=function, config=config, dtype=dtype)


def _product_forward(x, weight, bias, residual, activation, keep: bool):
    """x [..., I], weight [J,I], residual [..., J] -> y [..., J] and, where the backward pass needs it, what the slope is taken at."""
    lib = _lib.load()
    poll_errors()
    J, I = weight.shape
    M, dev = x.numel() // I, x.device
    plan = _lib.product_plan(M, J, I, dev.index)
    y = x.new_empty((*x.shape[:-1], J))
    z = torch.empty((M, J), dtype=torch.float16, device=dev) if keep and activation is not None else None
    work = torch.empty(plan.forward_work_bytes // 4, dtype=torch.float32, device=dev) if plan.forward_work_bytes else None
    err, word = _launch_word(dev) if plan.forward_waits else (None, None)
    rc = lib.frnn_b200_product_forward(
        x.data_ptr(), weight.data_ptr(), _ptr(bias), bias is not None and bias.dtype == torch.bfloat16, _ptr(residual),
        _lib.ACTIVATIONS[activation], y.data_ptr(), _ptr(z), M, J, I, _ptr(work), err, _stream(dev))
    if word is not None:
        _launched(word, "frnn_b200_product_forward")   # the tiles have the word, whether the pass behind them was accepted or not
    if rc:
        _lib.check(rc, "frnn_b200_product_forward")
    return y, z


def _whole_vectors(x, weight, bias, residual):
    """The operands as the kernels take them: contiguous, aligned, features padded with zeros to multiples of 8."""
    J, I = weight.shape
    if I % 8 or J % 8:
        pad, pad_i, pad_j = torch.nn.functional.pad, -I % 8, -J % 8
        x, weight = pad(x, (0, pad_i)), pad(weight, (0, pad_i, 0, pad_j))
        bias = None if bias is None else pad(bias, (0, pad_j))
        residual = None if residual is None else pad(residual, (0, pad_j))
    return _dense(x), _dense(weight), None if bias is None else _dense(bias), None if residual is None else _dense(residual)


class _FusedProjection(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        _note_stream(ctx, x.device)
        need = ctx.needs_input_grad
        J, I = weight.shape
        x, weight, bias, residual = _whole_vectors(x, weight, bias, residual)
        y, z = _product_forward(x, weight, bias, residual, activation, need[0] or need[1] or need[2])
        ctx.save_for_backward(x if need[1] else None, weight if need[0] else None, z)
        ctx.activation, ctx.shapes, ctx.features = activation, (x.shape, weight.shape), (J, I)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y[..., :J].contiguous() if J % 8 else y

    @staticmethod
    def backward(ctx, dy):
        _refuse_second_derivative(dy)
        if _current_device() != dy.device.index:
            with torch.cuda.device(dy.device):
                return _FusedProjection._backward(ctx, dy, dy.device)
        return _FusedProjection._backward(ctx, dy, dy.device)

    @staticmethod
    def _backward(ctx, dy, dev):
        _refuse_capture(ctx)
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        if not (need_x or need_w or need_b):
            return None, None, None, dy, None
        lib = _lib.load()
        poll_errors()
        x, weight, z = ctx.saved_tensors
        x_shape, w_shape = ctx.shapes
        features, (J, I) = ctx.features, w_shape
        g = _dense(dy if features[0] == J else torch.nn.functional.pad(dy, (0, J - features[0])))
        M = g.numel() // J
        plan = _lib.product_plan(M, J, I, dev.index)
        dx = g.new_empty(x_shape) if need_x else None
        dw = g.new_empty(w_shape) if need_w else None
        db = torch.empty(J, dtype=ctx.bias_dtype, device=dev) if need_b else None
        # dz, the partial sums of dbias and of the products: one allocation, each part on a 16-byte boundary
        dz_bytes = 2 * M * J if z is not None else 0
        part_bytes = (plan.dbpart_bytes + 15) // 16 * 16 if need_b else 0
        total = dz_bytes + part_bytes + plan.backward_work_bytes
        at = None
        if total:
            scratch = torch.empty(total, dtype=torch.uint8, device=dev)
            at = scratch.data_ptr()
        err, word = _launch_word(dev)
        rc = lib.frnn_b200_product_backward(
            g.data_ptr(), _ptr(z), _ptr(x), _ptr(weight), _lib.ACTIVATIONS[ctx.activation], at if dz_bytes else None, _ptr(dx), _ptr(dw),
            _ptr(db), ctx.bias_dtype == torch.bfloat16, at + dz_bytes if part_bytes else None, M, J, I,
            at + dz_bytes + part_bytes if plan.backward_work_bytes else None, err, _stream(dev))
        _launched(word, "frnn_b200_product_backward")   # earlier launches of the call have the word, whether a later one was accepted or not
        if rc:
            _lib.check(rc, "frnn_b200_product_backward")
        if features != (J, I):
            dx = None if dx is None else dx[..., :features[1]]
            dw = None if dw is None else dw[:features[0], :features[1]]
            db = None if db is None else db[:features[0]]
        return dx, dw, db, dy if need_r else None, None


def fused_projection(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                     residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``activation(x[..., I] @ weight[J,I].T + bias[J]) + residual[..., J]`` in one kernel, bf16 operands and result, fp32 sums.

    ``activation`` is None, ``"relu"``, ``"silu"`` or ``"gelu_tanh"`` (the tanh form of gelu). x, weight and residual are cast to
    bf16 where they are of another type, ``bias`` is bf16 or fp32 (others are cast to fp32). Nothing is rounded before the result.
    Differentiable in all four (once): the gradient at the product, ``dy * activation'(z)``, is rounded to bf16 for the tensor
    cores; the bias's gradient sums it unrounded. Features that are no multiple of 8 are padded with zeros, at the price of copies of operands and result."""
    if activation not in _lib.ACTIVATIONS:
        raise ValueError(f"Unknown activation {activation}: None, 'relu', 'silu' or 'gelu_tanh'")
    dev, shape = x.device, x.shape
    if len(shape) < 1 or weight.ndim != 2 or weight.shape[1] != shape[-1]:
        raise ValueError("expected x [..., I] and weight [J, I]")
    J, I = weight.shape
    if x.numel() < 1 or J < 1:
        raise ValueError("rows and features must be positive")
    ok = x.is_floating_point() and weight.is_floating_point()
    strided = x.layout == torch.strided and weight.layout == torch.strided
    same = weight.device == dev
    requires = x.requires_grad or weight.requires_grad
    if bias is not None:
        if bias.shape != (J,):
            raise ValueError("expected bias [J]")
        ok, strided, same = ok and bias.is_floating_point(), strided and bias.layout == torch.strided, same and bias.device == dev
        requires = requires or bias.requires_grad
    if residual is not None:
        if residual.shape != (*shape[:-1], J):
            raise ValueError("expected residual [..., J]")
        ok, same = ok and residual.is_floating_point(), same and residual.device == dev
        strided = strided and residual.layout == torch.strided
        requires = requires or residual.requires_grad
    if not strided:
        raise ValueError("inputs must have strided tensor layout")
    if not ok:
        raise ValueError("inputs must be floating-point tensors")
    if not same:
        raise ValueError("all inputs must be on the same device")
    if not x.is_cuda:
        raise RuntimeError("flashrnn_b200 runs on CUDA devices only (sm_100a); there is no CPU path")
    requires = requires and torch.is_grad_enabled()
    if _current_device() != dev.index:
        with torch.cuda.device(dev):
            return _run_product(x, weight, bias, activation, residual, requires)
    return _run_product(x, weight, bias, activation, residual, requires)


def _bf16(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.bfloat16 else t.to(torch.bfloat16)


def _run_product(x, weight, bias, activation, residual, grad: bool):
    J = weight.shape[0]
    x, weight = _bf16(x), _bf16(weight)
    if residual is not None:
        residual = _bf16(residual)
    if bias is not None and bias.dtype != torch.bfloat16 and bias.dtype != torch.float32:
        bias = bias.to(torch.float32)
    if grad:
        return _FusedProjection.apply(x, weight, bias, residual, activation)
    y = _product_forward(*_whole_vectors(x, weight, bias, residual), activation, False)[0]
    return y[..., :J].contiguous() if J % 8 else y
