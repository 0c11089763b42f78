"""Gradients of a bias: the sum of the terms that the same backward pass hands out, over few and over many parts."""

import pytest
import torch

from tests import _bias_sums as S
from tests import _linear_error as E
from tests.test_gpu_linear_precision import run
from tests.test_linear_error import inputs

pytestmark = pytest.mark.gpu


# one CTA and eight for the parts, of tiles and of walks
@pytest.mark.parametrize("shape", [(3, 300, 1, 36), (80, 3400, 1, 8), (70, 9, 2, 33), (2500, 2, 1, 30), (2500, 2, 1, 300)], ids=str)
@pytest.mark.parametrize("function", ["leaky", "lstm"])
def test_of_the_recurrence(function, shape, cuda_device):
    from flashrnn_b200 import _lib

    B, T, N, D = shape
    wx, b, s, n, dh, dl = inputs(function, "plain", *shape, seed=21)
    if n is None:
        n = torch.randint(T + 1, (B,), generator=torch.Generator().manual_seed(5))
    got = run(function, wx, b, s, n, dh, dl, cuda_device, torch.float32)
    plan = _lib.linear_plan(function, *shape)
    walk = plan.tile_steps == 8
    rows, columns = B * plan.tiles, plan.gates * N * D
    splits = 8 if rows >= 2048 and columns <= 1024 else 1
    in_part = T // 8 + 9 if walk else 16 + 5 + 8       # groups of eight steps; a thread's steps, lanes, warps
    # rows of terms in the order of the parts
    terms = got["d_wx"].flatten(0, 1)
    S.check(got["d_b"], terms, S.depth(rows, in_part, splits), -(-B // splits) * T if splits > 1 else None)
    E.check(got, E.evaluate(wx, b, s, function, n, dh, dl))
    half = run(function, wx.bfloat16(), b, s, n, dh.bfloat16(), dl, cuda_device, torch.bfloat16)
    E.check(half, E.evaluate(wx.bfloat16(), b, s, function, n, dh.bfloat16(), dl))


# 64 rows to a part: 3, 2049 and, over more columns than the eight CTAs take, 2049 again
@pytest.mark.parametrize("shape", [(130, 40), (131109, 40), (131109, 1032)], ids=str)
@pytest.mark.parametrize("bias", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("activation", [None, "relu"])
def test_of_the_product(activation, bias, shape, cuda_device):
    """Without an activation the terms are dy, behind a relu those of them whose result is not zero."""
    from flashrnn_b200 import fused_projection

    rows, outputs = shape
    g = torch.Generator(device=cuda_device).manual_seed(3)
    randn = lambda *size: torch.randn(size, generator=g, device=cuda_device)  # noqa: E731
    x, w, dy = randn(rows, 16).bfloat16(), (randn(outputs, 16) / 4).bfloat16(), randn(rows, outputs).bfloat16()
    b = randn(outputs).to(bias).requires_grad_(True)
    y = fused_projection(x, w, b, activation)
    d, = torch.autograd.grad(y, b, dy)
    terms = dy if activation is None else torch.where(y > 0, dy, 0)
    parts = -(-rows // 64)
    splits = 8 if parts >= 2048 and outputs <= 1024 else 1
    S.check(d, terms, S.depth(parts, 8 + 8, splits), -(-parts // splits) * 64 if splits > 1 else None)
