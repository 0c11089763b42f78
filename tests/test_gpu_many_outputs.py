"""A product of more outputs than one dimension of a grid has blocks for: its backward call takes what its forward call took."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("activation", [None, "relu"])
def test_gradients(activation, cuda_device):
    """Two rows of integers: sums are exact, each result is rounded once."""
    from flashrnn_b200 import fused_projection

    rows, inputs, outputs = 2, 8, 65535 * 256 + 264
    g = torch.Generator(device=cuda_device).manual_seed(0)
    ints = lambda *size: torch.randint(-3, 4, size, generator=g, device=cuda_device).bfloat16()  # noqa: E731
    x, w, b, dy = (ints(*s).requires_grad_(True) for s in ((rows, inputs), (outputs, inputs), (outputs,), (rows, outputs)))
    y = fused_projection(x, w, b, activation)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy.detach())
    with torch.no_grad():
        z = x.float() @ w.float().t() + b.float()
        dz = dy.float() if activation is None else torch.where(z > 0, dy.float(), 0)
        assert torch.equal(y, (z if activation is None else z.clamp(min=0)).bfloat16())
        assert torch.equal(dw, (dz.t() @ x.float()).bfloat16()) and torch.equal(db, dz.sum(0).bfloat16())
        want = dz.double() @ w.double()      # fp32 sums stay exact below 2^24
        assert want.abs().max() < 2 ** 24 and torch.equal(dx, want.float().bfloat16())
