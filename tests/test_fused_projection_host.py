"""fused_projection on the host: what it refuses, and its plan."""

import pytest
import torch

from flashrnn_b200 import _lib, fused_projection


def test_refusals():
    x, w, b, r = torch.zeros((2, 3, 16)), torch.zeros((24, 16)), torch.zeros(24), torch.zeros((2, 3, 24))
    bad = [
        ("Unknown activation", dict(activation="gelu")),
        (r"x \[..., I\] and weight", dict(weight=w.t())),
        (r"x \[..., I\] and weight", dict(weight=w[0])),
        (r"x \[..., I\] and weight", dict(x=torch.zeros(()))),
        ("must be positive", dict(x=x[:, :0], residual=None)),
        ("must be positive", dict(weight=w[:0], bias=None, residual=None)),
        (r"bias \[J\]", dict(bias=b[:8])),
        (r"bias \[J\]", dict(bias=b[None])),
        (r"residual \[..., J\]", dict(residual=r[:1])),
        (r"residual \[..., J\]", dict(residual=r.flatten(0, 1))),
        ("floating-point", dict(weight=w.int())),
        ("same device", dict(bias=b.to("meta"))),
        ("strided", dict(residual=r.to_sparse())),
    ]
    for message, change in bad:
        with pytest.raises(ValueError, match=message):
            fused_projection(**{"x": x, "weight": w, "bias": b, "residual": r, **change})
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        fused_projection(x, w, b, "silu", r)


def test_plan():
    big = _lib.product_plan(32768, 4096, 2048, -1)
    assert big.forward_work_bytes == 0 and big.dbpart_bytes > 0
    few = _lib.product_plan(300, 256, 8192, -1)            # two tiles and a long sum: cut into parts
    assert few.forward_work_bytes >= 2 * 4 * 300 * 256 and few.forward_waits
    assert not _lib.product_plan(16, 8192, 8192, -1).forward_waits and not _lib.product_plan(256, 1024, 1024, -1).forward_waits
    assert _lib.product_plan(257, 1024, 1024, -1).forward_waits and _lib.product_plan(17, 4096, 4096, -1).forward_waits
    tall = _lib.product_plan(9000, 24, 72, -1)             # dW has one tile and sums 9000 rows
    assert tall.backward_work_bytes >= 2 * 4 * 24 * 72
    lib, out = _lib.load(), _lib.ProductPlan()
    for a, rc in (((0, 8, 8), -5), ((8, 0, 8), -5), ((8, 8, -8), -5), ((8, 12, 8), -2), ((8, 8, 20), -2), ((2 ** 31, 8, 8), -2)):
        assert lib.frnn_b200_product_plan(*a, out) == rc, a


@pytest.mark.skipif(torch.cuda.is_available(), reason="calls with pointers to nothing")
def test_c_entries_refuse_before_any_launch():
    lib = _lib.load()
    f = lambda x=16, w=16, bias=16, y=16, act=1, M=8, J=8, I=8, err=16: lib.frnn_b200_product_forward(  # noqa: E731
        x, w, bias, 1, None, act, y, None, M, J, I, None, err, None)
    assert f(x=None) == f(w=None) == f(y=None) == f(err=None, M=300) == f(act=4) == f(M=0) == f(x=8) == f(bias=4) == f(y=24) == -5
    assert f(J=12) == f(I=4) == f(M=1 << 31) == -2
    g = lambda dy=16, z=16, x=16, w=16, act=1, dz=16, dx=16, part=16, I=8: lib.frnn_b200_product_backward(  # noqa: E731
        dy, z, x, w, act, dz, dx, 16, 16, 1, part, 8, 8, I, None, 16, None)
    assert g(dy=None) == g(z=None) == g(dz=None) == g(x=None) == g(w=None) == g(part=None) == g(act=-1) == g(dx=8) == -5
    assert g(I=9) == -2
