"""A product whose waits run out: the call ends, reports it, and the next one is right. With err[4] = 1 nothing is multiplied; every wait
is bounded."""

import pytest
import torch

from tests.test_gpu_fused_projection import make, step

pytestmark = pytest.mark.gpu

CODES = (102, 103, 104, 105)


# rows, inputs, outputs: whole tiles; tiles cut along the inputs; more tiles than pairs of CTAs
@pytest.mark.parametrize("shape", [(600, 512, 512), (300, 8192, 256), (9000, 128, 1024)], ids=str)
@pytest.mark.parametrize("direction", ["forward", "backward"])
def test_through_the_c_entries(direction, shape, cuda_device):
    from flashrnn_b200 import _lib

    M, I, J = shape
    x, w, b, r, dy = make(M, I, J, 3, cuda_device, bias=torch.bfloat16, residual=True)
    want = step(x, w, b, r, dy, "silu")
    lib, plan = _lib.load(), _lib.product_plan(M, J, I, 0)
    assert plan.forward_waits
    floats = lambda n: torch.zeros(max(n, 16) // 4, device=cuda_device)  # noqa: E731
    work, part = floats(max(plan.forward_work_bytes, plan.backward_work_bytes)), floats(plan.dbpart_bytes)
    y, z, dz = torch.empty_like(dy), torch.zeros((M, J), dtype=torch.float16, device=cuda_device), torch.empty_like(dy)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    err, clean = (torch.zeros(32, dtype=torch.int32, device=cuda_device) for _ in range(2))

    def call():
        stream, act = torch.cuda.current_stream().cuda_stream, _lib.ACTIVATIONS["silu"]
        rc = lib.frnn_b200_product_forward(x.data_ptr(), w.data_ptr(), b.data_ptr(), 1, r.data_ptr(), act, y.data_ptr(), z.data_ptr(), M, J, I,
                                           work.data_ptr(), (err if direction == "forward" else clean).data_ptr(), stream)
        if rc == 0 and direction == "backward":
            rc = lib.frnn_b200_product_backward(dy.data_ptr(), z.data_ptr(), x.data_ptr(), w.data_ptr(), act, dz.data_ptr(), dx.data_ptr(),
                                                dw.data_ptr(), db.data_ptr(), 1, part.data_ptr(), M, J, I, work.data_ptr(), err.data_ptr(), stream)
        assert rc == 0
        torch.cuda.synchronize()

    err[4] = 1
    call()
    assert err[0].item() in CODES and clean[0].item() == 0
    err.zero_()
    call()
    assert err[0].item() == 0 and torch.equal(y, want["y"])
    if direction == "backward":
        assert torch.equal(dx, want["x"]) and torch.equal(dw, want["weight"]) and torch.equal(db, want["bias"])


def test_through_fused_projection(cuda_device, monkeypatch):
    from flashrnn_b200 import functional, fused_projection, poll_errors, projection

    x, w, b, _, _ = make(600, 512, 512, 4, cuda_device, bias=torch.bfloat16)
    poll_errors(block=True)
    want = fused_projection(x, w, b, "relu")
    word = torch.zeros(32, dtype=torch.int32, device=cuda_device)
    word[4] = 1
    monkeypatch.setattr(projection, "_launch_word", lambda device: (word.data_ptr(), word))
    monkeypatch.setattr(projection, "_launched", functional._track)
    fused_projection(x, w, b, "relu")
    monkeypatch.undo()
    with pytest.raises(RuntimeError, match=r"frnn_b200_product_forward: device-side wait ran out \(code 10[2-5]"):
        poll_errors(block=True)
    assert torch.equal(fused_projection(x, w, b, "relu"), want)
    poll_errors(block=True)
