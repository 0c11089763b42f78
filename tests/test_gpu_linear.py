"""flashrnn_linear against the recurrence in 64 bits: values, gradients, padding, strides, streams, graphs."""

import pytest
import torch

from tests import _linear_reference as L

pytestmark = pytest.mark.gpu

B16, F32 = torch.bfloat16, torch.float32


def make(function, B, T, N, D, dtype, seed, device, states=True, lengths=None, forget=6.0):
    g = torch.Generator().manual_seed(seed)
    G = L.GATES[function]
    wx = torch.randn((B, T, G, N, D), generator=g).to(dtype)
    b = torch.randn((G, N, D), generator=g) * 0.1
    b[0 if function == "leaky" else 1] = torch.rand((N, D), generator=g) * forget
    s = torch.randn((1, B, 1, N, D), generator=g) * 0.5 if states else None
    dh, dl = torch.randn((B, T, N, D), generator=g).to(dtype), torch.randn((1, B, 1, N, D), generator=g)
    n = None
    if lengths == "ragged":
        n = (torch.rand(B, generator=g) * (T + 1)).to(torch.int32)
        n[B // 2] = 0
        n[0] = T
    return [None if t is None else t.to(device) for t in (wx, b, s, n, dh, dl)]


def step(function, wx, b, s, n, dh, dl):
    from flashrnn_b200 import flashrnn_linear

    leaves = [t.detach().requires_grad_(True) for t in (wx, b, s) if t is not None]   # strides and alignment as they are
    hidden, last = flashrnn_linear(leaves[0], leaves[1], leaves[2] if s is not None else None, function, n)
    outs, grads = ([hidden, last], [dh, dl]) if dl is not None else ([hidden], [dh])
    d = torch.autograd.grad(outs, leaves, grads)
    return {"hidden": hidden, "last": last, **dict(zip(("d_wx", "d_b", "d_states"), d))}


# one step; less than, exactly and just over a span of four or eight, a tile of 128; channels that end inside a block of 64 or
# 32; widths that are no multiple of four; two tiles and more; more than one group of 16 tiles
SHAPES = [(1, 1, 1, 1), (4, 1, 3, 256), (2, 3, 1, 7), (3, 4, 1, 64), (2, 5, 2, 34), (2, 9, 1, 33), (3, 17, 1, 68), (2, 18, 1, 31),
          (2, 33, 1, 130), (1, 64, 1, 72), (2, 127, 1, 20),
          (2, 128, 1, 65), (2, 129, 2, 32), (3, 300, 1, 36), (1, 385, 1, 5), (1, 2048, 1, 4), (1, 2049, 1, 3), (2, 4500, 1, 8)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [B16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("function", ["leaky", "lstm"])
def test_values_and_gradients(function, dtype, shape, cuda_device):
    from flashrnn_b200 import poll_errors

    B, T, N, D = shape
    odd = (B + T + D) % 2 == 1            # with and without a first state, a gradient of the last, padding
    wx, b, s, n, dh, dl = make(function, *shape, dtype, T + D, cuda_device, states=not odd, lengths="ragged" if B > 1 and odd else None)
    dl = dl if T % 3 else None
    ref = L.run_reference(wx, b, s, function, n, dh, dl)
    got = step(function, wx, b, s, n, dh, dl)
    torch.cuda.synchronize()
    poll_errors(block=True)
    assert got["hidden"].dtype == dtype and got["last"].dtype == F32 and got["last"].shape == (1, B, 1, N, D)
    L.check(got, ref, L.bounds(ref, wx, b, s, T, dh, dl))


# so many channels that a thread walks the whole sequence: even and odd widths, lengths around the 8 and 16 steps that it has on
# their way
@pytest.mark.parametrize("shape", [(512, 1, 1, 128), (512, 7, 2, 64), (512, 8, 1, 128), (256, 9, 2, 129), (200, 17, 1, 330), (410, 41, 5, 33),
                                   (1100, 25, 1, 30), (512, 19, 1, 256)], ids=str)
@pytest.mark.parametrize("dtype", [B16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("function", ["leaky", "lstm"])
def test_many_channels(function, dtype, shape, cuda_device):
    from flashrnn_b200 import _lib

    B, T, N, D = shape
    assert _lib.linear_plan(function, *shape).exchange_bytes == 0 and _lib.linear_plan(function, *shape).tile_steps == 8
    wx, b, s, n, dh, dl = make(function, *shape, dtype, T + D, cuda_device, states=T % 3 > 0, lengths="ragged" if T % 2 else None)
    got = step(function, wx, b, s, n, dh, dl)
    ref = L.run_reference(wx, b, s, function, n, dh, dl)
    L.check(got, ref, L.bounds(ref, wx, b, s, T, dh, dl))


# so many rows and tiles that the parts of db are summed by several CTAs
@pytest.mark.parametrize("shape", [(2500, 2, 1, 30), (80, 3400, 1, 8)], ids=str)
@pytest.mark.parametrize("function", ["leaky", "lstm"])
def test_many_parts_of_db(function, shape, cuda_device):
    from flashrnn_b200 import _lib

    B, T, N, D = shape
    assert _lib.linear_plan(function, *shape).dbpart_bytes >= 4 * 2048 * L.GATES[function] * N * D
    wx, b, s, n, dh, dl = make(function, *shape, B16, 21, cuda_device, lengths="ragged")
    got = step(function, wx, b, s, n, dh, dl)
    ref = L.run_reference(wx, b, s, function, n, dh, dl)
    L.check(got, ref, L.bounds(ref, wx, b, s, T, dh, dl))


@pytest.mark.parametrize("function", ["leaky", "lstm"])
@pytest.mark.parametrize("T", [7, 130, 2100])
def test_padding_is_never_read(function, T, cuda_device):
    """What lies behind a row's end, NaN and infinities in this case, reaches no result; an empty row hands its state through."""
    wx, b, s, n, dh, dl = make(function, 5, T, 1, 24, B16, 3, cuda_device, lengths="ragged")
    n[1], n[3] = T + 9, -2               # clamped
    lens = n.clamp(0, T)
    behind = torch.arange(T, device=cuda_device) >= lens[:, None]
    clean = step(function, wx, b, s, lens.long(), dh, dl)
    for bad in (float("nan"), float("inf"), torch.finfo(B16).min):
        wx2, dh2 = wx.clone(), dh.clone()
        wx2[behind], dh2[behind] = bad, bad
        got = step(function, wx2, b, s, n, dh2, dl)
        for key in clean:
            assert torch.equal(got[key], clean[key]), (bad, key)
    assert (clean["hidden"][behind] == 0).all() and (clean["d_wx"][behind] == 0).all()
    empty = (lens == 0).nonzero().flatten()
    assert len(empty) >= 2
    assert torch.equal(clean["last"][:, empty], s[:, empty]) and torch.equal(clean["d_states"][:, empty], dl[:, empty])


@pytest.mark.parametrize("function", ["leaky", "lstm"])
def test_infinite_and_extreme_gates(function, cuda_device):
    """Gates at either end of their range: a state kept for good, one that is replaced in every step, a NaN that stays in its channel."""
    from flashrnn_b200 import flashrnn_linear

    wx, b, s, _, _, _ = make(function, 2, 300, 1, 16, F32, 4, cuda_device)
    f = 0 if function == "leaky" else 1
    b.zero_()
    wx[:, :, f, :, 0], wx[:, :, f, :, 1] = float("inf"), -float("inf")
    wx[:, :, f, :, 2], wx[:, :, f, :, 3] = 1e30, -1e30
    wx[0, 150, f, 0, 5] = float("nan")
    if function == "lstm":
        wx[:, :, 0, :, 0] = wx[:, :, 0, :, 2] = -float("inf")
    h, last = flashrnn_linear(wx, b, s, function)
    for keeps in (0, 2):
        assert torch.equal(last[..., keeps], s[..., keeps])
    z = wx[:, -1, 1, 0] if function == "leaky" else torch.sigmoid(wx[:, -1, 0, 0]) * torch.tanh(wx[:, -1, 2, 0])
    for forgets in (1, 3):
        assert torch.allclose(last[0, :, 0, 0, forgets], z[:, forgets], rtol=2.0 ** -20, atol=2.0 ** -22)
    assert torch.isnan(last[0, 0, 0, 0, 5]) and torch.isfinite(h[0, :150]).all()
    ok = torch.ones_like(last, dtype=torch.bool)
    ok[0, 0, 0, 0, 5] = False
    assert torch.isfinite(last[ok]).all() and torch.isnan(h[0, 150:, 0, 5]).all()


@pytest.mark.parametrize("cut", [1, 128, 200])
def test_pieces_make_a_whole(cut, cuda_device):
    """A sequence in two calls, the state handed on, gives the values and gradients of one call, up to where sums are cut."""
    from flashrnn_b200 import flashrnn_linear

    wx, b, s, _, dh, dl = make("lstm", 2, 300, 2, 20, F32, 8, cuda_device)
    whole = step("lstm", wx, b, s, None, dh, dl)
    leaves = [t.clone().requires_grad_(True) for t in (wx, b, s)]
    h1, c1 = flashrnn_linear(leaves[0][:, :cut], leaves[1], leaves[2], "lstm")
    h2, c2 = flashrnn_linear(leaves[0][:, cut:], leaves[1], c1, "lstm")
    d = torch.autograd.grad([torch.cat((h1, h2), 1), c2], leaves, [dh, dl])
    got = {"hidden": torch.cat((h1, h2), 1), "last": c2, **dict(zip(("d_wx", "d_b", "d_states"), d))}
    ref = {k: v.detach().cpu().double() for k, v in whole.items()}
    limits = {k: 2 * v for k, v in L.bounds(ref, wx, b, s, 300, dh, dl).items()}   # both sides are off
    L.check(got, ref, limits)


def test_it_is_the_lstm_without_its_recurrent_matrix(cuda_device):
    from flashrnn_b200 import flashrnn, flashrnn_linear

    wx, b, s, _, _, _ = make("lstm", 4, 60, 2, 32, F32, 5, cuda_device, forget=2.0)
    hidden, last = flashrnn_linear(wx, b, s, "lstm")
    both = torch.cat((torch.zeros_like(s), s))
    ref, ref_last = flashrnn(wx, torch.zeros((4, 2, 32, 32), device=cuda_device), b, both, "lstm", dtype="float32")
    # those cells' tanh.approx is good to 2^-10.9, four of them in a step, a forget gate of sigmoid(2) adds up over 8 steps
    assert (hidden - ref[0]).abs().max() < 8 * 4 * 2.0 ** -10.9 and (last - ref_last[1:]).abs().max() < 8 * 4 * 2.0 ** -10.9


@pytest.mark.parametrize("T", [1, 100, 700, 3000])
@pytest.mark.parametrize("B", [6, 400])
@pytest.mark.parametrize("function", ["leaky", "lstm"])
def test_same_bits_every_time(function, B, T, cuda_device):
    wx, b, s, n, dh, dl = make(function, B, min(T, 100000 // B), 3, 100, B16, 6, cuda_device, lengths="ragged")
    first = step(function, wx, b, s, n, dh, dl)
    for _ in range(5):
        again = step(function, wx, b, s, n, dh, dl)
        assert all(torch.equal(first[k], again[k]) for k in first)


def test_strides_offsets_and_other_types(cuda_device):
    from flashrnn_b200 import flashrnn_linear

    wx, b, s, n, dh, dl = make("leaky", 3, 140, 2, 20, B16, 7, cuda_device, lengths="ragged")
    want = step("leaky", wx, b, s, n, dh, dl)
    turned = wx.permute(1, 0, 4, 3, 2).contiguous().permute(1, 0, 4, 3, 2)
    odd = torch.empty(wx.numel() + 1, dtype=B16, device=cuda_device)[1:].view_as(wx).copy_(wx)
    every = torch.stack((wx, wx), -1)[..., 0]
    assert odd.data_ptr() % 16
    long = torch.stack((n, n), 1).long()[:, 0]
    for other in (turned, odd, every):
        got = step("leaky", other, b, s, long, dh.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3), dl)
        assert all(torch.equal(got[k], want[k]) for k in want)
    # a gradient that broadcasts, as a sum hands it back, and parameters of another type
    leaves = [wx.clone().requires_grad_(True), b.to(B16).requires_grad_(True), s.to(B16).requires_grad_(True)]
    h, c = flashrnn_linear(leaves[0], leaves[1], leaves[2], "leaky", n)
    (h.sum() + c.sum()).backward()
    ones = step("leaky", wx, b.to(B16).float(), s.to(B16).float(), n, torch.ones_like(dh), torch.ones_like(dl))
    assert torch.equal(leaves[0].grad, ones["d_wx"]) and leaves[1].grad.dtype == B16 and leaves[2].grad.dtype == B16
    assert torch.equal(leaves[1].grad, ones["d_b"].to(B16)) and torch.equal(leaves[2].grad, ones["d_states"].to(B16))
    # one output used, the other not
    w = wx.clone().requires_grad_(True)
    flashrnn_linear(w, b, s, "leaky", n)[1].backward(dl)
    only = step("leaky", wx, b, s, n, torch.zeros_like(dh), dl)
    assert torch.equal(w.grad, only["d_wx"])
    with pytest.raises(RuntimeError):                      # no second derivatives, and no silent zeros in their place
        w = wx.clone().requires_grad_(True)
        g, = torch.autograd.grad(flashrnn_linear(w, b, s, "leaky", n)[0].float().sum(), w, create_graph=True)
        g.float().sum().backward()


@pytest.mark.parametrize("shape", [(3, 140, 2, 20), (2, 5, 1, 24), (500, 20, 1, 140)], ids=str)
def test_every_tensor_may_start_anywhere(shape, cuda_device):
    """Contiguous views that start four bytes behind a vector's boundary."""
    from flashrnn_b200 import flashrnn_linear

    def moved(t):
        out = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view_as(t)
        assert out.data_ptr() % 8 and out.is_contiguous()
        return out.copy_(t)

    wx, b, s, n, dh, dl = make("leaky", *shape, F32, 7, cuda_device, lengths="ragged")
    want = step("leaky", wx, b, s, n, dh, dl)
    got = step("leaky", *(moved(t) for t in (wx, b, s, n, dh, dl)))
    assert all(torch.equal(got[k], want[k]) for k in want)
    last, first = moved(s), moved(s)
    with torch.no_grad():
        assert flashrnn_linear(wx, b, first, "leaky", n, last_out=last)[1] is last and torch.equal(last, want["last"])
        flashrnn_linear(wx, b, first, "leaky", n, last_out=first)
    assert torch.equal(first, want["last"])


@pytest.mark.parametrize("T", [1, 60, 400])
def test_last_out_in_place_and_on_another_stream(T, cuda_device):
    from flashrnn_b200 import flashrnn_linear

    wx, b, s, _, _, _ = make("lstm", 4, T, 2, 40, B16, 9, cuda_device)
    hidden, last = flashrnn_linear(wx, b, s, "lstm")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    state = s.clone()
    torch.cuda.current_stream().synchronize()
    with torch.cuda.stream(side), torch.no_grad():
        h, out = flashrnn_linear(wx, b, state, "lstm", last_out=state)
    side.synchronize()
    assert out is state and torch.equal(state, last) and torch.equal(h, hidden)
    room = torch.cat((s.flatten(), s.flatten()))          # a view that overlaps the states without being them
    shifted, views = room[8:8 + s.numel()].view_as(s), room[:s.numel()].view_as(s)
    want = views.clone()
    _, w = flashrnn_linear(wx, b, want, "lstm")
    with torch.no_grad():
        flashrnn_linear(wx, b, views, "lstm", last_out=shifted)
    assert torch.equal(shifted, w)


def test_captured_decoding_and_training(cuda_device):
    """A decoding step that updates its state in place and a training step of a longer sequence, replayed from graphs on new data."""
    from flashrnn_b200 import flashrnn_linear, poll_errors

    wx, b, s, _, _, _ = make("leaky", 4, 8, 2, 32, B16, 10, cuda_device)
    want, end = flashrnn_linear(wx, b, s, "leaky")
    token, state = wx[:, :1].clone(), s.clone()
    side = torch.cuda.Stream()
    with torch.no_grad(), torch.cuda.stream(side):
        flashrnn_linear(token, b, state.clone(), "leaky")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            h, _ = flashrnn_linear(token, b, state, "leaky", last_out=state)
    torch.cuda.synchronize()
    state.copy_(s)
    for t in range(8):
        token.copy_(wx[:, t:t + 1])
        graph.replay()
        # a step at a time rounds states in other places than a tile of eight: (T 2^-23 + 2^-19) of the inputs, half a step of bf16
        assert ((h[:, 0] - want[:, t]).abs().float() <= 2.0 ** -7 * want[:, t].abs().float() + 1e-4).all()
    assert (state - end).abs().max() < 1e-4

    shapes = ("leaky", 3, 700, 2, 40, B16)
    wx, b, s, n, dh, dl = make(*shapes, 11, cuda_device, lengths="ragged")
    leaves = [t.clone().requires_grad_(True) for t in (wx, b, s)]

    def train():
        hidden, last = flashrnn_linear(*leaves, "leaky", n)
        return (hidden, last, *torch.autograd.grad([hidden, last], leaves, [dh, dl]))

    with torch.cuda.stream(side):
        for _ in range(2):
            train()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = train()
    for seed in (12, 13):
        wx2, b2, s2, n2, dh2, dl2 = make(*shapes, seed, cuda_device, lengths="ragged")
        with torch.no_grad():
            for t, v in zip((*leaves, n, dh, dl), (wx2, b2, s2, n2, dh2, dl2)):
                t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        want = step("leaky", wx2, b2, s2, n2, dh2, dl2)
        assert all(torch.equal(a, w) for a, w in zip(out, want.values()))
    poll_errors(block=True)
    del graph


@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "bf16"])
def test_capture_beside_an_eager_graph(dtype, cuda_device):
    """Autograd runs a leaf's node on the stream of the oldest graph that lives: the default one, which a capture must not wait for."""
    from flashrnn_b200 import flashrnn_linear

    torch.manual_seed(20)
    leaves = [torch.randn(shape, device=cuda_device, dtype=dtype).requires_grad_(True) for shape in ((3, 300, 2, 1, 40), (2, 1, 40))]
    call = lambda: flashrnn_linear(*leaves)[0]  # noqa: E731
    out, graph = call(), torch.cuda.CUDAGraph()
    want = torch.autograd.grad(out.float().sum(), leaves, retain_graph=True)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="cannot capture this backward pass"), torch.cuda.graph(graph):
        torch.autograd.grad(call().float().sum(), leaves)
    out.float().sum().backward()   # the eager graph is as it was
    assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))
    del out, graph
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(call().float().sum(), leaves)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    del graph


def test_words_of_a_graph_that_was_never_replayed(cuda_device, monkeypatch):
    """Nothing has zeroed them: what lies there is no error, unless it is a kernel's code."""
    from flashrnn_b200 import flashrnn_linear, functional, poll_errors

    words = []
    monkeypatch.setattr(functional, "_captured_errors", words)
    wx, b, s, _, _, _ = make("leaky", 2, 300, 1, 40, B16, 22, cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        flashrnn_linear(wx, b, s, "leaky")
    assert len(words) == 1
    for left_there in (-1, 1065353216):
        words[0][0].fill_(left_there)
        poll_errors(block=True)
    words[0][0][0] = 106
    with pytest.raises(RuntimeError, match="replayed CUDA graph"):
        poll_errors(block=True)
    graph.replay()                     # zeroes it
    poll_errors(block=True)
    del graph


@pytest.mark.parametrize("mute", [0, 1, 7])
@pytest.mark.parametrize("backward", [False, True], ids=["forward", "backward"])
def test_a_wait_that_runs_out_is_reported(backward, mute, cuda_device):
    """Tiles that hand nothing out (7: the state between two groups): the call ends within its limit, says so, and the next one is right."""
    from flashrnn_b200 import _lib

    B, T, N, D = 2, 1300, 1, 64
    wx, b, s, _, dh, dl = make("leaky", B, T, N, D, B16, 14, cuda_device)
    want = step("leaky", wx, b, s, None, dh, dl)
    lib, plan = _lib.load(), _lib.linear_plan("leaky", B, T, N, D)
    assert plan.tiles > 9
    exchange, err = torch.empty(plan.exchange_bytes, dtype=torch.uint8, device=cuda_device), torch.zeros(32, dtype=torch.int32, device=cuda_device)
    starts, part = torch.zeros(plan.starts_bytes // 4, device=cuda_device), torch.zeros(plan.dbpart_bytes // 4, device=cuda_device)
    out, last, db, d_init = torch.empty_like(dh), torch.empty_like(s), torch.empty_like(b), torch.empty_like(s)
    d_wx = torch.empty_like(wx)

    def call():
        stream = torch.cuda.current_stream().cuda_stream
        rc = lib.frnn_b200_linear_forward(0, wx.data_ptr(), 1, b.data_ptr(), s.data_ptr(), None, out.data_ptr(), last.data_ptr(),
                                          starts.data_ptr(), exchange.data_ptr(), B, T, N, D, 30, (clean if backward else err).data_ptr(), stream)
        if rc == 0 and backward:
            rc = lib.frnn_b200_linear_backward(0, wx.data_ptr(), 1, b.data_ptr(), s.data_ptr(), None, starts.data_ptr(), dh.data_ptr(),
                                               dl.data_ptr(), d_wx.data_ptr(), db.data_ptr(), d_init.data_ptr(), part.data_ptr(),
                                               exchange.data_ptr(), B, T, N, D, 30, err.data_ptr(), stream)
        assert rc == 0
        torch.cuda.synchronize()

    clean = torch.zeros_like(err)
    err[4], err[5] = 1, mute
    call()
    assert err[0].item() == 106 and clean[0].item() == 0
    err.zero_()
    call()
    assert err[0].item() == 0 and torch.equal(out, want["hidden"]) and torch.equal(last, want["last"])
    if backward:
        assert torch.equal(d_wx, want["d_wx"]) and torch.equal(db, want["d_b"]) and torch.equal(d_init, want["d_states"])


def test_offsets_past_32_bits(cuda_device):
    """More than 2^32 bytes and 2^31 elements of Wx: the far end of the sequence is that of a call of its own."""
    from flashrnn_b200 import flashrnn_linear

    B, T, N, D, tail = 2, 33000, 16, 1040, 300
    assert B * T * 2 * N * D > 2 ** 31
    g = torch.Generator(device=cuda_device).manual_seed(0)
    wx = torch.randn((B, T, 2, N, D), generator=g, device=cuda_device, dtype=B16)
    b = torch.zeros((2, N, D), device=cuda_device)
    s = torch.ones((1, B, 1, N, D), device=cuda_device)
    leaf = wx.requires_grad_(True)
    hidden, last = flashrnn_linear(leaf, b, s, "leaky")
    end = wx.detach()[:, T - tail:].contiguous().requires_grad_(True)
    h, c = flashrnn_linear(end, b, None, "leaky")        # sigmoid of a normal variable forgets a state within 100 steps for good
    assert torch.equal(h[:, 150:], hidden[:, T - 150:]) or (h[:, 150:] - hidden[:, T - 150:]).abs().max() <= 2.0 ** -7 * h.abs().max()
    assert (c - last).abs().max() < 1e-5
    dh = torch.zeros_like(hidden)
    dh[:, T - 100:] = 1
    d, = torch.autograd.grad(hidden, leaf, dh)
    d_end, = torch.autograd.grad(h, end, dh[:, T - tail:])
    assert (d[:, T - 150:] - d_end[:, 150:]).abs().max() <= 2.0 ** -7 * d_end.abs().max() and d[:, T - 150:].abs().max() > 0
    assert d[:, :16000].abs().max() == 0
