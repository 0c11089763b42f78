"""fused_projection against the product in 64 bits: values and gradients, ragged sizes, strides, graphs."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

B16 = torch.bfloat16
ACTS = {None: lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu,
        "gelu_tanh": lambda z: 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))}
CURVE = {None: 0.0, "relu": 0.0, "silu": 0.5, "gelu_tanh": 1.2}   # largest second derivative, rounded up


def make(M, I, J, seed, device, bias=None, residual=False):
    g = torch.Generator().manual_seed(seed)
    x, w = torch.randn((M, I), generator=g).to(B16), (torch.randn((J, I), generator=g) * I ** -0.5).to(B16)
    b = torch.randn(J, generator=g).to(bias) if bias is not None else None
    r = torch.randn((M, J), generator=g).to(B16) if residual else None
    dy = torch.randn((M, J), generator=g).to(B16)
    return [None if t is None else t.to(device) for t in (x, w, b, r, dy)]


def reference(x, w, b, r, dy, act):
    """Results and gradients in 64 bits on the CPU, and the largest error of each before its last rounding.

    A product sums K terms in fp32, whatever the order: at most (K + 8) 2^-23 of the sum of the terms' sizes (a tensor core may cut
    what it adds instead of rounding it). An activation scales an error by at most 1.13 and adds 2^-19 of |z| of its own. The slope is
    taken at z rounded to 11 bits, dz rounded to 8: half a step each."""
    x, w, b, r, dy = [None if t is None else t.detach().cpu().double() for t in (x, w, b, r, dy)]
    leaves = [t.requires_grad_(True) for t in (x, w, b, r) if t is not None]
    z = x @ w.t()
    if b is not None:
        z = z + b
    y = ACTS[act](z)
    if r is not None:
        y = y + r
    names = [n for n, t in zip(("x", "weight", "bias", "residual"), (x, w, b, r)) if t is not None]
    ref = {"y": y.detach(), **dict(zip(names, torch.autograd.grad(y, leaves, dy)))}
    with torch.no_grad():
        zs = z.detach().requires_grad_(True)
        with torch.enable_grad():
            slope, = torch.autograd.grad(ACTS[act](zs).sum(), zs)
        K, eps = x.shape[1], 2.0 ** -23
        ez = (K + 8) * eps * (x.abs() @ w.abs().t() + (0 if b is None else b.abs()))
        lim = {"y": 1.13 * ez + 2.0 ** -19 * z.abs() + (0 if r is None else 2.0 ** -23 * (z.abs() + r.abs()))}
        if act is None:
            edz, unrounded = torch.zeros_like(z), torch.zeros_like(z)
        else:
            unrounded = dy.abs() * (CURVE[act] * (ez + 2.0 ** -11 * z.abs()) + 2.0 ** -19 * (1 + z.abs()))
            if act == "relu":
                unrounded = torch.where(z.abs() <= ez, dy.abs(), torch.zeros_like(z))
            edz = unrounded + 2.0 ** -8 * (dy * slope).abs() * 1.01
        dz = (dy * slope).abs() + edz
        M, J = z.shape
        lim["x"] = edz @ w.abs() + (J + 8) * eps * (dz @ w.abs())
        lim["weight"] = edz.t() @ x.abs() + (M + 8) * eps * (dz.t() @ x.abs())
        lim["bias"] = unrounded.sum(0) + (M + 8) * eps * dz.sum(0)
        lim["residual"] = torch.zeros(())
    return ref, lim


def step(x, w, b, r, dy, act):
    from flashrnn_b200 import fused_projection

    named = [(n, t.detach().requires_grad_(True)) for n, t in zip(("x", "weight", "bias", "residual"), (x, w, b, r)) if t is not None]
    leaf = dict(named)
    y = fused_projection(leaf["x"], leaf["weight"], leaf.get("bias"), act, leaf.get("residual"))
    return {"y": y, **dict(zip(leaf, torch.autograd.grad(y, list(leaf.values()), dy)))}


def check(got, ref, lim):
    for key, want in ref.items():
        t = got[key].detach().cpu()
        off = (t.double() - want).abs() - torch.finfo(t.dtype).eps / 2 * want.abs()
        # a result that is off before its rounding may fall on the other side of a step: the rounding is that of a value near `want`
        allowed = lim[key] * (1 + torch.finfo(t.dtype).eps) + torch.finfo(torch.float32).tiny
        assert torch.isfinite(t).all() and (off <= allowed).all(), (key, (off - allowed).max().item())


# one row; less than, exactly and just over tiles of 128 and 256; K shorter than a stage and no multiple of one; more tiles than the
# GPU holds; few tiles with a long K (cut into parts); features that are no multiple of eight
# (few rows take a kernel of their own: up to 8, 16, 32 and more to a CTA, K up to 1024 and longer, either side of where it ends)
SHAPES = [(8, 2048, 264), (16, 1104, 40), (33, 520, 48), (70, 1032, 88), (256, 1024, 1024), (257, 1024, 1024), (260, 520, 1016), (17, 4096, 4096), (1, 8, 8), (1, 768, 1536), (3, 40, 24), (16, 264, 72), (17, 64, 136), (31, 72, 40), (128, 64, 128), (129, 200, 136), (256, 64, 256),
          (257, 520, 264), (300, 2048, 200), (1000, 768, 768), (5000, 128, 2504), (9000, 72, 24), (20, 1032, 16), (5, 33, 17), (130, 1001, 259)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("act", list(ACTS), ids=str)
def test_values_and_gradients(act, shape, cuda_device):
    from flashrnn_b200 import poll_errors

    M, I, J = shape
    kind = (M + I + list(ACTS).index(act)) % 4
    args = make(M, I, J, M + J, cuda_device, bias=(None, B16, torch.float32, B16)[kind], residual=kind in (0, 3))
    got = step(*args, act)
    torch.cuda.synchronize()
    poll_errors(block=True)
    assert got["y"].dtype == B16 and got["y"].shape == (M, J)
    check(got, *reference(*args, act))
    from flashrnn_b200 import fused_projection

    with torch.no_grad():                                      # the same values where nothing is kept for a backward pass
        assert torch.equal(fused_projection(args[0], args[1], args[2], act, args[3]), got["y"])


@pytest.mark.parametrize("bias", [B16, torch.float32], ids=["bf16", "f32"])
def test_many_parts_of_dbias(bias, cuda_device):
    """So many rows that their parts of dbias are summed by several CTAs."""
    args = make(131109, 16, 40, 21, cuda_device, bias=bias)
    check(step(*args, "silu"), *reference(*args, "silu"))


def test_extreme_values(cuda_device):
    """Products past the range of fp16 keep their slopes, NaN and infinities stay in their rows."""
    from flashrnn_b200 import fused_projection

    x = torch.zeros((6, 8), device=cuda_device, dtype=B16)
    x[:, 0] = torch.tensor([1e6, -1e6, 1e-9, -1e-9, float("nan"), float("inf")], device=cuda_device)
    w = torch.zeros((8, 8), device=cuda_device, dtype=B16)
    w[0, 0] = 1
    for act in ("relu", "silu", "gelu_tanh"):
        xl = x.clone().requires_grad_(True)
        y = fused_projection(xl, w, None, act)
        dx, = torch.autograd.grad(y, xl, torch.ones_like(y))
        y, dx = y[:, 0].float().cpu(), dx[:, 0].float().cpu()
        half = 0.5 if act != "relu" else 1.0
        assert y[0] == x[0, 0].float().cpu() and y[1] == 0 and torch.isnan(y[4]) and y[5] == float("inf"), (act, y)
        assert dx[0] == 1 and dx[1] == 0 and abs(dx[2] - half) < 1e-2 and abs(dx[3] - (half if half < 1 else 0)) < 1e-2, (act, dx)
        if act != "relu":
            assert torch.isnan(dx[4])


def test_strides_types_and_unwanted_gradients(cuda_device):
    from flashrnn_b200 import fused_projection

    x, w, b, r, dy = make(96, 72, 56, 3, cuda_device, bias=B16, residual=True)
    want = step(x, w, b, r, dy, "silu")
    odd = torch.empty(x.numel() + 1, dtype=B16, device=cuda_device)[1:].view_as(x).copy_(x)
    pair = [torch.stack((t, t), -1)[..., 0] for t in (w, b, r, dy)]
    got = step(odd, *pair, "silu")
    assert all(torch.equal(got[k], want[k]) for k in want)
    got = step(x.t().contiguous().t(), w.t().contiguous().t(), b, r.t().contiguous().t(), dy.t().contiguous().t(), "silu")
    assert all(torch.equal(got[k], want[k]) for k in want)
    # leading dimensions of any number, none of them: a vector
    y = fused_projection(x.view(4, 8, 3, 72), w, b, "silu", r.view(4, 8, 3, 56))
    assert y.shape == (4, 8, 3, 56) and torch.equal(y.view(96, 56), want["y"])
    assert fused_projection(x[0], w, b, "silu", r[0]).shape == (56,)
    # fp32 parameters: operands rounded to bf16, gradients in fp32
    leaves = [t.float().requires_grad_(True) for t in (x, w, b, r)]
    y = fused_projection(leaves[0], leaves[1], leaves[2], "silu", leaves[3])
    d = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(y, want["y"]) and all(t.dtype == torch.float32 for t in d)
    assert torch.equal(d[0], want["x"].float()) and torch.equal(d[2].to(B16), want["bias"])
    # each gradient alone is what it is among the others
    for i, name in enumerate(("x", "weight", "bias", "residual")):
        args = [t.detach().clone() for t in (x, w, b, r)]
        args[i].requires_grad_(True)
        d, = torch.autograd.grad(fused_projection(args[0], args[1], args[2], "silu", args[3]), args[i], dy)
        assert torch.equal(d, want[name]), name
    # a gradient that broadcasts
    xl = x.clone().requires_grad_(True)
    fused_projection(xl, w).sum().backward()
    assert torch.equal(xl.grad, step(x, w, None, None, torch.ones_like(dy), None)["x"])


@pytest.mark.parametrize("J", [24, 25])
def test_the_result_is_dense_and_may_be_changed(J, cuda_device):
    from flashrnn_b200 import fused_projection

    x, w, _, _, dy = make(40, 33, J, 4, cuda_device)
    leaf = x.clone().requires_grad_(True)
    y = fused_projection(leaf, w)
    assert y.is_contiguous() and y.view(5, 8, J).shape == (5, 8, J)
    y += 1
    d, = torch.autograd.grad(y, leaf, dy)
    with torch.no_grad():
        assert torch.equal(fused_projection(x, w) + 1, y) and fused_projection(x, w).is_contiguous()
    assert torch.equal(d, step(x, w, None, None, dy, None)["x"])


@pytest.mark.parametrize("shape", [(300, 2048, 200), (5000, 128, 2504), (2, 768, 768)], ids=str)
def test_same_bits_every_time(shape, cuda_device):
    args = make(*shape, 5, cuda_device, bias=torch.float32, residual=True)
    first = step(*args, "gelu_tanh")
    for _ in range(5):
        again = step(*args, "gelu_tanh")
        assert all(torch.equal(first[k], again[k]) for k in first)


def test_captured_training_step(cuda_device):
    from flashrnn_b200 import fused_projection, poll_errors

    shape = (300, 520, 264)
    x, w, b, r, dy = make(*shape, 6, cuda_device, bias=B16, residual=True)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]

    def train():
        y = fused_projection(leaves[0], leaves[1], leaves[2], "silu", leaves[3])
        return (y, *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        train()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = train()
    for seed in (7, 8):
        new = make(*shape, seed, cuda_device, bias=B16, residual=True)
        with torch.no_grad():
            for t, v in zip((*leaves, dy), new):
                t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, v) for a, v in zip(out, step(*new, "silu").values()))
    poll_errors(block=True)
    del graph


@pytest.mark.parametrize("dtype", [B16, torch.float32], ids=["bf16", "f32"])
def test_capture_beside_an_eager_graph(dtype, cuda_device):
    """Autograd runs a leaf's node on the stream of the oldest graph that lives: the default one, which a capture must not wait for."""
    from flashrnn_b200 import fused_projection

    torch.manual_seed(20)
    leaves = [torch.randn(shape, device=cuda_device, dtype=dtype).requires_grad_(True) for shape in ((70, 136), (264, 136), (264,))]
    call = lambda: fused_projection(*leaves, "silu")  # noqa: E731
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


@pytest.mark.parametrize("function", ["leaky", "lstm"])
def test_a_layer(function, cuda_device):
    """Product into the gates, recurrence, product back into the residual stream: a layer's values and all of its gradients."""
    from flashrnn_b200 import flashrnn_linear, fused_projection, poll_errors
    from tests import _linear_reference as L

    B, T, I, N, D = 3, 150, 40, 2, 24
    G = L.GATES[function]
    g = torch.Generator().manual_seed(9)
    rand = lambda *s, scale=1.0: torch.randn(s, generator=g) * scale  # noqa: E731
    p = {"x": rand(B, T, I).to(B16), "w_in": rand(G * N * D, I, scale=I ** -0.5).to(B16), "b": rand(G, N, D), "s": rand(1, B, 1, N, D),
         "w_out": rand(I, N * D, scale=(N * D) ** -0.5).to(B16)}
    dy = rand(B, T, I).to(B16)
    leaf = {k: v.to(cuda_device).requires_grad_(True) for k, v in p.items()}
    gates = fused_projection(leaf["x"], leaf["w_in"]).view(B, T, G, N, D)
    hidden, _ = flashrnn_linear(gates, leaf["b"], leaf["s"], function)
    y = fused_projection(hidden.view(B, T, N * D), leaf["w_out"], residual=leaf["x"])
    got = dict(zip(leaf, torch.autograd.grad(y, list(leaf.values()), dy.to(cuda_device))))
    poll_errors(block=True)
    ref = {k: v.double().requires_grad_(True) for k, v in p.items()}
    h, _ = L.reference((ref["x"] @ ref["w_in"].t()).view(B, T, G, N, D), ref["b"], ref["s"], function)
    want_y = h.reshape(B, T, N * D) @ ref["w_out"].t() + ref["x"]
    want = dict(zip(ref, torch.autograd.grad(want_y, list(ref.values()), dy.double())))
    # gates, hidden states and their gradients are rounded to bf16 between the operators: five roundings of half a step, relative to
    # the size of what is rounded, in root-mean-square terms no more than their sum
    for key, w in {"y": want_y.detach(), **want}.items():
        t = (y if key == "y" else got[key]).detach().cpu().double()
        assert (t - w).norm() <= 5 * 2.0 ** -8 * w.norm(), (key, ((t - w).norm() / w.norm()).item())
