"""mx.linear and mx.swiglu: forward and backward against float64, and as they are used together."""
import numpy as np
import pytest
import torch

import mx_plain as P

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]

LINEAR = [(P.E4M3, P.E4M3), (P.E4M3, P.E5M2), (P.E2M1, P.E4M3), (P.E2M1, P.E5M2)]


def randn(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(torch.bfloat16)


def leaf(t):
    return t.cuda().requires_grad_()


def linear_forms(x, w, dy, fmt, grad_fmt):
    """[(exact, bound)] of y, dx, dw in float64"""
    q = P.quantized_values
    return [P.product_bound(q(x, fmt), q(w, fmt)), P.product_bound(q(dy, grad_fmt), q(w.T, fmt)),
            P.product_bound(q(dy.T, grad_fmt), q(x.T, P.E4M3))]


@pytest.mark.parametrize("fmts", LINEAR, ids=str)
@pytest.mark.parametrize("shape", [(1, 32, 32), (31, 64, 96), (32, 96, 64), (33, 160, 128), (77, 1056, 992), (300, 256, 544)], ids=str)
def test_linear(shape, fmts):
    from mor_amd import mx
    t, k, n = shape
    x, w, dy = randn(1, t, k), randn(2, n, k, scale=0.02), randn(3, t, n, scale=1e-3)
    x[:, 3] *= 30
    w[0, :32] = 0
    xd, wd = leaf(x), leaf(w)
    y = mx.linear(xd, wd, *fmts)
    dx, dw = torch.autograd.grad(y, (xd, wd), dy.cuda())
    assert y.dtype == dx.dtype == dw.dtype == torch.bfloat16 and dx.shape == x.shape and dw.shape == w.shape
    for got, (want, bound) in zip((y, dx, dw), linear_forms(*map(P.to64, (x, w, dy)), *fmts)):
        assert (np.abs(P.to64(got) - want) <= bound).all()
    with torch.no_grad():
        assert torch.equal(mx.linear(xd, wd, *fmts), y)
    assert torch.equal(mx.linear(x.cuda(), w.cuda(), *fmts), y)


def test_linear_on_representable_values_is_the_plain_layer():
    """Values that every format holds (0, +-1, +-2) pass the quantisers unchanged, so the layer and its gradients are the
    plain ones; and since the layer is then linear, differences give the gradient exactly."""
    from mor_amd import mx
    g = torch.Generator().manual_seed(4)
    pick = lambda *s: torch.tensor([0.0, 0.0, 1.0, -1.0, 2.0, -2.0])[torch.randint(0, 6, s, generator=g)].to(torch.bfloat16)  # noqa: E731
    x, w, dy = pick(70, 64), pick(96, 64), pick(70, 96)
    for fmt, grad_fmt in LINEAR:
        xd, wd = leaf(x), leaf(w)
        y = mx.linear(xd, wd, fmt, grad_fmt)
        dx, dw = torch.autograd.grad(y, (xd, wd), dy.cuda())
        x64, w64, dy64 = map(P.to64, (x, w, dy))
        for got, want in ((y, x64 @ w64.T), (dx, dy64 @ w64), (dw, dy64.T @ x64)):
            assert np.array_equal(P.to64(got), P.to64(P.bf16(want)))          # integers up to 256 and their bf16 neighbours
        # f(x) = sum(dy * y): the difference for a step in one element that keeps x representable
        step = torch.zeros(70, 64, dtype=torch.bfloat16)
        step[5, 9] = 1.0 if float(x[5, 9]) != 2.0 else -1.0
        moved = P.to64(mx.linear((x + step).cuda(), w.cuda(), fmt, grad_fmt)) - P.to64(y)
        assert (moved * dy64).sum() == float(step[5, 9]) * (dy64 @ w64)[5, 9]


def test_linear_shapes_strides_and_partial_gradients():
    from mor_amd import mx
    x, w, dy = randn(11, 2, 19, 64), randn(12, 96, 64), randn(13, 2, 19, 96)
    flat = mx.linear(x.cuda().view(38, 64), w.cuda())
    xd, wd = leaf(x), leaf(w)
    y = mx.linear(xd, wd)
    assert y.shape == (2, 19, 96) and torch.equal(y.view(38, 96), flat)
    dx, dw = torch.autograd.grad(y, (xd, wd), dy.cuda())
    only_w = mx.linear(x.cuda(), wd)
    assert torch.equal(torch.autograd.grad(only_w, wd, dy.cuda())[0], dw)
    only_x = mx.linear(xd, w.cuda())
    assert torch.equal(torch.autograd.grad(only_x, xd, dy.cuda())[0], dx)
    # a transposed x, a weight that starts at an odd element, an expanded gradient
    xt = x.view(38, 64).t().contiguous().cuda().t().requires_grad_()
    odd = torch.cat([w.new_zeros(1), w.flatten()]).cuda()[1:].view(96, 64).requires_grad_()
    y2 = mx.linear(xt, odd)
    assert torch.equal(y2, flat)
    one = torch.ones((), dtype=torch.bfloat16, device="cuda").expand(38, 96)
    got = torch.autograd.grad(y2, (xt, odd), one)
    want = torch.autograd.grad(mx.linear(xd, wd), (xd, wd), one.contiguous().view(2, 19, 96))
    assert torch.equal(got[0], want[0].view(38, 64)) and torch.equal(got[1], want[1])
    # the same tensor used twice: the gradients add up
    y3 = mx.linear(xd, wd) + mx.linear(xd, wd)
    twice = torch.autograd.grad(y3, (xd, wd), dy.cuda())
    assert torch.equal(twice[0], dx + dx) and torch.equal(twice[1], dw + dw)


def test_linear_without_tokens():
    from mor_amd import mx
    x, w = torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True), leaf(randn(14, 32, 64))
    y = mx.linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros(0, 32, dtype=torch.bfloat16, device="cuda"))
    assert y.shape == (0, 32) and dx.shape == (0, 64) and dw.shape == (32, 64) and (dw == 0).all()


def test_linear_token_limit():
    """The weight's gradient sums over the tokens, of which a product takes fewer than 2^23: more are refused when they
    come in, not when the gradient is asked for; without that gradient they are rows like any others."""
    from mor_amd import mx
    x, w = torch.zeros(2 ** 23, 32, dtype=torch.bfloat16, device="cuda"), leaf(randn(33, 32, 32))
    x[-1] = 1
    with pytest.raises(RuntimeError, match="tokens"):
        mx.linear(x, w)
    y = mx.linear(x, w.detach())
    assert y.shape == (2 ** 23, 32) and (y[:-1] == 0).all() and torch.equal(y[-1:], mx.linear(x[-1:], w.detach()))


def test_linear_keeps_its_activation_in_8_bits():
    from mor_amd import mx, wire
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        mx.linear(leaf(randn(15, 70, 64)), leaf(randn(16, 96, 64)), wire.E2M1)
    # x^T [64, 96] in E4M3 and weight^T [64, 96] in E2M1, with a scale byte per block, each part filled up to 256 bytes
    assert [(t.dtype, t.numel()) for t in kept] == [(torch.uint8, 64 * 96 + 256 + 64 * 48 + 256)]


def test_linear_passes_nans_on():
    """A NaN or an infinity in x reaches its row of y and, through its column of x^T, its column of dw; nothing else."""
    from mor_amd import mx
    for fmt in (P.E4M3, P.E2M1):
        for bad in (float("nan"), float("inf")):
            x, w, dy = randn(17, 40, 64), randn(18, 32, 64), randn(19, 40, 32)
            x[7, 5] = bad
            xd, wd = leaf(x), leaf(w)
            y = mx.linear(xd, wd, fmt)
            dx, dw = torch.autograd.grad(y, (xd, wd), dy.cuda())
            assert torch.isnan(y[7]).all() and torch.isfinite(y[torch.arange(40) != 7]).all(), (fmt, bad)
            assert torch.isnan(dw[:, 5]).all() and torch.isfinite(dw[:, torch.arange(64) != 5]).all(), (fmt, bad)
            assert torch.isfinite(dx).all()


def swiglu_forms(g, u, dh):
    """[(exact, bound)] of h, dg, du.  One rounding to bf16 each; in fp32 exp(-g) is off by |g| 2^-23 and an ulp or two, so
    the sigmoid by (|g| + 4) 2^-23 of itself, 1 - s by as much of s, and 1 + g (1 - s) by (1 + |g|)^2 2^-22; past |g| = 88
    the sigmoid may be 0 instead of something below 2^-126."""
    half = P.BF16_HALF_STEP
    with np.errstate(over="ignore"):
        sig = lambda v: 1 / (1 + np.exp(-v))  # noqa: E731
        s = sig(g)
        h = g * s * u
        bounds = [(h, half * np.abs(h) + np.abs(h) * (np.abs(g) + 8) * 2.0 ** -22 + np.abs(g * u) * 2.0 ** -126 + 2.0 ** -133)]
        kg, ku = P.quantized_values(g, P.E4M3), P.quantized_values(u, P.E4M3)
        s, rest = sig(kg), sig(-kg)
        dg, du = dh * ku * s * (1 + kg * rest), dh * kg * s
        size = np.abs(dh * ku) * (s * (1 + np.abs(kg)) ** 2 * 2.0 ** -20 + (1 + np.abs(kg)) * 2.0 ** -126)
        bounds.append((dg, half * np.abs(dg) + size + 2.0 ** -133))
        bounds.append((du, half * np.abs(du) + np.abs(dh * kg) * (s * (np.abs(kg) + 8) * 2.0 ** -22 + 2.0 ** -126) + 2.0 ** -133))
    return bounds


@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 8), (5, 31), (4, 32), (9, 33), (2, 4096), (300, 1111), (64, 1024), (1, 100001)], ids=str)
@pytest.mark.parametrize("layout", ["apart", "halves", "shifted"])
def test_swiglu(shape, layout):
    from mor_amd import mx
    rows, cols = shape
    g, u, dh = randn(21, rows, cols, scale=3.0), randn(22, rows, cols), randn(23, rows, cols, scale=1e-2)
    g[0, 0], g[-1, -1] = -100.0, 120.0
    if rows * cols > 64:
        g.view(-1)[5:9] = torch.tensor([0.0, -0.0, -1.2784, 1e-30], dtype=torch.bfloat16)
    if layout == "apart":
        gd, ud = g.cuda(), u.cuda()
    else:
        lead = 0 if layout == "halves" else 3          # rows that begin at odd elements
        both = torch.cat([torch.zeros(rows, lead, dtype=torch.bfloat16), g, u], 1).cuda()
        gd, ud = both[:, lead:lead + cols], both[:, lead + cols:]
    gd, ud = gd.detach().requires_grad_(), ud.detach().requires_grad_()
    h = mx.swiglu(gd, ud)
    dg, du = torch.autograd.grad(h, (gd, ud), dh.cuda())
    for got, (want, bound) in zip((h, dg, du), swiglu_forms(*map(P.to64, (g, u, dh)))):
        assert (np.abs(P.to64(got) - want) <= bound).all(), np.max(np.abs(P.to64(got) - want) / bound)
    with torch.no_grad():
        assert torch.equal(mx.swiglu(gd, ud), h)


def test_swiglu_gradient_against_differences():
    """At values that E4M3 holds, the gradient is the derivative of h: central differences in float64."""
    from mor_amd import mx
    g = P.bf16(np.linspace(-6, 6, 97)[None].round(0) + np.tile([0, 0.5], 49)[None, :97])
    u, dh = P.bf16(np.tile([1.0, -2.0, 0.5], 33)[None, :97]), P.bf16(np.ones((1, 97)))
    gd, ud = leaf(g), leaf(u)
    dg, du = torch.autograd.grad(mx.swiglu(gd, ud), (gd, ud), dh.cuda())
    f = lambda a, b: a / (1 + np.exp(-a)) * b  # noqa: E731
    g64, u64, e = P.to64(g), P.to64(u), 1e-5
    assert np.array_equal(P.quantized_values(g64, P.E4M3), g64) and np.array_equal(P.quantized_values(u64, P.E4M3), u64)
    for got, diff in ((dg, (f(g64 + e, u64) - f(g64 - e, u64)) / (2 * e)), (du, (f(g64, u64 + e) - f(g64, u64 - e)) / (2 * e))):
        assert (np.abs(P.to64(got) - diff) <= P.BF16_HALF_STEP * np.abs(diff) + 1e-5).all()      # differences: e^2 |f'''| and 1e-16 / e


def test_swiglu_infinities_and_nans():
    """Forward as the formula; backward the block that holds one comes back as NaNs, the others are not touched."""
    from mor_amd import mx
    g, u, dh = randn(24, 4, 96), randn(25, 4, 96), randn(26, 4, 96)
    g[1, 40], u[2, 3] = float("nan"), float("inf")
    gd, ud = leaf(g), leaf(u)
    h = mx.swiglu(gd, ud)
    want = (g.float() / (1 + torch.exp(-g.float())) * u.float()).to(torch.bfloat16)
    assert torch.equal(torch.isnan(h.cpu()), torch.isnan(want)) and torch.equal(torch.isinf(h.cpu()), torch.isinf(want))
    dg, du = torch.autograd.grad(h, (gd, ud), dh.cuda())
    block = torch.zeros(4, 96, dtype=torch.bool)
    block[1, 32:64] = True
    block[2, 0:32] = True
    only_g = block.clone()
    only_g[2] = False
    assert torch.equal(torch.isnan(dg.cpu()), block) and torch.equal(torch.isnan(du.cpu()), only_g)


def test_swiglu_keeps_8_bits_and_takes_any_rank():
    from mor_amd import mx
    kept = []
    g, u = leaf(randn(27, 2, 3, 40)), leaf(randn(28, 2, 3, 40))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        h = mx.swiglu(g, u)
    assert h.shape == (2, 3, 40) and [(t.dtype, t.numel()) for t in kept] == [(torch.uint8, 2 * (512 + 12))]      # 6 rows of two blocks
    assert torch.equal(mx.swiglu(g.detach()[0, 0], u.detach()[0, 0]), h[0, 0])
    empty = torch.zeros(0, 5, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    out = mx.swiglu(empty, empty)
    assert out.shape == (0, 5) and torch.autograd.grad(out.sum(), empty)[0].shape == (0, 5)
    same = leaf(randn(29, 5, 64))                                  # one tensor for both: its gradients add up
    dh = randn(30, 5, 64).cuda()
    a, b = leaf(same.detach().cpu()), leaf(same.detach().cpu())
    da, db = torch.autograd.grad(mx.swiglu(a, b), (a, b), dh)
    assert torch.equal(torch.autograd.grad(mx.swiglu(same, same), same, dh)[0], da + db)


def test_no_second_derivative():
    from mor_amd import mx
    x, w = leaf(randn(31, 32, 64)), leaf(randn(32, 32, 64))
    y = mx.linear(x, w)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(mx.swiglu(x, x).float().sum(), x, create_graph=True)


def mlp(x, weights, fmt, grad_fmt):
    from mor_amd import mx
    gate, up, down = weights
    return mx.linear(mx.swiglu(mx.linear(x, gate, fmt, grad_fmt), mx.linear(x, up, fmt, grad_fmt)), down, fmt, grad_fmt)


@pytest.mark.parametrize("fmts", LINEAR, ids=str)
def test_run_together(fmts):
    """A gated feed-forward block, forward and backward.  Each stage is held to its own formula at the inputs it got, so
    that no bound has to follow an error through a quantiser."""
    from mor_amd import mx
    t, k, n = 45, 128, 224
    x, gw, uw, dw_ = randn(41, t, k), randn(42, n, k, scale=0.1), randn(43, n, k, scale=0.1), randn(44, k, n, scale=0.1)
    dy = randn(45, t, k, scale=1e-2)
    xd, weights = leaf(x), [leaf(v) for v in (gw, uw, dw_)]
    g, u = mx.linear(xd, weights[0], *fmts), mx.linear(xd, weights[1], *fmts)
    h = mx.swiglu(g, u)
    y = mx.linear(h, weights[2], *fmts)
    for v in (g, u, h):
        v.retain_grad()
    y.backward(dy.cuda())
    down = linear_forms(*map(P.to64, (h, dw_, dy)), *fmts)
    act = swiglu_forms(*map(P.to64, (g, u, h.grad)))
    gate, up = linear_forms(*map(P.to64, (x, gw, g.grad)), *fmts), linear_forms(*map(P.to64, (x, uw, u.grad)), *fmts)
    checks = [(y, *down[0]), (h.grad, *down[1]), (weights[2].grad, *down[2]), (h, *act[0]), (g.grad, *act[1]), (u.grad, *act[2]),
              (g, *gate[0]), (weights[0].grad, *gate[2]), (u, *up[0]), (weights[1].grad, *up[2])]
    both = gate[1][0] + up[1][0]
    checks.append((xd.grad, both, gate[1][1] + up[1][1] + P.BF16_HALF_STEP * (np.abs(both) + gate[1][1] + up[1][1])))
    for got, want, bound in checks:
        assert (np.abs(P.to64(got) - want) <= bound).all()
    assert torch.equal(mlp(x.cuda(), [w.detach() for w in weights], *fmts), y)


def test_training_step_captured_and_replayed():
    """Forward and backward of the block in one graph, replayed on changing inputs with eager steps between."""
    fmts = (P.E2M1, P.E4M3)
    weights = [leaf(randn(51 + i, *s, scale=0.1)) for i, s in enumerate(((224, 128), (224, 128), (128, 224)))]
    inputs = [(randn(60 + i, 45, 128).cuda(), randn(70 + i, 45, 128, scale=1e-2).cuda()) for i in range(4)]

    def step(x, dy):
        x = x.detach().requires_grad_()
        return torch.autograd.grad(mlp(x, weights, *fmts), [x, *weights], dy)

    want = [step(*i) for i in inputs]
    static = [t.clone() for t in inputs[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*static)
    for i in (1, 2, 3, 1):
        for dst, src in zip(static, inputs[i]):
            dst.copy_(src)
        graph.replay()
        eager = step(*inputs[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(outs, want[i], eager)), i


def test_capture_beside_a_live_eager_graph():
    """Torch adds a leaf's gradient on the stream of the graph that holds it, and the default stream cannot join a capture:
    the call is refused under capture while such a graph lives, and captured once it is freed."""
    from mor_amd import mx
    x, w = leaf(randn(84, 64, 64)), leaf(randn(85, 96, 64))
    deep = leaf(randn(86, 2, 3, 64))
    dh = randn(87, 64, 96).cuda()
    want = torch.autograd.grad(mx.swiglu(mx.linear(x, w), mx.linear(x, w)), (x, w), dh)
    for alive, calls in ((lambda: mx.linear(x, w), (lambda: mx.linear(x, w.detach()), lambda: mx.linear(x.detach(), w), lambda: mx.swiglu(x, x))),
                         (lambda: mx.swiglu(deep, deep), (lambda: mx.linear(deep, w), lambda: mx.swiglu(deep.detach(), deep)))):
        held = alive()
        torch.cuda.synchronize()
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            for call in calls:
                with pytest.raises(RuntimeError, match="default stream"):
                    call()
            with torch.no_grad():
                calls[0]()
        del held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(mx.swiglu(mx.linear(x, w), mx.linear(x, w)), (x, w), dh)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradients_on_another_stream():
    from mor_amd import mx
    x, w, dy = leaf(randn(81, 100, 512)), leaf(randn(82, 256, 512)), randn(83, 100, 256).cuda()
    want = torch.autograd.grad(mx.linear(x, w), (x, w), dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [torch.autograd.grad(mx.linear(x, w), (x, w), dy) for _ in range(4)]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
