"""y = act(x W^T + b) + residual and its gradients against the formulas in float64.

What a result may be off by, elementwise.  Sums: K products add up with an error of at most K 2^-24 of the sum of their magnitudes
(|x| |W|^T), which an activation passes on by at most its steepest slope (1.13; 2 |z| for the squared relu).  Rounding to bf16: 2^-8
of the value.  The gradient at z, dz = dy act'(z): the slope is kept with 2^-10 of itself (fp16: 2^-11, and 2^-25 below its
normal numbers) and computed from a z that is off by the sum's error, times the largest second derivative (1.2; 2 for the
squared relu; a jump of 1 where relu's sign is open), plus 4e-6 for exponentials and quotients; dz is rounded to bf16 for dx and dW, and every
product passes the errors of its operand on through the other's magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
ACTS = [None, "relu", "relu_squared", "gelu", "gelu_tanh", "silu"]


def act64(z, act):
    """(act(z), act'(z)) in float64."""
    if act is None:
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "relu_squared":
        return z.clamp_min(0) ** 2, 2 * z.clamp_min(0)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-z / 2 ** 0.5)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    c = (2 / torch.pi) ** 0.5
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def expected(x, w, b, act, r, dy):
    """{name: (value, what it may be off by)}"""
    x, w, dy = x.double(), w.double(), dy.double()
    k = x.shape[1]
    z = x @ w.t()
    z_off = (k + 2) * 2.0 ** -24 * (x.abs() @ w.abs().t())
    if b is not None:
        z = z + b.double()
        z_off = z_off + 2.0 ** -23 * b.double().abs()
    a, slope = act64(z, act)
    steep = 1.13 if act != "relu_squared" else 2 * (z.abs() + z_off)
    a_off = z_off * steep + (4e-6 * a.abs() + 1e-30 if act else 0)
    y = a if r is None else a + r.double()
    half = 2.0 ** -8
    out = {"y": (y, a_off + 2.0 ** -23 * a.abs() + half * (y.abs() + a_off))}
    dz = dy * slope
    if act is None:
        dz_off = torch.zeros_like(dz)
    elif act == "relu":
        dz_off = dy.abs() * (z.abs() <= z_off)
    else:
        curve = 2.0 if act == "relu_squared" else 1.2
        dz_off = dy.abs() * (slope.abs() * 2.0 ** -10 + 2.0 ** -25 + 4e-6 * (1 + z.abs()) + curve * z_off)
    t, n = dz.shape
    dz_sum = dz_off + 2.0 ** -23 * dz.abs()
    db = dz.sum(0)
    out["db"] = (db, dz_sum.sum(0) + t * 2.0 ** -24 * dz.abs().sum(0))
    kept = dz_off + (half * (dz.abs() + dz_off) if act else 0)
    for name, v, off, mag, terms in (("dx", dz @ w, kept @ w.abs(), dz.abs() @ w.abs(), n),
                                     ("dw", dz.t() @ x, kept.t() @ x.abs(), dz.abs().t() @ x.abs(), t)):
        off = off + (terms + 2) * 2.0 ** -24 * mag
        out[name] = (v, off + half * (v.abs() + off))
    return out


def check(got, want, name, extra=0.0):
    v, off = want
    bad = (got.double() - v).abs() > off * 1.001 + extra * v.abs() + 1e-37
    assert got.shape == v.shape and not bool(bad.any()), (name, int(bad.sum()), float(((got.double() - v).abs() / (off + 1e-37)).max()))


def make(t, k, n, bias, residual, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed + t * 7 + k * 3 + n)
    rnd = lambda *s, std=1.0: torch.empty(*s, device=DEV).normal_(0, std, generator=gen).bfloat16()  # noqa: E731
    x, w, dy = rnd(t, k), rnd(n, k, std=k ** -0.5), rnd(t, n, std=0.1)
    b = None if bias is None else rnd(n).to(bias)
    return x, w, b, rnd(t, n) if residual else None, dy


def run_and_check(x, w, b, act, r, dy):
    from dion_amd import linear

    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b, r)]
    y = linear(leaves[0], leaves[1], leaves[2], activation=act, residual=leaves[3])
    want = expected(x, w, b, act, r, dy)
    check(y, want["y"], "y")
    have = [t for t in leaves if t is not None]
    grads = dict(zip([i for i, t in enumerate(leaves) if t is not None], torch.autograd.grad(y, have, dy)))
    check(grads[0], want["dx"], "dx")
    check(grads[1], want["dw"], "dw")
    if b is not None:
        assert grads[2].dtype == b.dtype
        check(grads[2], want["db"], "db", extra=2.0 ** -8 if b.dtype == torch.bfloat16 else 0.0)
    if r is not None:
        assert torch.equal(grads[3], dy)
    plain = linear(x, w, b, activation=act, residual=r)
    assert torch.equal(plain, y)


SMALL = [(1, 1, 1), (1, 64, 64), (3, 7, 5), (16, 40, 24), (17, 1000, 130), (33, 129, 257), (64, 512, 48), (65, 64, 128),
         (65, 72, 136), (130, 200, 264), (257, 1000, 300), (300, 2730, 77), (512, 512, 512), (1024, 4096, 256), (1, 8192, 24)]


@pytest.mark.parametrize("t,k,n", SMALL)
@pytest.mark.parametrize("act,bias,residual", [(None, None, False), (None, torch.float32, True), ("relu", torch.bfloat16, True),
                                               ("relu_squared", None, False), ("gelu", torch.bfloat16, True),
                                               ("gelu_tanh", torch.float32, False), ("silu", None, True)])
def test_sizes(t, k, n, act, bias, residual):
    x, w, b, r, dy = make(t, k, n, bias, residual)
    run_and_check(x, w, b, act, r, dy)


@pytest.mark.parametrize("t,k,n", [(2600, 520, 4104), (2561, 700, 2050), (4096, 64, 4096), (700, 6000, 700), (9000, 200, 264)])
@pytest.mark.parametrize("act,bias,residual", [(None, torch.float32, True), ("gelu_tanh", torch.bfloat16, True), ("relu_squared", None, False)])
def test_large_tiles_and_split_reductions(t, k, n, act, bias, residual):
    x, w, b, r, dy = make(t, k, n, bias, residual)
    run_and_check(x, w, b, act, r, dy)


@pytest.mark.parametrize("t,k,n", [(5, 64, 32), (200, 136, 264), (300, 77, 130)])
@pytest.mark.parametrize("form", ["wide_rows", "odd_rows", "offset", "transposed", "one_column_apart"])
def test_strides_and_addresses(t, k, n, form):
    def lay(m):
        rows, cols = m.shape
        if form == "wide_rows":
            big = torch.full((rows, cols + 24), float("nan"), device=DEV, dtype=m.dtype)
            v = big[:, 8:8 + cols]
        elif form == "odd_rows":
            v = torch.full((rows, cols + 3), float("nan"), device=DEV, dtype=m.dtype)[:, :cols]
        elif form == "offset":
            v = torch.full((rows * cols + 5,), float("nan"), device=DEV, dtype=m.dtype)[5:].view(rows, cols)
        elif form == "transposed":
            v = torch.empty(cols, rows, device=DEV, dtype=m.dtype).t()
        else:
            v = torch.empty(rows, cols, 2, device=DEV, dtype=m.dtype)[:, :, 0]
        return v.copy_(m)

    x, w, b, r, dy = make(t, k, n, torch.bfloat16, True)
    run_and_check(lay(x), lay(w), b, "silu", lay(r), lay(dy))
    run_and_check(lay(x), lay(w), b, None, lay(r), lay(dy))


def test_leading_dimensions_expanded_gradients_and_partial_needs():
    from dion_amd import linear

    x, w, b, r, _dy = make(6 * 5, 72, 40, torch.bfloat16, True)
    x3, r3 = x.view(6, 5, 72), r.view(6, 5, 40)
    want = linear(x, w, b, activation="gelu", residual=r)
    assert torch.equal(linear(x3, w, b, activation="gelu", residual=r3), want.view(6, 5, 40))
    assert linear(x[0], w, b).shape == (40,)
    wl = w.detach().requires_grad_()
    y = linear(x3, wl, b, activation="gelu", residual=r3)
    y.sum().backward()  # (a gradient with strides of zero)
    full = torch.autograd.grad(linear(x, wl, b, activation="gelu", residual=r), wl, torch.ones_like(want))[0]
    assert torch.equal(wl.grad, full)
    for only in range(4):
        leaves = [t.detach().requires_grad_(i == only) for i, t in enumerate((x, w, b, r))]
        y = linear(leaves[0], leaves[1], leaves[2], activation="silu", residual=leaves[3])
        assert torch.autograd.grad(y, leaves[only], torch.ones_like(y))[0].shape == leaves[only].shape
    xl = x3.detach().requires_grad_()
    (gx,) = torch.autograd.grad(linear(xl, w, activation="silu").sum(), xl, create_graph=True)
    with pytest.raises(RuntimeError):  # differentiable once
        torch.autograd.grad(gx.sum(), xl)


def test_no_tokens():
    from dion_amd import linear

    x, w, b = (torch.zeros(s, device=DEV, dtype=torch.bfloat16).requires_grad_() for s in ((0, 24), (40, 24), (40,)))
    y = linear(x, w, b, activation="relu")
    assert y.shape == (0, 40)
    for g, t in zip(torch.autograd.grad(y, (x, w, b), torch.zeros_like(y)), (x, w, b)):
        assert g.shape == t.shape and not g.any()


@pytest.mark.parametrize("act", ACTS)
def test_values_at_the_ends_of_the_range(act):
    """Infinities, NaN and huge values stay in their own row and column; a saturated activation has no NaN."""
    from dion_amd import linear

    z = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 60.0, -60.0, 3e4, -3e4, 1e9, -1e9], device=DEV).bfloat16()
    t = z.numel()
    x = torch.zeros(t + 2, 8, device=DEV, dtype=torch.bfloat16)
    x[:t, 0] = z
    x[t, 0], x[t + 1, 0] = float("nan"), float("inf")
    w = torch.zeros(9, 8, device=DEV, dtype=torch.bfloat16)
    w[:, 0] = 1
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = linear(xl, wl, activation=act)
    a, slope = act64(z.double(), act)
    assert bool(((y[:t, 0].double() - a).abs() <= a.abs() * 2.0 ** -7 + 1e-35).all()), y[:t, 0]
    assert bool(y[t].isnan().all()) and bool((y[t + 1] == float("inf")).all())
    dy = torch.zeros_like(y)
    dy[:t] = 1
    dx = torch.autograd.grad(y, xl, dy)[0][:t, 0].double() / 9
    assert bool(((dx - slope).abs() <= slope.abs() * 2.0 ** -7 + 1e-5).all()), (dx, slope)


def test_gradients_against_differences():
    """One direction for every input: (L(p + h d) - L(p - h d)) / 2h of the float64 formulas against <gradient, d>."""
    from dion_amd import linear

    for act in ACTS:
        x, w, b, r, dy = make(40, 48, 56, torch.float32, True, seed=11)
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        grads = torch.autograd.grad(linear(*leaves[:3], activation=act, residual=leaves[3]), leaves, dy)

        def loss(ps):
            z = ps[0] @ ps[1].t() + ps[2]
            return float(((act64(z, act)[0] + ps[3]) * dy.double()).sum())

        for i, g in enumerate(grads):
            # along the gradient itself, whose norm dwarfs what its rounding can do to the product
            d = g.double() / g.double().norm()
            h, ps = 1e-4, [p.double() for p in (x, w, b, r)]
            up, down = list(ps), list(ps)
            up[i], down[i] = ps[i] + h * d, ps[i] - h * d
            slope = (loss(up) - loss(down)) / (2 * h)
            # rounding to bf16, twice, 2^-8 each; relu's kinks move the difference by a few of 2240 terms
            assert abs(slope - float((g.double() * d).sum())) <= 2.5e-2 * abs(slope), (act, i)


def test_streams_and_graph():
    """Two calls side by side on streams of their own, and a captured forward and backward pass that is replayed on new values."""
    from dion_amd import linear, ops

    a, b2 = make(300, 520, 264, torch.bfloat16, True, seed=1), make(257, 1003, 130, torch.bfloat16, True, seed=2)
    alone = [linear(x, w, b, activation="gelu", residual=r) for x, w, b, r, _ in (a, b2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, (x, w, b, r, _dy) in enumerate((a, b2)):
            with torch.cuda.stream(streams[i]):
                got[i] = linear(x, w, b, activation="gelu", residual=r)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(alone, got))

    x, w, b, r, dy = b2

    def both():
        y, slope = ops.linear_forward(x, w, b, "relu_squared", r, True)
        return (y, *ops.linear_backward(dy, slope, "relu_squared", x, w, True, True, b.dtype))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for k in range(4):
        x.copy_(torch.randn(x.shape, device=DEV))
        dy.copy_(torch.randn(dy.shape, device=DEV))
        eager = [t.clone() for t in both()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager)), k
        x.mul_(0.5)


def test_a_block_is_trained_through_products_and_step():
    """The pieces together as a training step uses them: two products and their gradients, Muon on the matrices, AdamW with
    8-bit moments on the biases and the embedding.  Gradients of the first step against float64; then eight steps run."""
    from dion import Muon
    from dion_amd import linear

    gen = torch.Generator(device=DEV).manual_seed(5)
    rnd = lambda *s, std: torch.nn.Parameter(torch.empty(*s, device=DEV).normal_(0, std, generator=gen).bfloat16())  # noqa: E731
    emb, up, down = rnd(50, 96, std=1.0), rnd(384, 96, std=0.1), rnd(96, 384, std=0.05)
    bu, bd = rnd(384, std=0.1), rnd(96, std=0.1)
    opt = Muon([{"params": [up, down]}, {"params": [emb, bu, bd], "algorithm": "adamw", "lr": 1e-3, "state_bits": 8}], lr=0.02)
    tokens = torch.randint(0, 50, (4, 33), device=DEV, generator=gen)
    target = torch.empty(4, 33, 96, device=DEV).normal_(0, 1, generator=gen)

    def forward():
        h = emb[tokens]
        return linear(linear(h, up, bu, activation="relu_squared"), down, bd, residual=h)

    for k in range(8):
        opt.zero_grad()
        loss = (forward().float() - target).square().mean()
        loss.backward()
        if k == 0:
            ps = [p.detach().double().requires_grad_() for p in (emb, up, down, bu, bd)]
            h = ps[0][tokens]
            z = (h @ ps[1].t() + ps[3]).clamp_min(0).square() @ ps[2].t() + ps[4] + h
            grads = torch.autograd.grad((z - target.double()).square().mean(), ps)
            for p, g in zip((emb, up, down, bu, bd), grads):
                # hidden values, y and dy are rounded to bf16 on the way (2^-8 each, at random), a result once more
                assert float((p.grad.double() - g).norm() / g.norm()) < 4 * 2.0 ** -8
        before = [p.detach().clone() for p in (emb, up, down, bu, bd)]
        opt.step()
        assert all(p.isfinite().all() and not torch.equal(p, q) for p, q in zip((emb, up, down, bu, bd), before))


def test_no_tokens_and_a_weight_past_one_launch():
    """2^28 and more elements of a gradient of zeros."""
    from dion_amd import linear

    x = torch.zeros(0, 16400, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(16400, 16400, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    (g,) = torch.autograd.grad(linear(x, w), w, torch.zeros(0, 16400, device=DEV, dtype=torch.bfloat16))
    assert g.shape == w.shape and not bool(g.any())


@pytest.mark.parametrize("k,n,act", [(8192, 64, None), (64, 8192, "gelu")])
def test_more_elements_than_32_bits_count(k, n, act):
    """Operands and results of 4.9 GB: the last rows, which alone carry a gradient, against the formulas."""
    from dion_amd import linear

    t, tail = 300000, 200
    x, w, b, _r, dy = make(tail, k, n, torch.bfloat16, False, seed=3)
    big = torch.ones(t, k, device=DEV, dtype=torch.bfloat16)
    big[-tail:] = x
    dys = torch.zeros(t, n, device=DEV, dtype=torch.bfloat16)
    dys[-tail:] = dy
    leaves = [p.requires_grad_() for p in (big, w, b)]
    y = linear(*leaves, activation=act)
    dx, dw, db = torch.autograd.grad(y, leaves, dys)
    want = expected(x, w.detach(), b.detach(), act, None, dy)
    check(y[-tail:], want["y"], "y")
    check(dx[-tail:], want["dx"], "dx")
    check(dw, want["dw"], "dw")
    check(db, want["db"], "db", extra=2.0 ** -8)
    assert torch.equal(y[0], y[t - tail - 1]) and not bool(dx[:-tail].any())


@pytest.mark.parametrize("act", ACTS)
def test_nan_reaches_the_gradients(act):
    """A row of x that is NaN: its row of dx and all of dW are NaN (with relu, whose derivative is a number there, the gradient goes
    on instead of ending); the other rows are as without it."""
    from dion_amd import linear

    x, w, b, _r, dy = make(40, 64, 48, torch.bfloat16, False, seed=9)
    bad = x.clone()
    bad[7] = float("nan")
    grads = []
    for v in (x, bad):
        leaves = [p.detach().requires_grad_() for p in (v, w, b)]
        y = linear(*leaves, activation=act)
        grads.append((y, *torch.autograd.grad(y, leaves, dy)))
    (y0, dx0, _, _), (y1, dx1, dw1, db1) = grads
    rest = torch.arange(40, device=DEV) != 7
    assert torch.equal(y0[rest], y1[rest]) and torch.equal(dx0[rest], dx1[rest])
    assert bool(y1[7].isnan().all()) and bool(dw1.isnan().all())
    if act in (None, "relu"):
        assert torch.equal(dx1[7], linear(dy[7], w.t().contiguous()))
    else:
        assert bool(dx1[7].isnan().all()) and bool(db1.isnan().all())


def test_a_captured_pass_through_autograd():
    """Forward and backward through autograd, recorded and replayed; not while an eager graph of the same leaves lives, whose
    stream the recorded pass would have to wait for."""
    from dion_amd import linear

    x, w, b, r, dy = make(160, 264, 1000, torch.float32, True, seed=4)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]

    def both():
        y = linear(*leaves[:3], activation="gelu", residual=leaves[3])
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, device=DEV))
        eager = [t.clone() for t in both()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager)), k

    alive = linear(x.detach(), leaves[1])
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="still has its graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            linear(x.detach(), leaves[1])
    del alive
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2):
        again = both()
    graph2.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(again, both()))


def test_operator_calls_are_checked():
    """The calls below the autograd function refuse what does not fit instead of reading past it."""
    from dion_amd import ops

    x, w, _b, _r, dy = make(12, 40, 24, None, False)
    y, slope = ops.linear_forward(x, w, None, "silu", None, True)
    good = dict(dy=dy, slope=slope, activation="silu", x=x, weight=w, need_dx=True, need_dw=True, bias_dtype=torch.float32)
    ops.linear_backward(**good)
    for bad in ({"dy": dy[:, :16]}, {"x": x[:8]}, {"x": None}, {"slope": None}, {"slope": slope[:8]}, {"activation": None},
                {"slope": slope.view(torch.uint8)}, {"weight": w[:16]}):
        with pytest.raises(ValueError, match="linear"):
            ops.linear_backward(**{**good, **bad})
    for bad in ({"dy": dy.float()}, {"x": x.half()}, {"bias_dtype": torch.float64}):
        with pytest.raises(TypeError):
            ops.linear_backward(**{**good, **bad})
    with pytest.raises(ValueError, match="does not fit"):
        ops.linear_forward(x, w[:, :32], None, None, None, False)
    with pytest.raises(ValueError, match="residual"):
        ops.linear_forward(x, w, None, None, y[:8], False)
