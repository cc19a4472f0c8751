"""Layer norm and its gradients against the formulas in float64.

What a result may be off by, elementwise.  A sum over a row runs through at most `deep` additions one after the other (32 in a thread,
6 over a wavefront, 16 over a workgroup, or width / 1024 in a thread of the widest rows) and is off by that times 2^-24 of the sum of
magnitudes.  So is the mean; centred values pass that on to the variance (twice the mean of |c| times it), whose relative
error counts half in 1 / sqrt, beside four roundings; everything else is elementwise roundings of 2^-24, and one of
half a step of the result's type.  Sums over the rows: `far` additions, rows / 128 and 64."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
E = 2.0 ** -24
BF, FP = torch.bfloat16, torch.float32


def half(t):
    return torch.finfo(t).eps / 2


def expected(x, w, b, eps, dtype, dy):
    rows, d = x.shape
    deep, far = max(64, d / 1024 + 32), rows / 128 + 64
    x64 = x.double()
    mean = x64.mean(1, keepdim=True)
    mean_off = deep * E * x64.abs().mean(1, keepdim=True)
    c = x64 - mean
    c_off = mean_off + E * (c.abs() + mean_off)
    var = (c * c).mean(1, keepdim=True)
    var_off = (2 * c.abs() * c_off + c_off * c_off).mean(1, keepdim=True) + deep * E * var
    r = 1 / (var + eps).sqrt()
    r_rel = 0.5 * var_off / (var + eps) * (1 + var_off / (var + eps)) + 4 * E
    xh = c * r
    xh_off = c_off * r * (1 + r_rel) + xh.abs() * (r_rel + E)
    w64 = torch.ones(d, device=DEV, dtype=torch.float64) if w is None else w.double()
    b64 = torch.zeros(d, device=DEV, dtype=torch.float64) if b is None else b.double()
    y = xh * w64 + b64
    y_off = xh_off * w64.abs() + 2 * E * ((xh * w64).abs() + b64.abs())
    out = {"y": (y, y_off + half(dtype) * (y.abs() + y_off))}
    dy = dy.double()
    g = dy * w64
    s0, s1 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    s0_off = (deep + 2) * E * g.abs().mean(1, keepdim=True)
    s1_off = (g.abs() * xh_off).mean(1, keepdim=True) + (deep + 2) * E * (g * xh).abs().mean(1, keepdim=True)
    dx = r * (g - s0 - xh * s1)
    inner = s0_off + xh_off * s1.abs() + (xh.abs() + xh_off) * s1_off + 4 * E * (g.abs() + s0.abs() + (xh * s1).abs())
    dx_off = r * (1 + r_rel) * inner + dx.abs() * (r_rel + E)
    out["x"] = (dx, dx_off + half(x.dtype) * (dx.abs() + dx_off))
    for name, t, v, off, mag in (("weight", w, (dy * xh).sum(0), (dy.abs() * xh_off).sum(0), (dy * xh).abs().sum(0)),
                                 ("bias", b, dy.sum(0), 0.0, dy.abs().sum(0))):
        if t is not None:
            off = off + (far + 2) * E * mag
            out[name] = (v, off + half(t.dtype) * (v.abs() + off))
    return out


def check(got, want, name):
    v, off = want
    bad = (got.double() - v).abs() > off * 1.001 + 1e-37
    assert got.shape == v.shape and not bool(bad.any()), (name, int(bad.sum()), float(((got.double() - v).abs() / (off + 1e-37)).max()))


def make(rows, d, x=BF, w=FP, b=FP, y=None, seed=0, shift=0.0):
    gen = torch.Generator(device=DEV).manual_seed(seed + rows * 5 + d)
    rnd = lambda *s: torch.empty(*s, device=DEV).normal_(0, 1, generator=gen)  # noqa: E731
    size = rnd(rows, 1).exp()
    return ((rnd(rows, d) + shift) * size).to(x), None if w is None else (1 + 0.3 * rnd(d)).to(w), None if b is None else rnd(d).to(b), \
        rnd(rows, d).to(y or x)


def run_and_check(x, w, b, dy, eps=1e-5):
    from dion_amd import layer_norm

    print("layer_norm", tuple(x.shape), x.dtype, dy.dtype, flush=True)
    leaves = {n: t.detach().requires_grad_() for n, t in (("x", x), ("weight", w), ("bias", b)) if t is not None}
    y = layer_norm(leaves["x"], leaves.get("weight"), leaves.get("bias"), eps=eps, dtype=dy.dtype)
    assert y.dtype == dy.dtype
    want = expected(x, w, b, eps, dy.dtype, dy)
    check(y, want["y"], "y")
    grads = torch.autograd.grad(y, list(leaves.values()), dy)
    for (name, t), g in zip(leaves.items(), grads):
        assert g.dtype == t.dtype
        check(g, want[name], name)
    assert torch.equal(layer_norm(x, w, b, eps=eps, dtype=dy.dtype), y)
    again = layer_norm(leaves["x"], leaves.get("weight"), leaves.get("bias"), eps=eps, dtype=dy.dtype)
    assert all(torch.equal(p, q) for p, q in zip(grads, torch.autograd.grad(again, list(leaves.values()), dy)))


# every number of threads a row and its edges, rows that are read again, odd widths
SIZES = [(1, 1), (3, 2), (5, 7), (1, 768), (2, 64), (63, 511), (64, 512), (65, 513), (33, 1000), (300, 1024), (7, 1025), (129, 2048),
         (20, 2050), (600, 4096), (9, 4097), (31, 8192), (5, 8200), (17, 16384), (3, 16391), (4, 32768), (300, 20000), (2, 40003)]


@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("x,w,b,y", [(BF, FP, FP, BF), (FP, FP, FP, FP), (FP, BF, None, BF), (BF, None, BF, FP), (BF, BF, FP, BF),
                                     (FP, None, None, FP)])
def test_sizes_and_types(rows, d, x, w, b, y):
    run_and_check(*make(rows, d, x, w, b, y))


@pytest.mark.parametrize("rows,d", [(5000, 96), (3001, 768), (2500, 2730)])
def test_many_rows(rows, d):
    run_and_check(*make(rows, d))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("form", ["wide_rows", "odd_rows", "offset", "one_column_apart", "transposed", "repeated"])
def test_strides_and_addresses(form, dtype):
    def lay(m):
        rows, cols = m.shape
        if form == "wide_rows":
            v = torch.full((rows, cols + 24), float("nan"), device=DEV, dtype=m.dtype)[:, 8:8 + cols]
        elif form == "odd_rows":
            v = torch.full((rows, cols + 3), float("nan"), device=DEV, dtype=m.dtype)[:, :cols]
        elif form == "offset":
            v = torch.full((rows * cols + 5,), float("nan"), device=DEV, dtype=m.dtype)[5:].view(rows, cols)
        elif form == "transposed":
            v = torch.empty(cols, rows, device=DEV, dtype=m.dtype).t()
        elif form == "repeated":
            return m[:1].expand(rows, cols)
        else:
            v = torch.empty(rows, cols, 2, device=DEV, dtype=m.dtype)[:, :, 0]
        return v.copy_(m)

    for d in (768, 77):
        x, w, b, dy = make(30, d, dtype, dtype, dtype)
        odd = torch.empty(d + 1, device=DEV, dtype=dtype)[1:].copy_(w)  # a weight off its line
        run_and_check(lay(x), odd, b, lay(dy))
        run_and_check(x, w, b, lay(dy))


def test_leading_dimensions_and_partial_needs():
    from dion_amd import layer_norm

    x, w, b, dy = make(30, 72)
    y = layer_norm(x, w, b)
    assert torch.equal(layer_norm(x.view(6, 5, 72), w, b), y.view(6, 5, 72)) and layer_norm(x[0], w, b).shape == (72,)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    every = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    for only in range(3):
        some = [t.detach().requires_grad_(i == only) for i, t in enumerate((x, w, b))]
        assert torch.equal(torch.autograd.grad(layer_norm(*some), some[only], dy)[0], every[only])
    g = torch.autograd.grad(layer_norm(*leaves).sum(), leaves)  # (a gradient with strides of zero)
    full = torch.autograd.grad(layer_norm(*leaves), leaves, torch.ones_like(dy))
    assert all(torch.equal(p, q) for p, q in zip(g, full))
    (gx,) = torch.autograd.grad(layer_norm(*leaves).sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError):  # differentiable once
        torch.autograd.grad(gx.sum(), leaves[0])


@pytest.mark.parametrize("d", [24, 9000, 20000])
def test_no_rows(d):
    from dion_amd import layer_norm

    ops = [torch.ones(s, device=DEV).requires_grad_() for s in ((0, d), (d,), (d,))]
    y = layer_norm(*ops)
    assert y.shape == (0, d)
    for g, t in zip(torch.autograd.grad(y, ops, torch.zeros_like(y)), ops):
        assert g.shape == t.shape and not bool(g.any())


@pytest.mark.parametrize("d", [100, 768, 3000, 6000, 40000])
def test_far_from_zero_and_constant_rows(d):
    """A mean a thousand times the deviation, and rows without any: what the difference of mean squares would lose."""
    run_and_check(*make(20, d, FP, seed=3, shift=1000.0))
    x, w, b, dy = make(4, d, FP)
    x[1] = 3.0
    x[2] = 0.0
    run_and_check(x, w, b, dy)
    run_and_check(x, w, b, dy, eps=1e-2)


@pytest.mark.parametrize("d", [96, 2048, 5000, 9000, 40000])
def test_values_that_are_not_finite_stay_in_their_row(d):
    from dion_amd import layer_norm

    x, w, b, dy = make(40, d, BF)
    bad = x.clone()
    bad[7, 3], bad[9, 5] = float("nan"), float("inf")
    outs = []
    for v in (x, bad):
        leaf = v.detach().requires_grad_()
        y = layer_norm(leaf, w, b)
        outs.append((y, *torch.autograd.grad(y, leaf, dy)))
    rest = torch.tensor([i not in (7, 9) for i in range(40)], device=DEV)
    for p, q in zip(*outs):
        assert torch.equal(p[rest], q[rest]) and bool(q[7].isnan().all()) and bool(q[9].isnan().any())


def test_gradients_against_differences():
    from dion_amd import layer_norm

    x, w, b, dy = make(30, 130, FP, seed=5)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, dy)

    def loss(x, w, b):
        c = x - x.mean(1, keepdim=True)
        return float(((c / ((c * c).mean(1, keepdim=True) + 1e-5).sqrt() * w + b) * dy.double()).sum())

    for i, g in enumerate(grads):
        d, h, ps = g.double() / g.double().norm(), 1e-4, [p.double() for p in (x, w, b)]
        up, down = list(ps), list(ps)
        up[i], down[i] = ps[i] + h * d, ps[i] - h * d
        slope = (loss(*up) - loss(*down)) / (2 * h)
        assert abs(slope - float((g.double() * d).sum())) <= 1e-5 * abs(slope), i


def test_a_captured_pass_and_streams():
    from dion_amd import layer_norm

    x, w, b, dy = make(300, 777, BF)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def both():
        y = layer_norm(*leaves, dtype=FP)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy.float()))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = both()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(beside, both()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, device=DEV))
            dy.copy_(torch.randn(dy.shape, device=DEV))
        eager = [t.clone() for t in both()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager)), i
    alive = layer_norm(*leaves)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="layer_norm: captured while"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            layer_norm(*leaves)
    del alive


def test_more_elements_than_32_bits_count():
    """x and dx of 4.9 GB: the last rows, which alone carry a gradient, against the formulas."""
    from dion_amd import layer_norm

    t, tail, d = 300000, 50, 8192
    x, w, b, dy = make(tail, d, seed=3)
    big = torch.ones(t, d, device=DEV, dtype=BF)
    big[-tail:] = x
    dys = torch.zeros(t, d, device=DEV, dtype=BF)
    dys[-tail:] = dy
    leaves = [p.requires_grad_() for p in (big, w, b)]
    y = layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dys)
    want = expected(x, w.detach(), b.detach(), 1e-5, BF, dy)
    check(y[-tail:], want["y"], "y")
    check(dx[-tail:], want["x"], "x")
    check(dw, want["weight"], "weight")
    check(db, want["bias"], "bias")
    assert not bool(dx[:-tail].any())


def test_operator_calls_are_checked():
    from dion_amd import ops

    x, w, b, dy = make(12, 40)
    _y, stats = ops.layer_norm_forward(x, w, b, 1e-5, None, True)
    good = dict(dy=dy, x=x, weight=w, stats=stats, need_dx=True, need_dw=True, bias_dtype=FP)
    ops.layer_norm_backward(**good)
    for bad in ({"dy": dy[:, :16]}, {"dy": dy[:5]}, {"weight": None}, {"weight": w[:8]}, {"stats": stats[:, :4]}, {"stats": stats.double()}):
        with pytest.raises(ValueError, match="layer_norm"):
            ops.layer_norm_backward(**{**good, **bad})
    for bad in ({"dy": dy.half()}, {"x": x.half()}, {"bias_dtype": torch.float64}):
        with pytest.raises(TypeError, match="layer_norm"):
            ops.layer_norm_backward(**{**good, **bad})
