"""h = act(g) u, g = x Wg^T + bg, u = x Wu^T + bu, and its gradients against the formulas in float64.

What a result may be off by, elementwise.  Sums: K products add up with an error of at most K 2^-24 of the sum of their magnitudes, and
a bias is added with 2^-24 of either.  The activation passes its sum's error on by at most its steepest slope (1.13; 2 |g| for the squared
relu), with 4e-6 of itself for exponentials and quotients; act' by its largest second derivative (1.2; 2 for the squared relu; a jump
of 1 where relu's sign is open), with 4e-6 (1 + |g|).  Rounding to bf16: 2^-8 of the value.  Kept are act'(g) u and act(g) in 24 bits, 2^-16 of
them, or beside an fp32 bias as they are; dh times these is rounded to bf16 for the products, which pass the errors of an operand on through the other's magnitudes."""
import pytest
import torch

from test_gpu_linear import act64, check

pytestmark = pytest.mark.gpu
DEV = "cuda"
ACTS = [None, "relu", "relu_squared", "gelu", "gelu_tanh", "silu"]
HALF = 2.0 ** -8
NAMES = ("x", "weight_gate", "weight_up", "bias_gate", "bias_up")


def expected(x, wg, wu, bg, bu, act, dh):
    """{name: (value, what it may be off by)}"""
    x, wg, wu, dh = (t.double() for t in (x, wg, wu, dh))
    (t, k), n = x.shape, wg.shape[0]

    def projection(w, b):
        z, off = x @ w.t(), (k + 2) * 2.0 ** -24 * (x.abs() @ w.abs().t())
        return (z, off) if b is None else (z + b.double(), off + 2.0 ** -23 * (b.double().abs() + z.abs()))

    (g, g_off), (u, u_off) = projection(wg, bg), projection(wu, bu)
    a, slope = act64(g, act)
    steep = {None: 1.0, "relu_squared": 2 * (g.abs() + g_off)}.get(act, 1.13)
    a_off = g_off * steep + (4e-6 * a.abs() + 1e-30 if act else 0)
    if act is None:
        slope_off = torch.zeros_like(g)
    elif act == "relu":
        slope_off = (g.abs() <= g_off).double()
    else:
        slope_off = (2.0 if act == "relu_squared" else 1.2) * g_off + 4e-6 * (1 + g.abs())

    def times(p, p_off, q, q_off):
        off = p_off * q.abs() + p.abs() * q_off + p_off * q_off
        return p * q, off + 2.0 ** -24 * ((p * q).abs() + off)

    def rounded(v, off, half=HALF):
        return v, off + half * (v.abs() + off)

    zero = torch.zeros((), device=x.device, dtype=torch.float64)
    out = {"h": rounded(*times(a, a_off, u, u_off))}
    kept = 0.0 if any(b is not None and b.dtype == torch.float32 for b in (bg, bu)) else 2.0 ** -16
    dg, dg_off = times(dh, zero, *rounded(*times(slope, slope_off, u, u_off), kept))
    du, du_off = times(dh, zero, *rounded(a, a_off, kept))
    for name, d, off in (("bias_gate", dg, dg_off), ("bias_up", du, du_off)):
        out[name] = (d.sum(0), off.sum(0) + t * 2.0 ** -24 * (d.abs() + off).sum(0))
    dg, dg_off = rounded(dg, dg_off)
    du, du_off = rounded(du, du_off)
    for name, v, off, mag, terms in (
            ("x", dg @ wg + du @ wu, dg_off @ wg.abs() + du_off @ wu.abs(), dg.abs() @ wg.abs() + du.abs() @ wu.abs(), 2 * n),
            ("weight_gate", dg.t() @ x, dg_off.t() @ x.abs(), dg.abs().t() @ x.abs(), t),
            ("weight_up", du.t() @ x, du_off.t() @ x.abs(), du.abs().t() @ x.abs(), t)):
        out[name] = rounded(v, off + (terms + 2) * 2.0 ** -24 * (mag + off))
    return out


def make(t, k, n, bias=(None, None), seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed + t * 7 + k * 3 + n)
    rnd = lambda *s, std=1.0: torch.empty(*s, device=DEV).normal_(0, std, generator=gen).bfloat16()  # noqa: E731
    x, wg, wu = rnd(t, k), rnd(n, k, std=k ** -0.5), rnd(n, k, std=k ** -0.5)
    bg, bu = (None if b is None else rnd(n).to(b) for b in bias)
    return [x, wg, wu, bg, bu], rnd(t, n, std=0.1)


def run_and_check(ops, act, dh):
    from dion_amd import gated_linear

    print("gated_linear", tuple(ops[0].shape), tuple(ops[1].shape), act, flush=True)
    leaves = [t.detach().requires_grad_() if t is not None else None for t in ops]
    h = gated_linear(*leaves, activation=act)
    want = expected(*ops, act, dh)
    check(h, want["h"], "h")
    there = {n: t for n, t in zip(NAMES, leaves) if t is not None}
    for (name, t), g in zip(there.items(), torch.autograd.grad(h, list(there.values()), dh)):
        assert g.dtype == t.dtype
        check(g, want[name], name, extra=HALF if "bias" in name and t.dtype == torch.bfloat16 else 0.0)
    assert torch.equal(gated_linear(*ops, activation=act), h)


SMALL = [(1, 1, 1), (1, 64, 64), (3, 7, 5), (16, 40, 24), (17, 1000, 130), (33, 129, 257), (64, 512, 48), (65, 64, 128),
         (65, 72, 136), (130, 200, 264), (257, 1000, 300), (300, 2730, 77), (512, 512, 512), (1024, 4096, 256), (1, 8192, 24),
         (5, 96, 4100), (32, 64, 40)]


@pytest.mark.parametrize("t,k,n", SMALL)
@pytest.mark.parametrize("act,bias", [(None, (None, torch.float32)), ("relu", (torch.bfloat16, torch.bfloat16)),
                                      ("relu_squared", (None, None)), ("gelu", (torch.bfloat16, None)),
                                      ("gelu_tanh", (torch.float32, torch.bfloat16)), ("silu", (None, None))])
def test_sizes(t, k, n, act, bias):
    ops, dh = make(t, k, n, bias)
    run_and_check(ops, act, dh)


# 256-wide, 256 x 128 and 128-wide tiles, whole and with a split reduction, an odd number of slabs in either half of the pair
@pytest.mark.parametrize("t,k,n", [(2600, 520, 2056), (2561, 700, 1030), (4096, 64, 2048), (700, 6000, 700), (9000, 200, 264),
                                   (2048, 2048, 192), (64, 4096, 5000), (300, 64, 4160), (2049, 1024, 1088), (128, 300, 2000)])
@pytest.mark.parametrize("act,bias", [(None, (torch.float32, None)), ("silu", (None, None))])
def test_large_tiles_and_split_reductions(t, k, n, act, bias):
    ops, dh = make(t, k, n, bias)
    run_and_check(ops, act, dh)


@pytest.mark.parametrize("t,k,n", [(5, 64, 32), (200, 136, 264), (300, 77, 130)])
@pytest.mark.parametrize("form", ["wide_rows", "odd_rows", "offset", "transposed", "one_column_apart"])
def test_strides_and_addresses(t, k, n, form):
    def lay(m, form=form):
        rows, cols = m.shape
        if form == "wide_rows":
            v = torch.full((rows, cols + 24), float("nan"), device=DEV, dtype=m.dtype)[:, 8:8 + cols]
        elif form == "odd_rows":
            v = torch.full((rows, cols + 3), float("nan"), device=DEV, dtype=m.dtype)[:, :cols]
        elif form == "offset":
            v = torch.full((rows * cols + 5,), float("nan"), device=DEV, dtype=m.dtype)[5:].view(rows, cols)
        elif form == "transposed":
            v = torch.empty(cols, rows, device=DEV, dtype=m.dtype).t()
        else:
            v = torch.empty(rows, cols, 2, device=DEV, dtype=m.dtype)[:, :, 0]
        return v.copy_(m)

    ops, dh = make(t, k, n, (torch.bfloat16, torch.float32))
    for which in ((0, 1, 2), (1,), (2,)):  # (weights that lie differently have rows of different lengths between them)
        laid = [lay(t) if i in which else t for i, t in enumerate(ops)]
        run_and_check(laid, "silu", lay(dh) if 0 in which else dh)


def test_halves_of_one_weight_and_leading_dimensions():
    from dion_amd import gated_linear

    ops, dh = make(6 * 5, 72, 40)
    packed = torch.cat(ops[1:3]).requires_grad_()
    h = gated_linear(ops[0].view(6, 5, 72), packed[:40], packed[40:], activation="gelu")
    assert torch.equal(h.view(30, 40), gated_linear(*ops, activation="gelu"))
    (g,) = torch.autograd.grad(h, packed, dh.view(6, 5, 40))
    leaves = [t.detach().requires_grad_() for t in ops[1:3]]
    two = torch.autograd.grad(gated_linear(ops[0], *leaves, activation="gelu"), leaves, dh)
    assert torch.equal(g, torch.cat(two))
    x, wg, wu = ops[:3]
    same = wg.detach().requires_grad_()  # one weight for both
    (g,) = torch.autograd.grad(gated_linear(x, same, same, activation=None), same, dh)
    want = expected(x, wg, wg, None, None, None, dh)
    check(g, (want["weight_gate"][0] + want["weight_up"][0], 2 * (want["weight_gate"][1] + want["weight_up"][1])), "shared")
    assert gated_linear(x[0], wg, wu).shape == (40,)
    xs = x[:1].expand(30, 72).detach().requires_grad_()  # rows of a distance of zero
    assert torch.equal(gated_linear(xs, wg, wu)[7], gated_linear(x[:1].repeat(30, 1), wg, wu)[7])
    for only in range(5):
        ops5, dh = make(20, 72, 41, (torch.bfloat16, torch.float32))
        all_leaves = [t.detach().requires_grad_() for t in ops5]
        every = torch.autograd.grad(gated_linear(*all_leaves), all_leaves, dh)
        leaves = [t.detach().requires_grad_(i == only) for i, t in enumerate(ops5)]
        assert torch.equal(torch.autograd.grad(gated_linear(*leaves), leaves[only], dh)[0], every[only])
    xl = x.detach().requires_grad_()
    (gx,) = torch.autograd.grad(gated_linear(xl, wg, wu).sum(), xl, create_graph=True)
    with pytest.raises(RuntimeError):  # differentiable once
        torch.autograd.grad(gx.sum(), xl)


def test_no_tokens():
    from dion_amd import gated_linear

    shapes = ((0, 24), (41, 24), (41, 24), (41,), (41,))
    ops = [torch.ones(s, device=DEV, dtype=torch.bfloat16).requires_grad_() for s in shapes]
    h = gated_linear(*ops)
    assert h.shape == (0, 41)
    for g, t in zip(torch.autograd.grad(h, ops, torch.zeros_like(h)), ops):
        assert g.shape == t.shape and not bool(g.any())


@pytest.mark.parametrize("act", ACTS)
def test_values_that_are_not_finite_stay_in_their_row(act):
    from dion_amd import gated_linear

    ops, dh = make(40, 64, 48, (torch.bfloat16, torch.bfloat16), seed=9)
    bad = ops[0].clone()
    bad[7, 3] = float("nan")
    bad[9, 5] = float("inf")
    grads = []
    for v in (ops[0], bad):
        leaves = [p.detach().requires_grad_() for p in (v, *ops[1:])]
        h = gated_linear(*leaves, activation=act)
        grads.append((h, *torch.autograd.grad(h, leaves, dh)))
    rest = torch.tensor([i not in (7, 9) for i in range(40)], device=DEV)
    assert torch.equal(grads[0][0][rest], grads[1][0][rest]) and torch.equal(grads[0][1][rest], grads[1][1][rest])
    assert bool(grads[1][0][7].isnan().all()) and not bool(grads[1][0][9].isfinite().all())
    assert bool(grads[1][2].isnan().any()) and bool(grads[1][3].isnan().all())


@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(act):
    """(L(p + e d) - L(p - e d)) / 2e of the float64 formulas against <gradient, d>, d along the gradient."""
    from dion_amd import gated_linear

    ops, dh = make(40, 48, 56, (torch.float32, torch.float32), seed=11)
    leaves = [t.detach().requires_grad_() for t in ops]
    grads = torch.autograd.grad(gated_linear(*leaves, activation=act), leaves, dh)

    def loss(p):
        return float((act64(p[0] @ p[1].t() + p[3], act)[0] * (p[0] @ p[2].t() + p[4]) * dh.double()).sum())

    for i, g in enumerate(grads):
        d = g.double() / g.double().norm()
        e, ps = 1e-4, [p.double() for p in ops]
        up, down = list(ps), list(ps)
        up[i], down[i] = ps[i] + e * d, ps[i] - e * d
        slope = (loss(up) - loss(down)) / (2 * e)
        # three roundings to bf16, 2^-8 each; relu's kinks move the difference by a few of 2240 terms
        assert abs(slope - float((g.double() * d).sum())) <= 3e-2 * abs(slope), (act, NAMES[i])


def test_streams():
    from dion_amd import gated_linear

    cases = [make(300, 520, 264, (torch.bfloat16, None), seed=1)[0], make(20, 1003, 130, seed=2)[0]]
    alone = [gated_linear(*c, activation="gelu") for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i] = gated_linear(*c, activation="gelu")
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(alone, got))


@pytest.mark.parametrize("t,k,n", [(160, 264, 1000), (8, 77, 40)])
def test_a_captured_pass(t, k, n):
    """Forward and backward through autograd, recorded and replayed on new values; refused beside a living eager graph."""
    from dion_amd import gated_linear

    ops, dh = make(t, k, n, (torch.float32, torch.bfloat16), seed=4)
    leaves = [t.requires_grad_() for t in ops]

    def both():
        h = gated_linear(*leaves, activation="gelu")
        return (h.detach(), *torch.autograd.grad(h, leaves, dh))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for i in range(4):
        with torch.no_grad():
            ops[0].copy_(torch.randn(ops[0].shape, device=DEV))
            dh.copy_(torch.randn(dh.shape, device=DEV))
        eager = [t.clone() for t in both()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager)), i
    alive = gated_linear(ops[0].detach(), leaves[1], leaves[2].detach())
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="gated_linear: captured while"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            gated_linear(ops[0].detach(), leaves[1], leaves[2].detach())
    del alive


@pytest.mark.parametrize("k,n", [(64, 8192), (8192, 64)])
def test_more_elements_than_32_bits_count(k, n):
    """Operands or results of 4.9 GB: the last rows, which alone carry a gradient, against the formulas."""
    from dion_amd import gated_linear

    t, tail = 300000, 200
    ops, dh = make(tail, k, n, seed=3)
    big = torch.ones(t, k, device=DEV, dtype=torch.bfloat16)
    big[-tail:] = ops[0]
    dhs = torch.zeros(t, n, device=DEV, dtype=torch.bfloat16)
    dhs[-tail:] = dh
    leaves = [p.requires_grad_() for p in (big, ops[1], ops[2])]
    h = gated_linear(*leaves)
    dx, dwg, dwu = torch.autograd.grad(h, leaves, dhs)
    want = expected(big[-tail:].detach(), ops[1].detach(), ops[2].detach(), None, None, "silu", dh)
    check(h[-tail:], want["h"], "h")
    check(dx[-tail:], want["x"], "x")
    check(dwg, want["weight_gate"], "weight_gate")
    check(dwu, want["weight_up"], "weight_up")
    assert torch.equal(h[0], h[t - tail - 1]) and not bool(dx[:-tail].any())


def test_operator_calls_are_checked():
    from dion_amd import ops as o

    (x, wg, wu, _bg, _bu), dh = make(12, 40, 24)
    _h, kept = o.gated_forward(x, wg, wu, None, None, "silu", 24)
    good = dict(dh=dh, kept=kept, keep=24, x=x, weight_gate=wg, weight_up=wu, need_dx=True, need_dgate=True, need_dup=True,
                bias_gate_dtype=torch.float32, bias_up_dtype=None)
    o.gated_backward(**good)
    for bad in ({"dh": dh[:, :16]}, {"x": x[:8]}, {"x": None}, {"kept": None}, {"kept": kept[:-1]}, {"kept": kept.view(torch.int16)}, {"keep": 32}, {"keep": 16},
                {"weight_gate": wg[:16]}, {"weight_up": wu[:16]}):
        with pytest.raises(ValueError, match="gated_linear"):
            o.gated_backward(**{**good, **bad})
    for bad in ({"dh": dh.float()}, {"x": x.half()}, {"bias_up_dtype": torch.float64}):
        with pytest.raises(TypeError, match="gated_linear"):
            o.gated_backward(**{**good, **bad})
