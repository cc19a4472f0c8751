"""Rows of a table and the table's gradient against the formulas in float64.

y: one product in fp32 (the factor rounded to it) and one rounding, 2^-23 and half a step of its type.  A row of the gradient: n
additions in fp32 and the factor, (n + 2) 2^-24 of the sum of magnitudes, and half a step of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
E = 2.0 ** -24
BF, FP = torch.bfloat16, torch.float32


def half(t):
    return torch.finfo(t).eps / 2


def check(got, v, off, name):
    bad = (got.double() - v).abs() > off * 1.001 + 1e-37
    assert got.shape == v.shape and not bool(bad.any()), (name, int(bad.sum()), float(((got.double() - v).abs() / (off + 1e-37)).max()))


def make(ids, vocab, d, table=FP, y=None, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed + vocab + d)
    rnd = lambda *s: torch.empty(*s, device=DEV).normal_(0, 1, generator=gen)  # noqa: E731
    return rnd(vocab, d).to(table), rnd(*ids.shape, d).to(y or table)


def zipf(tokens, vocab, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    u = torch.rand(tokens, device=DEV, dtype=torch.float64, generator=gen)
    return ((vocab + 1.0) ** u).long().sub_(1).clamp_(0, vocab - 1)


def run_and_check(ids, w, dy, scale=1.0, padding=None):
    from dion_amd import embedding

    print("embedding", tuple(ids.shape), ids.dtype, tuple(w.shape), w.dtype, dy.dtype, padding, flush=True)
    leaf = w.detach().requires_grad_()
    y = embedding(ids, leaf, scale=scale, padding_idx=padding, dtype=dy.dtype)
    want = scale * w.double()[ids.long()]
    check(y, want, (half(dy.dtype) + 2 * E) * want.abs(), "y")
    (g,) = torch.autograd.grad(y, leaf, dy)
    flat, dflat = ids.reshape(-1).long(), dy.reshape(-1, w.shape[1]).double()
    if padding is not None:
        keep = flat != padding % w.shape[0]
        flat, dflat = flat[keep], dflat[keep]
    sums = lambda v: torch.zeros(w.shape, device=DEV, dtype=torch.float64).index_add_(0, flat, v)  # noqa: E731
    value, mag = scale * sums(dflat), abs(scale) * sums(dflat.abs())
    n = torch.bincount(flat, minlength=w.shape[0])[:, None]
    off = (n + 2) * E * mag
    assert g.dtype == w.dtype
    check(g, value, off + half(w.dtype) * (value.abs() + off), "gradient")
    assert not bool(g[(n == 0).squeeze(1)].any())
    assert torch.equal(embedding(ids, w, scale=scale, dtype=dy.dtype), y)
    for again in (ids, ids.to(torch.int32 if ids.dtype == torch.int64 else torch.int64)):  # the same bits, whatever type the ids are
        y = embedding(again, leaf, scale=scale, padding_idx=padding, dtype=dy.dtype)
        assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], g)
    return g


SIZES = [(1, 1, 1), (1, 5, 8), (3, 7, 5), (64, 1, 24), (65, 1, 24), (64, 300, 77), (65, 300, 512), (1000, 3, 520), (1000, 257, 513),
         (1023, 5000, 64), (1025, 200, 1000), (3000, 131073, 96), (5000, 70, 768), (20000, 1001, 264), (17000, 40000, 128), (700, 90, 1254), (300, 50, 10), (2000, 3, 2050)]


@pytest.mark.parametrize("tokens,vocab,d", SIZES)
@pytest.mark.parametrize("table,y,scale,padding", [(FP, BF, 1.0, None), (BF, BF, 27.7, 0), (BF, FP, 1.0, -1), (FP, FP, -0.5, None)])
def test_sizes_and_types(tokens, vocab, d, table, y, scale, padding):
    ids = zipf(tokens, vocab, seed=tokens)
    run_and_check(ids, *make(ids, vocab, d, table, y), scale, padding)


@pytest.mark.parametrize("tokens", [1, 63, 64, 65, 128, 129, 1024, 1025, 4096, 30000, 50000])
@pytest.mark.parametrize("form", ["same", "same_but_one", "two_in_turn", "ascending", "one_workgroup", "blocks_of_65"])
def test_runs_of_equal_tokens(tokens, form):
    """Rows whose tokens end and start inside a run, all tokens in one row, and many rows of one workgroup of the index, with more tokens
    of a wavefront's run than its list has room for (2147 of 3136, at 50000)."""
    vocab = 40001
    at = torch.arange(tokens, device=DEV)
    ids = {"same": torch.full((tokens,), 33333, device=DEV), "same_but_one": torch.where(at == tokens // 2, 7, 256 * 7),
           "two_in_turn": torch.where(at % 2 == 0, 5, 5 + 256), "ascending": at % vocab, "one_workgroup": (at * 256 + 3) % (40000 // 256 * 256),
           "blocks_of_65": (at // 65 * 977) % vocab}[form]
    run_and_check(ids, *make(ids, vocab, 40, FP, FP))
    run_and_check(ids, *make(ids, vocab, 24, BF, BF), 2.0, int(ids[0]))


@pytest.mark.parametrize("form", ["wide_rows", "odd_rows", "offset", "transposed", "one_column_apart", "repeated"])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_strides_and_addresses(form, dtype):
    def lay(m):
        (rows, cols), fill = m.shape, float("nan") if m.is_floating_point() else 7
        if form == "wide_rows":
            v = torch.full((rows, cols + 24), fill, device=DEV, dtype=m.dtype)[:, 8:8 + cols]
        elif form == "odd_rows":
            v = torch.full((rows, cols + 3), fill, device=DEV, dtype=m.dtype)[:, :cols]
        elif form == "offset":
            v = torch.full((rows * cols + 5,), fill, device=DEV, dtype=m.dtype)[5:].view(rows, cols)
        elif form == "transposed":
            v = torch.empty(cols, rows, device=DEV, dtype=m.dtype).t()
        elif form == "repeated":
            return m[:1].expand(rows, cols)
        else:
            v = torch.empty(rows, cols, 2, device=DEV, dtype=m.dtype)[:, :, 0]
        return v.copy_(m)

    for d in (520, 77):
        ids = zipf(300, 100)
        w, dy = make(ids, 100, d, dtype)
        run_and_check(lay(ids[:, None].expand(300, 3))[:, 1] if form != "repeated" else ids, lay(w), lay(dy))


def test_shapes_of_ids_and_no_tokens():
    from dion_amd import embedding

    w, _ = make(torch.zeros(1), 50, 24, FP)
    ids = zipf(60, 50)
    y = embedding(ids, w)
    assert torch.equal(embedding(ids.view(3, 4, 5), w), y.view(3, 4, 5, 24)) and torch.equal(embedding(ids[0], w), y[0])
    leaf = w.requires_grad_()
    (g,) = torch.autograd.grad(embedding(ids.view(3, 20).t(), leaf).sum(), leaf)  # (a gradient with strides of zero)
    assert torch.equal(g, torch.bincount(ids, minlength=50)[:, None].float().expand(50, 24))
    (g,) = torch.autograd.grad(embedding(ids[0], leaf), leaf, torch.ones(24, device=DEV))
    assert float(g.sum()) == 24 and bool((g[ids[0]] == 1).all())
    for empty in (ids[:0], ids[:0].view(0, 7)):
        y = embedding(empty, leaf)
        assert y.shape == (*empty.shape, 24)
        (g,) = torch.autograd.grad(y, leaf, torch.zeros_like(y))
        assert g.shape == w.shape and not bool(g.any())


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("d", [64, 77])
def test_ids_outside_the_table(dtype, d):
    """They read and write nothing: NaN in their rows, no gradient, everything else as without them."""
    from dion_amd import embedding

    good = zipf(500, 40)
    w, dy = make(good, 40, d, FP)
    leaf = w.detach().requires_grad_()
    top = torch.iinfo(dtype)
    bad = torch.tensor([-1, 40, 41, top.max, top.min, -100, 1 << 20, top.max - 39], device=DEV, dtype=dtype)
    ids = good.to(dtype).clone()
    ids[100:108] = bad
    y = embedding(ids, leaf)
    ok = torch.ones(500, dtype=torch.bool, device=DEV)
    ok[100:108] = False
    assert bool(y[~ok].isnan().all()) and torch.equal(y[ok], w[good[ok]])
    (g,) = torch.autograd.grad(y, leaf, dy)
    (want,) = torch.autograd.grad(embedding(good[ok], leaf), leaf, dy[ok])
    assert torch.equal(g, want)


def test_padding_rows_of_nan_do_not_reach_the_gradient():
    from dion_amd import embedding

    ids = zipf(400, 30)
    w, dy = make(ids, 30, 48, FP)
    dy[ids == 4] = float("nan")
    leaf = w.detach().requires_grad_()
    (g,) = torch.autograd.grad(embedding(ids, leaf, padding_idx=4), leaf, dy)
    assert bool(g.isfinite().all()) and not bool(g[4].any())
    (g,) = torch.autograd.grad(embedding(ids, leaf), leaf, dy)
    assert bool(g[4].isnan().all()) and bool(g[[i for i in range(30) if i != 4]].isfinite().all())


def test_a_captured_pass_and_streams():
    from dion_amd import embedding

    ids = zipf(2000, 900)
    w, dy = make(ids, 900, 96, FP, BF)
    leaf = w.requires_grad_()

    def both():
        y = embedding(ids, leaf, scale=3.0, padding_idx=0, dtype=BF)
        return y.detach(), torch.autograd.grad(y, leaf, dy)[0]

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
        ids.copy_(zipf(2000, 900, seed=10 + i) if i % 2 else torch.full_like(ids, i + 1))
        dy.copy_(torch.randn(dy.shape, device=DEV))
        eager = [t.clone() for t in both()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager)), i
    alive = embedding(ids, leaf)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="embedding: captured while"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            embedding(ids, leaf)
    del alive


def test_more_elements_than_32_bits_count():
    """A table, and results, past 2^31 elements."""
    from dion_amd import embedding

    vocab, d = 560000, 4096
    w = torch.zeros(vocab, d, device=DEV, dtype=BF)
    w[-1], w[-2] = 3.0, 5.0
    leaf = w.requires_grad_()
    ids = torch.tensor([vocab - 1, 0, vocab - 2, vocab - 1], device=DEV)
    y = embedding(ids, leaf)
    assert y[:, 7].tolist() == [3.0, 0.0, 5.0, 3.0]
    (g,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert g[-2:, 9].tolist() == [1.0, 2.0] and float(g[0, 0]) == 1.0 and not bool(g[1:-2].any())
    del g, y, leaf, w
    t = 560000
    table = torch.arange(8, device=DEV, dtype=FP)[:, None].expand(8, d).contiguous().requires_grad_()
    ids = torch.arange(t, device=DEV) % 8
    y = embedding(ids, table, dtype=BF)
    assert bool((y[-8:, -1] == torch.arange(8, device=DEV)).all())
    dy = torch.zeros(1, d, device=DEV, dtype=BF).expand(t, d).contiguous()
    dy[-1] = 2.0
    (g,) = torch.autograd.grad(y, table, dy)
    assert bool((g[(t - 1) % 8] == 2).all()) and float(g.sum()) == 2 * d


def test_operator_calls_are_checked():
    from dion_amd import ops

    ids = zipf(12, 20)
    w, dy = make(ids, 20, 40)
    good = dict(dy=dy, ids=ids, vocab=20, scale=1.0, padding_idx=None, dtype=FP)
    ops.embedding_backward(**good)
    for bad in ({"dy": dy[:5]}, {"vocab": 0}, {"padding_idx": 20}):
        with pytest.raises(ValueError, match="embedding"):
            ops.embedding_backward(**{**good, **bad})
    for bad in ({"dy": dy.half()}, {"ids": ids.to(torch.int16)}, {"dtype": torch.float16}):
        with pytest.raises(TypeError, match="embedding"):
            ops.embedding_backward(**{**good, **bad})
