"""AdamW with moments in 8 bits, and in float32 beside bfloat16 parameters, against the formulas in float64.

What they may be off by.  m = m0 + w1 (g - m0) carries four roundings of 2^-24, each of at most |m0| + |g|: 2^-22 (|m0| + |g|).  A
maximum is off by no more than the largest error of what it is taken over, so a scale by 1 / 127 of the block's largest such
bound and its own rounding; in a block of many elements whose largest m is at least a tenth of its largest |m0| and |g| that is 3e-6
of the scale, in one of a single element, where m0 and g can cancel, it is not.  sqrt(v) has no cancellation: 1e-6.  A code differs from float64's only where the value lies within 127 x 3e-6 or 255 x 1e-6
of a border between two, and then by one: at most 0.2 % of the elements.  x carries m's error over the denominator and 2e-6 of the
move (roundings of the powers, quotients and roots), and its own rounding."""
import copy

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
B1, B2, EPS = 0.9, 0.95, 1e-8


def mix(h):
    h = np.asarray(h, dtype=np.uint64) & 0xFFFFFFFF
    h ^= h >> np.uint64(16)
    h = h * np.uint64(0x6A09E667) & np.uint64(0xFFFFFFFF)
    h ^= h >> np.uint64(15)
    h = h * np.uint64(0xBB67AE85) & np.uint64(0xFFFFFFFF)
    return h ^ (h >> np.uint64(16))


def noise(seed, step, n):
    key = mix(mix(seed & 0xFFFFFFFF) + np.uint64(step))
    i = np.arange(n, dtype=np.uint64)
    h = mix(key ^ (i >> np.uint64(3)))
    h = h + (i & np.uint64(7)) * np.uint64(0x9E3779B9) & np.uint64(0xFFFFFFFF)
    return (h >> np.uint64(8)).astype(np.float64) / 2.0 ** 24


def blocks(x, pad=0.0):
    n = -(-x.size // 128) * 128
    return np.concatenate([x, np.full(n - x.size, pad)]).reshape(-1, 128)


def oracle(x, g, c, s, k, q, lr, wd, step, cautious, seed):
    """One update in float64: (x, what x may be off by, codes, scales, what those may be off by, codes, scales)."""
    n = x.size
    m = (blocks(c) * s[:, None]).ravel()[:n]
    v = ((blocks(k) * q[:, None]) ** 2).ravel()[:n]
    m_off = 2.0 ** -22 * (np.abs(m) + np.abs(g))
    m = B1 * m + (1 - B1) * g
    v = B2 * v + (1 - B2) * g * g
    off = lr / (1 - B1 ** step) * m_off / (np.sqrt(v / (1 - B2 ** step)) + EPS)
    x_off = 2.0 ** -23 * np.abs(x)  # of the decay: 1 - lr wd is rounded, and its product with x, which the move may cancel
    upd = m / (1 - B1 ** step) / (np.sqrt(v / (1 - B2 ** step)) + EPS)
    if cautious:  # where m is smaller than what it is off by, its sign is open, and with it whether x decays
        x_off = x_off + lr * wd * np.abs(x) * (np.abs(m) <= m_off)
    x = np.where(upd * x >= 0, x * (1 - lr * wd), x) if cautious else x * (1 - lr * wd)
    x = x - lr * upd
    off = off + 2e-6 * np.abs(lr * upd) + x_off + 2.0 ** -24 * np.abs(x)
    s = np.abs(blocks(m)).max(1) / 127
    s_off = blocks(m_off).max(1) / 127 + 2.0 ** -22 * s
    q = np.sqrt(blocks(v)).max(1) / 255
    u = noise(seed, step, n)
    each = lambda a: np.repeat(a, 128)[:n]  # noqa: E731
    t = np.divide(m, each(s), out=np.zeros(n), where=each(s) > 0)
    c = np.clip(np.floor(t + u), -127, 127)
    r = np.divide(np.sqrt(v), each(q), out=np.zeros(n), where=each(q) > 0)
    low = np.floor(r)
    k = np.where(u * (2 * low + 1) < r * r - low * low, low + 1, low)
    k = np.where(v > 0, np.maximum(k, 1), k)
    return x, off, c, s, s_off, np.minimum(k, 255), q


def state(sizes, xdt, gdt, seed, offset=0):
    """Tensors of the given sizes, ``offset`` elements into their allocations."""
    gen = torch.Generator().manual_seed(seed)

    def make(n, std, dtype):
        t = torch.zeros(n + offset, dtype=dtype)
        t[offset:] = (torch.randn(n, generator=gen) * std).to(dtype)
        return t.to(DEV)[offset:]

    X = [make(n, 0.1, xdt) for n in sizes]
    G = [make(n, 0.02, gdt) for n in sizes]
    M = [torch.randint(-127, 128, (n + offset,), generator=gen, dtype=torch.int8).to(DEV)[offset:] for n in sizes]
    V = [torch.randint(1, 256, (n + offset,), generator=gen, dtype=torch.uint8).to(DEV)[offset:] for n in sizes]
    MS = [(torch.rand(-(-n // 128), generator=gen) * 1e-4).to(DEV) for n in sizes]
    VS = [(torch.rand(-(-n // 128), generator=gen) * 1e-4).to(DEV) for n in sizes]
    return X, G, M, MS, V, VS


def npy(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("sizes,offset", [([1], 0), ([0, 3, 0], 0), ([127, 128, 129], 0), ([1000, 2048, 2049, 7], 0), ([5000, 640], 3),
                                          ([70000], 1), ([2048] * 50, 0), ([(4 << 20) + 77, 300], 0)])
@pytest.mark.parametrize("xdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gdt,cautious", [(torch.bfloat16, False), (torch.float32, True)])
def test_update_against_float64(sizes, offset, xdt, gdt, cautious):
    from dion_amd import ops

    X, G, M, MS, V, VS = state(sizes, xdt, gdt, 5, offset)
    before = [[npy(t) for t in ts] for ts in (X, G, M, MS, V, VS)]
    steps = [torch.full((), 9.0, device=DEV) for _ in sizes]
    ops.adamw8_step(X, G, M, MS, V, VS, steps, torch.tensor(0.01, device=DEV), B1, B2, 0.1, EPS, cautious, seed=77)
    for i, n in enumerate(sizes):
        x, off, c, s, s_off, k, q = oracle(*(b[i] for b in before), 0.01, 0.1, 10, cautious, 77)
        assert float(steps[i]) == 10.0
        if not n:
            continue
        half = 0 if xdt == torch.float32 else 2.0 ** -8
        assert np.all(np.abs(npy(X[i]) - x) <= np.abs(x) * half + 1.01 * off), (i, n)
        assert np.all(np.abs(npy(MS[i]) - s) <= s_off) and np.all(np.abs(npy(VS[i]) - q) <= 1e-6 * q)
        for got, want in ((M[i], c), (V[i], k)):
            d = np.abs(npy(got) - want)
            assert d.max() <= 1 and np.mean(d) <= 2e-3 + 1.0 / n * (n < 500), (i, n, d.max(), np.mean(d))
        assert npy(V[i]).min() >= 1


def test_repeats_bit_for_bit_and_the_seed_counts():
    from dion_amd import ops

    def run(seed):
        X, G, M, MS, V, VS = state([3000, 515], torch.float32, torch.float32, 6)
        steps = [torch.zeros((), device=DEV) for _ in X]
        for _ in range(3):
            ops.adamw8_step(X, G, M, MS, V, VS, steps, torch.tensor(0.01, device=DEV), B1, B2, 0.0, EPS, seed=seed)
        return X + M + MS + V + VS

    a, b, c, d = run(1), run(1), run(2), run(1 + (1 << 32))
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and all(torch.equal(x, y) for x, y in zip(a, d))
    assert not all(torch.equal(x, y) for x, y in zip(a, c))


def test_rounding_is_unbiased_where_nearest_would_stand_still():
    """g = 0 for 400 steps at beta2 = 0.999: v decays by 0.1 % a step, an eighth of a code.  A code is +-1 at random each
    step: the mean over 12800 elements of v after t steps is off by about sqrt(t / 6) / 128 / sqrt(12800) relative, 0.06 %; bound 1 %."""
    from dion_amd import ops

    n = 12800
    x, g = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    M, MS = torch.zeros(n, dtype=torch.int8, device=DEV), torch.zeros(n // 128, device=DEV)
    V, VS = torch.full((n,), 128, dtype=torch.uint8, device=DEV), torch.full((n // 128,), 1e-3, device=DEV)
    V[::128] = 255
    g[::128] = 0.255  # keeps the scale where it is
    step = torch.zeros((), device=DEV)
    for _ in range(400):
        ops.adamw8_step([x], [g], [M], [MS], [V], [VS], [step], torch.tensor(0.0, device=DEV), 0.9, 0.999, 0.0, EPS, seed=3)
    v = ops.state8_values(V, VS).view(-1, 128)
    assert abs(float(v[:, 0].mean()) / 0.255 ** 2 - 1) < 1e-2
    assert abs(float(v[:, 1:].double().mean()) / (0.128 ** 2 * 0.999 ** 400) - 1) < 1e-2


def test_blocks_that_are_zero_tiny_or_not_finite():
    from dion_amd import ops

    n = 128 * 5 + 4
    X, G, M, MS, V, VS = ([t] for t in (torch.ones(n, device=DEV), torch.zeros(n, device=DEV),
                                        torch.zeros(n, dtype=torch.int8, device=DEV), torch.zeros(6, device=DEV),
                                        torch.zeros(n, dtype=torch.uint8, device=DEV), torch.zeros(6, device=DEV)))
    G[0][128:256] = 1e-32           # first moments below 1e-30; the squares vanish in fp32
    G[0][256 + 5] = float("nan")
    G[0][384 + 7] = float("inf")
    G[0][512:640] = 1.0
    G[0][513] = 1e-6                # second moment 1e-12 of the block's largest: keeps a code
    G[0][640:] = 2.0                # a short block
    step = [torch.zeros((), device=DEV)]
    ops.adamw8_step(X, G, M, MS, V, VS, step, torch.tensor(0.1, device=DEV), B1, B2, 0.0, EPS, seed=0)
    m, v = ops.state8_values(M[0], MS[0]), ops.state8_values(V[0], VS[0])
    assert torch.equal(X[0][:128], torch.ones(128, device=DEV)) and not m[:256].any() and not v[:256].any()
    assert m[256:384].isnan().all() and v[256:384].isnan().all() and m[384:512].isnan().all() and v[384:512].isnan().all()
    fine = X[0][256:512].isfinite()
    assert int((~fine).sum()) == 2 and not fine[5] and not fine[128 + 7]
    assert int(V[0][513]) == 1 and torch.equal(V[0][640:], torch.full((4,), 255, dtype=torch.uint8, device=DEV))
    assert torch.equal(M[0][640:], torch.full((4,), 127, dtype=torch.int8, device=DEV))


@pytest.mark.parametrize("n,offset", [(0, 0), (1, 0), (129, 0), (5000, 0), (5000, 5), ((1 << 22) + 3, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_of_codes(n, offset, dtype):
    from dion_amd.functional import state8_blocks, state8_values

    scales = torch.rand(state8_blocks(n), device=DEV) + 0.1
    signed = torch.randint(-127, 128, (n + offset,), dtype=torch.int8, device=DEV)[offset:]
    plain = torch.randint(0, 256, (n + offset,), dtype=torch.uint8, device=DEV)[offset:]
    each = scales.repeat_interleave(128)[:n]
    assert torch.equal(state8_values(signed, scales, dtype), (signed.float() * each).to(dtype))
    assert torch.equal(state8_values(plain, scales, dtype), (plain.float() * each).square().to(dtype))


@pytest.mark.parametrize("gdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cautious", [False, True])
@pytest.mark.parametrize("sizes", [[1, 129, 5000], [3000000, 7], [(5 << 20) + 8192, 12], [(34 << 20) + 5]])
def test_fp32_moments_beside_bf16_parameters(sizes, gdt, cautious):
    """The moments equal those of an all-fp32 step bit for bit, and so do the parameters once they are rounded."""
    from dion_amd.functional import adamw_update_foreach

    gen = torch.Generator(device=DEV).manual_seed(3)
    rnd = lambda n, s: torch.empty(n, device=DEV).normal_(0, s, generator=gen)  # noqa: E731
    X = [rnd(n, 0.1).bfloat16() for n in sizes]
    G = [rnd(n, 0.02).to(gdt) for n in sizes]
    M, V = [rnd(n, 0.01) for n in sizes], [rnd(n, 0.01).square() for n in sizes]
    X32, M32, V32 = [x.float() for x in X], [m.clone() for m in M], [v.clone() for v in V]
    for xs, ms, vs in ((X, M, V), (X32, M32, V32)):
        adamw_update_foreach(xs, G, ms, vs, 0.01, B1, B2, 0.1, cautious_wd=cautious,
                             state_steps=[torch.full((), 4.0, device=DEV) for _ in sizes])
    for x, x32 in zip(X, X32):
        assert torch.equal(x, x32.bfloat16())
    assert all(torch.equal(a, b) for a, b in zip(M + V, M32 + V32))


def _param(t):
    p = torch.nn.Parameter(t)
    p.grad_dtype = None
    return p


@pytest.mark.parametrize("bits,dtype", [(8, torch.float32), (8, torch.bfloat16), (32, torch.bfloat16), (32, torch.float32)])
def test_group_option_state_dict_and_graph(bits, dtype):
    """An AdamW group with ``state_bits`` beside a Muon group: a checkpoint goes on where the run was, bit for bit, and so does a
    replayed graph."""
    from dion import Muon
    from dion_amd import HipGraphOptimizer

    def make():
        gen = torch.Generator().manual_seed(8)
        rnd = lambda *s: (torch.randn(*s, generator=gen) * 0.1).to(dtype).to(DEV)  # noqa: E731
        mats, rest = [_param(rnd(64, 128))], [_param(rnd(300, 33)), _param(rnd(257))]
        opt = Muon([{"params": mats}, {"params": rest, "algorithm": "adamw", "lr": 0.01, "state_bits": bits, "state_seed": 4}], lr=0.02)
        return mats + rest, opt

    def grads(params, k):
        gen = torch.Generator().manual_seed(100 + k)
        for p in params:
            g = (torch.randn(*p.shape, generator=gen) * 0.1).to(dtype).to(DEV)
            if p.grad is None:
                p.grad = g
            else:
                p.grad.copy_(g)

    params, opt = make()
    want = {8: {"momentum", "momentum_scale", "variance", "variance_scale", "step_dev"},
            32: {"momentum", "variance", "step_dev"}}[bits]
    assert set(opt.state[params[1]]) == want
    for k in range(2):
        grads(params, k)
        opt.step()
    saved = copy.deepcopy(opt.state_dict())  # (loading shares tensors of the right dtype, here Muon's momentum)
    held = [p.detach().clone() for p in params]
    other, opt2 = make()
    opt2.load_state_dict(saved)
    for p, h in zip(other, held):
        p.data.copy_(h)
    assert opt2.state[other[1]]["momentum"].dtype == (torch.int8 if bits == 8 else torch.float32)
    for k in range(2, 5):
        for ps, o in ((params, opt), (other, opt2)):
            grads(ps, k)
            o.step()
    assert all(torch.equal(a, b) for a, b in zip(params, other))

    third, inner = make()
    graph = HipGraphOptimizer(inner, warmup_steps=1)
    for k in range(5):
        grads(third, k)
        graph.step()
        torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(params, third))


def test_a_parameter_twice_and_counters_of_another_kind_are_refused():
    from dion_amd.functional import adamw8_update_foreach

    x, g = torch.zeros(300, device=DEV), torch.zeros(300, device=DEV)
    state = lambda: (torch.zeros(300, dtype=torch.int8, device=DEV), torch.zeros(3, device=DEV),  # noqa: E731
                     torch.zeros(300, dtype=torch.uint8, device=DEV), torch.zeros(3, device=DEV))
    lists = [list(t) for t in zip(state(), state())]
    steps = [torch.zeros((), device=DEV) for _ in range(2)]
    with pytest.raises(ValueError, match="twice"):
        adamw8_update_foreach([x, x], [g, g], *lists, 0.1, 0.9, 0.95, 0.0, state_steps=steps)
    with pytest.raises(TypeError, match="steps"):
        adamw8_update_foreach([x, x.clone()], [g, g], *lists, 0.1, 0.9, 0.95, 0.0, state_steps=[steps[0], torch.zeros(())])
    none = torch.zeros(0, device=DEV)  # (two empty parameters share an address, and nothing else)
    empty = [[t[:0], t[:0]] for t in state()]
    adamw8_update_foreach([none, none.clone()], [none, none], *empty, 0.1, 0.9, 0.95, 0.0, state_steps=steps)
    assert [float(s) for s in steps] == [1.0, 1.0]
