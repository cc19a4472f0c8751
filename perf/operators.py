"""The operators around an optimizer step, as cases that can be timed and compared.

Two kinds of case:

  ``linear``  the product a weight matrix stands for, ``y = act(x W^T + b) + residual``: its forward pass, or with
              ``train`` the forward pass and the gradients of x, W, b and the residual;
  ``adamw``   one AdamW update of many tensors whose first and second moments are kept in 8 bits (codes with a scale for
              every 128 elements) or in fp32 beside bf16 parameters.

The tensors of an ``adamw`` case lie in one allocation per kind, every tensor at a multiple of 128 elements, so that a pass
returns a few whole buffers instead of several hundred tensors.
"""
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BLOCK = 128  # elements that share a scale
BETA1, BETA2, EPSILON, LR, WEIGHT_DECAY, SEED = 0.9, 0.95, 1e-8, 1e-3, 0.01, 1234


def _linear(name, tokens, fan_in, fan_out, act, *, bias="none", residual=False, train=False):
    return {"name": name, "kind": "linear", "tokens": tokens, "fan_in": fan_in, "fan_out": fan_out, "act": act, "bias": bias,
            "residual": residual, "train": train}


def _adamw(name, layers, width, vocab, *, bits=8, param="fp32", grad="bf16", cautious=False):
    return {"name": name, "kind": "adamw", "layers": layers, "width": width, "vocab": vocab, "bits": bits, "param": param,
            "grad": grad, "cautious": cautious}


def listed():
    return [
        # One token through an attention output projection of a small model: nothing but latency.
        _linear("linear_1x768x768", 1, 768, 768, "none", bias="bf16", residual=True),
        # One token through the up projection of an 8B model: reads the weight once.
        _linear("linear_1x4096x14336", 1, 4096, 14336, "silu"),
        # A small batch of sequences that are decoded together, down projection of a 1.3B model.
        _linear("linear_32x8192x2048", 32, 8192, 2048, "none", bias="bf16", residual=True),
        # A ragged training batch of a gated model whose sizes fit no tile.
        _linear("linear_train_777x1000x2730", 777, 1000, 2730, "gelu", bias="bf16", residual=True, train=True),
        # Attention output projection of a 1.3B model, 2 sequences of 2048, fp32 bias.
        _linear("linear_train_4096x2048x2048", 4096, 2048, 2048, "none", bias="fp32", residual=True, train=True),
        # Up projection of the same model in training, squared ReLU: the three products of a weight.
        _linear("linear_train_8192x2048x8192", 8192, 2048, 8192, "relu_squared", train=True),
        # Up projection of an 8B model over a long prompt: the largest product.
        _linear("linear_16384x4096x14336", 16384, 4096, 14336, "silu"),
        # The norm weights of a 24-layer model alone, as beside matrices that Muon holds: launches, not bytes.
        _adamw("adamw8_norms_49x2048", 24, 2048, 0),
        # Embedding, head and norms of GPT-small: fp32 parameters, bf16 gradients.
        _adamw("adamw8_gpt_small", 12, 768, 50304),
        # A model kept in bf16 whose sizes fit no block, cautious weight decay.
        _adamw("adamw8_bf16_ragged", 6, 1001, 32003, param="bf16", cautious=True),
        # bf16 parameters whose moments stay in fp32, embedding and head of a 1.3B model.
        _adamw("adamw32_bf16_gpt_1p3b", 24, 2048, 50304, bits=32, param="bf16", grad="bf16"),
        # Embedding and head of an 8B model, fp32 gradients: the largest update.
        _adamw("adamw8_llama3_8b", 32, 4096, 32000, grad="fp32"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _extent(rng, lo, hi):
    v = _log_uniform(rng, lo, hi)
    grain = rng.choice((64, 64, 8, 1))
    return max(grain, (v + grain // 2) // grain * grain)


def draw(rng):
    top = {c["kind"]: work(c) for c in listed() if c["name"] in ("linear_16384x4096x14336", "adamw8_llama3_8b")}
    while True:
        if rng.random() < 0.6:
            act = rng.choice(("none", "none", "relu", "relu_squared", "gelu", "gelu_tanh", "silu"))
            case = _linear("", _log_uniform(rng, 1, 16384), _extent(rng, 64, 14336), _extent(rng, 64, 14336), act,
                           bias=rng.choice(("none", "bf16", "fp32" if act == "none" else "bf16")),
                           residual=rng.random() < 0.5, train=rng.random() < 0.5)
        else:
            bits = rng.choice((8, 8, 32))
            case = _adamw("", _log_uniform(rng, 1, 40), _extent(rng, 64, 4096), rng.choice((0, _log_uniform(rng, 256, 64000))),
                          bits=bits, param="bf16" if bits == 32 else rng.choice(("fp32", "bf16")),
                          grad=rng.choice(("bf16", "bf16", "fp32")), cautious=rng.random() < 0.3)
        del case["name"]
        w, most = work(case), top[case["kind"]]
        if w["flops"] <= most["flops"] and w["bytes"] <= most["bytes"]:
            return case


def _sizes(case):
    """Elements of each tensor of an ``adamw`` case: embedding, head, norms."""
    table = [case["vocab"] * case["width"]] * 2 if case["vocab"] else []
    return table + [case["width"]] * (2 * case["layers"] + 1)


def _placed(sizes):
    """(first element of each tensor, elements of the buffer)."""
    at, starts = 0, []
    for n in sizes:
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    return starts, at


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=gen).to(dtype)

    if case["kind"] == "linear":
        t, k, n = case["tokens"], case["fan_in"], case["fan_out"]
        state = {"case": case, "x": normal(t, k), "weight": normal(n, k, std=k ** -0.5), "bias": None, "residual": None}
        if case["bias"] != "none":
            state["bias"] = normal(n, std=0.1, dtype=DTYPES[case["bias"]])
        if case["residual"]:
            state["residual"] = normal(t, n)
        if case["train"]:
            state["dy"] = normal(t, n, std=0.01)
            for name in ("x", "weight", "bias", "residual"):
                if state[name] is not None:
                    state[name].requires_grad_()
        return state

    sizes = _sizes(case)
    starts, total = _placed(sizes)
    pdt, gdt = DTYPES[case["param"]], DTYPES[case["grad"]]
    # gradients differ from row to row as token frequencies do: a scale for each block, over two decades
    level = torch.empty(total // BLOCK, 1, device="cuda").normal_(-4.0, 1.0, generator=gen).exp_() * 0.02
    inside = torch.zeros(total, dtype=torch.bool, device="cuda")
    for s, n in zip(starts, sizes):
        inside[s:s + n] = True
    inside = inside.view(-1, BLOCK)
    x = (normal(total // BLOCK, BLOCK, std=0.02, dtype=torch.float32) * inside).to(pdt).view(-1)
    g = (normal(total // BLOCK, BLOCK, dtype=torch.float32) * level * inside).to(gdt).view(-1)
    m = normal(total // BLOCK, BLOCK, std=0.3, dtype=torch.float32) * level * inside
    v = (normal(total // BLOCK, BLOCK, std=0.25, dtype=torch.float32).exp_() * level * inside).square_()
    steps = torch.full((len(sizes),), 100.0, device="cuda")
    state = {"case": case, "x": x, "g": g, "steps": steps, "lr": torch.tensor(LR, device="cuda")}
    if case["bits"] == 8:
        ms = m.abs().amax(1) / 127
        vs = v.sqrt().amax(1) / 255
        state["m"] = (m / ms.clamp_min(1e-30)[:, None]).round_().to(torch.int8).view(-1)
        state["v"] = (v.sqrt() / vs.clamp_min(1e-30)[:, None]).round_().to(torch.uint8).view(-1)
        state["m_scale"], state["v_scale"] = ms, vs
        # where each block lies in its tensor
        first = torch.zeros(total // BLOCK, dtype=torch.int64, device="cuda")
        first[torch.tensor(starts, device="cuda") // BLOCK] = torch.tensor(starts, device="cuda") // BLOCK
        state["block"] = torch.arange(total // BLOCK, device="cuda") - first.cummax(0).values
    else:
        state["m"], state["v"] = m.view(-1), v.view(-1)

    def views(buffer):
        return [buffer[s:s + n] for s, n in zip(starts, sizes)]

    state["lists"] = {name: views(state[name]) for name in ("x", "g", "m", "v")}
    if case["bits"] == 8:
        for name in ("m_scale", "v_scale"):
            state["lists"][name] = [state[name][s // BLOCK:(s + n + BLOCK - 1) // BLOCK] for s, n in zip(starts, sizes)]
    state["lists"]["steps"] = list(steps.unbind(0))
    return state


def run(state):
    with torch.enable_grad():
        if state["case"]["kind"] == "linear":
            return _run_linear(state)
    with torch.no_grad():
        return _run_adamw(state)


# ---------------------------------------------------------------------------------------------- the product of a weight
def _act(z, act):
    """(act(z), act'(z))"""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if act == "relu_squared":
        p = z.clamp_min(0)
        return p * p, 2 * p
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    c, d = 0.7978845608028654, 0.044715
    t = torch.tanh(c * (z + d * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * d * z * z)


def _run_linear(state):
    case = state["case"]
    act = None if case["act"] == "none" else case["act"]
    x, weight, bias, residual = (state[k] for k in ("x", "weight", "bias", "residual"))
    leaves = {k: state[k] for k in ("x", "weight", "bias", "residual") if state[k] is not None}
    if own:
        from dion_amd import linear

        if not case["train"]:
            with torch.no_grad():
                return linear(x, weight, bias, activation=act, residual=residual)
        y = linear(x, weight, bias, activation=act, residual=residual)
        grads = torch.autograd.grad(y, list(leaves.values()), state["dy"])
        return {"y": y.detach(), **dict(zip(leaves, grads))}
    with torch.no_grad():
        xf, wf = x.float(), weight.float()
        z = xf @ wf.t()
        if bias is not None:
            z = z + bias.float()
        a, slope = _act(z, case["act"])
        y = (a if residual is None else a + residual.float()).to(torch.bfloat16)
        if not case["train"]:
            return y
        dz = state["dy"].float() * slope
        grads = {"x": (dz @ wf).to(x.dtype), "weight": (dz.t() @ xf).to(weight.dtype)}
        if bias is not None:
            grads["bias"] = dz.sum(0).to(bias.dtype)
        if residual is not None:
            grads["residual"] = state["dy"].to(residual.dtype)
        return {"y": y, **grads}


def _exact_linear(case, state):
    with torch.enable_grad():
        d = {k: state[k].detach().double().requires_grad_(case["train"])
             for k in ("x", "weight", "bias", "residual") if state[k] is not None}
        z = torch.nn.functional.linear(d["x"], d["weight"], d.get("bias"))
        a = {"none": lambda: z, "relu": lambda: z.relu(), "relu_squared": lambda: z.relu().square(),
             "silu": lambda: z * z.sigmoid(), "gelu": lambda: torch.nn.functional.gelu(z),
             "gelu_tanh": lambda: torch.nn.functional.gelu(z, approximate="tanh")}[case["act"]]()
        y = a + d["residual"] if "residual" in d else a
        if not case["train"]:
            return y
        grads = torch.autograd.grad(y, list(d.values()), state["dy"].double())
        return {"y": y.detach(), **dict(zip(d, grads))}


# ---------------------------------------------------------------------------------------------------------------- AdamW
def _mix(h):
    """A 32-bit number from a 32-bit number (held in int64)."""
    h = h ^ (h >> 16)
    h = (h * 0x6A09E667) & 0xFFFFFFFF
    h = h ^ (h >> 15)
    h = (h * 0xBB67AE85) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _noise(step, block):
    """[blocks, 128] numbers in [0, 1), multiples of 2^-24: one hash for eight neighbours of a tensor, then equal steps."""
    seed = _mix(torch.full((), SEED, dtype=torch.int64, device=block.device))
    key = _mix((seed + step.to(torch.int64)) & 0xFFFFFFFF)
    eight = torch.arange(BLOCK // 8, device=block.device)
    h = _mix(key ^ (block[:, None] * (BLOCK // 8) + eight))
    h = (h[:, :, None] + torch.arange(8, device=block.device) * 0x9E3779B9) & 0xFFFFFFFF
    return (h >> 8).view(-1, BLOCK)


def _codes(m, v, u):
    """First and second moments [blocks, 128] as (int8 codes, scales, uint8 codes, scales), rounded up or down by u."""
    top = m.abs().amax(1, keepdim=True)
    held = top >= 1e-30
    c = torch.floor(m * torch.where(held, 127 / top, 0.0) + u).clamp(-127, 127)
    r = v.sqrt()
    rtop = r.amax(1, keepdim=True)
    rheld = rtop >= 1e-30
    t = r * torch.where(rheld, 255 / rtop, 0.0)
    k = torch.floor(t).clamp_max(255)
    k = torch.where(u * (2 * k + 1) < (t - k) * (t + k), k + 1, k).clamp_max(255)
    k = torch.where((v > 0) & rheld, k.clamp_min(1), k)
    return c, torch.where(held, top / 127, 0.0), k, torch.where(rheld, rtop / 255, 0.0)


def _run_adamw(state):
    case, lists = state["case"], state["lists"]
    x, g, m, v, steps = (state[k] for k in ("x", "g", "m", "v", "steps"))
    if own:
        from dion_amd.functional import adamw8_update_foreach, adamw_update_foreach, state8_values

        if case["bits"] == 8:
            adamw8_update_foreach(lists["x"], lists["g"], lists["m"], lists["m_scale"], lists["v"], lists["v_scale"],
                                  state["lr"], BETA1, BETA2, WEIGHT_DECAY, state_steps=lists["steps"], epsilon=EPSILON,
                                  cautious_wd=case["cautious"], seed=SEED)
            return {"x": x, "steps": steps, "m": state8_values(m, state["m_scale"], torch.bfloat16),
                    "v": state8_values(v, state["v_scale"], torch.bfloat16)}
        adamw_update_foreach(lists["x"], lists["g"], lists["m"], lists["v"], state["lr"], BETA1, BETA2, WEIGHT_DECAY,
                             epsilon=EPSILON, cautious_wd=case["cautious"], state_steps=lists["steps"])
        return {"x": x, "steps": steps, "m": m, "v": v}

    steps += 1
    step = steps[0]
    b1, b2 = torch.tensor(BETA1, device="cuda"), torch.tensor(BETA2, device="cuda")
    xf, gf = x.float().view(-1, BLOCK), g.float().view(-1, BLOCK)
    if case["bits"] == 8:
        mf = m.float().view(-1, BLOCK) * state["m_scale"][:, None]
        vf = (v.float().view(-1, BLOCK) * state["v_scale"][:, None]).square()
    else:
        mf, vf = m.view(-1, BLOCK), v.view(-1, BLOCK)
    mf = mf + (1 - b1) * (gf - mf)
    vf = vf * b2 + (1 - b2) * (gf * gf)
    denom = vf.sqrt() * (1 / (1 - b2 ** step).sqrt()) + EPSILON
    update = mf / denom
    decay = state["lr"] * WEIGHT_DECAY
    if case["cautious"]:
        xf = torch.where(update * xf >= 0, xf - xf * decay, xf)
    else:
        xf = xf * (1 - decay)
    x.copy_((xf - state["lr"] / (1 - b1 ** step) * update).view(-1))
    if case["bits"] != 8:
        m.copy_(mf.view(-1))
        v.copy_(vf.view(-1))
        return {"x": x, "steps": steps, "m": m, "v": v}
    c, ms, k, vs = _codes(mf, vf, _noise(step, state["block"]).float() * 2.0 ** -24)
    m.copy_(c.view(-1))
    v.copy_(k.view(-1))
    state["m_scale"].copy_(ms.view(-1))
    state["v_scale"].copy_(vs.view(-1))
    return {"x": x, "steps": steps, "m": (c * ms).to(torch.bfloat16).view(-1),
            "v": (k * vs).square().to(torch.bfloat16).view(-1)}


def _exact_adamw(case, state):
    step = int(state["steps"][0]) + 1
    x, g = (state[k].double().view(-1, BLOCK) for k in ("x", "g"))
    lr = float(state["lr"])
    m, v = (state[k].double().view(-1, BLOCK) for k in ("m", "v"))
    if case["bits"] == 8:
        m = m * state["m_scale"].double()[:, None]
        v = v.mul(state["v_scale"].double()[:, None]) ** 2
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g ** 2
    update = (m / (1 - BETA1 ** step)) / ((v / (1 - BETA2 ** step)) ** 0.5 + EPSILON)
    keep = 1 - lr * WEIGHT_DECAY
    x = torch.where(update * x >= 0, x * keep, x) if case["cautious"] else x * keep
    x = x - lr * update
    if case["bits"] == 8:
        u = _noise(torch.tensor(step, device="cuda"), state["block"]).double() / 2 ** 24
        s = m.abs().amax(1, keepdim=True) / 127
        m = s * torch.nan_to_num(torch.floor(m / s + u)).clamp(-127, 127)
        q = v.amax(1, keepdim=True).sqrt() / 255
        w = torch.nan_to_num(v / q ** 2)  # between the squares of two codes
        low = w.sqrt().floor()
        code = torch.where(u < (w - low ** 2) / (2 * low + 1), low + 1, low).clamp(max=255)
        code = torch.where(v > 0, code.clamp(min=1), code)
        v = (code * q) ** 2
    return {"x": x.view(-1), "steps": state["steps"].double() + 1, "m": m.reshape(-1), "v": v.reshape(-1)}


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "linear":
        return _exact_linear(case, state)
    with torch.no_grad():
        return _exact_adamw(case, state)


def work(case):
    if case["kind"] == "linear":
        t, k, n = case["tokens"], case["fan_in"], case["fan_out"]
        nbytes = 2 * (t * k + n * k + t * n) + n * {"none": 0, "bf16": 2, "fp32": 4}[case["bias"]]
        nbytes += 2 * t * n if case["residual"] else 0
        if not case["train"]:
            return {"bytes": float(nbytes), "flops": 2.0 * t * n * k}
        # dy read, the gradients of x, W and b written
        nbytes += 2 * (t * n + t * k + n * k) + n * {"none": 0, "bf16": 2, "fp32": 4}[case["bias"]]
        return {"bytes": float(nbytes), "flops": 6.0 * t * n * k}
    p, g = (2 if case[k] == "bf16" else 4 for k in ("param", "grad"))
    # 8 bits: two codes and 1/128 of two scales read and written, and the values they stand for written in bf16
    per = 2 * p + g + (4 + 16 / BLOCK + 4 if case["bits"] == 8 else 16)
    return {"bytes": float(sum(_sizes(case)) * per), "flops": 30.0 * sum(_sizes(case))}
