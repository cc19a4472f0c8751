"""The layers around the matrices that the optimizers update, as cases that can be timed and compared.

Three kinds of case:

  ``gated``      both projections of a gated feed-forward block, ``h = act(x Wg^T + bg) * (x Wu^T + bu)``;
  ``norm``       layer norm, ``y = (x - mean) / sqrt(var + eps) * w + b``;
  ``embedding``  rows of a table, ``y[t] = scale W[ids[t]]``, whose gradient adds the rows of equal tokens.

Each runs its forward pass, or with ``train`` the forward pass and the gradients of all its inputs.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp32": 4, "int32": 4, "int64": 8}
EPS = 1e-5


def _gated(name, tokens, fan_in, fan_out, act, *, bias="none", train=False):
    return {"name": name, "kind": "gated", "tokens": tokens, "fan_in": fan_in, "fan_out": fan_out, "act": act, "bias": bias,
            "train": train}


def _norm(name, rows, width, *, x="bf16", y="bf16", param="fp32", weight=True, bias=True, train=False):
    return {"name": name, "kind": "norm", "rows": rows, "width": width, "x": x, "y": y, "param": param, "weight": weight,
            "bias": bias, "train": train}


def _embedding(name, tokens, vocab, width, *, table="fp32", y="bf16", ids="int64", scaled=False, padded=False, train=False):
    return {"name": name, "kind": "embedding", "tokens": tokens, "vocab": vocab, "width": width, "table": table, "y": y,
            "ids": ids, "scaled": scaled, "padded": padded, "train": train}


def listed():
    return [
        # One token through a small model: nothing but latency.
        _gated("gated_1x768x2048", 1, 768, 2048, "silu"),
        # One token through an 8B model: reads both weights once.
        _gated("gated_1x4096x14336", 1, 4096, 14336, "silu"),
        # Sequences that are decoded together, a 1.3B model with biases.
        _gated("gated_24x2048x8192", 24, 2048, 8192, "gelu_tanh", bias="bf16"),
        # A ragged training batch whose sizes fit no tile.
        _gated("gated_train_777x1000x2730", 777, 1000, 2730, "gelu", bias="fp32", train=True),
        # A training step of a 1.3B model, 4 sequences of 2048.
        _gated("gated_train_8192x2048x5632", 8192, 2048, 5632, "silu", train=True),
        # An 8B model over a long prompt: the largest products.
        _gated("gated_8192x4096x14336", 8192, 4096, 14336, "silu"),
        # One token of a small model.
        _norm("norm_1x768", 1, 768),
        # A ragged batch in full precision.
        _norm("norm_train_777x1001", 777, 1001, x="fp32", y="fp32", train=True),
        # A training batch of an 8B model, the weight's and the bias's gradients reduced over 16384 rows.
        _norm("norm_train_16384x4096", 16384, 4096, train=True),
        # The next tokens of 32 sequences, a table whose sizes fit no chunk.
        _embedding("embedding_32x32003x1001", 32, 32003, 1001, table="bf16"),
        # GPT-small, 16 padded sequences of 512: most of the table's gradient is zeros.
        _embedding("embedding_train_8192x50304x768", 8192, 50304, 768, padded=True, train=True),
        # An 8B model, 16 sequences of 2048, a table kept in bf16 and scaled as a tied head needs it.
        _embedding("embedding_train_32768x32000x4096", 32768, 32000, 4096, table="bf16", scaled=True, train=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _extent(rng, lo, hi):
    v = _log_uniform(rng, lo, hi)
    grain = rng.choice((64, 64, 8, 1))
    return max(grain, (v + grain // 2) // grain * grain)


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        top = most.setdefault(c["kind"], {"bytes": 0.0, "flops": 0.0})
        for k in top:
            top[k] = max(top[k], w[k])
    while True:
        kind = rng.choice(("gated", "gated", "norm", "embedding"))
        if kind == "gated":
            act = rng.choice(("none", "relu", "relu_squared", "gelu", "gelu_tanh", "silu", "silu"))
            case = _gated("", _log_uniform(rng, 1, 16384), _extent(rng, 64, 8192), _extent(rng, 64, 14336), act,
                          bias=rng.choice(("none", "none", "bf16", "fp32")), train=rng.random() < 0.5)
        elif kind == "norm":
            x = rng.choice(("bf16", "bf16", "fp32"))
            weight = rng.random() < 0.8
            case = _norm("", _log_uniform(rng, 1, 65536), _extent(rng, 64, 16384), x=x, y=rng.choice((x, "bf16")),
                         param=rng.choice(("fp32", "bf16")), weight=weight, bias=weight and rng.random() < 0.7,
                         train=rng.random() < 0.6)
        else:
            table = rng.choice(("fp32", "bf16"))
            case = _embedding("", _log_uniform(rng, 1, 131072), _log_uniform(rng, 256, 131072), _extent(rng, 64, 4096),
                              table=table, y=rng.choice((table, "bf16")), ids=rng.choice(("int64", "int32")),
                              scaled=rng.random() < 0.5, padded=rng.random() < 0.4, train=rng.random() < 0.7)
        del case["name"]
        w = work(case)
        if all(w[k] <= most[kind][k] for k in w):
            return case


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=gen).to(dtype)

    state = {"case": case}
    if case["kind"] == "gated":
        t, k, n = case["tokens"], case["fan_in"], case["fan_out"]
        leaves = {"x": normal(t, k), "weight_gate": normal(n, k, std=k ** -0.5), "weight_up": normal(n, k, std=k ** -0.5)}
        if case["bias"] != "none":
            leaves["bias_gate"] = normal(n, std=0.1, dtype=DTYPES[case["bias"]])
            leaves["bias_up"] = normal(n, std=0.1, dtype=DTYPES[case["bias"]])
        if case["train"]:
            state["dy"] = normal(t, n, std=0.01)
    elif case["kind"] == "norm":
        t, d = case["rows"], case["width"]
        # a residual stream: rows of different sizes, a few columns that stand out in all of them
        size = normal(t, 1, std=0.5, dtype=torch.float32).exp_()
        column = normal(1, d, std=0.3, dtype=torch.float32)
        column = torch.where(column.abs() > 0.9, 10 * column, column)
        leaves = {"x": ((normal(t, d, dtype=torch.float32) + column) * size).to(DTYPES[case["x"]])}
        if case["weight"]:
            leaves["weight"] = (1 + normal(d, std=0.2, dtype=torch.float32)).to(DTYPES[case["param"]])
        if case["bias"]:
            leaves["bias"] = normal(d, std=0.1, dtype=DTYPES[case["param"]])
        if case["train"]:
            state["dy"] = normal(t, d, std=0.01, dtype=DTYPES[case["y"]])
    else:
        t, v, d = case["tokens"], case["vocab"], case["width"]
        # tokens as frequent as one over their rank, the most frequent ones first in the table
        u = torch.empty(t, device="cuda", dtype=torch.float64).uniform_(0.0, 1.0, generator=gen)
        ids = ((v + 1.0) ** u).long().sub_(1).clamp_(0, v - 1)
        state["padding_idx"] = None
        if case["padded"]:  # sequences of up to 512
            length = torch.empty(t // 512 + 1, device="cuda").uniform_(200.0, 513.0, generator=gen).long()
            at = torch.arange(t, device="cuda")
            ids = torch.where(at % 512 >= length[at // 512], v - 1, ids)
            state["padding_idx"] = v - 1
        state["ids"] = ids.to(torch.int32 if case["ids"] == "int32" else torch.int64)
        state["scale"] = math.sqrt(d) if case["scaled"] else 1.0
        leaves = {"weight": normal(v, d, std=0.02, dtype=DTYPES[case["table"]])}
        if case["train"]:
            state["dy"] = normal(t, d, std=0.01, dtype=DTYPES[case["y"]])
    if case["train"]:
        for leaf in leaves.values():
            leaf.requires_grad_()
    state["leaves"] = leaves
    return state


def run(state):
    case, leaves = state["case"], state["leaves"]
    if not own:
        with torch.no_grad():
            return {"gated": _plain_gated, "norm": _plain_norm, "embedding": _plain_embedding}[case["kind"]](state)
    from dion_amd import embedding, gated_linear, layer_norm

    with torch.set_grad_enabled(case["train"]):
        if case["kind"] == "gated":
            act = None if case["act"] == "none" else case["act"]
            y = gated_linear(leaves["x"], leaves["weight_gate"], leaves["weight_up"], leaves.get("bias_gate"),
                             leaves.get("bias_up"), activation=act)
        elif case["kind"] == "norm":
            y = layer_norm(leaves["x"], leaves.get("weight"), leaves.get("bias"), eps=EPS, dtype=DTYPES[case["y"]])
        else:
            y = embedding(state["ids"], leaves["weight"], scale=state["scale"], padding_idx=state["padding_idx"],
                          dtype=DTYPES[case["y"]])
        if not case["train"]:
            return {"y": y}
        grads = torch.autograd.grad(y, list(leaves.values()), state["dy"])
        return {"y": y.detach(), **dict(zip(leaves, grads))}


# ------------------------------------------------------------------------------------------------------------ plain forms
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


def _plain_gated(state):
    case, leaves = state["case"], state["leaves"]
    x, wg, wu = (leaves[k].float() for k in ("x", "weight_gate", "weight_up"))
    g, u = x @ wg.t(), x @ wu.t()
    if case["bias"] != "none":
        g, u = g + leaves["bias_gate"].float(), u + leaves["bias_up"].float()
    a, slope = _act(g, case["act"])
    out = {"y": (a * u).to(torch.bfloat16)}
    if not case["train"]:
        return out
    dy = state["dy"].float()
    dg, du = dy * u * slope, dy * a
    out["x"] = (dg @ wg + du @ wu).to(torch.bfloat16)
    out["weight_gate"] = (dg.t() @ x).to(torch.bfloat16)
    out["weight_up"] = (du.t() @ x).to(torch.bfloat16)
    if case["bias"] != "none":
        out["bias_gate"] = dg.sum(0).to(leaves["bias_gate"].dtype)
        out["bias_up"] = du.sum(0).to(leaves["bias_up"].dtype)
    return out


def _plain_norm(state):
    case, leaves = state["case"], state["leaves"]
    x = leaves["x"].float()
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    rstd = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPS)
    xhat = centred * rstd
    y = xhat
    if case["weight"]:
        y = y * leaves["weight"].float()
    if case["bias"]:
        y = y + leaves["bias"].float()
    out = {"y": y.to(DTYPES[case["y"]])}
    if not case["train"]:
        return out
    dy = state["dy"].float()
    dxhat = dy * leaves["weight"].float() if case["weight"] else dy
    dx = rstd * (dxhat - dxhat.mean(1, keepdim=True) - xhat * (dxhat * xhat).mean(1, keepdim=True))
    out["x"] = dx.to(leaves["x"].dtype)
    if case["weight"]:
        out["weight"] = (dy * xhat).sum(0).to(leaves["weight"].dtype)
    if case["bias"]:
        out["bias"] = dy.sum(0).to(leaves["bias"].dtype)
    return out


def _plain_embedding(state):
    case, weight, ids = state["case"], state["leaves"]["weight"], state["ids"]
    out = {"y": (weight[ids].float() * state["scale"]).to(DTYPES[case["y"]])}
    if not case["train"]:
        return out
    dy = state["dy"].float()
    if case["padded"]:
        dy = torch.where((ids == state["padding_idx"])[:, None], 0.0, dy)
    sums = torch.zeros(weight.shape, device=weight.device).index_add_(0, ids, dy)
    out["weight"] = (sums * state["scale"]).to(weight.dtype)
    return out


# ----------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    leaves = {k: v.detach().double().requires_grad_(case["train"]) for k, v in state["leaves"].items()}
    with torch.enable_grad():
        if case["kind"] == "gated":
            g = torch.nn.functional.linear(leaves["x"], leaves["weight_gate"], leaves.get("bias_gate"))
            a = {"none": lambda: g, "relu": lambda: g.relu(), "relu_squared": lambda: g.relu().square(),
                 "silu": lambda: g * g.sigmoid(), "gelu": lambda: torch.nn.functional.gelu(g),
                 "gelu_tanh": lambda: torch.nn.functional.gelu(g, approximate="tanh")}[case["act"]]()
            y = a * torch.nn.functional.linear(leaves["x"], leaves["weight_up"], leaves.get("bias_up"))
        elif case["kind"] == "norm":
            var, mean = torch.var_mean(leaves["x"], dim=1, correction=0, keepdim=True)
            y = (leaves["x"] - mean) * torch.rsqrt(var + EPS)
            y = y * leaves.get("weight", 1.0) + leaves.get("bias", 0.0)
        else:
            y = state["scale"] * leaves["weight"].detach().index_select(0, state["ids"])
        if not case["train"]:
            return {"y": y.detach()}
        dy = state["dy"].double()
        if case["kind"] == "embedding":
            keep = torch.ones_like(state["ids"], dtype=torch.bool)
            if state["padding_idx"] is not None:
                keep = state["ids"] != state["padding_idx"]
            grad = torch.zeros_like(leaves["weight"].detach())
            return {"y": y, "weight": grad.index_add_(0, state["ids"][keep], dy[keep], alpha=state["scale"])}
        return {"y": y.detach(), **dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))}


def _distinct(tokens, vocab, padded):
    """How many rows of the table the tokens are expected to name."""
    rank = torch.arange(1, vocab + 1, dtype=torch.float64)
    share = torch.log1p(1 / rank) / math.log(vocab + 1)
    return min(float(vocab), float((1 - (1 - share) ** (0.7 * tokens if padded else tokens)).sum()) + padded)


def work(case):
    train = case["train"]
    if case["kind"] == "gated":
        t, k, n = case["tokens"], case["fan_in"], case["fan_out"]
        bias = 2 * n * BYTES.get(case["bias"], 0)
        nbytes = 2 * (t * k + 2 * n * k + t * n) + bias
        if train:  # dy read, the gradients of x, both weights and both biases written
            nbytes += 2 * (t * n + t * k + 2 * n * k) + bias
        return {"bytes": float(nbytes), "flops": (12.0 if train else 4.0) * t * n * k}
    if case["kind"] == "norm":
        t, d = case["rows"], case["width"]
        params = d * BYTES[case["param"]] * (case["weight"] + case["bias"])
        nbytes = t * d * (BYTES[case["x"]] + BYTES[case["y"]]) + params
        if train:  # dy read, the gradients written; x once for both passes
            nbytes += t * d * (BYTES[case["x"]] + BYTES[case["y"]]) + params
        return {"bytes": float(nbytes), "flops": (20.0 if train else 8.0) * t * d}
    t, v, d = case["tokens"], case["vocab"], case["width"]
    nbytes = t * BYTES[case["ids"]] + _distinct(t, v, case["padded"]) * d * BYTES[case["table"]] + t * d * BYTES[case["y"]]
    if train:  # dy read, the whole gradient of the table written
        nbytes += t * d * BYTES[case["y"]] + v * d * BYTES[case["table"]]
    return {"bytes": float(nbytes), "flops": (2.0 if train else 1.0) * t * d}
