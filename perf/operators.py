"""Sequence-policy layers and losses: what one pass of each costs.

Three operators of ``d3rlpy_amd.torch_ops``, forward alone and with their
gradients: the layer norm, the gated feed-forward block, and the softmax
cross entropy of a linear head over a large vocabulary of discrete actions.

``listed()`` names the cases, ``prepare`` makes one case's inputs on the GPU,
``run`` is one pass.  With ``own`` false a pass is the plain form, elementary
torch operations in float32; with ``own`` true it is the framework's call.
``exact`` is the definition in float64.
"""
import math

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
_EPS = 1e-5
_IGNORE = -100


# ------------------------------------------------------------------- the cases
def _norm(name, rows, width, dtype, train, members=1):
    return {"name": name, "op": "layer_norm", "members": members, "rows": rows, "width": width,
            "dtype": dtype, "train": train}


def _gated(name, rows, width, hidden, dtype, train, members=1, bias=False, activation="silu"):
    return {"name": name, "op": "gated_mlp", "members": members, "rows": rows, "width": width,
            "hidden": hidden, "dtype": dtype, "train": train, "bias": bias,
            "activation": activation}


def _entropy(name, rows, width, vocab, dtype, train, ignored=0.0, bias=False):
    return {"name": name, "op": "linear_cross_entropy", "rows": rows, "width": width,
            "vocab": vocab, "dtype": dtype, "train": train, "ignored": ignored, "bias": bias}


def listed():
    return [
        # two critics' hidden layer of 256 over one minibatch of 256: launches bound it
        _norm("norm_critics_f32", 256, 256, "float32", True, members=2),
        # one decoded token's normalisation
        _norm("norm_token_bf16", 1, 2048, "bfloat16", False),
        # a training batch of 8192 tokens: memory bound
        _norm("norm_train_bf16", 8192, 2048, "bfloat16", True),
        # odd rows and an odd width, so that no row but the first is aligned
        _norm("norm_ragged_f32", 3001, 1537, "float32", True),
        # two gated critics of hidden width 256 with biases, one minibatch
        _gated("gated_critics_f32", 256, 256, 512, "float32", True, members=2, bias=True),
        # one decoded token: the weights are read once
        _gated("gated_token_bf16", 1, 2048, 5632, "bfloat16", False),
        # a training batch of 8192 tokens: matrix products
        _gated("gated_train_bf16", 8192, 1024, 4096, "bfloat16", True),
        # odd everything, at full precision
        _gated("gated_ragged_f32", 1999, 513, 1366, "float32", True, bias=True,
               activation="gelu"),
        # a minibatch of discrete actions behind a 256 wide trunk
        _entropy("entropy_batch_f32", 256, 256, 1024, "float32", True, bias=True),
        # scoring a few tokens against the whole vocabulary: the weights are read once
        _entropy("entropy_score_bf16", 8, 1024, 65536, "bfloat16", False),
        # a training batch of 8192 tokens, some of them padding
        _entropy("entropy_train_bf16", 8192, 1024, 32768, "bfloat16", True, ignored=0.1),
        # an odd vocabulary and width at full precision, a third of it padding
        _entropy("entropy_ragged_f32", 1500, 777, 10007, "float32", True, ignored=0.33,
                 bias=True),
    ]


def _size(rng, low, high):
    """Whole numbers from low to high, even over their logarithm; two in five are round."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.4:
        for step in (256, 64, 16):
            if v >= 2 * step:
                v -= v % step
                break
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(("layer_norm", "gated_mlp", "linear_cross_entropy"))
    dtype = rng.choice(("float32", "bfloat16"))
    train = rng.random() < 0.7
    if op == "layer_norm":
        case = _norm("", _size(rng, 1, 8192), _size(rng, 16, 4096), dtype, train,
                     rng.choice((1, 1, 2, 3)))
        most, axis = 8192 * 2048, "rows"

        def cost(c):
            return c["members"] * c["rows"] * c["width"]
    elif op == "gated_mlp":
        case = _gated("", _size(rng, 1, 8192), _size(rng, 16, 2048), _size(rng, 16, 5632), dtype,
                      train, rng.choice((1, 1, 2)), rng.random() < 0.5,
                      rng.choice(("silu", "silu", "gelu", "relu")))
        most, axis = 8192 * 1024 * 4096 // (8 if dtype == "float32" else 1), "rows"

        def cost(c):
            return c["members"] * c["rows"] * c["width"] * c["hidden"]
    else:
        case = _entropy("", _size(rng, 1, 8192), _size(rng, 16, 1024), _size(rng, 2, 65536),
                        dtype, train, rng.choice((0.0, 0.1, 0.5)), rng.random() < 0.3)
        most, axis = 8192 * 1024 * 32768 // (16 if dtype == "float32" else 1), "rows"

        def cost(c):
            return c["rows"] * c["width"] * c["vocab"]
    if cost(case) > most:
        case[axis] = max(1, int(case[axis] * most / cost(case)))
    del case["name"]
    return case


# ------------------------------------------------------------------- the inputs
def _normal(gen, shape, dtype, scale=1.0, shift=0.0):
    t = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return t.mul_(scale).add_(shift).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    state = dict(case)
    D, R = case["width"], case["rows"]
    lead = (case["members"],) if case.get("members", 1) > 1 else ()
    if case["op"] == "layer_norm":
        # residual-stream values: features of unlike scales and means
        x = _normal(gen, lead + (R, D), torch.float32)
        x = x.mul_(_normal(gen, (D,), torch.float32).abs_().add_(0.3))
        x = x.add_(_normal(gen, (D,), torch.float32, 0.5)).to(dtype)
        state |= {"x": x, "weight": _normal(gen, lead + (D,), dtype, 0.1, 1.0),
                  "bias": _normal(gen, lead + (D,), dtype, 0.1),
                  "dy": _normal(gen, x.shape, dtype, 0.05)}
        leaves = ("x", "weight", "bias")
    elif case["op"] == "gated_mlp":
        F = case["hidden"]
        state |= {"x": _normal(gen, lead + (R, D), dtype),
                  "Wg": _normal(gen, lead + (F, D), dtype, D ** -0.5),
                  "Wu": _normal(gen, lead + (F, D), dtype, D ** -0.5),
                  "Wd": _normal(gen, lead + (D, F), dtype, F ** -0.5),
                  "dy": _normal(gen, lead + (R, D), dtype, 0.05)}
        leaves = ("x", "Wg", "Wu", "Wd")
        if case["bias"]:
            state |= {"bg": _normal(gen, lead + (F,), dtype, 0.1),
                      "bu": _normal(gen, lead + (F,), dtype, 0.1),
                      "bd": _normal(gen, lead + (D,), dtype, 0.1)}
            leaves += ("bg", "bu", "bd")
    else:
        V = case["vocab"]
        target = torch.randint(0, V, (R,), generator=gen, device="cuda")
        pad = torch.rand((R,), generator=gen, device="cuda") < case["ignored"]
        state |= {"x": _normal(gen, (R, D), dtype), "W": _normal(gen, (V, D), dtype, 2 * D ** -0.5),
                  "target": target.masked_fill_(pad, _IGNORE)}
        leaves = ("x", "W")
        if case["bias"]:
            state["b"] = _normal(gen, (V,), dtype, 0.5)
            leaves += ("b",)
    state["leaves"] = leaves
    if case["train"]:
        for k in leaves:
            state[k].requires_grad_(True)
    return state


# --------------------------------------------------------------- the plain forms
def _out(values, dtype):
    return {k: v.to(dtype) for k, v in values.items()}


def _plain_layer_norm(s):
    x, w = s["x"].float(), s["weight"].float().unsqueeze(-2)
    xc = x - x.mean(-1, keepdim=True)
    rstd = ((xc * xc).mean(-1, keepdim=True) + _EPS).rsqrt()
    xh = xc * rstd
    out = {"y": xh * w + s["bias"].float().unsqueeze(-2)}
    if s["train"]:
        dy = s["dy"].float()
        g = dy * w
        out["x"] = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
        out["weight"] = (dy * xh).sum(-2)
        out["bias"] = dy.sum(-2)
    return _out(out, s["x"].dtype)


def _act(name, g):
    """The activation and its derivative."""
    if name == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    sig = 1 / (1 + torch.exp(-g))
    return g * sig, sig * (1 + g * (1 - sig))


def _plain_gated_mlp(s):
    x, wg, wu, wd = (s[k].float() for k in ("x", "Wg", "Wu", "Wd"))
    g, u = x @ wg.transpose(-1, -2), x @ wu.transpose(-1, -2)
    if s["bias"]:
        g, u = g + s["bg"].float().unsqueeze(-2), u + s["bu"].float().unsqueeze(-2)
    a, da = _act(s["activation"], g)
    h = a * u
    y = h @ wd.transpose(-1, -2)
    out = {"y": y + s["bd"].float().unsqueeze(-2) if s["bias"] else y}
    if s["train"]:
        dy = s["dy"].float()
        dh = dy @ wd
        dg, du = dh * u * da, dh * a
        out["x"] = dg @ wg + du @ wu
        out["Wg"] = dg.transpose(-1, -2) @ x
        out["Wu"] = du.transpose(-1, -2) @ x
        out["Wd"] = dy.transpose(-1, -2) @ h
        if s["bias"]:
            out["bg"], out["bu"], out["bd"] = dg.sum(-2), du.sum(-2), dy.sum(-2)
    return _out(out, s["x"].dtype)


def _plain_linear_cross_entropy(s):
    x, w, t = s["x"].float(), s["W"].float(), s["target"]
    z = x @ w.transpose(0, 1)
    if s["bias"]:
        z = z + s["b"].float()
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    kept = t != _IGNORE
    at = torch.where(kept, t, 0).unsqueeze(-1)
    loss = (total.log() + top - z.gather(-1, at)).squeeze(-1)
    loss = torch.where(kept, loss, 0.0)
    if not s["train"]:
        return {"loss": loss}
    share = kept.float() / kept.sum().clamp(min=1)
    dz = e / total
    dz.scatter_add_(-1, at, torch.full_like(at, -1, dtype=dz.dtype))
    dz = dz * share.unsqueeze(-1)
    grads = {"x": dz @ w, "W": dz.transpose(0, 1) @ x}
    if s["bias"]:
        grads["b"] = dz.sum(0)
    return {"loss": (loss * share).sum()} | _out(grads, s["x"].dtype)


# -------------------------------------------------------------- the framework's
def _own_layer_norm(s):
    from d3rlpy_amd import torch_ops
    y = torch_ops.layer_norm(s["x"], s["weight"], s["bias"], _EPS)
    return "y", y, s["dy"]


def _own_gated_mlp(s):
    from d3rlpy_amd import torch_ops
    y = torch_ops.gated_mlp(s["x"], s["Wg"], s["Wu"], s["Wd"], s.get("bg"), s.get("bu"),
                            s.get("bd"), activation=s["activation"])
    return "y", y, s["dy"]


def _own_linear_cross_entropy(s):
    from d3rlpy_amd import torch_ops
    loss = torch_ops.linear_cross_entropy(s["x"], s["W"], s["target"], s.get("b"),
                                          ignore_index=_IGNORE,
                                          reduction="mean" if s["train"] else "none")
    return "loss", loss, None


def run(state):
    if own:
        name, out, dy = {"layer_norm": _own_layer_norm, "gated_mlp": _own_gated_mlp,
                         "linear_cross_entropy": _own_linear_cross_entropy}[state["op"]](state)
        if not state["train"]:
            return {name: out}
        grads = torch.autograd.grad(out, [state[k] for k in state["leaves"]], dy)
        return {name: out.detach()} | dict(zip(state["leaves"], grads))
    with torch.no_grad():
        return {"layer_norm": _plain_layer_norm, "gated_mlp": _plain_gated_mlp,
                "linear_cross_entropy": _plain_linear_cross_entropy}[state["op"]](state)


# ------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    leaf = {k: s[k].detach().double().requires_grad_(case["train"]) for k in s["leaves"]}
    if case["op"] == "layer_norm":
        var, mean = torch.var_mean(leaf["x"], -1, correction=0, keepdim=True)
        out = (leaf["x"] - mean) / torch.sqrt(var + _EPS) * leaf["weight"].unsqueeze(-2) \
            + leaf["bias"].unsqueeze(-2)
        name, dy = "y", s["dy"].double()
    elif case["op"] == "gated_mlp":
        def product(x, w, b):
            y = torch.matmul(x, leaf[w].transpose(-1, -2).contiguous())
            return y + leaf[b].unsqueeze(-2) if case["bias"] else y

        g = product(leaf["x"], "Wg", "bg")
        if case["activation"] == "silu":
            a = g / (1 + torch.exp(-g))
        elif case["activation"] == "gelu":
            a = g * torch.special.ndtr(g)
        else:
            a = g.clamp(min=0)
        out = product(a * product(leaf["x"], "Wu", "bu"), "Wd", "bd")
        name, dy = "y", s["dy"].double()
    else:
        z = torch.matmul(leaf["x"], leaf["W"].transpose(0, 1).contiguous())
        if case["bias"]:
            z = z + leaf["b"]
        kept = (s["target"] != _IGNORE).nonzero().squeeze(-1)
        rows = torch.logsumexp(z[kept], -1) - z[kept, s["target"][kept]]
        name, dy = "loss", None
        if case["train"]:
            out = rows.sum() / max(1, kept.numel())
        else:
            out = torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
            out[kept] = rows.detach()
    if not case["train"]:
        return {name: out}
    grads = torch.autograd.grad(out, list(leaf.values()), dy)
    return {name: out.detach()} | dict(zip(leaf, grads))


# ------------------------------------------------------------------------ work
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    R, D, C = case["rows"], case["width"], case.get("members", 1)
    train = case["train"]
    if case["op"] == "layer_norm":
        # x in, y out (training: dy in, dx out); weight and bias in (their gradients out)
        return {"bytes": size * C * D * ((4 if train else 2) * R + (4 if train else 2)),
                "flops": C * R * D * (19 if train else 8)}
    if case["op"] == "gated_mlp":
        F = case["hidden"]
        weights = 3 * D * F + (2 * F + D if case["bias"] else 0)
        return {"bytes": size * C * ((4 if train else 2) * R * D + (2 if train else 1) * weights),
                "flops": C * 6 * R * D * F * (3 if train else 1)}
    V = case["vocab"]
    weights = V * D + (V if case["bias"] else 0)
    # training: the logits once, and the two products of their gradient
    return {"bytes": size * ((2 if train else 1) * (R * D + weights)) + R * 8
            + (4 if train else 4 * R),
            "flops": (3 if train else 1) * 2 * R * D * V}
