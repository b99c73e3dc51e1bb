"""float64 forms of layer_norm, gated_mlp and linear_cross_entropy, each value
with a bound on how far a kernel may be from it.

A bound follows the kernel's roundings.  ``u`` is half a step of float32,
2^-24; ``ut`` half a step of the tensors' type (bfloat16: 2^-8).  A float32 sum
of n products whose magnitudes add up to S is off by at most (n / 16 + 40) u S:
a matrix instruction adds 16 at a time and the instructions chain, the split
of a float32 operand and the joins of partial sums are within the 40.  A value
stored in the tensors' type adds ut times its magnitude.  The kernels' exp,
reciprocal, erf and log are good to a few u: 8 u where one is used.
"""
import math

import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TINY = 1e-37  # results under the normal range


def acc(n):
    return (n / 16 + 40) * U


def within(got, want, bound, what):
    got = got.detach().double().cpu()
    want, bound = want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound + TINY)
    if bool(bad.any()):
        i = int(((got - want).abs() / (bound + TINY)).nan_to_num(nan=1e30).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst at {i}: "
                             f"{got.flatten()[i]} for {want.flatten()[i]}, bound "
                             f"{bound.flatten()[i]}")


def _t(a):
    return a.transpose(-1, -2)


def norm_reference(x, w, b, eps, dy):
    """{name: (value, bound)} of y, x, weight, bias gradients; w, b [.., 1, n]."""
    ut, uw = HALF[x.dtype], HALF[w.dtype]
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    n = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    var = (xc * xc).mean(-1, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    xh = xc * rstd
    # a lane's chain of up to 64 values (rows over 8192: n / 256), then a tree
    u = (80 + n / 256) * U
    e_mean = u * x.abs().mean(-1, keepdim=True)
    e_xc = e_mean + u * xc.abs()
    e_rstd = rstd * (u + 2 * (e_xc * xc.abs()).mean(-1, keepdim=True) * rstd * rstd)
    e_xh = e_xc * rstd + xc.abs() * e_rstd + 2 * U * xh.abs()
    y = xh * w + b
    out = {"y": (y, e_xh * w.abs() + 4 * U * (xh * w).abs() + (2 * U + ut) * y.abs())}
    t = dy * w
    m0, m1 = t.mean(-1, keepdim=True), (t * xh).mean(-1, keepdim=True)
    inner = t - m0 - xh * m1
    e_inner = (4 * U * t.abs() + u * t.abs().mean(-1, keepdim=True)
               + e_xh * m1.abs()
               + xh.abs() * ((e_xh * t.abs()).mean(-1, keepdim=True)
                             + u * (t * xh).abs().mean(-1, keepdim=True)) + 4 * U * inner.abs())
    dx = inner * rstd
    out["x"] = (dx, e_inner * rstd + inner.abs() * e_rstd + (2 * U + ut) * dx.abs())
    rows = x.shape[-2]
    dw, db = (dy * xh).sum(-2), dy.sum(-2)
    out["weight"] = (dw, (e_xh * dy.abs()).sum(-2) + (rows + 8) * U * (dy * xh).abs().sum(-2)
                     + uw * dw.abs())
    out["bias"] = (db, (rows + 8) * U * dy.abs().sum(-2) + uw * db.abs())
    return out


def _activation(name, g):
    """act, act', and bounds on |act'| and |act''| near g."""
    if name == "relu":
        on = (g > 0).double()
        return g * on, on, torch.ones_like(g), torch.zeros_like(g)
    if name == "gelu":
        cdf = torch.special.ndtr(g)
        pdf = torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
        return g * cdf, cdf + g * pdf, 1.13 * torch.ones_like(g), 0.8 * torch.ones_like(g)
    s = torch.sigmoid(g)
    return g * s, s * (1 + g * (1 - s)), 1.1 * torch.ones_like(g), 0.5 * torch.ones_like(g)


def gated_reference(p, dy, activation, shared=False):
    """{name: (value, bound)} for p = x, Wg, Wu, Wd (and bg, bu, bd), all of one
    type, with leading members or none."""
    ut = HALF[p["x"].dtype]
    one_plane = ut > U
    q = {k: v.double() for k, v in p.items()}
    x, wg, wu, wd, dy = q["x"], q["Wg"], q["Wu"], q["Wd"], dy.double()
    D, F, O, R = wg.shape[-1], wg.shape[-2], wd.shape[-2], x.shape[-2]

    def add(v, k):
        return v + q[k].unsqueeze(-2) if k in q else v

    g, u = add(x @ _t(wg), "bg"), add(x @ _t(wu), "bu")
    e_g = acc(D) * (x.abs() @ _t(wg.abs())) + 2 * U * g.abs()
    e_u = acc(D) * (x.abs() @ _t(wu.abs())) + 2 * U * u.abs()
    a, da, l1, l2 = _activation(activation, g)
    h = a * u
    up = ut if one_plane else 2 * U  # a product operand's rounding
    e_a = e_g * l1 + 8 * U * (a.abs() + g.abs())
    e_h = e_a * u.abs() + a.abs() * e_u + (2 * U + up) * h.abs()
    y = add(h @ _t(wd), "bd")
    out = {"y": (y, e_h @ _t(wd.abs()) + acc(F) * (h.abs() @ _t(wd.abs())) + (2 * U + ut) * y.abs())}

    # the backward goes by g and u as kept, in float32
    e_g, e_u = e_g + U * g.abs(), e_u + U * u.abs()
    e_a = e_g * l1 + 8 * U * (a.abs() + g.abs())
    e_da = e_g * l2 + 16 * U * (1 + g.abs())
    if activation == "relu":  # a gate this near zero may fall on either side
        e_da = e_da + (g.abs() <= e_g).double()
    e_h = e_a * u.abs() + (a.abs() + e_a) * e_u + (2 * U + up) * h.abs()
    dh = dy @ wd
    e_dh = acc(O) * (dy.abs() @ wd.abs())
    dg, du = dh * u * da, dh * a
    e_dg = (e_dh * (u * da).abs() + dh.abs() * (e_u * (da.abs() + e_da) + u.abs() * e_da)
            + (4 * U + up) * dg.abs())
    e_du = e_dh * a.abs() + dh.abs() * e_a + (2 * U + up) * du.abs()
    n = 2 * F
    dx = dg @ wg + du @ wu
    e_dx = (e_dg @ wg.abs() + e_du @ wu.abs()
            + acc(n * (x.dim() == 2 and wg.dim() == 3 and wg.shape[0] or 1))
            * (dg.abs() @ wg.abs() + du.abs() @ wu.abs()))
    if shared:
        dx, e_dx = dx.sum(0), e_dx.sum(0)
    out["x"] = (dx, e_dx + ut * dx.abs())
    for k, d, e in (("Wg", dg, e_dg), ("Wu", du, e_du)):
        v = _t(d) @ x
        out[k] = (v, _t(e) @ x.abs() + acc(R) * (_t(d.abs()) @ x.abs()) + ut * v.abs())
    v = _t(dy) @ h
    out["Wd"] = (v, _t(dy.abs()) @ e_h + acc(R) * (_t(dy.abs()) @ h.abs()) + ut * v.abs())
    for k, d, e in (("bg", dg, e_dg), ("bu", du, e_du), ("bd", dy, torch.zeros_like(dy))):
        if k in q:
            v = d.sum(-2)
            out[k] = (v, e.sum(-2) + (R + 8) * U * d.abs().sum(-2) + ut * v.abs())
    return out


def xent_reference(x, W, b, target, ignore, reduction, g):
    """{name: (value, bound)} of loss and the gradients of x, W, b; g: the
    loss's gradient (a number, or one a row for reduction 'none')."""
    ut = HALF[x.dtype]
    one_plane = ut > U
    x, W = x.double(), W.double()
    z = x @ _t(W)
    D, V, R = W.shape[1], W.shape[0], x.shape[0]
    e_z = acc(D) * (x.abs() @ _t(W.abs())) + 2 * U * z.abs()
    if b is not None:
        z = z + b.double()
        e_z = e_z + 2 * U * z.abs()
    on = target != ignore
    at = torch.where(on, target, 0)
    lse = torch.logsumexp(z, -1)
    p = torch.exp(z - lse[:, None])
    # the terms' exponentials err with their arguments; a lane's chain of up to
    # 32 terms, the joins of a wave's and then of the row's parts (8 a group)
    spread = (p * (z - z.amax(-1, keepdim=True)).abs()).sum(-1)
    e_lse = ((p * e_z).sum(-1) + U * (60 + V / 256 + 4 * spread + 2 * lse.abs()
                                      + 2 * z.amax(-1).abs()))
    rows = torch.where(on, lse - z.gather(-1, at[:, None])[:, 0], 0.0)
    e_rows = torch.where(on, e_lse + e_z.gather(-1, at[:, None])[:, 0] + 2 * U * (rows.abs() + lse.abs()), 0.0)
    share = on.double()
    if reduction == "mean":
        share = share / max(1, int(on.sum()))
    if reduction == "none":
        loss, e_loss = rows, e_rows
    else:
        loss = (rows * share).sum()
        e_loss = (e_rows * share).sum() + 2 * U * loss.abs()
    gr = share * (g if not torch.is_tensor(g) else g.double())
    onehot = torch.zeros_like(p).scatter_(-1, at[:, None], 1.0)
    d = (p - onehot) * gr[:, None]
    e_p = p * (e_z + e_lse[:, None] + U * (12 + 4 * (z - lse[:, None]).abs()))
    e_d = (e_p + 2 * U * (p - onehot).abs()) * gr.abs()[:, None] \
        + (4 * U + (ut if one_plane else 2 * U)) * d.abs()
    out = {"loss": (loss, e_loss)}
    v = d @ W
    out["x"] = (v, e_d @ W.abs() + acc(V) * (d.abs() @ W.abs()) + ut * v.abs())
    v = _t(d) @ x
    out["W"] = (v, _t(e_d) @ x.abs() + acc(R) * (_t(d.abs()) @ x.abs()) + ut * v.abs())
    if b is not None:
        v = d.sum(0)
        out["b"] = (v, e_d.sum(0) + (R + 8) * U * d.abs().sum(0) + ut * v.abs())
    return out
