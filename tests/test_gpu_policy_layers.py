"""layer_norm, gated_mlp and linear_cross_entropy of torch_ops against their
float64 forms, each output within the bound that its roundings give
(policy_layer_helpers): sizes from one row up, odd ones, strides, members,
masked rows, infinities, replays, streams."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from policy_layer_helpers import gated_reference, norm_reference, within, xent_reference

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
DEV = "cuda:0"


@pytest.fixture(scope="module")
def T():
    from d3rlpy_amd import torch_ops
    return torch_ops


def rnd(seed, *shape, dtype=F32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).to(DEV)


def check(got, ref, keys=None):
    for k in keys or ref:
        within(got[k], *ref[k], k)


# ------------------------------------------------------------------ layer norm
def run_norm(T, x, w, b, dy, eps=1e-5):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = T.layer_norm(*leaves, eps)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    return {"y": y, "x": dx, "weight": dw, "bias": db}


@pytest.mark.parametrize("rows,n", [(1, 1), (1, 64), (3, 17), (257, 256), (1000, 257), (5, 513),
                                    (130, 1024), (33, 1537), (9, 2048), (6, 2049), (7, 4100),
                                    (5, 8192), (3, 8193), (70, 12288), (4100, 24)])
@pytest.mark.parametrize("dtype,wtype", [(F32, F32), (BF16, BF16), (BF16, F32)])
def test_layer_norm(T, rows, n, dtype, wtype):
    x = rnd(1, rows, n, dtype=dtype, scale=2.0, shift=0.7)
    w, b = rnd(2, n, dtype=wtype, scale=0.3, shift=1.0), rnd(3, n, dtype=wtype)
    dy = rnd(4, rows, n, dtype=dtype)
    check(run_norm(T, x, w, b, dy), norm_reference(x, w, b, 1e-5, dy))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [96, 300, 9000])
def test_layer_norm_members(T, dtype, n):
    C, R = 3, 37
    x, dy = rnd(1, C, R, n, dtype=dtype), rnd(4, C, R, n, dtype=dtype)
    w, b = rnd(2, C, n, dtype=dtype), rnd(3, C, n, dtype=dtype)
    ref = norm_reference(x, w[:, None], b[:, None], 1e-5, dy)
    check(run_norm(T, x, w, b, dy), ref)


def test_layer_norm_strides_and_leading_axes(T):
    x = rnd(1, 6, 50, 128, dtype=BF16)
    w, b, dy = rnd(2, 64), rnd(3, 64), rnd(4, 6, 50, 64, dtype=BF16)
    for v in (x[:, :, :64], x[:, :, 64:], x[:, :, 1:65], x[:, :, ::2]):
        ref = norm_reference(v, w, b, 1e-5, dy)
        got = run_norm(T, v, w, b, dy)
        assert got["y"].is_contiguous()
        ref["weight"] = tuple(t.sum(0) for t in ref["weight"])
        ref["bias"] = tuple(t.sum(0) for t in ref["bias"])
        # 300 rows in all where the bound counted 50 a slice: the same sums
        check(got, ref)
    flat = x[0, :, :64]  # rows 128 apart
    ref = norm_reference(flat, w, b, 1e-5, dy[0])
    check(run_norm(T, flat, w, b, dy[0]), ref)
    # a gradient that is one value expanded, and rows of a transposed array
    one = torch.ones((), device=DEV, dtype=BF16).expand(50, 64)
    check(run_norm(T, flat, w, b, one), norm_reference(flat, w, b, 1e-5, one))
    tr = rnd(5, 64, 50, dtype=BF16).t()
    check(run_norm(T, tr, w, b, dy[0]), norm_reference(tr, w, b, 1e-5, dy[0]))


def test_layer_norm_without_weight_or_rows(T):
    x = rnd(1, 9, 40).requires_grad_(True)
    dy = rnd(2, 9, 40)
    one, zero = torch.ones(40, device=DEV), torch.zeros(40, device=DEV)
    y = T.layer_norm(x)
    (dx,) = torch.autograd.grad(y, [x], dy)
    ref = norm_reference(x, one, zero, 1e-5, dy)
    check({"y": y, "x": dx}, ref, ("y", "x"))
    w, b = one.clone().requires_grad_(True), zero.clone().requires_grad_(True)
    none = torch.empty(0, 40, device=DEV, requires_grad=True)
    y = T.layer_norm(none, w, b)
    grads = torch.autograd.grad(y, [none, w, b], torch.empty_like(y))
    assert y.shape == (0, 40) and grads[0].shape == (0, 40)
    assert not grads[1].any() and not grads[2].any()
    # one gradient alone
    (dw,) = torch.autograd.grad(T.layer_norm(x.detach(), w, b), [w], dy)
    within(dw, *ref["weight"], "weight")


@pytest.mark.parametrize("n", [8, 7])
def test_layer_norm_more_rows_than_a_launch_has_threads(T, n):
    """2^26 rows of 64 lanes each would be 2^32 threads."""
    R = (1 << 26) + 5
    x = rnd(1, 1 << 12, n, dtype=BF16).repeat((R >> 12) + 1, 1)[:R].requires_grad_(True)
    w, b = rnd(2, n), rnd(3, n)
    y = T.layer_norm(x, w, b)
    dy = torch.ones((), device=DEV, dtype=BF16).expand(R, n)
    (dx,) = torch.autograd.grad(y, [x], dy)
    x, y = x.detach(), y.detach()
    for rows in (slice(0, 9), slice(R - 9, R)):
        ref = norm_reference(x[rows], w, b, 1e-5, dy[rows])
        check({"y": y[rows], "x": dx[rows]}, ref, ("y", "x"))
    # the same rows give the same values, bit by bit
    for v in (y, dx):
        assert torch.equal(v[1 << 25:(1 << 25) + (1 << 20)], v[:1 << 20])


def test_layer_norm_constant_and_bad_rows(T):
    x = rnd(1, 4, 100)
    x[1] = 3.0
    x[2, 7] = float("inf")
    x[3, 9] = float("nan")
    w, b = torch.ones(100, device=DEV), torch.zeros(100, device=DEV)
    y = T.layer_norm(x, w, b)
    assert torch.isfinite(y[:2]).all() and y[2:].isnan().all()
    within(y[:2], *(t[:2] for t in norm_reference(x, w, b, 1e-5, x)["y"]), "y")


# ------------------------------------------------------------------ gated block
def gated_params(C, R, D, F, O, dtype, bias, shared=False):
    lead = (C,) if C else ()
    p = {"x": rnd(1, *(() if shared else lead), R, D, dtype=dtype),
         "Wg": rnd(2, *lead, F, D, dtype=dtype, scale=D ** -0.5),
         "Wu": rnd(3, *lead, F, D, dtype=dtype, scale=D ** -0.5),
         "Wd": rnd(4, *lead, O, F, dtype=dtype, scale=F ** -0.5)}
    if bias:
        p |= {"bg": rnd(5, *lead, F, dtype=dtype, scale=0.3),
              "bu": rnd(6, *lead, F, dtype=dtype, scale=0.3),
              "bd": rnd(7, *lead, O, dtype=dtype, scale=0.3)}
    return p, rnd(8, *lead, R, O, dtype=dtype)


def run_gated(T, p, dy, activation):
    q = {k: v.detach().requires_grad_(True) for k, v in p.items()}
    y = T.gated_mlp(q["x"], q["Wg"], q["Wu"], q["Wd"], q.get("bg"), q.get("bu"), q.get("bd"),
                    activation=activation)
    grads = torch.autograd.grad(y, list(q.values()), dy)
    return {"y": y} | dict(zip(q, grads))


SIZES = [(1, 8, 8, 8), (1, 1, 1, 1), (2, 3, 5, 7), (5, 64, 32, 48), (17, 40, 72, 24),
         (33, 129, 100, 65), (64, 256, 130, 256), (65, 72, 520, 71), (200, 256, 512, 256),
         (333, 130, 1000, 129)]
# an axis past 1024 and few rows: thin forward with the tiles' backward (R <= 16),
# or the tiles with most of each empty
THIN_SIZES = [(1, 40, 1100, 24), (7, 24, 1041, 33), (16, 1030, 72, 65), (17, 1030, 72, 24),
              (40, 33, 1100, 17), (200, 1030, 72, 1100), (1100, 40, 24, 33)]


@pytest.mark.parametrize("R,D,F,O", SIZES + THIN_SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("activation,bias", [("silu", False), ("gelu", True), ("relu", True)])
def test_gated_mlp(T, R, D, F, O, dtype, activation, bias):
    p, dy = gated_params(0, R, D, F, O, dtype, bias)
    check(run_gated(T, p, dy, activation), gated_reference(p, dy, activation))


# enough tiles for the larger ones
@pytest.mark.parametrize("R,D,F,O", [(2560, 192, 1280, 130), (3000, 136, 2056, 264),
                                     (4100, 264, 4100, 2100)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gated_mlp_large_tiles(T, R, D, F, O, dtype):
    p, dy = gated_params(0, R, D, F, O, dtype, False)
    check(run_gated(T, p, dy, "silu"), gated_reference(p, dy, "silu"))


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("R,D,F,O", [(1, 17, 40, 3), (40, 24, 100, 33), (300, 128, 512, 128),
                                     (3, 17, 1100, 9), (40, 24, 1100, 33), (33, 1030, 40, 40)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gated_mlp_members(T, R, D, F, O, dtype, shared):
    p, dy = gated_params(3, R, D, F, O, dtype, True, shared)
    got = run_gated(T, p, dy, "silu")
    assert got["y"].shape == (3, R, O)
    check(got, gated_reference(p, dy, "silu", shared))


@pytest.mark.parametrize("F", [96, 1104])  # products from the tensors, tiles
def test_gated_mlp_strides(T, F):
    R, D, O = 50, 64, 40
    p, dy = gated_params(0, R, D, F, O, BF16, False)
    ref = gated_reference(p, dy, "silu")

    def wide(t, by, off):  # the same values in rows `by` longer, `off` in
        big = torch.full((t.shape[0], t.shape[1] + by), 7.0, device=DEV, dtype=t.dtype)
        big[:, off:off + t.shape[1]] = t
        return big[:, off:off + t.shape[1]]

    for by, off in ((64, 0), (64, 8), (24, 16), (3, 1), (5, 0)):
        v = {k: wide(t, by, off) for k, t in p.items()}
        check(run_gated(T, v, wide(dy, by, off), "silu"), ref)
    # gate and up as halves of one array, down transposed, x rows far apart
    both = torch.cat([p["Wg"], p["Wu"]])
    v = {"x": wide(p["x"], 1000, 8), "Wg": both[:F], "Wu": both[F:], "Wd": p["Wd"].t().contiguous().t()}
    check(run_gated(T, v, dy, "silu"), ref)
    # three leading axes, an expanded gradient
    x3 = {"x": p["x"].view(5, 10, D)} | {k: p[k] for k in ("Wg", "Wu", "Wd")}
    got = run_gated(T, x3, dy.view(5, 10, O), "silu")
    assert got["y"].shape == (5, 10, O) and got["x"].shape == (5, 10, D)
    check({k: t.reshape(ref[k][0].shape) for k, t in got.items()}, ref)
    one = torch.ones((), device=DEV, dtype=BF16).expand(R, O)
    check(run_gated(T, p, one, "silu"), gated_reference(p, one, "silu"))


@pytest.mark.parametrize("F", [40, 1100])
@pytest.mark.parametrize("R", [20, 9])
def test_gated_mlp_one_gradient_and_no_rows(T, R, F):
    p, dy = gated_params(0, R, 24, F, 16, F32, True)
    ref = gated_reference(p, dy, "silu")
    for k in p:
        q = {n: t.detach().requires_grad_(n == k) for n, t in p.items()}
        y = T.gated_mlp(q["x"], q["Wg"], q["Wu"], q["Wd"], q["bg"], q["bu"], q["bd"])
        (d,) = torch.autograd.grad(y, [q[k]], dy)
        within(d, *ref[k], k)
    p["x"], dy = p["x"][:0], dy[:0]
    got = run_gated(T, p, dy, "silu")
    assert got["y"].shape == (0, 16) and got["x"].shape == (0, 24)
    assert not any(bool(got[k].any()) for k in got if k not in ("y", "x"))


def test_gated_mlp_rows_do_not_mix(T):
    """A row of infinities spoils its own outputs and no other row's."""
    p, _ = gated_params(0, 70, 40, 72, 24, BF16, False)
    args = (p["Wg"], p["Wu"], p["Wd"])
    y = T.gated_mlp(p["x"], *args)
    x = p["x"].clone()
    x[33] = float("inf")
    z = T.gated_mlp(x, *args)
    keep = torch.arange(70, device=DEV) != 33
    assert torch.equal(y[keep], z[keep]) and not torch.isfinite(z[33]).all()


# ------------------------------------------------------------- linear cross entropy
def run_xent(T, x, W, b, target, reduction, g, ignore=-100):
    q = {"x": x.detach().requires_grad_(True), "W": W.detach().requires_grad_(True)}
    if b is not None:
        q["b"] = b.detach().requires_grad_(True)
    loss = T.linear_cross_entropy(q["x"], q["W"], target, q.get("b"), ignore, reduction)
    grads = torch.autograd.grad(loss, list(q.values()),
                                g if torch.is_tensor(g) else torch.full_like(loss, g))
    return {"loss": loss} | dict(zip(q, grads))


def xent_inputs(R, D, V, dtype, bias, pad=0.2):
    gen = torch.Generator().manual_seed(R * 7 + V)
    t = torch.randint(0, V, (R,), generator=gen)
    t[torch.rand(R, generator=gen) < pad] = -100
    return (rnd(1, R, D, dtype=dtype), rnd(2, V, D, dtype=dtype, scale=2 * D ** -0.5),
            rnd(3, V, dtype=dtype) if bias else None, t.to(DEV))


@pytest.mark.parametrize("R,D,V", [(1, 1, 1), (1, 8, 2), (3, 17, 5), (8, 64, 1000), (33, 100, 257),
                                   (65, 40, 130), (130, 256, 64), (257, 33, 1031),
                                   (700, 128, 2050), (1, 8, 2100), (3, 17, 2101), (65, 40, 5003),
                                   (33, 1030, 257), (1030, 24, 5), (9, 40, 33011)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("reduction,bias", [("mean", False), ("sum", True), ("none", True)])
def test_linear_cross_entropy(T, R, D, V, dtype, reduction, bias):
    x, W, b, t = xent_inputs(R, D, V, dtype, bias)
    g = rnd(9, R) if reduction == "none" else 0.7
    check(run_xent(T, x, W, b, t, reduction, g), xent_reference(x, W, b, t, -100, reduction, g))


@pytest.mark.parametrize("R,D,V", [(4000, 136, 4099), (2049, 72, 10007), (33000, 24, 1100)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_cross_entropy_large_tiles(T, R, D, V, dtype):
    x, W, b, t = xent_inputs(R, D, V, dtype, True)
    check(run_xent(T, x, W, b, t, "mean", 1.0), xent_reference(x, W, b, t, -100, "mean", 1.0))


def test_linear_cross_entropy_pieces(T):
    """A vocabulary in several pieces (float32: 6 bytes a logit, 512 MiB a
    piece), the last one odd, is the sum of its pieces."""
    x, W, b, t = xent_inputs(6000, 24, 33001, F32, True)
    check(run_xent(T, x, W, b, t, "mean", 1.0), xent_reference(x, W, b, t, -100, "mean", 1.0))


@pytest.mark.parametrize("V", [77, 2201])  # products from the tensors, tiles
def test_linear_cross_entropy_masked_rows(T, V):
    x, W, b, t = xent_inputs(40, 24, V, F32, True)
    t[:] = -100
    for reduction in ("mean", "sum", "none"):
        got = run_xent(T, x, W, b, t, reduction, 1.0)
        assert not any(bool(v.any()) for v in got.values())
    # another ignored value, one that is a class; and rows whose logits are not numbers
    t = torch.arange(40, device=DEV) % 5
    ref = xent_reference(x, W, b, t, 3, "mean", 1.0)
    check(run_xent(T, x, W, b, t, "mean", 1.0, ignore=3), ref)
    bad = x.clone()
    bad[t == 3] = float("nan")
    bad[8] = float("inf")  # (target 3)
    got = run_xent(T, bad, W, b, t, "mean", 1.0, ignore=3)
    check({k: got[k] for k in ("loss", "b")}, ref, ("loss", "b"))
    assert torch.equal(got["x"][t == 3], torch.zeros_like(got["x"][t == 3]))


@pytest.mark.parametrize("n", [35, 1100])
def test_linear_cross_entropy_extreme_logits(T, n):
    """Logits of the type's lowest value and of -inf (a masked action), and a
    target outside the vocabulary."""
    x, W, b, t = xent_inputs(30, 16, 2 * n, F32, True, pad=0.0)
    t = t % n
    b[n:n + 15] = float("-inf")
    b[n + 15:] = torch.finfo(F32).min
    cut = xent_reference(x, W[:n], b[:n], t, -100, "mean", 1.0)
    got = run_xent(T, x, W, b, t, "mean", 1.0)
    within(got["loss"], *cut["loss"], "loss")
    within(got["x"], *cut["x"], "x")
    within(got["W"][:n], *cut["W"], "W")
    assert not got["W"][n:].any() and not got["b"][n:].any()
    for wrong in (-1, 2 * n, 1 << 40, -(1 << 40)):
        u = t.clone()
        u[4] = wrong
        got = run_xent(T, x, W, b, u, "none", 1.0)
        assert got["loss"][4].isnan() and got["x"][4].isnan().all()
        rest = torch.arange(30, device=DEV) != 4
        assert torch.isfinite(got["loss"][rest]).all() and torch.isfinite(got["x"][rest]).all()


@pytest.mark.parametrize("V", [77, 2201, 33011])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_cross_entropy_rows_that_are_not_numbers(T, V, dtype):
    """NaN in a row, or a logit of +inf: that row's loss and gradient are NaN, no
    other row's."""
    x, W, b, t = xent_inputs(70, 24, V, dtype, True)
    t[5] = t[69] = 1
    clean = run_xent(T, x, W, b, t, "none", 1.0)
    bad = x.clone()
    bad[5, 3] = float("nan")
    bad[69, 7] = float("inf")
    got = run_xent(T, bad, W, b, t, "none", 1.0)
    rest = torch.ones(70, dtype=torch.bool, device=DEV)
    rest[5] = rest[69] = False
    assert got["loss"][~rest].isnan().all() and got["x"][~rest].isnan().all()
    assert torch.equal(got["loss"][rest], clean["loss"][rest])
    assert torch.equal(got["x"][rest], clean["x"][rest])


@pytest.mark.parametrize("V", [90, 2190])
def test_linear_cross_entropy_shapes_and_strides(T, V):
    x, W, b, t = xent_inputs(48, 40, V, BF16, True)
    ref = xent_reference(x, W, b, t, -100, "mean", 1.0)
    got = run_xent(T, x.view(4, 12, 40), W, b, t.view(4, 12), "mean", 1.0)
    assert got["x"].shape == (4, 12, 40)
    got["x"] = got["x"].reshape(48, 40)
    check(got, ref)
    big = torch.full((48, 83), 5.0, device=DEV, dtype=BF16)
    big[:, 3:43] = x
    tied = rnd(11, V, 80, dtype=BF16)
    tied[:, 40:] = W
    got = run_xent(T, big[:, 3:43], tied[:, 40:], b, t, "mean", 1.0)
    check(got, ref)
    none = run_xent(T, x[:0], W, b, t[:0], "mean", 1.0)
    assert not none["loss"].detach().any() and not none["W"].any() and not none["b"].any()


def test_linear_cross_entropy_more_rows_than_a_launch_has_threads(T):
    """2^27 rows, 8 to a workgroup of 256, would be 2^32 threads."""
    R, D, V = (1 << 27) + 3, 8, 3
    x = rnd(1, 1 << 12, D, dtype=BF16).repeat((R >> 12) + 1, 1)[:R]
    W = rnd(2, V, D, dtype=BF16)
    t = (torch.arange(1 << 12, device=DEV) % V).repeat((R >> 12) + 1)[:R]
    loss = T.linear_cross_entropy(x, W, t, reduction="none")
    for rows in (slice(0, 9), slice(R - 9, R)):
        ref = xent_reference(x[rows], W, None, t[rows], -100, "none", 1.0)
        within(loss[rows], *ref["loss"], "loss")
    assert torch.equal(loss[1 << 26:(1 << 26) + (1 << 20)], loss[:1 << 20])


@pytest.mark.parametrize("V", [200, 4099])
def test_linear_cross_entropy_common_factor(T, V):
    """bfloat16, the mean over 510 rows: 1/510 would round to bfloat16 with
    2^-8 of it, in every row alike.  The gradients' common error, their
    component along the exact ones, is at most that of 1 - p at a target, 2^-9
    (the others' signs vary)."""
    x, W, _, t = xent_inputs(510, 64, V, BF16, False, pad=0.0)
    ref = xent_reference(x, W, None, t, -100, "mean", 1.0)
    got = run_xent(T, x, W, None, t, "mean", 1.0)
    check(got, ref)
    for k in ("x", "W"):
        want = ref[k][0]
        assert abs(float(((got[k].double() - want) * want).sum() / (want * want).sum())) <= 2.0 ** -9, k


# --------------------------------------------------------------- together, replays
def block_step(T, q, tokens, target):
    """A pre-norm gated residual block and a classification head: loss, gradients."""
    x = q["emb"][tokens]
    h = T.layer_norm(x, q["n1"], q["c1"])
    x = x + T.gated_mlp(h, q["Wg"], q["Wu"], q["Wd"])
    loss = T.linear_cross_entropy(T.layer_norm(x, q["n2"], q["c2"]), q["emb"], target)
    return loss, torch.autograd.grad(loss, list(q.values()))


def block_inputs(dtype):
    V, D, F, R = 300, 64, 160, 90
    gen = torch.Generator().manual_seed(5)
    q = {"emb": torch.randn(V, D, generator=gen), "n1": torch.ones(D), "c1": torch.zeros(D),
         "Wg": torch.randn(F, D, generator=gen) * D ** -0.5,
         "Wu": torch.randn(F, D, generator=gen) * D ** -0.5,
         "Wd": torch.randn(D, F, generator=gen) * F ** -0.5, "n2": torch.ones(D),
         "c2": torch.zeros(D)}
    q = {k: v.to(dtype).to(DEV).requires_grad_(True) for k, v in q.items()}
    tokens = torch.randint(0, V, (R,), generator=gen).to(DEV)
    target = torch.randint(0, V, (R,), generator=gen).to(DEV)
    target[::7] = -100
    return q, tokens, target


def test_block_trains_as_in_float64(T):
    """The three together, the embedding tied to the head: loss and gradients
    against the same network in float64 torch.  Every stage is good to the
    float32 bounds above; through three stages and a sum over 90 rows they
    stay under 2e-5 of the largest gradient (2^-24 times some 300 chained
    roundings)."""
    q, tokens, target = block_inputs(F32)
    loss, grads = block_step(T, q, tokens, target)
    d = {k: v.detach().double().requires_grad_(True) for k, v in q.items()}
    x = d["emb"][tokens]
    D = x.shape[1]
    nrm = torch.nn.functional.layer_norm
    h = nrm(x, (D,), d["n1"], d["c1"])
    g = h @ d["Wg"].t()
    x = x + (g * torch.sigmoid(g) * (h @ d["Wu"].t())) @ d["Wd"].t()
    ref = torch.nn.functional.cross_entropy(nrm(x, (D,), d["n2"], d["c2"]) @ d["emb"].t(), target)
    want = torch.autograd.grad(ref, list(d.values()))
    assert abs(float(loss) - float(ref)) <= 2e-5 * abs(float(ref))
    for k, a, b in zip(q, grads, want):
        assert float((a - b).abs().max()) <= 2e-5 * float(b.abs().max()), k


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_block_is_deterministic_and_replays(T, dtype):
    """Bit-identical from run to run, on another stream, and in a captured
    graph replayed between eager calls."""
    q, tokens, target = block_inputs(dtype)
    det = {k: v.detach() for k, v in q.items()}

    def step():
        # (forward and backward calls, not autograd: what a captured loop runs)
        ops = T.load()
        x = det["emb"][tokens]
        h, s1 = ops.layer_norm(x, det["n1"], det["c1"], 1e-5)
        y, kept = ops.gated_mlp(h, det["Wg"], det["Wu"], det["Wd"], None, None, None, "silu", True)
        r, s2 = ops.layer_norm(x + y, det["n2"], det["c2"], 1e-5)
        loss, lse, scale = ops.linear_cross_entropy(r, det["emb"], target, None, -100, "mean")
        dr, demb, _ = ops.linear_cross_entropy_backward(
            torch.ones_like(loss), r, det["emb"], target, None, lse, scale, -100, "mean",
            [True, True, False])
        dxy, dn2, dc2 = ops.layer_norm_backward(dr, x + y, det["n2"], det["c2"], s2, [True] * 3)
        dh, dWg, dWu, dWd = ops.gated_mlp_backward(
            dxy, h, det["Wg"], det["Wu"], det["Wd"], None, None, None, kept, "silu",
            [True] * 4 + [False] * 3)[:4]
        return [loss, demb, dn2, dc2, dh, dWg, dWu, dWd]

    want = step()
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert all(torch.equal(a, b) for a, b in zip(step(), want))


def test_captured_autograd(T):
    """Loss and torch.autograd.grad captured together, after warm-up passes on
    the capture's kind of stream whose graphs are gone: every replay, with new
    parameters between, is the eager pass."""
    q, tokens, target = block_inputs(F32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            block_step(T, q, tokens, target)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = block_step(T, q, tokens, target)
    for k in range(4):
        with torch.no_grad():
            q["Wg"].mul_(1.0 + 0.1 * k)
        graph.replay()
        torch.cuda.synchronize()
        got = [loss.detach().clone()] + [g.clone() for g in grads]
        want = block_step(T, q, tokens, target)
        assert torch.equal(got[0], want[0].detach())
        # (the embedding's gradient adds rows of the same token in torch's order)
        for n, a, b in zip(q, got[1:], want[1]):
            assert torch.equal(a, b) or n == "emb", n


def test_gradients_against_differences(T):
    """The losses' directional derivative, by central differences of the
    float32 loss: steps of 1e-2 leave 1e-4 of curvature and 1e-5 of rounding
    over 2e-2, so 2e-2 of the derivative's size."""
    q, tokens, target = block_inputs(F32)
    _, grads = block_step(T, q, tokens, target)
    for k, g in zip(q, grads):
        v = g / g.norm()
        ends = []
        for s in (1e-2, -1e-2):
            with torch.no_grad():
                moved = dict(q) | {k: q[k] + s * v}
                x = moved["emb"][tokens]
                h = T.layer_norm(x, moved["n1"], moved["c1"])
                x = x + T.gated_mlp(h, moved["Wg"], moved["Wu"], moved["Wd"])
                ends.append(float(T.linear_cross_entropy(
                    T.layer_norm(x, moved["n2"], moved["c2"]), moved["emb"], target)))
        slope = (ends[0] - ends[1]) / 2e-2
        assert abs(slope - float(g.norm())) <= 2e-2 * max(float(g.norm()), 1e-2), (k, slope, float(g.norm()))


def test_no_second_derivative(T):
    x = rnd(1, 4, 8).requires_grad_(True)
    (dx,) = torch.autograd.grad(T.layer_norm(x).sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


# -------------------------------------------------------- refusals, long arrays, memory
def test_refusals_on_the_gpu(T):
    x, w = rnd(1, 4, 8), rnd(2, 8)
    W, Wd, t = rnd(3, 6, 8), rnd(4, 8, 6), torch.zeros(4, dtype=torch.int64, device=DEV)
    for call, match in (
            (lambda: T.layer_norm(x.half(), w.half()), "float32 or bfloat16"),
            (lambda: T.layer_norm(x, w.bfloat16()), "weight and bias must"),
            (lambda: T.layer_norm(x, w.cpu()), "weight / bias on cpu"),
            (lambda: T.layer_norm(x, w, eps=-1.0), "eps"),
            (lambda: T.gated_mlp(x, W, W.bfloat16(), Wd), "Wu is"),
            (lambda: T.gated_mlp(x, W, W, Wd.cpu()), "Wd is on cpu"),
            (lambda: T.gated_mlp(x.double(), W.double(), W.double(), Wd.double()),
             "float32 or bfloat16"),
            (lambda: T.linear_cross_entropy(x, W, t.cpu()), "target is on cpu"),
            (lambda: T.linear_cross_entropy(x, W.bfloat16(), t), "W is"),
            (lambda: T.linear_cross_entropy(x, W, t, rnd(5, 6, dtype=BF16)), "b is")):
        with pytest.raises(RuntimeError, match=match):
            call()
    ops = T.load()
    y, stats = ops.layer_norm(x, w, None, 1e-5)
    with pytest.raises(RuntimeError, match="stats of another"):
        ops.layer_norm_backward(x, x, w, None, stats[:, :, :2].contiguous(), [True] * 3)
    y, kept = ops.gated_mlp(x, W, W, Wd, None, None, None, "silu", False)
    with pytest.raises(RuntimeError, match="keep = True"):
        ops.gated_mlp_backward(y, x, W, W, Wd, None, None, None, kept, "silu", [True] * 7)


def test_vocabulary_past_32_bit_offsets(T):
    """2.2 million classes of 1024 bfloat16 values: W's end lies past 2^32
    bytes and past 2^31 elements."""
    V, D, R = 2_200_003, 1024, 5
    W = torch.empty(V, D, device=DEV, dtype=BF16)
    W[:] = rnd(1, 1, D, dtype=BF16)
    W[V - 7] = rnd(2, D, dtype=BF16)
    x = rnd(3, R, D, dtype=BF16, scale=D ** -0.5)
    t = torch.tensor([V - 7, V - 1, 0, V - 7, -100], device=DEV)
    got = T.linear_cross_entropy(x, W, t, reduction="none")
    z = x.double() @ torch.stack([W[0], W[V - 7]]).double().t()
    lse = torch.logsumexp(torch.stack([z[:, 0] + torch.log(torch.tensor(V - 1.0, dtype=torch.float64)),
                                       z[:, 1]]), 0)
    want = lse - torch.stack([z[0, 1], z[1, 0], z[2, 0], z[3, 1], lse[4]])
    # lse near 15: sums over some 34000 parts joined 32 ways, each in float32
    within(got, want, torch.full_like(want, (V / 64 / 32 + 200) * 2.0 ** -24 * 2), "loss")


def test_norm_past_32_bit_offsets(T):
    rows, n = 2_200_001, 1024
    x = torch.empty(rows, n, device=DEV, dtype=BF16)
    x[:] = rnd(1, 1, n, dtype=BF16)
    x[-3:] = rnd(2, 3, n, dtype=BF16, scale=3.0)
    w, b = rnd(3, n, dtype=BF16), rnd(4, n, dtype=BF16)
    y = T.layer_norm(x, w, b)
    for part in (slice(0, 2), slice(rows - 3, rows)):
        within(y[part], *norm_reference(x[part], w, b, 1e-5, x[part])["y"], "y")


def test_logits_all_at_the_lowest_value(T):
    """A row whose every logit is the type's lowest value: uniform."""
    for dtype in (F32, BF16):
        x, W, b, t = xent_inputs(20, 16, 50, dtype, True, pad=0.0)
        b[:] = torch.finfo(dtype).min
        got = run_xent(T, torch.zeros_like(x), W, b, t, "sum", 1.0)
        # lse = lowest + log 50 rounds to lowest (steps of 2e31): the loss is 0,
        # and every exp(z - lse) is 1, as torch's float32 has it
        assert not got["loss"].any()
        p = 20.0 - torch.bincount(t, minlength=50).double()
        within(got["b"], p, 2.0 ** -8 * p.abs(), "b")
        dx, dW = got["x"], got["W"]
        assert torch.isfinite(dx).all() and torch.isfinite(dW).all()


def test_nothing_is_left_allocated(T):
    q, tokens, target = block_inputs(BF16)
    for _ in range(3):
        block_step(T, q, tokens, target)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(20):
        block_step(T, q, tokens, target)
    assert torch.cuda.memory_allocated() <= before


def test_two_streams_at_once(T):
    """The same calls on two streams at the same time, each with scratch of its
    own, give what each gives alone."""
    q, tokens, target = block_inputs(BF16)
    r = {k: (v.detach() * 0.5).requires_grad_(True) for k, v in q.items()}
    want = [block_step(T, p, tokens, target) for p in (q, r)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for p, s in zip((q, r), streams):
            with torch.cuda.stream(s):
                got.append(block_step(T, p, tokens, target))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and all(torch.equal(u, v) for u, v in zip(a[1], b[1]))
