"""layer_norm, gated_mlp and linear_cross_entropy at the ends of their ranges:
logits that share a large value, large and long arrays, parts and pieces.  Against
float64 forms with bounds from the kernels' roundings (policy_layer_helpers)."""
import ctypes
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from policy_layer_helpers import U, acc, gated_reference, within, xent_reference

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


def run_xent(T, x, W, b, target, reduction, g, ignore=-100):
    q = {"x": x.detach().requires_grad_(True), "W": W.detach().requires_grad_(True)}
    if b is not None:
        q["b"] = b.detach().requires_grad_(True)
    loss = T.linear_cross_entropy(q["x"], q["W"], target, q.get("b"), ignore, reduction)
    grads = torch.autograd.grad(loss, list(q.values()),
                                g if torch.is_tensor(g) else torch.full_like(loss, g))
    return {"loss": loss} | dict(zip(q, grads))


def rows_and_classes(R, D, V, dtype, pad=0.2):
    g = torch.Generator(DEV).manual_seed(R + V)
    x = torch.randn(R, D, device=DEV, generator=g).to(dtype)
    W = (torch.randn(V, D, device=DEV, generator=g) * D ** -0.5).to(dtype)
    b = torch.randn(V, device=DEV, generator=g).to(dtype)
    t = torch.randint(0, V, (R,), device=DEV, generator=g)
    t[torch.rand(R, device=DEV, generator=g) < pad] = -100
    return x, W, b, t


# ------------------------------------------------- logits that share a large value
def common_inputs(V, dtype, common, step):
    """Logits of ``common`` plus whole multiples of ``step``, exact in float32: x
    has one feature, which W does not weigh, so a logit is its bias."""
    R, D = 20, 16
    x, W = torch.zeros(R, D), torch.randn(V, D, generator=torch.Generator().manual_seed(V))
    x[:, 0] = torch.arange(1, R + 1)
    W[:, 0] = 0.0
    over = torch.randint(0, 8, (V,), generator=torch.Generator().manual_seed(1)) * step
    b = torch.full((V,), common).to(dtype).double() + over
    assert torch.equal(b.to(dtype).double(), b)
    t = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(2))
    t[3] = -100
    return x.to(dtype).to(DEV), W.to(dtype).to(DEV), b.to(dtype).to(DEV), over.to(DEV), t.to(DEV)


@pytest.mark.parametrize("V", [50, 2201, 33011])  # from the tensors; tiles; many parts a row
@pytest.mark.parametrize("dtype,common,step", [
    (F32, 0.0, 0.5), (F32, 1e5, 0.5), (F32, -1e6, 0.5), (F32, -1e9, 0.0),
    (F32, torch.finfo(F32).min, 0.0), (F32, torch.finfo(F32).max, 0.0),
    (BF16, -100.0, 0.5), (BF16, 1e6, 0.0), (BF16, torch.finfo(BF16).min, 0.0)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cross_entropy_of_logits_with_a_common_value(T, V, dtype, common, step, reduction):
    """A value that all of a row's logits share changes neither loss nor gradients:
    both are those of the logits without it, within the bounds that these have."""
    x, W, b, over, t = common_inputs(V, dtype, common, step)
    g = rnd(9, 20) if reduction == "none" else 0.7
    ref = xent_reference(x, W, over, t, -100, reduction, g)
    check(run_xent(T, x, W, b, t, reduction, g), ref)


def test_cross_entropy_of_uniform_rows_is_torchs(T):
    """Fifty logits of the lowest value: log 50 and 1/50, as torch has it."""
    b = torch.full((50,), torch.finfo(F32).min, device=DEV)
    x, W = torch.zeros(4, 8, device=DEV), torch.zeros(50, 8, device=DEV)
    t = torch.tensor([0, 7, 49, 7], device=DEV)
    got = run_xent(T, x, W, b, t, "sum", 1.0)
    c = b.cpu().requires_grad_(True)
    loss = torch.nn.functional.cross_entropy(c.expand(4, 50), t.cpu(), reduction="sum")
    loss.backward()
    # a logarithm and an exponential of a few steps each, and sums of four
    within(got["loss"], loss.detach(), 16 * U * loss.detach().abs(), "loss")
    within(got["b"], c.grad, 64 * U * torch.ones(50), "b")


def test_cross_entropy_lse_and_its_low_part(T):
    """lse is the logsumexp's float32 value, shape and all; the backward of the C
    entry without the low part goes by lse alone."""
    from d3rlpy_amd import _native as N
    x, W, b, over, t = common_inputs(50, F32, 1e5, 0.5)
    ops = T.load()
    loss, lse, scale = ops.linear_cross_entropy(x.view(4, 5, 16), W, t.view(4, 5), b, -100, "sum")
    want = torch.logsumexp(b.double(), 0)
    assert lse.shape == (4, 5)
    within(lse, want.expand(4, 5), (U * want.abs()).expand(4, 5), "lse")
    # and what it left: lse + low is the logarithm of the sum to a few steps of its own
    low = scale[1:].double()
    within(lse.flatten().double() + low, want.expand(20), torch.full((20,), 64 * U), "lse + low")

    d = N.LinearXentDesc()
    d.rows, d.n_in, d.vocab, d.ldx, d.ldW, d.ignore_index, d.reduction = 20, 16, 50, 16, 16, -100, 2
    one, db = torch.ones(1, device=DEV), torch.empty(50, device=DEV)
    for k, v in (("x", x), ("W", W), ("b", b), ("target", t), ("loss", loss), ("lse", lse),
                 ("out", loss), ("scale", scale), ("gloss", one), ("db", db)):
        setattr(d, k, v.data_ptr())
    size = ctypes.c_int64()
    assert N.lib().d3a_linear_xent_workspace(ctypes.byref(d), 1, ctypes.byref(size)) == 0
    ws = torch.empty(size.value, dtype=torch.uint8, device=DEV)
    d.ws, d.ws_bytes = ws.data_ptr(), size.value
    stream = torch.cuda.current_stream().cuda_stream
    assert N.lib().d3a_linear_xent_bwd(ctypes.byref(d), stream) == 0
    p = torch.softmax(over.double(), 0)
    count = torch.bincount(t[t >= 0], minlength=50).double()
    # every row's p is off by the same factor, exp(2^-24 |lse|) at most
    within(db, 19 * p - count, 19 * p * (1.1 * U * 1e5) + 64 * U * (19 * p + count), "b")


# ------------------------------------------------------------- gated block, few rows
@pytest.mark.parametrize("R,D,F,O", [(1, 64, 512, 48), (1, 256, 2816, 256), (5, 33, 1041, 70),
                                     (8, 72, 1100, 24)])
@pytest.mark.parametrize("C", [0, 3])
@pytest.mark.parametrize("train", [False, True])
def test_few_rows_are_rounded_once(T, R, D, F, O, C, train):
    """bfloat16, up to eight rows: y is float32's value rounded to bfloat16, with h held
    to 2^-16 in between (one bfloat16 h would be 2^-8 off, and sums of it are more than
    y's own rounding wherever y is small)."""
    lead = (C,) if C else ()
    x = rnd(1, *lead, R, D, dtype=BF16)
    Wg, Wu = (rnd(k, *lead, F, D, dtype=BF16, scale=D ** -0.5) for k in (2, 3))
    Wd = rnd(4, *lead, O, F, dtype=BF16, scale=F ** -0.5)
    bd = rnd(5, *lead, O, dtype=BF16)
    got = T.gated_mlp(x.requires_grad_(train), Wg, Wu, Wd, None, None, bd)
    x, Wg, Wu, Wd, bd = (t.detach().double() for t in (x, Wg, Wu, Wd, bd))
    g, u = x @ Wg.mT.contiguous(), x @ Wu.mT.contiguous()
    e_g = acc(D) * (x.abs() @ Wg.abs().mT.contiguous()) + 2 * U * g.abs()
    e_u = acc(D) * (x.abs() @ Wu.abs().mT.contiguous()) + 2 * U * u.abs()
    a = g * torch.sigmoid(g)
    h = a * u
    e_h = (1.1 * e_g + 8 * U * (a.abs() + g.abs())) * u.abs() + a.abs() * e_u \
        + (2 * U + 2.0 ** -16) * h.abs()
    WdT = Wd.mT.contiguous()
    y = h @ WdT + bd.unsqueeze(-2)
    bound = (e_h @ WdT.abs() + 2 * acc(F) * (h.abs() @ WdT.abs()) + (2 * U + 2.0 ** -8) * y.abs())
    within(got, y, bound, "y")


def test_few_rows_with_an_infinite_hidden_value(T):
    """An infinity of h is one of y, not NaN from its second part."""
    x = torch.ones(2, 8, device=DEV, dtype=BF16)
    W = torch.full((16, 8), 1e30, device=DEV, dtype=BF16)
    Wd = torch.full((8, 16), 0.5, device=DEV, dtype=BF16)
    assert T.gated_mlp(x, W, W, Wd).isposinf().all()


# ------------------------------------------------------------- cross entropy, few rows
@pytest.mark.parametrize("R,D,V", [(1, 64, 2), (1, 64, 50), (1, 112, 39680), (3, 33, 77), (16, 40, 2000),
                                   (1, 17, 2101), (9, 24, 5003), (17, 1030, 40), (32, 72, 4099)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_few_rows_gradients_are_rounded_once(T, R, D, V, reduction):
    """bfloat16, up to 16 rows (32 where an axis is too long for the products from the
    tensors): the gradients are float32's rounded to bfloat16, with dz held to 2^-16 in
    between.  (One part would be 2^-8 off, an error that all of one row's W gradient
    shares.)"""
    x, W, b, t = rows_and_classes(R, D, V, BF16, pad=0.0)
    W = (W.float() * 1.5).to(BF16)
    g = rnd(9, R) if reduction == "none" else 0.7
    got = run_xent(T, x, W, b, t, reduction, g)
    # float32's bounds on the same values, dz's two parts, the results' rounding
    ref = xent_reference(x.float(), W.float(), b.float(), t, -100, reduction, g)
    z = x.double() @ W.double().t() + b.double()
    d = torch.softmax(z, -1)
    d[torch.arange(R, device=DEV), t] -= 1.0
    d = d.abs() * (g.abs().double()[:, None] if reduction == "none" else 0.7 / R)
    two = {"x": d @ W.double().abs(), "W": d.t() @ x.double().abs(), "b": d.sum(0)}
    for k, s in two.items():
        want, bound = ref[k]
        within(got[k], want, bound + 2.0 ** -16 * s + 2.0 ** -8 * want.abs(), k)


# --------------------------------------------------------------- float32's whole range
def largest_inputs(R, D, N):
    """x whose first feature is float32's largest value, of either sign, times 2^-125
    in the weight: 8 in every product, exact, of operands that bfloat16 would round to
    infinities; the other features are ordinary."""
    x, W = rnd(1, R, D), rnd(2, N, D, scale=D ** -0.5)
    x[:, 0] = torch.finfo(F32).max
    x[1::2, 0] = -torch.finfo(F32).max
    W[:, 0] = 2.0 ** -125
    return x, W


@pytest.mark.parametrize("F", [72, 1100])  # products from the tensors, tiles
def test_gated_mlp_of_the_largest_values(T, F):
    R, D, O = 40, 24, 16
    x, Wg = largest_inputs(R, D, F)
    Wu, Wd, dy = rnd(3, F, D, scale=D ** -0.5), rnd(4, O, F, scale=F ** -0.5), rnd(5, R, O)
    Wu[:, 0] = 2.0 ** -126
    p = {"x": x, "Wg": Wg, "Wu": Wu, "Wd": Wd}
    q = {k: v.detach().requires_grad_(k in ("x", "Wd")) for k, v in p.items()}
    y = T.gated_mlp(*q.values())
    dx, dWd = torch.autograd.grad(y, [q["x"], q["Wd"]], dy)
    check({"y": y, "x": dx, "Wd": dWd}, gated_reference(p, dy, "silu"), ("y", "x", "Wd"))


@pytest.mark.parametrize("V", [77, 2201])
def test_cross_entropy_of_the_largest_values(T, V):
    x, W = largest_inputs(30, 24, V)
    t = torch.arange(30, device=DEV) % V
    q = x.detach().requires_grad_(True)
    loss = T.linear_cross_entropy(q, W, t)
    (dx,) = torch.autograd.grad(loss, [q])
    check({"loss": loss, "x": dx}, xent_reference(x, W, None, t, -100, "mean", 1.0), ("loss", "x"))


@pytest.mark.parametrize("V", [77, 2201])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_float32_infinities_spoil_their_rows_alone(T, V, bad):
    x, W, t = rnd(1, 30, 24), rnd(2, V, 24), torch.arange(30, device=DEV)
    x[7, 3] = bad
    loss = T.linear_cross_entropy(x, W, t, reduction="none")
    assert loss[7].isnan()
    rest = torch.arange(30, device=DEV) != 7
    want = T.linear_cross_entropy(x[rest], W, t[rest], reduction="none")
    assert torch.equal(loss[rest], want)


# ------------------------------------------------------------------ layer norm, long rows
def test_layer_norm_of_more_columns_than_a_launch_has_threads(T):
    """2^27 columns, of which the pass that adds their sums has 32 threads each, are 2^32
    threads."""
    n = (1 << 27) + 3
    x, dy = (torch.randn(1, n, device=DEV, generator=torch.Generator(DEV).manual_seed(k))
             for k in (1, 2))
    w, b = (torch.randn(n, device=DEV, generator=torch.Generator(DEV).manual_seed(k))
            for k in (3, 4))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = T.layer_norm(*leaves, 1e-5)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    y, x, w, b = (t.detach() for t in (y, x, w, b))
    # one row: b's gradient is dy itself, w's dy xh; the statistics are sums of 2^19
    # values a lane, (2^19 + 80) 2^-24 of their mean magnitude
    assert torch.equal(db, dy[0])
    mean = x.double().mean()
    var = ((x - mean) ** 2).double().mean()
    rstd = 1 / (var + 1e-5).sqrt()
    u = ((1 << 19) + 80) * U
    e_mean, e_rstd = u * x.abs().double().mean(), rstd * u * 2
    for part in (slice(0, 4096), slice((1 << 26) - 2048, (1 << 26) + 2048), slice(n - 4096, n)):
        xh = (x[0, part].double() - mean) * rstd
        e_xh = e_mean * rstd + xh.abs() * (e_rstd / rstd + 8 * U)
        within(dw[part], dy[0, part] * xh, (dy[0, part].abs() * (e_xh + 4 * U * xh.abs())), "weight")
        want = xh * w[part] + b[part]
        within(y[0, part], want, e_xh * w[part].abs() + 4 * U * (want.abs() + (xh * w[part]).abs()), "y")
    assert torch.isfinite(dx).all()


# ------------------------------------------- pieces of the vocabulary, blocks of the rows
@pytest.mark.parametrize("R,D,V,dtype,reduction", [
    (33000, 24, 9000, BF16, "mean"),    # two pieces, sums of columns by a pass of their own
    (33000, 24, 9000, BF16, "none"),
    (8000, 40, 36001, BF16, "none"),    # two pieces, their columns' sums in the epilogue
    (6000, 24, 33001, F32, "none"),     # three
    (400003, 24, 300, F32, "mean"),     # two pieces x two blocks of rows
    (400003, 17, 77, F32, "none"),      # one piece
    (400003, 17, 300, F32, "sum"),      # rows that are not 16-byte aligned, two x two
    ((1 << 20) + 4099, 8, 264, BF16, "sum"),
    ((1 << 20) + 4099, 8, 264, BF16, "none")])
def test_cross_entropy_in_pieces_and_blocks(T, R, D, V, dtype, reduction):
    x, W, b, t = rows_and_classes(R, D, V, dtype)
    g = torch.randn(R, device=DEV, generator=torch.Generator(DEV).manual_seed(9)) \
        if reduction == "none" else 1.0
    got = run_xent(T, x, W, b, t, reduction, g)
    again = run_xent(T, x, W, b, t, reduction, g)
    assert all(torch.equal(got[k], again[k]) for k in got)
    check(got, xent_reference(x, W, b, t, -100, reduction, g))


def test_cross_entropy_single_gradients_in_blocks(T):
    """A gradient alone is the one that comes with the others, bit by bit."""
    x, W, b, t = rows_and_classes(400003, 24, 300, F32)
    want = run_xent(T, x, W, b, t, "mean", 1.0)
    for k in ("x", "W", "b"):
        q = {n: v.detach().requires_grad_(n == k) for n, v in (("x", x), ("W", W), ("b", b))}
        loss = T.linear_cross_entropy(q["x"], q["W"], t, q["b"])
        (got,) = torch.autograd.grad(loss, [q[k]])
        assert torch.equal(got, want[k]), k


def test_cross_entropy_forward_in_blocks_of_rows(T):
    """2^17 rows of 33000 classes: the parts of 516 waves a row are over 512 MiB, so
    the rows come in two blocks (65792 and the rest)."""
    R, D, V = (1 << 17) + 3, 8, 33000
    x, W, b, t = rows_and_classes(R, D, V, BF16)
    loss = T.linear_cross_entropy(x, W, t, b, reduction="none")
    for rows in (slice(0, 20), slice(65782, 65802), slice(R - 20, R)):
        ref = xent_reference(x[rows], W, b, t[rows], -100, "none", 1.0)
        within(loss[rows], *ref["loss"], "loss")
    # each block alone gives the same rows, bit by bit, and their sums are all of them's
    for rows in (slice(0, 65792), slice(65792, R)):
        assert torch.equal(T.linear_cross_entropy(x[rows], W, t[rows], b, reduction="none"), loss[rows])
    total, kept = loss.double().sum(), int((t != -100).sum())
    for reduction, want in (("sum", total), ("mean", total / kept)):
        got = T.linear_cross_entropy(x, W, t, b, reduction=reduction)
        within(got, want, 2 * U * want.abs(), reduction)


# ------------------------------------------------------------- captures and eager graphs
CAPTURED = {
    "layer_norm": lambda T, p: T.layer_norm(p["x"], p["w"]),
    "gated_mlp": lambda T, p: T.gated_mlp(p["x"], p["W"], p["W2"], p["D"]),
    "linear_cross_entropy": lambda T, p: T.linear_cross_entropy(p["x"], p["W"], p["t"])}


@pytest.mark.parametrize("op", CAPTURED)
def test_capture_that_meets_an_eager_graph_is_refused(T, op):
    """A captured backward whose leaf has an accumulation node of the default stream,
    kept alive by an eager output, raises before it hands that node a gradient; with
    the eager output gone the same capture runs and replays."""
    call = CAPTURED[op]
    p = {"x": rnd(1, 20, 8), "w": rnd(2, 8), "W": rnd(3, 12, 8), "W2": rnd(4, 12, 8),
         "D": rnd(5, 8, 12), "t": torch.arange(20, device=DEV) % 12}
    leaf = p["w" if op == "layer_norm" else "W"].requires_grad_(True)
    (want,) = torch.autograd.grad(call(T, p).sum(), [leaf])
    eager = call(T, p)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match=f"{op}: a captured backward"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(call(T, p).sum(), [leaf])
    # a gradient that goes elsewhere does not touch that node
    x = p["x"].requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (dx,) = torch.autograd.grad(call(T, p).sum(), [x])
    graph.replay()
    del eager
    (again,) = torch.autograd.grad(call(T, p).sum(), [x])
    assert torch.equal(dx, again)
    del again
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(call(T, p).sum(), [leaf])
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_cross_entropy_of_few_rows_in_blocks(T):
    """2^26 classes are 2^20 parts a row, 8 MiB: 100 rows come in two blocks of 50."""
    R, D, V = 100, 8, (1 << 26) - 5
    g = torch.Generator(DEV).manual_seed(1)
    x = torch.randn(R, D, device=DEV, generator=g).to(BF16)
    W = torch.randn(V, D, device=DEV, generator=g).to(BF16)
    t = torch.randint(0, V, (R,), device=DEV, generator=g)
    loss = T.linear_cross_entropy(x, W, t, reduction="none")
    xd = x.double()
    lse = torch.stack([torch.logsumexp(xd @ w.double().t(), -1) for w in W.split(1 << 22)]).logsumexp(0)
    z = (xd * W[t].double()).sum(-1)
    # a part's 64 terms, then 4096 parts a thread and 256 threads' sums; logits to a few steps
    bound = U * (4096 + 200 + 64 * (xd.abs().sum(-1) * W.abs().max().double()))
    within(loss, lse - z, bound, "loss")


# ------------------------------------------------- layouts and cuts of the tiled products
@pytest.mark.parametrize("C", [0, 2])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("by", [8, 3])  # rows that the tiles read in place, and not
def test_gate_and_up_weights_of_unlike_strides(T, C, dtype, by):
    """The gate's weights in wider rows (and members further apart) than the up's."""
    R, D, F, O = 150, 64, 1104, 40
    lead = (C,) if C else ()
    p = {"x": rnd(1, *lead, R, D, dtype=dtype),
         "Wg": rnd(2, *lead, F, D, dtype=dtype, scale=D ** -0.5),
         "Wu": rnd(3, *lead, F, D, dtype=dtype, scale=D ** -0.5),
         "Wd": rnd(4, *lead, O, F, dtype=dtype, scale=F ** -0.5)}
    dy = rnd(5, *lead, R, O, dtype=dtype)
    ref = gated_reference(p, dy, "silu")

    def spread(t, rows, cols):  # the same values, `rows` and `cols` more around them
        big = torch.full((*t.shape[:-2], t.shape[-2] + rows, t.shape[-1] + cols), 7.0,
                         device=DEV, dtype=dtype)
        big[..., :t.shape[-2], :t.shape[-1]] = t
        return big[..., :t.shape[-2], :t.shape[-1]]

    for one, other in (((0, by), (0, 0)), ((0, 0), (0, by)), ((8, 0), (0, 0)), ((8, by), (16, 2 * by))):
        q = p | {"Wg": spread(p["Wg"], *one), "Wu": spread(p["Wu"], *other)}
        q = {k: v.detach().requires_grad_(True) for k, v in q.items()}
        y = T.gated_mlp(*q.values())
        grads = torch.autograd.grad(y, list(q.values()), dy)
        check({"y": y} | dict(zip(q, grads)), ref)


def test_weight_gradients_cut_over_k_with_members(T):
    """4096 rows are the weight gradients' k axis, cut over workgroups for each of two
    members: partial sums [split][member]."""
    from d3rlpy_amd import _native as N
    C, R, D, F, O = 2, 4096, 64, 1104, 24
    d = N.GatedMlpDesc()
    d.rows, d.n_in, d.n_hidden, d.n_out, d.members = R, D, F, O, C
    d.ldx, d.ldWg, d.ldWu, d.ldWd, d.lddy = D, D, D, F, O
    d.sx, d.sWg, d.sWu, d.sWd, d.sdy = R * D, F * D, F * D, O * F, R * O
    for k in ("x", "Wg", "Wu", "Wd", "y", "dy", "kept", "dWd"):
        setattr(d, k, 256)
    d.dtype = 1
    size = ctypes.c_int64()
    assert N.lib().d3a_gated_mlp_workspace(ctypes.byref(d), 1, ctypes.byref(size)) == 0
    assert size.value >= 2 * C * O * F * 4  # (all operands in place: the partial sums alone)
    for dtype in (BF16, F32):
        p = {"x": rnd(1, C, R, D, dtype=dtype), "Wg": rnd(2, C, F, D, dtype=dtype, scale=D ** -0.5),
             "Wu": rnd(3, C, F, D, dtype=dtype, scale=D ** -0.5),
             "Wd": rnd(4, C, O, F, dtype=dtype, scale=F ** -0.5)}
        dy = rnd(5, C, R, O, dtype=dtype)
        q = {k: v.detach().requires_grad_(True) for k, v in p.items()}
        y = T.gated_mlp(*q.values())
        grads = torch.autograd.grad(y, list(q.values()), dy)
        check({"y": y} | dict(zip(q, grads)), gated_reference(p, dy, "silu"))


@pytest.mark.parametrize("V", [300, 5003])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_head_and_its_gradients_replay(T, V, dtype):
    """A block with a head of its own, captured through autograd: every gradient of
    every replay, the head's among them, is the eager pass's bit by bit."""
    D, F, R = 64, 160, 90
    q = {"x": rnd(1, R, D), "w": rnd(2, D, scale=0.1, shift=1.0), "c": rnd(3, D, scale=0.1),
         "Wg": rnd(4, F, D, scale=D ** -0.5), "Wu": rnd(5, F, D, scale=D ** -0.5),
         "Wd": rnd(6, D, F, scale=F ** -0.5), "head": rnd(7, V, D, scale=D ** -0.5), "b": rnd(8, V)}
    q = {k: v.to(dtype).requires_grad_(True) for k, v in q.items()}
    t = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(9)).to(DEV)

    def step():
        h = T.layer_norm(q["x"], q["w"], q["c"])
        r = q["x"] + T.gated_mlp(h, q["Wg"], q["Wu"], q["Wd"])
        loss = T.linear_cross_entropy(r, q["head"], t, q["b"])
        return [loss.detach()] + list(torch.autograd.grad(loss, list(q.values())))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            q["head"].mul_(1.0 + 0.1 * k)
            q["x"].add_(0.05 * k)
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, want = [o.clone() for o in out], step()
        for name, a, b in zip(["loss"] + list(q), got, want):
            assert torch.equal(a, b), (k, name)
