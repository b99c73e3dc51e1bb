"""layer_norm, gated_mlp, linear_cross_entropy without a GPU: derivatives that they do
not have, and the scratch of large calls."""
import os

import pytest
import torch
import torch.autograd.forward_ad as fwad


@pytest.fixture(scope="module")
def T():
    from d3rlpy_amd import _build, torch_ops
    if not os.path.exists(torch_ops.library_path()):
        _build.build()
    torch_ops.load()
    return torch_ops


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


# every floating input of each operator: shapes, and the call
CALLS = {
    "layer_norm": (((4, 8), (8,), (8,)), lambda T, x, w, b: T.layer_norm(x, w, b)),
    "gated_mlp": (((4, 8), (5, 8), (5, 8), (3, 5), (5,), (5,), (3,)),
                  lambda T, *a: T.gated_mlp(*a)),
    "linear_cross_entropy": (((4, 8), (9, 8), (9,)),
                             lambda T, x, W, b: T.linear_cross_entropy(
                                 x, W, torch.empty(4, dtype=torch.int64, device="meta"), b)),
}
EACH = [(op, i) for op, (shapes, _) in CALLS.items() for i in range(len(shapes))]


@pytest.mark.parametrize("op,i", EACH)
@pytest.mark.parametrize("leaf", [False, True])
def test_forward_mode_is_refused(T, op, i, leaf):
    """A tangent of any input raises, as torch_ops.linear does; it is not dropped."""
    shapes, call = CALLS[op]
    a = [meta(*s).requires_grad_(leaf) for s in shapes]
    with fwad.dual_level():
        a[i] = fwad.make_dual(a[i], meta(*shapes[i]))
        with pytest.raises(NotImplementedError, match=f"{op} has no forward-mode"):
            call(T, *a)


@pytest.mark.parametrize("op,i", EACH)
def test_func_jvp_is_refused(T, op, i):
    shapes, call = CALLS[op]
    a = [meta(*s) for s in shapes]

    def f(t):
        return call(T, *(a[:i] + [t] + a[i + 1:]))
    with pytest.raises(NotImplementedError, match=f"{op} has no forward-mode"):
        torch.func.jvp(f, (a[i],), (meta(*shapes[i]),))


@pytest.mark.parametrize("op", CALLS)
def test_tangent_of_the_outputs_gradient_is_refused(T, op):
    """(linear in that gradient, but the backward kernels would drop it too)"""
    shapes, call = CALLS[op]
    a = [meta(*s).requires_grad_(True) for s in shapes]
    y = call(T, *a)
    with fwad.dual_level():
        g = fwad.make_dual(meta(*y.shape), meta(*y.shape))
        with pytest.raises(NotImplementedError, match=f"{op} has no forward-mode"):
            torch.autograd.grad(y, a, g)


@pytest.mark.parametrize("op", CALLS)
def test_calls_without_a_tangent_still_run_in_a_dual_level(T, op):
    shapes, call = CALLS[op]
    a = [meta(*s).requires_grad_(True) for s in shapes]
    with fwad.dual_level():
        y = call(T, *a)
        grads = torch.autograd.grad(y, a, meta(*y.shape))
    assert [g.shape for g in grads] == [t.shape for t in a]


def xent_workspace(rows, n_in, vocab, dtype, bwd, reduction=1):
    import ctypes
    from d3rlpy_amd import _native as N
    d = N.LinearXentDesc()
    d.rows, d.n_in, d.vocab, d.ldx, d.ldW, d.dtype, d.reduction = (rows, n_in, vocab, n_in, n_in,
                                                                   dtype, reduction)
    for k in ("x", "W", "b", "target", "loss", "lse", "out", "scale", "gloss", "dx", "dW", "db"):
        setattr(d, k, 256)
    n = ctypes.c_int64()
    assert N.lib().d3a_linear_xent_workspace(ctypes.byref(d), bwd, ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("dtype,planes", [(0, 3), (1, 1)])
@pytest.mark.parametrize("rows,vocab", [
    (6000, 29826), (8192, 32768), (8000, 33001), (8192, 1 << 20), (1 << 17, 65536),
    (1 << 20, 65536), (1 << 20, 300), (1 << 22, 65536), (1 << 23, 40), (1 << 24, 1 << 18),
    (37, 1 << 26), (100, 1 << 26), (300, 1 << 27), (1 << 26, 2000)])
def test_cross_entropy_scratch_does_not_grow_with_the_logits(T, dtype, planes, rows, vocab):
    """Either direction's scratch is 512 MiB for what has a value a logit (or a wave's
    64), whatever rows x vocabulary is, and what goes with x and W."""
    D = 8
    MiB, pad = 1 << 20, 1 << 16
    copies = 6 * (rows + vocab) * D if planes == 3 else 0  # float32 operands are packed
    per_row = 8 * rows  # the targets' logits
    assert xent_workspace(rows, D, vocab, dtype, 0) <= 512 * MiB + copies + per_row + pad
    # partial sums of at most 1280 tiles' rows of D; the columns' sums, of at least 32 rows
    # of a piece each, and of 256 columns x 256 chunks a block of rows
    blocks = rows * planes // (1 << 20) + 2
    extra = 1280 * 256 * 4 * D + 36 * MiB + blocks * 256 * 256 * 4
    sums = 4 * rows * D + 4 * 256 * D  # dx over pieces, dW over blocks
    assert xent_workspace(rows, D, vocab, dtype, 1) <= 512 * MiB + copies + sums + extra + pad


def test_cross_entropy_scratch_of_many_rows(T):
    """The forward's parts of 2^20 rows x 65536 classes are 8 GiB, dz's of 2^22 rows 2
    GiB a 256 columns: both within 512 MiB, by blocks of rows."""
    GiB = 1 << 30
    assert xent_workspace(1 << 20, 8, 65536, 1, 0) < 0.6 * GiB
    assert xent_workspace(1 << 22, 8, 65536, 1, 1) < 0.8 * GiB
    assert xent_workspace(1 << 20, 8, 65536, 0, 1) < 0.7 * GiB
    # and cut down, not up: two pieces of 15104 columns were 518.6 MiB
    assert xent_workspace(6000, 8, 29826, 0, 1) < 512 * (1 << 20) + 8 * (1 << 20)
