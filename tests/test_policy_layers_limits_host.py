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
