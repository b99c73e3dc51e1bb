"""layer_norm, gated_mlp, linear_cross_entropy without a GPU: output shapes on
the meta device, refused calls, the C descriptors' layouts, argument checks and
workspace sizes."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

HEADER = Path(__file__).resolve().parents[1] / "include" / "d3rlpy_amd.h"


@pytest.fixture(scope="module")
def T():
    from d3rlpy_amd import _build, torch_ops
    import os
    if not os.path.exists(torch_ops.library_path()):
        _build.build()
    torch_ops.load()
    return torch_ops


def meta(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_meta_shapes(T):
    ops = T.load()
    y, stats = ops.layer_norm(meta(4, 5, 8), meta(8), meta(8), 1e-5)
    assert y.shape == (4, 5, 8) and stats.shape == (2, 1, 20)
    y, stats = ops.layer_norm(meta(4, 5, 8, dtype=torch.bfloat16), meta(4, 8), None, 1e-5)
    assert y.dtype == torch.bfloat16 and stats.shape == (2, 4, 5) and stats.dtype == torch.float32
    assert T.gated_mlp(meta(7, 6), meta(12, 6), meta(12, 6), meta(3, 12)).shape == (7, 3)
    assert T.gated_mlp(meta(2, 7, 6), meta(12, 6), meta(12, 6), meta(3, 12)).shape == (2, 7, 3)
    W = meta(4, 12, 6), meta(4, 12, 6), meta(4, 3, 12)
    assert T.gated_mlp(meta(7, 6), *W).shape == (4, 7, 3)
    assert T.gated_mlp(meta(4, 7, 6), *W).shape == (4, 7, 3)
    y, kept = ops.gated_mlp(meta(7, 6), *W, None, None, None, "silu", True)
    # g, u float32 and h's three planes, rows of 12 rounded up to 16
    assert kept.shape == (4 * 7 * 16 * (8 + 6),) and kept.dtype == torch.uint8
    t = torch.empty(4, 5, dtype=torch.int64, device="meta")
    assert T.linear_cross_entropy(meta(4, 5, 8), meta(99, 8), t).shape == ()
    loss = T.linear_cross_entropy(meta(4, 5, 8, dtype=torch.bfloat16),
                                  meta(99, 8, dtype=torch.bfloat16), t, reduction="none")
    assert loss.shape == (4, 5) and loss.dtype == torch.float32


def test_meta_gradients(T):
    x, w = meta(4, 8).requires_grad_(True), meta(8).requires_grad_(True)
    dx, dw = torch.autograd.grad(T.layer_norm(x, w).sum(), [x, w])
    assert dx.shape == (4, 8) and dw.shape == (8,)
    W = [meta(12, 8).requires_grad_(True), meta(12, 8).requires_grad_(True),
         meta(5, 12).requires_grad_(True)]
    grads = torch.autograd.grad(T.gated_mlp(x, *W).sum(), [x] + W)
    assert [g.shape for g in grads] == [t.shape for t in [x] + W]
    t = torch.empty(4, dtype=torch.int64, device="meta")
    dW, = torch.autograd.grad(T.linear_cross_entropy(x, W[0], t), [W[0]])
    assert dW.shape == (12, 8)


@pytest.mark.parametrize("call,match", [
    (lambda T: T.layer_norm(meta(4, 8), meta(7)), "weight / bias of 7"),
    (lambda T: T.layer_norm(meta(4, 8), meta(3, 8)), "members"),
    (lambda T: T.layer_norm(meta(0, 4, 8), meta(0, 8)), "no member"),
    (lambda T: T.layer_norm(meta(4, 8), meta(8), meta(1, 8)), "one shape and dtype"),
    (lambda T: T.layer_norm(meta(4, 0)), "empty last"),
    (lambda T: T.gated_mlp(meta(4, 8), meta(5, 7), meta(5, 7), meta(8, 5)), "8 features"),
    (lambda T: T.gated_mlp(meta(4, 8), meta(5, 8), meta(6, 8), meta(8, 5)), "Wu must"),
    (lambda T: T.gated_mlp(meta(4, 8), meta(5, 8), meta(5, 8), meta(8, 6)), "Wd"),
    (lambda T: T.gated_mlp(meta(3, 4, 8), meta(2, 5, 8), meta(2, 5, 8), meta(2, 8, 5)), "members"),
    (lambda T: T.gated_mlp(meta(4, 8), meta(5, 8), meta(5, 8), meta(8, 5), meta(4)), "bias"),
    (lambda T: T.gated_mlp(meta(4, 8), meta(5, 8), meta(5, 8), meta(8, 5), activation="tanh"),
     "'silu', 'gelu' or 'relu'"),
    (lambda T: T.linear_cross_entropy(meta(4, 8), meta(9, 7), meta(4).long()), "8 features"),
    (lambda T: T.linear_cross_entropy(meta(4, 8), meta(9, 8), meta(5).long()), "one target"),
    (lambda T: T.linear_cross_entropy(meta(4, 8), meta(9, 8), meta(4)), "int64"),
    (lambda T: T.linear_cross_entropy(meta(4, 8), meta(9, 8), meta(4).long(), meta(8)), r"b \[vocab\]"),
    (lambda T: T.linear_cross_entropy(meta(4, 8), meta(9, 8), meta(4).long(), reduction="max"),
     "'none', 'mean' or 'sum'"),
])
def test_refused_shapes(T, call, match):
    with pytest.raises(RuntimeError, match=match):
        call(T)


def test_no_cpu_path(T):
    with pytest.raises((RuntimeError, NotImplementedError)):
        T.layer_norm(torch.zeros(2, 4), torch.ones(4), torch.zeros(4))


def test_struct_layouts_match_header(tmp_path):
    from d3rlpy_amd import _native as N
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    pairs = (("d3a_gated_mlp_desc", N.GatedMlpDesc), ("d3a_linear_xent_desc", N.LinearXentDesc),
             ("d3a_layer_norm_desc", N.LayerNormDesc))
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){"]
    for cname, cls in pairs:
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run([cc, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    at = dict(line.rsplit(" ", 1) for line in out.splitlines())
    for cname, cls in pairs:
        assert int(at[cname]) == ctypes.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert int(at[f"{cname}.{f}"]) == getattr(cls, f).offset, (cname, f)


def gated_desc(**kw):
    from d3rlpy_amd import _native as N
    d = N.GatedMlpDesc()
    d.rows, d.n_in, d.n_hidden, d.n_out, d.members = 100, 32, 64, 48, 1
    d.ldx, d.ldWg, d.ldWu, d.ldWd, d.lddy = 32, 32, 32, 64, 48
    for k in ("x", "Wg", "Wu", "Wd", "y", "dy", "kept"):
        setattr(d, k, 256)
    d.dtype = 1
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def error():
    from d3rlpy_amd import _native as N
    return N.lib().d3a_last_error().decode()


@pytest.mark.parametrize("kw,bwd,match", [
    (dict(dtype=2), False, "dtype"), (dict(act=3), False, "activation"),
    (dict(rows=-1), False, "positive"), (dict(n_hidden=0), False, "positive"),
    (dict(n_in=(1 << 21) + 1, ldx=1 << 22, ldWg=1 << 22, ldWu=1 << 22), False, "too large"),
    (dict(members=65536), False, "too large"), (dict(ldx=31), False, "row stride"),
    (dict(ldWd=63), False, "row stride"), (dict(Wu=None), False, "null weight"),
    (dict(x=None), False, "null operand"), (dict(y=None), False, "null operand"),
    (dict(kept=8), False, "16-byte"), (dict(dy=None), True, "null operand"),
    (dict(kept=None), True, "kept"), (dict(lddy=47), True, "row stride"),
    (dict(), False, "workspace of"), (dict(ws=256, ws_bytes=10), True, "workspace of"),
    (dict(ws=264, ws_bytes=1 << 30), True, "workspace of"),
])
def test_gated_descriptor_checks(kw, bwd, match):
    """(a call that would launch is never reached: every one is refused before)"""
    from d3rlpy_amd import _native as N
    if not bwd:
        kw = {"kept": None} | kw  # without kept the forward needs scratch for h
    d = gated_desc(**kw)
    d.dx = 256 if bwd else None
    fn = N.lib().d3a_gated_mlp_bwd if bwd else N.lib().d3a_gated_mlp
    assert fn(ctypes.byref(d), None) < 0 and match in error()


def test_gated_workspaces():
    from d3rlpy_amd import _native as N
    lib, n = N.lib(), ctypes.c_int64()

    def size(d, bwd):
        assert lib.d3a_gated_mlp_workspace(ctypes.byref(d), bwd, ctypes.byref(n)) == 0, error()
        return n.value
    # aligned bfloat16 operands are read in place: h alone, or nothing with kept
    assert size(gated_desc(kept=None), 0) == 100 * 64 * 2
    assert size(gated_desc(), 0) == 0
    # a minibatch reads unaligned operands as they lie; tiles have x packed
    wide = dict(n_hidden=1104, ldWd=1104)
    assert size(gated_desc(kept=None, x=258), 0) == 100 * 64 * 2
    assert size(gated_desc(**wide), 0) == 0
    assert size(gated_desc(kept=None, x=258, **wide), 0) >= 100 * (1104 + 32) * 2
    # the backward's dg and du, and nothing for gradients that nobody wants
    assert size(gated_desc(dx=256), 1) >= 2 * 100 * 64 * 2
    assert size(gated_desc(), 1) == 0
    # float32: three planes of every operand of a tile
    f = gated_desc(dtype=0, kept=None, **wide)
    assert size(f, 0) >= 3 * 2 * (100 * 1104 + 100 * 32 + 2 * 1104 * 32 + 48 * 1104)
    f = gated_desc(dtype=0, kept=None)
    assert size(f, 0) == 4 * 100 * 64
    assert lib.d3a_gated_mlp_kept(ctypes.byref(f), ctypes.byref(n)) == 0
    assert n.value == 100 * 64 * (8 + 6)


def test_xent_descriptor_checks():
    from d3rlpy_amd import _native as N
    lib = N.lib()

    def desc(**kw):
        d = N.LinearXentDesc()
        d.rows, d.n_in, d.vocab, d.ldx, d.ldW, d.dtype = 50, 32, 1000, 32, 32, 1
        for k in ("x", "W", "target", "loss", "lse", "out", "scale", "gloss"):
            setattr(d, k, 256)
        for k, v in kw.items():
            setattr(d, k, v)
        return d
    for kw, match in ((dict(dtype=5), "dtype"), (dict(reduction=3), "reduction"),
                      (dict(vocab=0), "positive"), (dict(ldW=31), "row stride"),
                      (dict(target=None), "null operand"), (dict(W=None), "null weight"),
                      (dict(reduction=1, out=None), "out and scale"),
                      (dict(n_in=1 << 22, ldx=1 << 22, ldW=1 << 22), "too large"),
                      (dict(), "workspace of")):
        assert lib.d3a_linear_xent(ctypes.byref(desc(**kw)), None) < 0 and match in error(), kw
    assert lib.d3a_linear_xent_bwd(ctypes.byref(desc(gloss=None, dx=256)), None) < 0
    assert "null gradient" in error()
    # the backward's scratch is bounded by the piece of the vocabulary, not by all of it
    n = ctypes.c_int64()
    big = desc(rows=8192, n_in=512, ldx=512, ldW=512, vocab=1 << 20, dx=256, dW=256, db=256)
    assert lib.d3a_linear_xent_workspace(ctypes.byref(big), 1, ctypes.byref(n)) == 0
    assert n.value < (1 << 30)


def test_norm_descriptor_checks():
    from d3rlpy_amd import _native as N
    lib = N.lib()

    def desc(**kw):
        d = N.LayerNormDesc()
        d.rows, d.n, d.members, d.ldx, d.lddy = 10, 64, 1, 64, 64
        for k in ("x", "w", "b", "y", "mean", "rstd", "dy", "dx", "dw", "db"):
            setattr(d, k, 256)
        for k, v in kw.items():
            setattr(d, k, v)
        return d
    for kw, match in ((dict(dtype=2), "dtype"), (dict(dtype=0, wtype=1), "weight and bias"),
                      (dict(n=0), "positive"), (dict(ldx=63), "row stride"),
                      (dict(y=None), "null operand"), (dict(mean=None), "go together"),
                      (dict(rows=1 << 31), "too large")):
        assert lib.d3a_layer_norm(ctypes.byref(desc(**kw)), None) < 0 and match in error(), kw
    for kw, match in ((dict(dy=None), "null operand"), (dict(mean=None, rstd=None), "mean and rstd"),
                      (dict(), "workspace of")):
        assert lib.d3a_layer_norm_bwd(ctypes.byref(desc(**kw)), None) < 0 and match in error(), kw
