"""Entry points of include/ptl_tuning.h without a GPU: blobs whose sizes do not fit together are refused, outputs untouched; what a call does not use is
not looked at."""
import ctypes

import numpy as np
import pytest

import tuning as tn
from test_tuning_args import np_type, refused


def accepted(pkg, name, a, n):
    """Not refused: an empty batch is fine, and without a device a batch fails for want of it (nothing here may reach one)."""
    import torch
    lib = pkg.load()
    assert getattr(lib, name)(ctypes.byref(a), 0) == 0
    if not torch.cuda.is_available():
        assert getattr(lib, name)(ctypes.byref(a), n) == 2 and b"no CPU fallback" in lib.ptl_last_error()


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_act_linear(pkg, dt):
    t = np_type(dt)
    fw, bw = ("ptl_act_linear_%s_%s_batched" % (dt, s) for s in ("fw", "bw"))
    x, w, y, b = np.ones((2, 6), t), np.ones((5, 6), t), np.full((2, 5), 7, t), np.ones(5, t)
    full = dict(x=x, dx=x.copy(), w=w, dw=w.copy(), b=b, db=b.copy(), h=y, dh=y.copy(), skip=y, y=y, dy=y.copy())
    for name in (fw, bw):
        for field, wrong in (("coeff", 29), ("coeff", 6), ("bias", 4), ("bias", 6), ("hidden", 4), ("hidden", 10), ("skip", 6)):
            if (name, field) == (bw, "skip"):
                continue  # (only the forward call reads it)
            a, keep = tn.act_args(pkg, 6, 5, 1, **full)
            getattr(a, field).contents.dim = wrong
            refused(pkg, name, a, 2, says="sizes")
        a, keep = tn.act_args(pkg, 6, 5, 1, **full)
        a.output.contents.dim = 4
        refused(pkg, name, a, 2, says="sizes")
        accepted(pkg, name, tn.act_args(pkg, 6, 5, 1, **full)[0], 2)
    a, keep = tn.act_args(pkg, 6, 5, 1, **full)  # what is not used
    a.bias.contents.dim, a.hidden.contents.dim, a.use_biases, a.hidden.contents.data = 0, 0, 0, None
    accepted(pkg, fw, a, 2)
    a, keep = tn.act_args(pkg, 6, 5, 4, **full)
    a.hidden.contents.dim, a.skip.contents.dim = 0, 0
    accepted(pkg, bw, a, 2)
    a, keep = tn.act_args(pkg, 6, 5, 4, **full, skip_wg=1)
    a.bias.contents.dim = 0
    accepted(pkg, bw, a, 2)
    a, keep = tn.act_args(pkg, 6, 5, 1, **full, skip_wg=1, skip_ig=1)
    a.bias.contents.dim = a.coeff.contents.dim = 0
    accepted(pkg, bw, a, 2)
    assert (y == 7).all() and (x == 1).all() and (w == 1).all()


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_norm_join(pkg, dt):
    t = np_type(dt)
    fw, bw = ("ptl_norm_join_%s_%s_batched" % (dt, s) for s in ("fw", "bw"))
    x, w, y, gates = np.ones((6, 8), t), np.ones(8, t), np.full((6, 8), 7, t), np.ones((3, 8), t)
    full = dict(b=x, db=y, x=x, dx=y, gate=gates, dgate=gates.copy(), w1=w, dw1=w.copy(), w2=w, dw2=w.copy(), s=y, ds=x, y=y, dy=x, per=2)
    for name in (fw, bw):
        for field, wrong in [(f, d) for f in ("skip", "sum", "coeff_post", "coeff_pre", "output") for d in (7, 16, 0)] + [("gate", 7), ("gate", 12), ("gate", 16), ("gate", 0)]:
            a, keep = tn.join_args(pkg, 8, **full)
            getattr(a, field).contents.dim = wrong
            refused(pkg, name, a, 6, says="sizes")
        for dim in (8, 24, 32):  # one gate's elements, all of them, more
            a, keep = tn.join_args(pkg, 8, **full)
            a.gate.contents.dim = dim
            accepted(pkg, name, a, 6)
        a, keep = tn.join_args(pkg, 8, **{**full, "w2": None, "dw2": None})  # what is not used
        a.output = ctypes.pointer(pkg.blob(y, None, dim=3))
        accepted(pkg, name, a, 6)
    a, keep = tn.join_args(pkg, 8, **full, skip_ig=1)
    a.skip.contents.dim = 0
    accepted(pkg, bw, a, 6)
    assert (y == 7).all() and (w == 1).all() and (x == 1).all()
