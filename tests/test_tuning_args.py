"""Entry points of include/ptl_tuning.h without a GPU: what the header declares is exported and listed, the ctypes mirrors match the
C layout, and calls are refused before any device work, outputs untouched."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

import tuning as tn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CLANG = "/opt/rocm/lib/llvm/bin/clang"
HEADER = os.path.join(ROOT, "include", "ptl_tuning.h")
STRUCTS = {"ActLinear_args": "ActLinearArgs", "NormJoin_args": "NormJoinArgs", "policy_loss_args": "PolicyLossArgs", "adamw_args": "AdamwArgs"}
SINGLE = {"adamw_state": "AdamwState", "adamw_step": "AdamwStep"}


def test_exports_and_lists(pkg):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"^int\s+(\w+)\s*\(", text, flags=re.M))
    assert len(names) == 12
    assert names == set(pkg.TUNING_ENTRY_POINTS + pkg.POLICY_ENTRY_POINTS + pkg.ADAMW_ENTRY_POINTS)
    assert all(hasattr(pkg.load(), n) for n in names)


def test_ctypes_mirrors_match_c_layout(pkg, tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "ptl_api.h"', "int main(void){"]
    pairs = [(c + sfx, py) for c, py in STRUCTS.items() for sfx in ("", "_fp16")] + list(SINGLE.items())
    for cname, py in pairs:
        for f, _ in getattr(pkg, py)._fields_:
            lines.append('printf("%s %s %%zu %%zu\\n", sizeof(struct %s), offsetof(struct %s, %s));' % (py, f, cname, cname, f))
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.check_call([CLANG, "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    for line in subprocess.check_output([str(exe)], text=True).split("\n")[:-1]:
        py, f, size, off = line.split()
        assert ctypes.sizeof(getattr(pkg, py)) == int(size), line
        assert getattr(getattr(pkg, py), f).offset == int(off), line


def refused(pkg, name, a, *more, says):
    lib = pkg.load()
    assert getattr(lib, name)(ctypes.byref(a) if a is not None else None, *more) == 1, name
    assert says in lib.ptl_last_error().decode(), lib.ptl_last_error()


def np_type(dt):
    return np.float32 if dt == "fp32" else np.float16


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_act_linear_refusals(pkg, dt):
    t = np_type(dt)
    fw, bw = ("ptl_act_linear_%s_%s_batched" % (dt, s) for s in ("fw", "bw"))
    x, w, y = np.ones((2, 6), t), np.ones((5, 6), t), np.full((2, 5), 7, t)

    def args(n_in=6, n_out=5, act=1, **k):
        return tn.act_args(pkg, n_in, n_out, act, **{**dict(x=x, w=w, y=y), **k})

    refused(pkg, fw, None, 2, says="null argument")
    for k, says in ((dict(n_in=0), "geometry"), (dict(n_out=0), "geometry"), (dict(act=5), "activation"), (dict(act=-1), "activation"),
                    (dict(n_in=2 ** 27 + 1), "geometry"), (dict(n_out=2 ** 30), "geometry"), (dict(x=None), "null buffer"), (dict(w=None), "null buffer"),
                    (dict(y=None), "null buffer"), (dict(db=y), "null buffer")):
        a, keep = args(**k)
        refused(pkg, fw, a, 2, says=says)
    a, keep = args(skip=y)
    a.skip.contents.data = None
    refused(pkg, fw, a, 2, says="null buffer")
    a, keep = args()
    a.use_biases = 1
    refused(pkg, fw, a, 2, says="null bias")
    full = dict(dx=x.copy(), dw=w.copy(), h=y, dh=y.copy(), dy=y.copy())
    a, keep = args(**{k: v for k, v in full.items() if k not in ("h", "dh")})
    refused(pkg, bw, a, 2, says="null argument")
    for gone in ("dx", "dw", "h", "dh", "dy", "x", "w"):
        a, keep = args(**{**full, gone: None})
        refused(pkg, bw, a, 2, says="null buffer")
    for n, n_in, n_out in ((2 ** 10, 2 ** 21, 1), (2 ** 10, 1, 2 ** 21), (1, 2 ** 20, 2 ** 11)):  # inputs, outputs, weights of 2^31
        a, keep = args(n_in, n_out, **full)
        refused(pkg, bw, a, n, says="2^31")
    for name in (fw, bw):
        a, keep = args(**full)
        refused(pkg, name, a, 2 ** 30 + 1, says="2^30")
        assert getattr(pkg.load(), name)(ctypes.byref(a), 0) == 0
    a, keep = args(act=4, dy=y, skip_wg=1, skip_ig=1)  # nothing is wanted
    assert getattr(pkg.load(), bw)(ctypes.byref(a), 0) == 0
    assert (y == 7).all() and (x == 1).all() and (w == 1).all()


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_norm_join_refusals(pkg, dt):
    t = np_type(dt)
    fw, bw = ("ptl_norm_join_%s_%s_batched" % (dt, s) for s in ("fw", "bw"))
    x, w, y = np.ones((2, 8), t), np.ones(8, t), np.full((2, 8), 7, t)

    def args(dim=8, **k):
        return tn.join_args(pkg, dim, **{**dict(b=x, x=x, w1=w, w2=w, s=y, y=y, gate=w), **k})

    refused(pkg, fw, None, 2, says="null argument")
    for k, says in ((dict(dim=0), "geometry"), (dict(dim=-1), "geometry"), (dict(dim=2 ** 24 + 1), "geometry"), (dict(eps=-1.0), "eps"),
                    (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(alpha=float("nan")), "skip_scale"),
                    (dict(alpha=float("inf")), "skip_scale"), (dict(per=-1), "rows_per_gate"), (dict(b=None), "null buffer"), (dict(x=None), "null buffer"),
                    (dict(w1=None), "null buffer"), (dict(s=None), "null buffer"), (dict(y=None), "null buffer"), (dict(w2=None, dw2=w), "null buffer"),
                    (dict(gate=None, dgate=w), "null buffer")):
        a, keep = args(**k)
        refused(pkg, fw, a, 2, says=says)
    for gone in ("input", "skip", "coeff_post", "sum", "output"):
        a, keep = args()
        setattr(a, gone, None)
        refused(pkg, fw, a, 2, says="null argument")
    full = dict(db=y, dx=y, dw1=w, dw2=w, dgate=w, ds=x, dy=x)
    for gone in ("db", "dx", "dw1", "dw2", "dgate", "dy", "s", "b"):
        a, keep = args(**{**full, gone: None})
        refused(pkg, bw, a, 2, says="null buffer")
    a, keep = args(**{**full, "w2": None, "dw2": None, "ds": None})  # no gradient comes in
    refused(pkg, bw, a, 2, says="null buffer")
    for name in (fw, bw):
        a, keep = args(**full)
        refused(pkg, name, a, 2 ** 30 + 1, says="2^30")
        assert getattr(pkg.load(), name)(ctypes.byref(a), 0) == 0
    a, keep = args(dy=x, skip_wg=1, skip_ig=1)  # nothing is wanted
    assert getattr(pkg.load(), bw)(ctypes.byref(a), 2) == 0
    assert (y == 7).all() and (w == 1).all() and (x == 1).all()


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_policy_refusals(pkg, dt):
    t = np_type(dt)
    name = "ptl_policy_loss_%s_batched" % dt
    z, g, c, f, loss = np.ones((2, 9), t), np.full((2, 9), 7, t), np.zeros(2, np.int32), np.ones(2, np.float32), np.full(2, 7, np.float32)

    def args(grad=g):
        return tn.policy_args(pkg, z, grad, c, f, f, f, f, loss, loss)

    refused(pkg, name, None, 2, 2, says="null argument")
    nan, inf = float("nan"), float("inf")
    for k, v, says in (("temperature", 0.0, "temperature"), ("temperature", nan, "temperature"), ("temperature", inf, "temperature"),
                       ("clip_low", -0.1, "border"), ("clip_high", -0.1, "border"), ("clip_low", nan, "border"), ("clip_high", nan, "border"),
                       ("beta", inf, "beta"), ("beta", nan, "beta"), ("weight", inf, "weight"), ("weight", nan, "weight"), ("actions", None, "null buffer"),
                       ("old_logp", None, "null buffer"), ("advantages", None, "null buffer"), ("wr_loss", None, "null buffer")):
        a, keep = args()
        setattr(a, k, v)
        refused(pkg, name, a, 2, 2, says=says)
    for step in (-1, 3):
        a, keep = args()
        refused(pkg, name, a, 2, step, says="step")
    a, keep = args()
    a.output.contents.dim = 0
    refused(pkg, name, a, 2, 2, says="geometry")
    a, keep = args(grad=None)
    refused(pkg, name, a, 2, 1, says="null buffer")
    a, keep = args()
    refused(pkg, name, a, 2 ** 30 + 1, 2, says="2^30")
    assert getattr(pkg.load(), name)(ctypes.byref(a), 0, 2) == 0
    assert (g == 7).all() and (loss == 7).all()


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_adamw_refusals(pkg, dt):
    t, lib, keep = np_type(dt), pkg.load(), []
    f = getattr(lib, "ptl_adamw_%s_multi" % dt)
    w, g, u = np.ones(300, t), np.ones(300, t), np.full(300, 7, t)
    m, v, q, p, s, sm = (np.full(300, 7, k) for k in (np.float32, np.float32, np.int8, np.uint8, np.float32, np.float32))
    wide = lambda **k: tn.state(pkg, keep, **{**dict(m=m, v=v), **k})  # noqa: E731
    eight = lambda **k: tn.state(pkg, keep, **{**dict(m_root=q, v_root=p, m_scale=s, v_scale=sm), **k})  # noqa: E731

    def one(state=None, new=None, data=w, diff=g, updated=u, dim=300, dim_u=300):
        a = (pkg.AdamwArgs * 1)()
        a[0].weights = ctypes.pointer(pkg.blob(data, diff, dim=dim))
        if updated is not None:
            a[0].updated = ctypes.pointer(pkg.blob(updated, None, dim=dim_u))
        if state is not None:
            a[0].state = state
        if new is not None:
            a[0].new_state = new
        a[0].learning_rate = 0.5
        return a

    def no(a, count, step, says):
        assert f(a, count, ctypes.byref(step) if step is not None else None) == 1
        assert says in lib.ptl_last_error().decode(), lib.ptl_last_error()

    ok = tn.adamw_step(pkg)
    no(None, 1, ok, "null argument")
    no(one(wide()), 1, None, "null argument")
    for k, says in ((dict(beta1=1.0), "beta"), (dict(beta2=-0.1), "beta"), (dict(beta1=float("nan")), "beta"), (dict(eps=0.0), "eps"),
                    (dict(eps=float("inf")), "eps"), (dict(eps=float("nan")), "eps"), (dict(t=0), "from 1 on")):
        no(one(wide()), 1, tn.adamw_step(pkg, **k), says)
    a = one(wide())
    a[0].weights = None
    no(a, 1, ok, "null argument")
    no(one(), 1, ok, "neither")
    for s_, n_ in ((wide(v=None), None), (wide(m_root=q), None), (eight(v_scale=None), None), (eight(m=m), None), (wide(), eight()), (eight(), wide())):
        no(one(s_, n_), 1, ok, "a state holds")
    no(one(wide(master=m), wide()), 1, ok, "master")
    no(one(wide(), wide(master=m)), 1, ok, "master")
    for k, says in ((dict(data=None), "null buffer"), (dict(diff=None), "null buffer"), (dict(dim=-1), "geometry"), (dict(dim_u=299), "geometry"),
                    (dict(data=None, updated=None), "null buffer")):
        no(one(wide(), **k), 1, ok, says)
    for field in ("learning_rate", "weight_decay"):
        a = one(wide())
        setattr(a[0], field, float("inf"))
        no(a, 1, ok, "rate")
    two = (pkg.AdamwArgs * 2)(one(wide())[0], one()[0])  # the second is wrong: the first is not worked on
    no(two, 2, ok, "neither")
    assert f(None, 0, None) == 0 and f(one(wide()), -1, ctypes.byref(ok)) == 0
    assert all((b == 7).all() for b in (u, m, v, q, p, s, sm)) and (w == 1).all()


def test_no_device_is_reported(pkg):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    x, w, y = np.ones((2, 8), np.float32), np.ones((4, 8), np.float32), np.full((2, 4), 7, np.float32)
    a, keep = tn.act_args(pkg, 8, 4, 4, x=x, w=w, y=y)
    assert pkg.load().ptl_act_linear_fp32_fw_batched(ctypes.byref(a), 2) == 2
    assert b"no CPU fallback" in pkg.load().ptl_last_error() and (y == 7).all()
