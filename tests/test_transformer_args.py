"""Entry points of include/ptl_transformer.h without a GPU: what the header declares is exported and listed, the ctypes mirrors
match the C layout, and calls are refused before any device work, outputs untouched."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

import transformer as tr

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CLANG = "/opt/rocm/lib/llvm/bin/clang"
HEADER = os.path.join(ROOT, "include", "ptl_transformer.h")
STRUCTS = {"RmsNorm_args": "RmsNormArgs", "GatedLinear_args": "GatedLinearArgs", "matMul_int8_args": "MatMulInt8Args",
           "distill_args": "DistillArgs"}


def test_exports_and_lists(pkg):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"^int\s+(\w+)\s*\(", text, flags=re.M))
    assert len(names) == 12
    assert names == set(pkg.ROW_ENTRY_POINTS + pkg.INT8_ENTRY_POINTS + pkg.DISTILL_ENTRY_POINTS)
    assert all(hasattr(pkg.load(), n) for n in names)


def test_ctypes_mirrors_match_c_layout(pkg, tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "ptl_api.h"', "int main(void){"]
    for cname, py in STRUCTS.items():
        for sfx in ("", "_fp16"):
            for f, _ in getattr(pkg, py)._fields_:
                lines.append('printf("%s %s %%zu %%zu\\n", sizeof(struct %s%s), offsetof(struct %s%s, %s));'
                             % (py, f, cname, sfx, cname, sfx, f))
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.check_call([CLANG, "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    for line in subprocess.check_output([str(exe)], text=True).split("\n")[:-1]:
        py, f, size, off = line.split()
        assert ctypes.sizeof(getattr(pkg, py)) == int(size), line
        assert getattr(getattr(pkg, py), f).offset == int(off), line


def refused(pkg, name, a, *more, says=None):
    lib = pkg.load()
    assert getattr(lib, name)(ctypes.byref(a) if a is not None else None, *more) == 1, name
    if says:
        assert says in lib.ptl_last_error().decode(), lib.ptl_last_error()


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_rms_norm_refusals(pkg, dt):
    t = np.float32 if dt == "fp32" else np.float16
    fw, bw = "ptl_rms_norm_%s_fw_batched" % dt, "ptl_rms_norm_%s_bw_batched" % dt
    x, w, y, q, s = np.ones((2, 8), t), np.ones(8, t), np.full((2, 8), 7, t), np.full((2, 8), 7, np.int8), np.full(2, 7, np.float32)

    def args(**k):
        return tr.norm_args(pkg, k.pop("dim", 8), **{**dict(x=x, w=w, y=y), **k})

    refused(pkg, fw, None, 2, says="null argument")
    for k, says in ((dict(dim=0), "geometry"), (dict(dim=-3), "geometry"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                    (dict(eps=float("inf")), "eps"), (dict(w=None), "null buffer"), (dict(x=None), "null buffer"),
                    (dict(y=None), "no output"), (dict(q=q), "both"), (dict(scale=s), "both"), (dict(skip=x), "sum"),
                    (dict(skip=x, has_sum=True), "sum"), (dict(has_skip=True, total=y), "null buffer")):
        a, keep = args(**k)
        refused(pkg, fw, a, 2, says=says)
    for k, says in ((dict(dy=None, dx=y, dw=w), "null buffer"), (dict(dy=x, dw=w), "null buffer"), (dict(dy=x, dx=y), "null buffer"),
                    (dict(dy=x, dx=y, dw=w, x=None), "null buffer"), (dict(dy=x, dx=y, dw=w, dskip=y), "sum")):
        a, keep = args(**k)
        refused(pkg, bw, a, 2, says=says)
    assert (y == 7).all() and (q == 7).all() and (s == 7).all() and (w == 1).all()
    for n in (0, -1):  # an empty batch
        a, keep = args()
        assert getattr(pkg.load(), fw)(ctypes.byref(a), n) == 0
    a, keep = args(dy=x, skip_wg=1, skip_ig=1)  # nothing is wanted
    assert getattr(pkg.load(), bw)(ctypes.byref(a), 2) == 0


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_gated_refusals(pkg, dt):
    t = np.float32 if dt == "fp32" else np.float16
    fw, bw = "ptl_gated_linear_%s_fw_batched" % dt, "ptl_gated_linear_%s_bw_batched" % dt
    x, w, y, h = np.ones((2, 6), t), np.ones((10, 6), t), np.full((2, 5), 7, t), np.full((2, 10), 7, t)

    def args(n_in=6, n_out=5, act=1, **k):
        return tr.gated_args(pkg, n_in, n_out, act, **{**dict(x=x, w=w, y=y), **k})

    refused(pkg, fw, None, 2, says="null argument")
    for k, says in ((dict(n_in=0), "geometry"), (dict(n_out=0), "geometry"), (dict(act=4), "activation"), (dict(act=-1), "activation"),
                    (dict(x=None), "null buffer"), (dict(w=None), "null buffer"), (dict(y=None), "null buffer"),
                    (dict(db=h), "null buffer")):
        a, keep = args(**k)
        refused(pkg, fw, a, 2, says=says)
    a, keep = args()
    a.use_biases = 1
    refused(pkg, fw, a, 2, says="null bias")
    full = dict(dx=x.copy(), dw=w.copy(), h=h, dh=h.copy(), dy=y.copy())
    a, keep = args(**{k: v for k, v in full.items() if k not in ("h", "dh")})
    refused(pkg, bw, a, 2, says="null argument")
    for gone in ("dx", "dw", "h", "dh", "dy", "x", "w"):
        a, keep = args(**{**full, gone: None})
        refused(pkg, bw, a, 2, says="null buffer")
    a, keep = args(**full)
    assert (y == 7).all() and (h == 7).all()
    a, keep = args()
    assert getattr(pkg.load(), fw)(ctypes.byref(a), 0) == 0


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_int8_refusals(pkg, dt):
    name = "ptl_mm_int8_" + dt
    A, B = np.ones((3, 4), np.int8), np.ones((5, 4), np.int8)
    C = np.full((3, 5), 7, np.float32 if dt == "fp32" else np.float16)
    refused(pkg, name, None, says="null argument")
    for f, v, says in (("N", -1, "geometry"), ("M", 0, "geometry"), ("K", 0, "geometry"), ("K", 131072, "131071"), ("A", None, "null buffer"),
                       ("B", None, "null buffer"), ("C", None, "null buffer"), ("USE_BIASES", 1, "null buffer")):
        a, keep = tr.int8_args(pkg, A, B, C)
        setattr(a, f, v)
        refused(pkg, name, a, says=says)
    assert (C == 7).all()
    a, keep = tr.int8_args(pkg, A, B, C)
    a.N = 0
    assert getattr(pkg.load(), name)(ctypes.byref(a)) == 0


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_distill_refusals(pkg, dt):
    t = np.float32 if dt == "fp32" else np.float16
    name = "ptl_distill_%s_batched" % dt
    z, u, c = np.ones((2, 9), t), np.ones((2, 3), t), np.zeros((2, 3), np.int32)
    g, loss = np.full((2, 9), 7, t), np.full(2, 7, np.float32)

    def args(temperature=1.0, weight=1.0):
        return tr.distill_args(pkg, z, g, u, c, loss, temperature, weight)

    refused(pkg, name, None, 2, 2, says="null argument")
    for f, v, says in (("n_top", 0, "n_top"), ("n_top", 2049, "n_top"), ("temperature", 0.0, "temperature"), ("temperature", -1.0, "temperature"),
                       ("temperature", float("nan"), "temperature"), ("temperature", float("inf"), "temperature"), ("temperature", 1e-7, "temperature"),
                       ("weight", float("inf"), "weight"), ("weight", float("nan"), "weight"), ("teacher", None, "null buffer"),
                       ("classes", None, "null buffer"), ("wr_loss", None, "null buffer")):
        a, keep = args()
        setattr(a, f, v)
        refused(pkg, name, a, 2, 2, says=says)
    for step in (-1, 3):
        a, keep = args()
        refused(pkg, name, a, 2, step, says="step")
    a, keep = args()
    a.output.contents.dim = 0
    refused(pkg, name, a, 2, 2, says="geometry")
    a, keep = tr.distill_args(pkg, z, None, u, c, loss, 1.0, 1.0)
    refused(pkg, name, a, 2, 1, says="null buffer")
    assert (g == 7).all() and (loss == 7).all()
    a, keep = args()
    assert getattr(pkg.load(), name)(ctypes.byref(a), 0, 2) == 0


def test_no_device_is_reported(pkg):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    A, C = np.ones((2, 4), np.int8), np.full((2, 2), 7, np.float32)
    a, keep = tr.int8_args(pkg, A, A, C)
    assert pkg.load().ptl_mm_int8_fp32(ctypes.byref(a)) == 2
    assert b"no CPU fallback" in pkg.load().ptl_last_error() and (C == 7).all()


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_more_samples_than_a_call_takes(pkg, dt):
    t = np.float32 if dt == "fp32" else np.float16
    many = 2 ** 30 + 1
    x, w, y = np.ones((2, 8), t), np.ones(8, t), np.full((2, 8), 7, t)
    a, keep = tr.norm_args(pkg, 8, x=x, w=w, y=y, dx=y, dw=w, dy=x)
    refused(pkg, "ptl_rms_norm_%s_fw_batched" % dt, a, many, says="2^30")
    refused(pkg, "ptl_rms_norm_%s_bw_batched" % dt, a, many, says="2^30")
    a, keep = tr.gated_args(pkg, 8, 4, 1, x=x, w=x.repeat(4, 0), y=y, h=y)
    refused(pkg, "ptl_gated_linear_%s_fw_batched" % dt, a, many, says="2^30")
    refused(pkg, "ptl_gated_linear_%s_bw_batched" % dt, a, many, says="2^30")
    a, keep = tr.distill_args(pkg, x, y, x, np.zeros((2, 8), np.int32), np.full(2, 7, np.float32), 1.0, 1.0)
    refused(pkg, "ptl_distill_%s_batched" % dt, a, many, 2, says="2^30")
    a, keep = tr.int8_args(pkg, np.ones((3, 4), np.int8), np.ones((5, 4), np.int8), y)
    a.N = many
    refused(pkg, "ptl_mm_int8_" + dt, a, says="geometry")
    assert (y == 7).all()


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_larger_layers_than_a_call_takes(pkg, dt):
    t = np.float32 if dt == "fp32" else np.float16
    x, y = np.ones((2, 8), t), np.full((2, 8), 7, t)
    for step in ("fw", "bw"):
        name = "ptl_gated_linear_%s_%s_batched" % (dt, step)
        for n_in, n_out in ((2 ** 27 + 1, 4), (8, 2 ** 29)):
            a, keep = tr.gated_args(pkg, n_in, n_out, 1, x=x, dx=y, w=x, dw=y, h=x, dh=y, y=y, dy=x)
            refused(pkg, name, a, 2, says="geometry")
    for n, n_in, n_out in ((2 ** 10, 2 ** 21, 1), (2 ** 10, 1, 2 ** 20), (1, 2 ** 20, 2 ** 10)):  # inputs, pre-activations, weights of 2^31
        a, keep = tr.gated_args(pkg, n_in, n_out, 1, x=x, dx=y, w=x, dw=y, h=x, dh=y, y=y, dy=x)
        refused(pkg, name, a, n, says="2^31")
    assert (y == 7).all() and (x == 1).all()
