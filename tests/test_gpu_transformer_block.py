"""The operators of include/ptl_transformer.h together, as a program uses them: a feed-forward block trained by a teacher - residual and
norm, gated layer, dense layer, residual and norm, classifier, distillation, all the way back and one step of gradient descent - and a
frozen one in 8 bits; eager, on another stream, and captured into a graph."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import helpers as hp
import transformer as tr

pytestmark = pytest.mark.gpu
EPS, T, LR = 1e-5, 2.0, 0.5


class Block:
    """Tensors and argument structs of a training step: x, skip -> sum1, y1 -> h, g -> y2 -> sum2, y3 -> logits -> loss, and back."""

    def __init__(self, pkg, dt, n, dim, hidden, classes, top, seed=1, flat=None):
        self.pkg, self.lib, self.n, self.keep = pkg, pkg.load(), n, []
        f = flat or (lambda t: t)
        r = lambda s, *sh, scale=1.0: f(tr.dev(tr.rand(seed * 100 + s, *sh, scale=scale, dt=dt)))
        e = lambda *sh: f(torch.full(sh, 7, dtype=tr.t_dtype(dt), device="cuda"))
        t = self.t = {"x": r(1, n, dim), "skip": r(2, n, dim), "w1": f(tr.dev(1 + tr.rand(seed * 100 + 3, dim, scale=0.1, dt=dt))),
                      "wg": r(4, 2 * hidden, dim, scale=dim ** -0.5), "bg": r(5, 2 * hidden, scale=0.1),
                      "wd": r(6, dim, hidden, scale=hidden ** -0.5), "w2": f(tr.dev(1 + tr.rand(seed * 100 + 7, dim, scale=0.1, dt=dt))),
                      "wc": r(8, classes, dim, scale=dim ** -0.5), "teacher": r(9, n, top, scale=2.0)}
        self.inputs = {k: v.clone() for k, v in t.items()}
        g = torch.Generator().manual_seed(seed)
        t["classes"] = torch.stack([torch.randperm(classes, generator=g)[:top] for _ in range(n)]).to(torch.int32).cuda()
        for k, sh in {"sum1": (n, dim), "y1": (n, dim), "h": (n, 2 * hidden), "g": (n, hidden), "y2": (n, dim), "sum2": (n, dim), "y3": (n, dim),
                      "z": (n, classes)}.items():
            t[k], t["d" + k] = e(*sh), e(*sh)
        for k in ("x", "w1", "wg", "bg", "wd", "w2", "wc"):
            t["d" + k] = e(*t[k].shape)
        t["loss"] = torch.full((n,), 7.0, device="cuda")
        n1, k1 = tr.norm_args(pkg, dim, x=t["x"], dx=t["dx"], skip=t["skip"], dskip=t["dx"], total=t["sum1"], dtotal=t["dsum1"], w=t["w1"],
                              dw=t["dw1"], y=t["y1"], dy=t["dy1"], eps=EPS)
        ga, k2 = tr.gated_args(pkg, dim, hidden, 1, x=t["y1"], dx=t["dy1"], w=t["wg"], dw=t["dwg"], b=t["bg"], db=t["dbg"], h=t["h"],
                               dh=t["dh"], y=t["g"], dy=t["dg"])
        down, k3 = hp.linear_args(pkg, t["g"], t["dg"], t["wd"], t["dwd"], t["y2"], t["dy2"], hidden, dim)
        # the second residual is the sum of the first: its gradient arrives there
        n2, k4 = tr.norm_args(pkg, dim, x=t["y2"], dx=t["dy2"], skip=t["sum1"], dskip=t["dsum1"], total=t["sum2"], w=t["w2"], dw=t["dw2"],
                              y=t["y3"], dy=t["dy3"], eps=EPS)
        head, k5 = hp.linear_args(pkg, t["y3"], t["dy3"], t["wc"], t["dwc"], t["z"], t["dz"], dim, classes)
        kd, k6 = tr.distill_args(pkg, t["z"], t["dz"], t["teacher"], t["classes"], t["loss"], T, T * T / n)
        opt = (pkg.OptimArgs if dt == "fp32" else pkg.OptimArgsFp16)
        steps = (opt * 6)()
        for a, k in zip(steps, ("w1", "wg", "bg", "wd", "w2", "wc")):
            one, held = hp.optim_args(pkg, dt, t[k], t["d" + k], None, None, LR, 0.0)
            a.weights, a.learning_rate, a.weight_decay_lambda = one.weights, one.learning_rate, one.weight_decay_lambda
            self.keep += [one, held]
        self.keep += [n1, ga, down, n2, head, kd, steps, k1, k2, k3, k4, k5, k6]
        f = lambda name, a, *more: (getattr(self.lib, name.replace("DT", dt)), (ctypes.byref(a),) + more)
        self.calls = [f("ptl_rms_norm_DT_fw_batched", n1, n), f("ptl_gated_linear_DT_fw_batched", ga, n), f("ptl_linear_DT_fw_batched", down, n),
                      f("ptl_rms_norm_DT_fw_batched", n2, n), f("ptl_linear_DT_fw_batched", head, n), f("ptl_distill_DT_batched", kd, n, 2),
                      f("ptl_linear_DT_bw_batched", head, n), f("ptl_rms_norm_DT_bw_batched", n2, n), f("ptl_linear_DT_bw_batched", down, n),
                      f("ptl_gated_linear_DT_bw_batched", ga, n), f("ptl_rms_norm_DT_bw_batched", n1, n),
                      (getattr(self.lib, "ptl_gradient_descent_%s_multi" % dt), (ctypes.byref(steps), 6))]

    def step(self):
        for f, args in self.calls:
            assert f(*args) == 0, (f.__name__, self.lib.ptl_last_error())

    def reset(self):
        for k, v in self.inputs.items():
            self.t[k].copy_(v)


def reference(b):
    """The same step in 64 bits, gradients by automatic differentiation."""
    p = {k: v.double().cpu().requires_grad_(k not in ("skip", "teacher")) for k, v in b.inputs.items()}
    s1 = p["x"] + p["skip"]
    y1 = tr.norm64(s1, p["w1"], EPS)
    h = y1 @ p["wg"].t() + p["bg"]
    o = h.shape[1] // 2
    y2 = (torch.nn.functional.silu(h[:, :o]) * h[:, o:]) @ p["wd"].t()
    s2 = y2 + s1
    z = tr.norm64(s2, p["w2"], EPS) @ p["wc"].t()
    log_q = torch.log_softmax(z / T, 1)
    log_p = torch.log_softmax(p["teacher"] / T, 1)
    loss = T * T / b.n * (log_p.exp() * (log_p - log_q.gather(1, b.t["classes"].cpu().long()))).sum(1)
    loss.sum().backward()
    return loss.detach(), {k: v.grad for k, v in p.items() if v.grad is not None}


def rel(got, ref):
    return float((got.double().cpu() - ref).norm() / ref.norm())


# Seven tensors lie between a weight's gradient and the loss and back, each of which rounds once to the tensor type: at most a
# dozen half steps one after the other in the 2-norm (fp32: the sums between them, up to 1500 terms of 2^-24, weigh more).
BOUND = {"fp32": 1500 * 2.0 ** -24, "fp16": 12 * 2.0 ** -11}


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,dim,hidden,classes,top", [(1, 64, 96, 300, 5), (37, 100, 150, 1000, 16), (300, 256, 700, 5000, 40), (512, 512, 1408, 2000, 64)])
def test_training_step(pkg, gpu, dt, n, dim, hidden, classes, top):
    b = Block(pkg, dt, n, dim, hidden, classes, top)
    b.step()
    assert gpu.ptl_sync() == 0
    loss, grads = reference(b)
    assert rel(b.t["loss"], loss) <= BOUND[dt]
    for k, g in grads.items():
        if dt == "fp16" and float(g.abs().max()) < 1e-4:
            continue  # (without a loss scale such gradients are subnormal fp16 numbers)
        assert rel(b.t["d" + k], g) <= BOUND[dt], k
        if k != "x":
            new = b.inputs[k].double().cpu() - LR * b.t["d" + k].double().cpu()
            tr.within(b.t[k], new, tr.step(new, dt) + 4 * tr.U * new.abs() + 2 * tr.step(LR * b.t["d" + k].double().cpu(), dt), k)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_captured_step(pkg, gpu, dt):
    """Captured on a stream of its own after an eager step of the same sizes, replayed with eager work between the replays: every replay
    leaves the bits of the eager step."""
    b = Block(pkg, dt, 256, 256, 704, 40000, 32)  # (the products of fp16 in one launch, rows of logits in parts)
    b.step()
    torch.cuda.synchronize()
    want = {k: v.clone() for k, v in b.t.items()}
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    gpu.ptl_set_stream(ctypes.c_void_p(side.cuda_stream))
    try:
        with torch.cuda.graph(graph, stream=side):
            b.step()
        for i in range(4):
            b.reset()
            for k in ("loss", "z", "dx", "dwg", "h"):
                b.t[k].fill_(7)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for k, v in want.items():
                assert torch.equal(b.t[k], v), (i, k)
            b.reset()
            torch.cuda.synchronize()
            b.step()  # eager, on the same stream, between the replays
            torch.cuda.synchronize()
            for k, v in want.items():
                assert torch.equal(b.t[k], v), (i, k)
    finally:
        gpu.ptl_set_stream(None)


def test_two_graphs_share_the_workspace(pkg, gpu):
    """Two captured steps of different sizes, replayed in turn."""
    blocks = [Block(pkg, "fp16", 200, 128, 300, 33000, 17, seed=2), Block(pkg, "fp16", 64, 512, 1408, 5000, 9, seed=3)]
    for b in blocks:
        b.step()
    torch.cuda.synchronize()
    want = [{k: v.clone() for k, v in b.t.items()} for b in blocks]
    side = torch.cuda.Stream()
    graphs = [torch.cuda.CUDAGraph() for _ in blocks]
    torch.cuda.synchronize()
    gpu.ptl_set_stream(ctypes.c_void_p(side.cuda_stream))
    try:
        for b, g in zip(blocks, graphs):
            with torch.cuda.graph(g, stream=side):
                b.step()
        for _ in range(3):
            for b in blocks:
                b.reset()
            torch.cuda.synchronize()
            for g in graphs:
                g.replay()
            torch.cuda.synchronize()
            for b, w in zip(blocks, want):
                assert all(torch.equal(b.t[k], v) for k, v in w.items())
    finally:
        gpu.ptl_set_stream(None)


def test_a_step_is_the_same_every_time(pkg, gpu):
    b = Block(pkg, "fp16", 300, 264, 700, 3000, 40)
    b.step()
    torch.cuda.synchronize()
    want = {k: v.clone() for k, v in b.t.items()}
    for _ in range(3):
        b.reset()
        b.step()
        torch.cuda.synchronize()
        assert all(torch.equal(b.t[k], v) for k, v in want.items())


def test_another_stream(pkg, gpu):
    b = Block(pkg, "fp32", 50, 96, 130, 700, 11)
    b.step()
    torch.cuda.synchronize()
    want = {k: v.clone() for k, v in b.t.items()}
    side = torch.cuda.Stream()
    b.reset()
    torch.cuda.synchronize()
    gpu.ptl_set_stream(ctypes.c_void_p(side.cuda_stream))
    try:
        b.step()
        assert gpu.ptl_sync() == 0
        assert all(torch.equal(b.t[k], v) for k, v in want.items())
    finally:
        gpu.ptl_set_stream(None)


@pytest.mark.parametrize("n", [1, 2, 3, 33, 700])
def test_frozen_layer_in_8_bits(pkg, gpu, n):
    """Residual and norm with an output in 8 bits, and the product that reads it, against the layer in 64 bits.  Each of the `dim`
    products is off by half a unit of either factor: the sum, of independent errors, by at most 6 standard deviations of that."""
    dim, outs = 520, 300
    x, skip, w1 = (tr.dev(t) for t in (tr.rand(1, n, dim, dt="fp16"), tr.rand(2, n, dim, dt="fp16"), 1 + tr.rand(3, dim, scale=0.1, dt="fp16")))
    w, bias = tr.rand(4, outs, dim, scale=dim ** -0.5).double(), tr.rand(5, outs, scale=0.1, dt="fp16")
    sb = w.abs().amax(1) / 127
    B = torch.round(w / sb[:, None]).to(torch.int8).cuda()
    total, q, sa = torch.empty_like(x), torch.empty(n, dim, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    a, k1 = tr.norm_args(pkg, dim, x=x, skip=skip, total=total, w=w1, q=q, scale=sa, eps=EPS)
    pkg.call("ptl_rms_norm_fp16_fw_batched", a, n)
    y = torch.empty(n, outs, dtype=torch.float16, device="cuda")
    m, k2 = tr.int8_args(pkg, q, B, y, sa, sb.float().cuda(), bias.cuda())
    assert gpu.ptl_mm_int8_fp16(ctypes.byref(m)) == 0 and gpu.ptl_sync() == 0
    v = tr.norm64(x.double().cpu() + skip.double().cpu(), w1.double().cpu(), EPS)
    ref = v @ w.t() + bias.double()
    unit_a, unit_b = v.abs().amax(1, keepdim=True) / 127, sb[None]
    spread = torch.sqrt((unit_a ** 2 * (w * w).sum(1)[None] + unit_b ** 2 * (v * v).sum(1, keepdim=True) + dim * unit_a ** 2 * unit_b ** 2 / 12) / 12)
    tr.within(y, ref, 6 * spread + tr.step(ref, "fp16"))


def growth_in_a_capture(what):
    """In a process of its own, whose workspace is as small as it is reserved: the call fails with status 2 and a text that names
    ptl_reserve, the capture stays valid; with the sizes that an eager call leaves reserved it is captured."""
    import __graft_entry__ as ge
    pkg = ge.load_package()
    gpu = pkg.load()
    assert gpu.ptl_init(0) == 0
    z = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")  # noqa: E731
    if what == "distill":  # the entries of 100 rows in parts: 6.5 MB
        n, v, top = 100, 70000, 2048
        a, keep = tr.distill_args(pkg, z(n, v), z(n, v), z(n, top), torch.zeros(n, top, dtype=torch.int32, device="cuda"),
                                  torch.zeros(n, device="cuda"), 1.0, 1.0)
        call = lambda: gpu.ptl_distill_fp16_batched(ctypes.byref(a), n, 2)  # noqa: E731
    elif what == "norm":  # 1024 shares of 4096
        a, keep = tr.norm_args(pkg, 4096, x=z(1100, 4096), dx=z(1100, 4096), w=z(4096), dw=z(4096), dy=z(1100, 4096))
        call = lambda: gpu.ptl_rms_norm_fp16_bw_batched(ctypes.byref(a), 1100)  # noqa: E731
    elif what == "gated":  # products in parts
        n, i, o = 256, 2048, 2048
        a, keep = tr.gated_args(pkg, i, o, 1, x=z(n, i), dx=z(n, i), w=z(2 * o, i), dw=z(2 * o, i), h=z(n, 2 * o), dh=z(n, 2 * o), dy=z(n, o))
        call = lambda: gpu.ptl_gated_linear_fp16_bw_batched(ctypes.byref(a), n)  # noqa: E731
    else:  # copies of rows that do not start on 16 bytes
        A, B = torch.zeros(4096, 2045, dtype=torch.int8, device="cuda"), torch.zeros(2048, 2045, dtype=torch.int8, device="cuda")
        a, keep = tr.int8_args(pkg, A, B, z(4096, 2048))
        call = lambda: gpu.ptl_mm_int8_fp16(ctypes.byref(a))  # noqa: E731
    after, side = torch.zeros(1, device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    gpu.ptl_set_stream(ctypes.c_void_p(side.cuda_stream))
    for reserved in (False, True):
        if reserved:
            assert call() == 0 and gpu.ptl_sync() == 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            rc, text = call(), gpu.ptl_last_error().decode()
            after.add_(1)
        assert rc == (0 if reserved else 2) and (reserved or "ptl_reserve" in text), (rc, text)
        graph.replay()
        torch.cuda.synchronize()
        assert float(after) == (2 if reserved else 1)
    gpu.ptl_set_stream(None)
    print("finished", flush=True)


@pytest.mark.parametrize("what", ["distill", "norm", "gated", "int8"])
def test_growth_is_refused_in_a_capture(gpu, what):
    here = os.path.dirname(os.path.abspath(__file__))
    code = "import sys; sys.path[:0] = [%r, %r]; import test_gpu_transformer_block as t; t.growth_in_a_capture(%r)" % (here, os.path.dirname(here), what)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "finished" in r.stdout, r.stdout + r.stderr


def refused_in_place(sizes):
    """In a process of its own: a gated layer's way back in a capture whose workspace (whose copies' memory is there) may not grow,
    hidden->diff in the place of hidden->data.  The refused call leaves the pre-activations as they are, also when what was captured is
    replayed, and an eager call behind it has its results."""
    import __graft_entry__ as ge
    pkg = ge.load_package()
    gpu = pkg.load()
    assert gpu.ptl_init(0) == 0
    dt, n, i, o, path, bias = sizes
    r = lambda s, *sh: tr.dev(tr.rand(s, *sh, dt=dt))  # noqa: E731
    x, w, h, dy = r(1, n, i), r(2, 2 * o, i), r(3, n, 2 * o), r(4, n, o)
    dx, dw, db = torch.full_like(x, 7), torch.full_like(w, 7), torch.full((2 * o,), 7, dtype=x.dtype, device="cuda") if bias else None
    a, keep = tr.gated_args(pkg, i, o, 1, x=x, dx=dx, w=w, dw=dw, db=db, h=h, dh=h, dy=dy)
    call = lambda: getattr(gpu, "ptl_gated_linear_%s_bw_batched" % dt)(ctypes.byref(a), n)  # noqa: E731
    gpu.ptl_set_gemm_path(path)
    assert gpu.ptl_reserve(0, 256 << 20) == 0
    ws = ctypes.c_size_t(1)
    before, after, side, graph = h.clone(), torch.zeros(1, device="cuda"), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    gpu.ptl_set_stream(ctypes.c_void_p(side.cuda_stream))
    with torch.cuda.graph(graph, stream=side):
        rc, text = call(), gpu.ptl_last_error().decode()
        after.add_(1)
    assert rc == 2 and "ptl_reserve" in text, (rc, text)
    graph.replay()
    torch.cuda.synchronize()
    assert float(after) == 1 and torch.equal(h, before)
    assert call() == 0 and gpu.ptl_sync() == 0
    gpu.ptl_reserved(ctypes.byref(ws), None)
    assert ws.value > 0
    over = [t.clone() for t in (h, dx, dw) + ((db,) if bias else ())]
    again = torch.cuda.CUDAGraph()  # with what the eager call has left reserved it is captured
    with torch.cuda.graph(again, stream=side):
        assert call() == 0, gpu.ptl_last_error()
    for _ in range(3):
        h.copy_(before)
        for t in (dx, dw):
            t.fill_(7)
        torch.cuda.synchronize()
        again.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(over, (h, dx, dw)))
    h2, dh = before.clone(), torch.full_like(before, 7)
    a, keep = tr.gated_args(pkg, i, o, 1, x=x, dx=dx, w=w, dw=dw, db=db, h=h2, dh=dh, dy=dy)
    assert call() == 0 and gpu.ptl_sync() == 0
    assert all(torch.equal(p, q) for p, q in zip(over, (dh, dx, dw) + ((db,) if bias else ())))
    gpu.ptl_set_stream(None)
    gpu.ptl_set_gemm_path(0)
    print("finished", flush=True)


# both products in one launch, in parts; as copies, with the sums of the bias; in two halves; a dense layer's call, by three of its routes; one kernel
@pytest.mark.parametrize("sizes", [("fp16", 256, 2048, 2048, 0, 0), ("fp16", 257, 2045, 2047, 0, 1), ("fp16", 20, 1000, 400, 0, 0), ("fp32", 40, 300, 2000, 0, 0),
                                   ("fp32", 200, 300, 2000, 1, 1), ("fp16", 64, 512, 1408, 0, 0), ("fp32", 2, 300, 2000, 0, 1)])
def test_a_refused_call_leaves_what_it_reads(gpu, sizes):
    here = os.path.dirname(os.path.abspath(__file__))
    code = "import sys; sys.path[:0] = [%r, %r]; import test_gpu_transformer_block as t; t.refused_in_place(%r)" % (here, os.path.dirname(here), sizes)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "finished" in r.stdout, r.stdout + r.stderr
