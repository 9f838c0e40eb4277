"""The operators of include/ptl_tuning.h together, as a program uses them: blocks with plain feed-forward layers and norms on both sides tuned by
rewards - layer with activation, layer, norms with gate and residual between, classifier, policy loss, all the way back and a step of AdamW over all
weights; eager, on another stream, and captured into a graph."""
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

import transformer as tr
import tuning as tn

pytestmark = pytest.mark.gpu
EPS, ALPHA, T, LOW, HIGH, BETA, LR, DECAY = 1e-5, 0.75, 0.75, 0.25, 0.25, 0.125, 2.0 ** -6, 0.125
WEIGHTS = ["w1", "b1", "w2", "b2", "gate", "post", "pre", "w3", "b3"]


class Block:
    """Tensors and argument structs of a step: x -> h -> a (gelu) -> f -> joined with the residual: s, y -> y W3^T + s2 (the residual of a second
    layer) -> logits -> loss, and back."""

    def __init__(self, pkg, dt, n, dim, hidden, classes, per, seed=1, scale=1.0):
        self.pkg, self.lib, self.n, self.keep, self.per = pkg, pkg.load(), n, [], per
        r = lambda s, *sh, scale=1.0: tr.dev(tr.rand(seed * 100 + s, *sh, scale=scale, dt=dt))  # noqa: E731
        e = lambda *sh: torch.full(sh, 7, dtype=tr.t_dtype(dt), device="cuda")  # noqa: E731
        f = lambda *sh: torch.full(sh, 7.0, device="cuda")  # noqa: E731
        gates = 1 if per == 0 else -(-n // per)
        t = self.t = {"x": r(1, n, dim), "skip": r(2, n, dim), "w1": r(3, hidden, dim, scale=dim ** -0.5), "b1": r(4, hidden, scale=0.1),
                      "w2": r(5, dim, hidden, scale=hidden ** -0.5), "b2": r(6, dim, scale=0.1), "gate": r(7, gates, dim, scale=0.5),
                      "post": tr.dev(1 + tr.rand(seed * 100 + 8, dim, scale=0.1, dt=dt)), "pre": tr.dev(1 + tr.rand(seed * 100 + 9, dim, scale=0.1, dt=dt)),
                      "w3": r(10, classes, dim, scale=dim ** -0.5), "b3": r(11, classes, scale=0.1)}
        self.inputs = {k: v.clone() for k, v in t.items()}
        g = torch.Generator().manual_seed(seed)
        t["action"] = torch.randint(0, classes, (n,), generator=g).to(torch.int32).cuda()
        t["old"] = torch.full((n,), -math.log(classes), device="cuda")
        t["ref"] = t["old"] + 0.25
        t["adv"], t["rw"] = torch.randn(n, generator=g).cuda(), (torch.rand(n, generator=g) + 0.5).cuda()
        if n > 3:
            t["action"][3::7] = -1
        for k, sh in {"h": (n, hidden), "a": (n, hidden), "f": (n, dim), "s": (n, dim), "y": (n, dim), "z": (n, classes)}.items():
            t[k] = e(*sh)
        t["loss"], t["logp"] = f(n), f(n)
        for k in list(self.inputs) + ["h", "a", "f", "y", "s", "z"]:
            t["d" + k] = torch.full_like(t[k], 7)
        # the classifier's gradient is all that reaches y; what reaches s from the rest of a model:
        t["ds"] = r(12, n, dim, scale=0.01 * scale)
        self.weight = scale / n
        p = lambda k, d, rows=1: tr.ptr(self.keep, pkg, t[k], t["d" + k], d, rows)  # noqa: E731
        up, down, head = pkg.ActLinearArgs(), pkg.ActLinearArgs(), pkg.ActLinearArgs()
        up.input, up.coeff, up.bias, up.hidden, up.output = p("x", dim), p("w1", dim, hidden), p("b1", hidden), p("h", hidden), p("a", hidden)
        up.activation, up.use_biases = 2, 1
        down.input, down.coeff, down.bias, down.output = p("a", hidden), p("w2", hidden, dim), p("b2", dim), p("f", dim)
        down.activation, down.use_biases = 4, 1
        j = pkg.NormJoinArgs()
        j.input, j.skip, j.gate, j.coeff_post, j.coeff_pre, j.sum, j.output = p("f", dim), p("skip", dim), p("gate", dim, gates), p("post", dim), p("pre", dim), p("s", dim), p("y", dim)
        j.skip_scale, j.eps, j.rows_per_gate = ALPHA, EPS, per
        head.input, head.coeff, head.bias, head.output = p("y", dim), p("w3", dim, classes), p("b3", classes), p("z", classes)
        head.activation, head.use_biases = 4, 1
        l, keep = tn.policy_args(pkg, t["z"], t["dz"], t["action"], t["old"], t["adv"], t["ref"], t["rw"], t["loss"], t["logp"], LOW, HIGH, BETA, T, self.weight)
        steps = (pkg.AdamwArgs * len(WEIGHTS))()
        self.moments = []
        for i, k in enumerate(WEIGHTS):
            m = t[k].numel()
            eight = m >= 1024
            t["n" + k] = torch.full_like(t[k], 7)
            if eight:
                st = dict(m_root=torch.full((m,), 7, dtype=torch.int8, device="cuda"), v_root=torch.full((m,), 7, dtype=torch.uint8, device="cuda"),
                          m_scale=f(-(-m // 256)), v_scale=f(-(-m // 256)))
            else:
                st = dict(m=f(m), v=f(m))
            st["master"] = f(m)
            self.moments.append(st)
            t["master" + k] = st["master"]
            steps[i].weights, steps[i].updated, steps[i].new_state = tr.ptr(self.keep, pkg, t[k], t["d" + k], m), tr.ptr(self.keep, pkg, t["n" + k], None, m), tn.state(pkg, self.keep, **st)
            steps[i].learning_rate, steps[i].weight_decay = LR, DECAY
        t["factor"] = torch.tensor([1.0 / scale], device="cuda")
        h = tn.adamw_step(pkg, factor=t["factor"], eps=1e-6)
        self.keep += [up, down, head, j, l, keep, steps, h]
        c = lambda name, a, *more: (getattr(self.lib, name.replace("DT", dt)), (ctypes.byref(a),) + more)  # noqa: E731
        self.calls = [c("ptl_act_linear_DT_fw_batched", up, n), c("ptl_act_linear_DT_fw_batched", down, n), c("ptl_norm_join_DT_fw_batched", j, n),
                      c("ptl_act_linear_DT_fw_batched", head, n), c("ptl_policy_loss_DT_batched", l, n, 2), c("ptl_act_linear_DT_bw_batched", head, n),
                      c("ptl_norm_join_DT_bw_batched", j, n), c("ptl_act_linear_DT_bw_batched", down, n), c("ptl_act_linear_DT_bw_batched", up, n),
                      (getattr(self.lib, "ptl_adamw_%s_multi" % dt), (ctypes.byref(steps), len(WEIGHTS), ctypes.byref(h)))]

    def step(self):
        for f, args in self.calls:
            assert f(*args) == 0, (f.__name__, self.lib.ptl_last_error())

    def results(self):
        return {**self.t, **{(i, k): v for i, m in enumerate(self.moments) for k, v in m.items()}}


def reference(b, scale=1.0):
    """The same step in 64 bits, gradients by automatic differentiation."""
    p = {k: v.double().cpu().requires_grad_(True) for k, v in b.inputs.items()}
    c = {k: b.t[k].cpu().double() for k in ("old", "ref", "adv", "rw", "ds")}
    a = torch.nn.functional.gelu(p["x"] @ p["w1"].t() + p["b1"], approximate="tanh")
    f = a @ p["w2"].t() + p["b2"]
    s, y = tn.join64(f, p["skip"], p["gate"], p["post"], p["pre"], ALPHA, EPS, b.per or b.n)
    z = y @ p["w3"].t() + p["b3"]
    loss, _ = tn.policy64(z, b.t["action"].cpu(), c["old"], c["adv"], c["ref"], c["rw"], LOW, HIGH, BETA, T, b.weight)
    (loss.sum() + (s * c["ds"]).sum()).backward()
    return loss.detach(), {k: v.grad for k, v in p.items()}


def rel(got, ref):
    """What is off in the 2-norm; gradients in fp16 that the loss scale takes beyond 65504 are infinite."""
    got = got.double().cpu()
    over = (ref.abs() > 65504 * 0.97) & torch.isinf(got)
    assert not torch.isinf(got[~over]).any() and torch.equal(got[over].sign(), ref[over].sign())
    return float((got - ref)[~over].norm() / ref[~over].norm())


# Eight tensors lie between a weight's gradient and the loss and back, each of which rounds once to the tensor type: at most a
# dozen half steps one after the other in the 2-norm (fp32: the sums between them, up to 1500 terms of 2^-24, weigh more).  A clipped
# row's gradient is all or nothing: rows whose ratio the roundings of z may take over a border are left out of the inputs' range by
# their advantages' sign in no way, so that ratios are checked to be further from the borders than that.
BOUND = {"fp32": 1500 * 2.0 ** -24, "fp16": 16 * 2.0 ** -11}


def clear_of_borders(b, dt):
    """Moves old log-probabilities so that no ratio of the step in 64 bits is within 2 % of a border: z rounds to some 2^-9."""
    p = {k: v.double().cpu() for k, v in b.inputs.items()}
    a = torch.nn.functional.gelu(p["x"] @ p["w1"].t() + p["b1"], approximate="tanh")
    _, y = tn.join64(a @ p["w2"].t() + p["b2"], p["skip"], p["gate"], p["post"], p["pre"], ALPHA, EPS, b.per or b.n)
    z = y @ p["w3"].t() + p["b3"]
    at = b.t["action"].cpu().long().clamp(min=0)[:, None]
    lp = torch.log_softmax(z / T, 1).gather(1, at)[:, 0]
    g = torch.Generator().manual_seed(5)
    moved = torch.randn(b.n, generator=g, dtype=torch.float64) * 0.3
    for border in (math.log(1 - LOW), math.log(1 + HIGH)):
        moved = torch.where((moved - border).abs() < 0.03, moved + 0.06, moved)
    b.t["old"].copy_((lp - moved).float())
    b.t["ref"].copy_((lp + 0.3 * torch.randn(b.n, generator=g, dtype=torch.float64)).float())


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,dim,hidden,classes,per", [(1, 64, 96, 300, 0), (37, 100, 150, 1000, 10), (300, 256, 700, 5000, 100), (512, 512, 1408, 2000, 0)])
def test_training_step(pkg, gpu, dt, n, dim, hidden, classes, per):
    scale = 1024.0 * n if dt == "fp16" else 1.0
    b = Block(pkg, dt, n, dim, hidden, classes, per, scale=min(scale, 65536.0))
    clear_of_borders(b, dt)
    torch.cuda.synchronize()
    b.step()
    assert gpu.ptl_sync() == 0
    loss, grads = reference(b)
    assert rel(b.t["loss"], loss) <= 4 * BOUND[dt]  # (a sum of terms of both signs)
    for k, g in grads.items():
        assert rel(b.t["d" + k], g) <= 2 * BOUND[dt], k
    factor = float(b.t["factor"])
    for i, k in enumerate(WEIGHTS):
        g = b.t["d" + k].double().cpu().view(-1)
        w0 = b.inputs[k].double().cpu().view(-1)
        new, m, v, up = tn.adamw64(w0, g * factor, torch.zeros_like(w0), torch.zeros_like(w0), 1, LR, DECAY, eps=1e-6)
        tol = 30 * tr.U * up.abs() + 6 * tr.U * (w0.abs() + new.abs())
        tr.within(b.t["n" + k].view(-1), new, tol + tr.step(new, dt), k)
        tr.within(b.moments[i]["master"], new, tol, k)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_captured_step(pkg, gpu, dt):
    """Captured on a stream of its own after an eager step of the same sizes, replayed with eager work between the replays: every replay
    leaves the bits of the eager step."""
    b = Block(pkg, dt, 256, 264, 704, 40000, 100)  # (products in parts, sums of rows in a workspace)
    b.step()
    torch.cuda.synchronize()
    want = {k: v.clone() for k, v in b.results().items()}
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    gpu.ptl_set_stream(ctypes.c_void_p(side.cuda_stream))
    try:
        with torch.cuda.graph(graph, stream=side):
            b.step()
        for i in range(4):
            for again in (graph.replay, b.step):  # (an eager step on the same stream between the replays)
                for k in ("loss", "logp", "z", "h", "s", "dx", "dw1", "dgate", "nw2"):
                    b.t[k].fill_(7)
                torch.cuda.synchronize()
                again()
                torch.cuda.synchronize()
                for k, v in b.results().items():
                    assert torch.equal(v, want[k]), (i, k)
    finally:
        gpu.ptl_set_stream(None)


def test_two_graphs_share_the_workspace(pkg, gpu):
    """Two captured steps of different sizes, replayed in turn."""
    blocks = [Block(pkg, "fp16", 200, 128, 300, 33000, 7, seed=2), Block(pkg, "fp16", 64, 512, 1408, 5000, 0, seed=3)]
    for b in blocks:
        b.step()
    torch.cuda.synchronize()
    want = [{k: v.clone() for k, v in b.results().items()} for b in blocks]
    side = torch.cuda.Stream()
    graphs = [torch.cuda.CUDAGraph() for _ in blocks]
    torch.cuda.synchronize()
    gpu.ptl_set_stream(ctypes.c_void_p(side.cuda_stream))
    try:
        for b, g in zip(blocks, graphs):
            with torch.cuda.graph(g, stream=side):
                b.step()
        for _ in range(3):
            for g in graphs:
                g.replay()
            torch.cuda.synchronize()
            for b, w in zip(blocks, want):
                assert all(torch.equal(v, w[k]) for k, v in b.results().items())
                for k in ("loss", "z", "dx", "dw1", "dgate", "nw2"):
                    b.t[k].fill_(7)
            torch.cuda.synchronize()
    finally:
        gpu.ptl_set_stream(None)


def test_a_step_is_the_same_every_time_and_on_another_stream(pkg, gpu):
    b = Block(pkg, "fp16", 300, 264, 700, 3000, 40)
    b.step()
    torch.cuda.synchronize()
    want = {k: v.clone() for k, v in b.results().items()}
    for _ in range(3):
        b.step()
        torch.cuda.synchronize()
        assert all(torch.equal(v, want[k]) for k, v in b.results().items())
    side = torch.cuda.Stream()
    for k in ("loss", "z", "h", "dx", "dw1", "dgate", "nw2"):
        b.t[k].fill_(7)
    torch.cuda.synchronize()
    gpu.ptl_set_stream(ctypes.c_void_p(side.cuda_stream))
    try:
        b.step()
        assert gpu.ptl_sync() == 0
        assert all(torch.equal(v, want[k]) for k, v in b.results().items())
    finally:
        gpu.ptl_set_stream(None)


def growth_in_a_capture(what):
    """In a process of its own, whose workspace is as small as it is reserved: the call fails with status 2 and a text that names
    ptl_reserve, what it reads stays as it was, the capture stays valid; with the sizes that an eager call leaves reserved it is captured."""
    import __graft_entry__ as ge
    pkg = ge.load_package()
    gpu = pkg.load()
    assert gpu.ptl_init(0) == 0
    seeds = iter(range(1, 100))
    z = lambda *s: tr.dev(tr.rand(next(seeds), *s, dt="fp16"))  # noqa: E731
    if what == "policy":  # parts of rows; the smallest workspace has 8 MB
        n, v = 128, 131072
        t = z(1, v).expand(n, v).contiguous()
        f = torch.zeros(n, device="cuda")
        assert gpu.ptl_reserve(0, 0) == 0
        a, keep = tn.policy_args(pkg, t, t, torch.zeros(n, dtype=torch.int32, device="cuda"), f, f, None, None, f.clone(), None)
        call, held = (lambda: gpu.ptl_policy_loss_fp16_batched(ctypes.byref(a), n, 2)), [t]
    elif what == "norm":  # shares of 4096 columns, in the place of what is read
        n, dim = 1100, 4096
        b, s, w = z(n, dim), z(n, dim), z(dim)
        a, keep = tn.join_args(pkg, dim, b=b, db=b, w1=w, dw1=z(dim), w2=w, dw2=z(dim), gate=z(1, dim), dgate=z(1, dim), s=s, dx=s, dy=z(n, dim), ds=z(n, dim))
        call, held = (lambda: gpu.ptl_norm_join_fp16_bw_batched(ctypes.byref(a), n)), [b, s]
    else:  # products in parts; a dense layer's call; one kernel; each with the gradients in the place of what they are formed from
        dt, n, i, o, over = {"products": ("fp16", 256, 2048, 4096, "h"), "dense": ("fp16", 64, 512, 1408, "dy"), "few": ("fp32", 2, 300, 4000, "dy")}[what]
        r = lambda *s: tr.dev(tr.rand(next(seeds), *s, dt=dt))  # noqa: E731
        x, w, h, dy = r(n, i), r(o, i), r(n, o), r(n, o)
        a, keep = tn.act_args(pkg, i, o, 2, x=x, dx=r(n, i), w=w, dw=r(o, i), db=r(o), h=h, dh=h if over == "h" else dy, dy=dy)
        call, held = (lambda: getattr(gpu, "ptl_act_linear_%s_bw_batched" % dt)(ctypes.byref(a), n)), [h, dy]
    after, side = torch.zeros(1, device="cuda"), torch.cuda.Stream()
    before = [t.clone() for t in held]
    torch.cuda.synchronize()
    gpu.ptl_set_stream(ctypes.c_void_p(side.cuda_stream))
    for reserved in (False, True):
        if reserved:
            assert call() == 0 and gpu.ptl_sync() == 0
            for t, b in zip(held, before):
                t.copy_(b)
            torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            rc, text = call(), gpu.ptl_last_error().decode()
            after.add_(1)
        assert rc == (0 if reserved else 2) and (reserved or "ptl_reserve" in text), (rc, text)
        graph.replay()
        torch.cuda.synchronize()
        assert float(after) == (2 if reserved else 1)
        if not reserved:
            assert all(torch.equal(t, b) for t, b in zip(held, before))
    gpu.ptl_set_stream(None)
    print("finished", flush=True)


@pytest.mark.parametrize("what", ["policy", "norm", "products", "dense", "few"])
def test_growth_is_refused_in_a_capture(gpu, what):
    here = os.path.dirname(os.path.abspath(__file__))
    code = "import sys; sys.path[:0] = [%r, %r]; import test_gpu_tuning_block as t; t.growth_in_a_capture(%r)" % (here, os.path.dirname(here), what)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "finished" in r.stdout, r.stdout + r.stderr
