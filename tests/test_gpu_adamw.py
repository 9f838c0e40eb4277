"""AdamW over many tensors against its formula in 64 bits.  u = 2^-24: a moment rounds three products and sums; the step a dozen operations,
the root and the inverse of which are off by a step (2 u)."""
import ctypes

import pytest
import torch

import transformer as tr
import tuning as tn

pytestmark = pytest.mark.gpu
U = tr.U
LR, DECAY = 1e-2, 0.1


def pack(m, v):
    """The form in 8 bits of moments in 64: codes and scales of 256 elements each (fp32 as they are held)."""
    n = m.numel()
    pad = -n % 256
    m, v = (torch.nn.functional.pad(t, (0, pad)).view(-1, 256) for t in (m.double(), v.double()))
    a, c = m.abs().sqrt(), v.sqrt().sqrt()
    ms, vs = (a.amax(1) / 127).float(), (c.amax(1) / 255).float()
    inv = lambda s: torch.where(s > 0, 1 / s.double(), torch.zeros_like(s.double()))[:, None]  # noqa: E731
    q = (torch.round(a * inv(ms)) * m.sign()).to(torch.int8).view(-1)[:n]
    p = torch.round(c * inv(vs))
    p = torch.where((v > 0) & (p < 1), torch.ones_like(p), p).to(torch.uint8).view(-1)[:n]
    return q, p, ms, vs


def unpack(q, p, ms, vs):
    a = q.double() * ms.double().repeat_interleave(256)[:q.numel()]
    c = p.double() * vs.double().repeat_interleave(256)[:q.numel()]
    return a * a.abs(), c ** 4


class Case:
    """Tensors of `sizes`, some with moments in 8 bits, some without earlier ones; placed one after the other with an odd gap, so that most
    start inside a 16-byte piece."""

    def __init__(self, pkg, dt, sizes, eight, master=False, fresh=False, place=True, seed=1, **k):
        self.pkg, self.dt, self.sizes, self.k, self.keep, self.bufs = pkg, dt, sizes, k, [], []
        self.lib = pkg.load()
        def put(t):  # behind an element of its type
            if not place:
                return t.clone()
            buf = torch.full((t.numel() + 2,), 7, dtype=t.dtype, device="cuda")
            buf[1:-1] = t.to("cuda")
            self.bufs.append(buf)
            return buf[1:-1]

        self.host, self.dev, self.out = [], [], []
        for i, n in enumerate(sizes):
            r = lambda s, scale=1.0: tr.rand(seed * 1000 + 10 * i + s, n, scale=scale)  # noqa: E731
            h = {"w": r(1).to(tr.t_dtype(dt)), "g": (r(2) * torch.exp(r(3))).mul(1e-2).to(tr.t_dtype(dt))}
            h["master"] = h["w"].float() + r(7, 1e-5) if master else None
            m, v = r(4, 3e-3), r(5, 1e-2).square() * 0.1
            if n > 3:
                v[3], m[3], h["g"][3] = 0, 0, 0
            h["eight"] = eight(i)
            if h["eight"]:
                h["codes"] = pack(m, v)
                m, v = unpack(*h["codes"])
            h["m"], h["v"] = (torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)) if fresh else (m.double(), v.double())
            d = {"w": put(h["w"]), "g": put(h["g"]), "master": None if h["master"] is None else put(h["master"])}
            if not fresh:
                if h["eight"]:
                    d["mq"], d["vq"], d["ms"], d["vs"] = (put(t) for t in h["codes"])
                else:
                    d["m"], d["v"] = put(m.float()), put(v.float())
            blocks = -(-n // 256)
            o = {"w": put(torch.full((n,), 7, dtype=tr.t_dtype(dt))), "master": put(torch.full((n,), 7.0)) if master else None}
            if h["eight"]:
                o["mq"], o["vq"] = put(torch.full((n,), 7, dtype=torch.int8)), put(torch.full((n,), 7, dtype=torch.uint8))
                o["ms"], o["vs"] = put(torch.full((blocks,), 7.0)), put(torch.full((blocks,), 7.0))
            else:
                o["m"], o["v"] = put(torch.full((n,), 7.0)), put(torch.full((n,), 7.0))
            self.host.append(h)
            self.dev.append(d)
            self.out.append(o)
        self.fresh, self.master = fresh, master

    def state(self, t):
        names = {"m": "m", "v": "v", "mq": "m_root", "vq": "v_root", "ms": "m_scale", "vs": "v_scale", "master": "master"}
        return tn.state(self.pkg, self.keep, **{names[k]: v for k, v in t.items() if k in names})

    def run(self, in_place=False, **k):
        a = (self.pkg.AdamwArgs * len(self.sizes))()
        for i, (n, d, o) in enumerate(zip(self.sizes, self.dev, self.out)):
            a[i].weights = tr.ptr(self.keep, self.pkg, d["w"], d["g"], n)
            if not self.fresh:
                a[i].state = self.state(d)
            if not in_place:
                a[i].updated, a[i].new_state = tr.ptr(self.keep, self.pkg, o["w"], None, n), self.state(o)
            a[i].learning_rate, a[i].weight_decay = LR, DECAY if i % 2 == 0 else 0.0
        s = tn.adamw_step(self.pkg, **{**self.k, **k})
        self.keep += [a, s]
        f = getattr(self.lib, "ptl_adamw_%s_multi" % self.dt)
        assert f(a, len(self.sizes), ctypes.byref(s)) == 0, self.lib.ptl_last_error()
        assert self.lib.ptl_sync() == 0
        return self.dev if in_place else self.out

    def untouched(self):
        for buf in self.bufs:
            assert buf[0] == 7 and buf[-1] == 7

    def check(self, got, t=1, factor=1.0, **k):
        for i, (n, h, o) in enumerate(zip(self.sizes, self.host, got)):
            what = (i, n)
            g = h["g"].double() * tn.f32(factor)
            start = (h["w"] if h["master"] is None or self.fresh else h["master"]).double()
            w, m, v, up = tn.adamw64(start, g, h["m"], h["v"], t, LR, DECAY if i % 2 == 0 else 0.0, **k)
            b1, b2 = k.get("beta1", 0.9), k.get("beta2", 0.999)
            e_m = 4 * U * (b1 * h["m"].abs() + (1 - b1) * g.abs())  # of the first moment, whose two terms may cancel
            lr = tn.f32(LR)
            rest = torch.where(up != 0, (up / torch.where(m != 0, m, torch.ones_like(m))).abs(), torch.zeros_like(up))
            tol = up.abs() * U * 20 + rest * e_m * 1.1 + 4 * U * (start.abs() + w.abs() + lr * DECAY * start.abs())
            tr.within(o["w"], w, tol + tr.step(w, self.dt), what)
            if h["master"] is not None:
                tr.within(o["master"], w, tol + 2 * U * w.abs(), what)
            e_v = v * U * 6 + 2.0 ** -149
            if not h["eight"]:
                tr.within(o["m"], m, e_m + 2 * U * m.abs() + 2.0 ** -149, what)
                tr.within(o["v"], v, e_v, what)
                continue
            pad = -n % 256
            for code, scale, root, e, most in ((o["mq"].cpu().double(), o["ms"], m.abs().sqrt(), e_m + 4 * U * m.abs(), 127), (o["vq"].cpu().double(), o["vs"], v ** 0.25, None, 255)):
                blocks = torch.nn.functional.pad(root, (0, pad)).view(-1, 256)
                top = blocks.amax(1)
                # the root halves the relative error of what it is of, the fourth root quarters it
                rel = 8 * U if e is None else 8 * U + float((e / m.abs().clamp(min=1e-30))[m.abs() >= 1e-3 * m.abs().max()].max()) if n else 0
                tr.within(scale, top / most, top / most * rel + 1e-30, what)
                unit = torch.where(top > 0, most / top, torch.zeros_like(top)).repeat_interleave(256)[:n]
                off = (code.abs() - root * unit).abs()
                # a root within its own error of a border may fall on either side: of m where it is near 0, by what its terms leave
                slack = most * 16 * U + (0 if e is None else (torch.sqrt(m.abs() + e) - torch.sqrt((m.abs() - e).clamp(min=0))) * unit)
                small = (code == 1) & (most == 255)
                assert (off - slack <= torch.where(small, torch.ones_like(off), torch.full_like(off, 0.5))).all(), what
                if most == 127:
                    assert (torch.sign(code) * torch.sign(m) >= 0).all(), what
                else:
                    assert ((code > 0) == (v > 0)).all(), what
        self.untouched()


SIZES = [1, 3, 4, 5, 255, 256, 257, 1000, 1023, 4095, 4096, 4097, 10001, 2, 70000]


@pytest.mark.parametrize("dt,master", [("fp32", False), ("fp16", False), ("fp16", True), ("fp32", True)])
@pytest.mark.parametrize("bits", [8, 32, 40])
def test_step(pkg, gpu, dt, master, bits):
    """Moments in 8 bits, in 32, and tensors of both in one call."""
    for t, fresh in ((1, True), (3, False), (5000, False)):
        c = Case(pkg, dt, SIZES, lambda i: bits == 8 or (bits == 40 and i % 3 != 0), master=master, fresh=fresh)
        c.check(c.run(t=t), t=t)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_many_tensors(pkg, gpu, dt):
    """More tensors than one launch takes, a few of them empty."""
    c = Case(pkg, dt, [(7 * i) % 50 * (i % 5) + 300 * (i % 7) for i in range(130)], lambda i: i % 4 == 1, master=dt == "fp16")
    c.check(c.run(t=2), t=2)


@pytest.mark.parametrize("dt,master", [("fp32", False), ("fp16", True), ("fp16", False)])
@pytest.mark.parametrize("eight", [False, True])
def test_in_place(pkg, gpu, dt, master, eight):
    want = Case(pkg, dt, SIZES, lambda i: eight, master=master).run(t=4)
    c = Case(pkg, dt, SIZES, lambda i: eight, master=master)
    got = c.run(in_place=True, t=4)
    for a, b in zip(want, got):
        assert all(torch.equal(a[k], b[k]) for k in a if a[k] is not None)
    c.check(got, t=4)


@pytest.mark.parametrize("betas", [(0.0, 0.0), (0.5, 0.9), (0.9, 0.99999)])
def test_other_rates(pkg, gpu, betas):
    k = dict(beta1=betas[0], beta2=tn.f32(betas[1]), eps=1e-5)
    for t in (1, 7):
        c = Case(pkg, "fp32", SIZES, lambda i: False)
        c.check(c.run(t=t, **k), t=t, **k)


def test_steps_behind_one_another(pkg, gpu):
    """Ten steps with the moments in 32 bits against ten steps in 64, and in 8 bits near them: the codes hold roots to 1 / 254 and
    1 / 510 of the largest of 256 at every step."""
    n = 5000
    w0, keep = tr.rand(1, n), []
    w64, m, v = w0.double(), torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    W = [w0.cuda(), w0.cuda()]
    M, V = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    eight = dict(m_root=torch.empty(n, dtype=torch.int8, device="cuda"), v_root=torch.empty(n, dtype=torch.uint8, device="cuda"),
                 m_scale=torch.empty(20, device="cuda"), v_scale=torch.empty(20, device="cuda"))
    states = [tn.state(pkg, keep, m=M, v=V), tn.state(pkg, keep, **eight)]
    path = torch.zeros(n, dtype=torch.float64)
    for t in range(1, 11):
        g = tr.rand(100 + t, n) + 0.5 * tr.rand(99, n)
        w64, m, v, up = tn.adamw64(w64, g.double(), m, v, t, LR, DECAY)
        path += up.abs()
        G, a = g.cuda(), (pkg.AdamwArgs * 2)()
        for i in range(2):
            a[i].weights = tr.ptr(keep, pkg, W[i], G, n)
            if t > 1:
                a[i].state = states[i]
            a[i].new_state, a[i].learning_rate, a[i].weight_decay = states[i], LR, DECAY
        assert gpu.ptl_adamw_fp32_multi(a, 2, ctypes.byref(tn.adamw_step(pkg, t=t))) == 0 and gpu.ptl_sync() == 0
    tr.within(W[0], w64, 10 * U * (30 * path + 4 * w64.abs() + 1))
    assert float((W[1].double().cpu() - w64).norm() / (w64 - w0.double()).norm()) < 0.1


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_step_and_factor_in_memory(pkg, gpu, dt):
    """The number of the step and the factor of the gradients are read when the step runs; without a finite factor nothing changes."""
    for eight in (False, True):
        mk = lambda **k: Case(pkg, dt, SIZES, lambda i: eight, master=dt == "fp16", **k)  # noqa: E731
        c = mk()
        t, f = torch.tensor([9], dtype=torch.int32, device="cuda"), torch.tensor([0.25], device="cuda")
        c.check(c.run(t=1, step_data=t, factor=f), t=9, factor=0.25)
        for bad in (float("nan"), float("inf")):
            f.fill_(bad)
            c = mk()
            before = [{k: v.clone() for k, v in d.items() if v is not None} for d in c.dev]
            got = c.run(t=9, factor=f, in_place=True)
            assert all(torch.equal(d[k], v) for d, b in zip(got, before) for k, v in b.items())
            c = mk()
            got = c.run(t=9, factor=f)
            for o, d in zip(got, c.dev):
                for k, v in o.items():
                    if k == "w" and d["master"] is not None:
                        assert torch.equal(v, d["master"].to(v.dtype))
                    elif v is not None:
                        assert torch.equal(v, d[k])
            c = mk(fresh=True)
            got = c.run(t=1, factor=f)
            for o, d in zip(got, c.dev):
                assert torch.equal(o["w"], d["w"]) and all((o[k] == 0).all() for k in o if k not in ("w", "master"))
                assert o["master"] is None or torch.equal(o["master"], d["w"].float())
            c.untouched()


def test_captured_step(pkg, gpu):
    """One graph, replayed with the step's number and the gradients changed between the replays."""
    n, keep = 3000, []
    w, g = tr.rand(1, n).cuda(), tr.rand(2, n).cuda()
    m, v, t = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    eager = [w.clone(), m.clone(), v.clone()]

    def args(w, m, v):
        a = (pkg.AdamwArgs * 1)()
        a[0].weights, a[0].state, a[0].learning_rate, a[0].weight_decay = tr.ptr(keep, pkg, w, g, n), tn.state(pkg, keep, m=m, v=v), LR, DECAY
        keep.append(a)
        return a

    captured, plain, s = args(w, m, v), args(*eager), tn.adamw_step(pkg, step_data=t)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    gpu.ptl_set_stream(ctypes.c_void_p(side.cuda_stream))
    try:
        with torch.cuda.graph(graph, stream=side):
            assert gpu.ptl_adamw_fp32_multi(captured, 1, ctypes.byref(s)) == 0
        for i in range(4):
            t.fill_(i + 1)
            g.copy_(tr.rand(10 + i, n))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert gpu.ptl_adamw_fp32_multi(plain, 1, ctypes.byref(tn.adamw_step(pkg, step_data=t))) == 0
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip((w, m, v), eager)), i
    finally:
        gpu.ptl_set_stream(None)


@pytest.mark.parametrize("eight", [False, True])
def test_values(pkg, gpu, eight):
    """Gradients that are no numbers reach their own element, in 8 bits the scale of their 256; gradients of 0 leave weights to the decay."""
    n, bad = 2000, 300
    c = Case(pkg, "fp32", [n], lambda i: eight, fresh=True)
    c.dev[0]["g"][:] = 0
    c.dev[0]["g"][bad] = float("nan")
    c.dev[0]["g"][bad + 1] = float("inf")
    o = c.run(t=1)[0]
    w = c.host[0]["w"].double()
    good = [i for i in range(n) if i not in (bad, bad + 1)]
    assert not torch.isfinite(o["w"][bad]) and not torch.isfinite(o["w"][bad + 1])
    assert ((o["w"].double().cpu() - w * (1 - tn.f32(LR) * tn.f32(DECAY)))[good].abs() <= 3 * U * w[good].abs()).all()
    if eight:
        assert not torch.isfinite(o["ms"][1]) and not torch.isfinite(o["vs"][1])
        rest = [0, 2, 3, 4, 5, 6, 7]
        assert (o["ms"][rest] == 0).all() and (o["vs"][rest] == 0).all() and (o["mq"][:256] == 0).all() and (o["vq"][512:] == 0).all()
    else:
        assert (o["m"][good] == 0).all() and (o["v"][good] == 0).all() and torch.isnan(o["m"][bad]) and torch.isinf(o["v"][bad + 1])


def test_tiny_and_large_gradients(pkg, gpu):
    """Squares near fp32's smallest values and roots of them: the step is that of any gradient (eps far below)."""
    n = 1024
    c = Case(pkg, "fp32", [n], lambda i: False, fresh=True, eps=1e-30)
    g = torch.logspace(-17, 17, n, dtype=torch.float64).float()
    c.host[0]["g"] = g
    c.dev[0]["g"][:] = g.cuda()
    c.check(c.run(t=1), t=1, eps=1e-30)


@pytest.mark.parametrize("eight", [False, True])
def test_host_arrays(pkg, gpu, eight):
    want = Case(pkg, "fp16", [300, 5000], lambda i: eight, master=True).run(t=2)
    c = Case(pkg, "fp16", [300, 5000], lambda i: eight, master=True, place=False)
    got = c.run(t=2)
    for a, b in zip(want, got):
        assert all(torch.equal(a[k].cpu(), b[k]) for k in a)
    got = Case(pkg, "fp16", [300, 5000], lambda i: eight, master=True, place=False).run(t=2, in_place=True)
    for a, b in zip(want, got):
        assert all(torch.equal(a[k].cpu(), b[k]) for k in a)
    # a step that is not taken: host arrays stay as they are
    c = Case(pkg, "fp16", [300, 5000], lambda i: eight, master=True, place=False)
    before = [{k: v.clone() for k, v in d.items() if v is not None} for d in c.dev]
    got = c.run(t=2, in_place=True, factor=torch.tensor([float("inf")]))
    assert all(torch.equal(d[k], v) for d, b in zip(got, before) for k, v in b.items())


@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("shared", [("m", "mq"), ("v", "vq", "ms"), ("ms",), ("vs", "mq", "vq"), ("master",)])
def test_some_places_shared_without_a_step(pkg, gpu, eight, master, shared):
    """Without a finite factor every part of a new state that is not the old one's place receives what that holds, whichever others are."""
    c = Case(pkg, "fp16", [5, 700], lambda i: eight, master=master)
    for d, o in zip(c.dev, c.out):
        for k in shared:
            if o.get(k) is not None:
                o[k] = d[k]
    before = [{k: v.clone() for k, v in d.items() if v is not None} for d in c.dev]
    for o, d, b in zip(c.run(t=3, factor=torch.tensor([float("nan")], device="cuda")), c.dev, before):
        assert all(torch.equal(d[k], b[k]) for k in b)
        assert torch.equal(o["w"], (b["master"] if master else b["w"]).to(o["w"].dtype))
        assert all(torch.equal(v, b[k]) for k, v in o.items() if k != "w" and v is not None)
    c.untouched()
    for d, o in zip(c.dev, c.out):
        for k in shared:
            assert o.get(k) is None or o[k] is d[k]
