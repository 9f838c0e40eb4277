"""The norms between two blocks, their gate and residual, against their formula in 64 bits.  u = 2^-24.  A sum of n positive terms that
is formed in chains of at most c additions is at most c u of itself off; a row's sums are formed in chains of 8 values a piece, up to 8
pieces a thread (long rows: dim / 1024 a thread), 6 folds of a wave and 15 of its workgroup."""
import ctypes

import pytest
import torch

import transformer as tr
import tuning as tn

pytestmark = pytest.mark.gpu
U = tr.U
EPS, ALPHA = 1e-5, 0.75


def chain(dim):
    return 64 + 21 + dim / 1024


def gates(n, per):
    return 1 if per == 0 else -(-n // per)


def make(seed, dt, n, dim, per=0, gate=True, pre=True):
    r = lambda k, *s, **a: tr.rand(seed * 50 + k, *s, dt=dt, **a)  # noqa: E731
    return {"b": r(1, n, dim), "x": r(2, n, dim, scale=2.0), "w1": 1 + r(3, dim, scale=0.2), "w2": 1 + r(4, dim, scale=0.2) if pre else None,
            "gate": r(5, gates(n, per), dim, scale=0.5) if gate else None, "s": r(6, n, dim, scale=2.0), "dy": r(7, n, dim, scale=0.5) if pre else None,
            "ds": r(8, n, dim, scale=0.5)}


def rows_of(gate, n, per):
    return 1.0 if gate is None else gate.double() if per == 0 or per >= n else gate.double()[torch.arange(n) // per]


def forward(pkg, gpu, dt, t, per=0, alpha=ALPHA, eps=EPS, over=False):
    n, dim = t["b"].shape
    d = {k: None if t[k] is None else tr.dev(t[k]) for k in ("b", "x", "w1", "w2", "gate")}
    s = d["x"] if over else torch.full((n + 1, dim), 7, dtype=d["b"].dtype, device="cuda")
    y = None if d["w2"] is None else d["b"] if over else torch.full((n + 1, dim), 7, dtype=d["b"].dtype, device="cuda")
    a, keep = tn.join_args(pkg, dim, s=s, y=y, alpha=alpha, eps=eps, per=per, **d)
    pkg.call("ptl_norm_join_%s_fw_batched" % dt, a, n)
    assert gpu.ptl_sync() == 0
    if not over:
        assert (s[n] == 7).all() and (y is None or (y[n] == 7).all())
    return s[:n], None if y is None else y[:n]


def check_forward(dt, t, s, y, per=0, alpha=ALPHA, eps=EPS):
    n, dim = t["b"].shape
    d = {k: None if t[k] is None else t[k].double() for k in ("b", "x", "w1", "w2", "gate")}
    ref, ry = tn.join64(d["b"], d["x"], d["gate"], d["w1"], d["w2"], alpha, eps, per or n)
    # b, the weight and the gate round three products, the root and the quotient half of the sum's error
    gu = (ref - alpha * d["x"]).abs()
    off = gu * U * (chain(dim) / 2 + 9) + 2 * U * (alpha * d["x"]).abs() + U * ref.abs()
    tr.within(s, ref, off + tr.step(ref, dt), "s")
    if y is None:
        return
    rms = torch.sqrt((ref * ref).mean(1, keepdim=True) + eps)
    # s as it is before it is rounded, off by that, and the root by what the row's sum is
    tol = off / rms * d["w2"].abs() + ry.abs() * (torch.sqrt((off * off).mean(1, keepdim=True)) / rms + U * (chain(dim) / 2 + 8))
    tr.within(y, ry, tol + tr.step(ry, dt), "y")


DIMS = [1, 3, 4, 7, 8, 9, 63, 64, 257, 512, 785, 1000, 1024, 2056, 4095, 4096, 4100, 8200, 16384, 16400]


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("dim", DIMS)
def test_forward(pkg, gpu, dt, dim):
    for n, per, gate, pre in ((1, 0, 1, 1), (5, 2, 1, 1), (67, 0, 0, 1), (67, 10, 1, 0)):
        t = make(dim + n, dt, n, dim, per, gate, pre)
        check_forward(dt, t, *forward(pkg, gpu, dt, t, per), per)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,dim,per", [(9000, 64, 7), (9001, 200, 0), (4500, 1001, 1), (2100, 2056, 300), (1025, 4096, 64), (3, 33000, 1), (5, 70001, 2)])
def test_forward_many_rows_and_long_rows(pkg, gpu, dt, n, dim, per):
    """Walkers of several rows, also across the borders of gates; rows that no workgroup holds."""
    t = make(n, dt, n, dim, per)
    check_forward(dt, t, *forward(pkg, gpu, dt, t, per), per)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,dim", [(3, 77), (2, 4096), (9000, 72), (2, 40001)])
def test_forward_in_place(pkg, gpu, dt, n, dim):
    t = make(1, dt, n, dim)
    s, y = forward(pkg, gpu, dt, t)
    s2, y2 = forward(pkg, gpu, dt, t, over=True)
    assert torch.equal(s, s2) and torch.equal(y, y2)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_forward_values(pkg, gpu, dt):
    """Rows of zeros (with eps 0 too), infinities and NaN stay in their rows."""
    n, dim = 8, 100
    t = make(2, dt, n, dim)
    t["b"][1] = 0
    t["b"][2, 5], t["x"][3, 7], t["b"][4, 99] = float("inf"), float("nan"), float("nan")
    t["b"][5], t["x"][5] = 0, 0
    for eps in (EPS, 0.0):
        s, y = forward(pkg, gpu, dt, t, eps=eps)
        good = [0, 6, 7]
        check_forward(dt, {k: v if v is None or v.shape[0] != n else v[good] for k, v in t.items()}, s[good], y[good], eps=eps)
        assert torch.equal(s[1].cpu(), (t["x"][1].double() * ALPHA).to(s.dtype)) and torch.isfinite(y[1]).all()
        assert (s[5] == 0).all() and (y[5] == 0).all()
        assert torch.isnan(s[2, 5]) and torch.isnan(s[4]).all() and torch.isnan(s[3, 7]) and torch.isfinite(s[3, :7]).all() and torch.isnan(y[3]).all()


def backward(pkg, gpu, dt, t, per=0, alpha=ALPHA, eps=EPS, places=None, **skips):
    n, dim = t["b"].shape
    d = {k: None if t[k] is None else tr.dev(t[k]) for k in ("b", "s", "w1", "w2", "gate", "dy", "ds")}
    full = lambda v: None if v is None else torch.full_like(v, 7)  # noqa: E731
    out = {"db": full(d["b"]), "dx": full(d["b"]), "dw1": full(d["w1"]), "dw2": full(d["w2"]), "dgate": full(d["gate"])}
    for k, v in (places or {}).items():
        out[k] = d[v]
    a, keep = tn.join_args(pkg, dim, alpha=alpha, eps=eps, per=per, **d, **out, **skips)
    pkg.call("ptl_norm_join_%s_bw_batched" % dt, a, n)
    assert gpu.ptl_sync() == 0
    return out


def check_backward(dt, t, got, per=0, alpha=ALPHA, eps=EPS, only=None):
    n, dim = t["b"].shape
    b, w1 = t["b"].double(), t["w1"].double()
    gate = rows_of(t["gate"], n, per)
    mean = lambda v: v.mean(1, keepdim=True)  # noqa: E731
    r1 = 1 / torch.sqrt(mean(b * b) + eps)
    c = U * (chain(dim) + 16)
    d = torch.zeros_like(b) if t["ds"] is None else t["ds"].double()
    g = s = m2 = torch.zeros_like(b)
    r2 = 0.0
    if t["w2"] is not None:
        s, dy = t["s"].double(), t["dy"].double()
        r2 = 1 / torch.sqrt(mean(s * s) + eps)
        g = dy * t["w2"].double()
        m2 = r2 * r2 * mean(g * s)
    ds = d + r2 * (g - s * m2)
    off = c * ((r2 * g).abs() + r2 ** 3 * mean((g * s).abs()) * s.abs()) + 2 * U * (ds.abs() + d.abs())
    k = gate * w1 * ds
    k0 = (gate * w1 * b).abs()
    am = r2 * r2 * mean((g * s).abs())  # of m2
    e_mean = 2 * c * (mean(k0 * d.abs()) + r2 * mean(k0 * g.abs()) + r2 * am * mean(k0 * s.abs()))
    db = r1 * (k - b * r1 * r1 * mean(k * b))
    tol = r1 * ((gate * w1).abs() * off + 3 * U * k.abs() + b.abs() * r1 * r1 * e_mean) + c * (r1 * k.abs() + r1 ** 3 * b.abs() * mean(k * b).abs())
    u, hat = b * r1 * w1, b * r1
    sums = {"dw1": (gate * ds * hat, (gate * hat).abs() * off + (gate * ds * hat).abs() * U * (chain(dim) / 2 + 10))}
    if t["w2"] is not None:
        sums["dw2"] = (t["dy"].double() * s * r2, (t["dy"].double() * s * r2).abs() * U * (chain(dim) / 2 + 8))
    if t["gate"] is not None:
        sums["dgate"] = (ds * u, u.abs() * off + (ds * u).abs() * U * (chain(dim) / 2 + 10))
    for name in only or ("db", "dx", "dw1", "dw2", "dgate"):
        if name == "db":
            tr.within(got["db"], db, tol + tr.step(db, dt), "db")
        elif name == "dx":
            tr.within(got["dx"], alpha * ds, abs(alpha) * off + 2 * U * (alpha * ds).abs() + tr.step(alpha * ds, dt), "dx")
        elif name in sums:
            each, e = sums[name]
            if name == "dgate":
                at = torch.arange(n) // (per or n)
                fold = lambda v: torch.zeros(gates(n, per), dim, dtype=torch.float64).index_add_(0, at, v)  # noqa: E731
            else:
                fold = lambda v: v.sum(0)  # noqa: E731
            ref = fold(each)
            tr.within(got[name], ref, fold(e) + U * (n + 4) * fold(each.abs()) + tr.step(ref, dt), name)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("dim", DIMS)
def test_backward(pkg, gpu, dt, dim):
    for n, per, gate, pre in ((1, 0, 1, 1), (3, 1, 1, 1), (5, 2, 1, 1), (67, 0, 1, 1), (67, 0, 0, 0), (67, 10, 1, 0)):
        t = make(dim + n, dt, n, dim, per, gate, pre)
        check_backward(dt, t, backward(pkg, gpu, dt, t, per), per)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,dim,per", [(3000, 64, 0), (3001, 72, 1), (3001, 200, 5), (2500, 100, 700), (1030, 500, 1000), (1100, 1001, 3), (1025, 2056, 0),
                                       (1025, 2056, 256), (515, 4096, 2), (515, 4100, 500), (300, 8200, 0), (300, 8200, 90), (130, 20000, 0), (130, 20000, 1),
                                       (130, 20000, 3), (130, 20000, 100), (2, 33001, 1)])
def test_backward_many_rows_and_gates(pkg, gpu, dt, n, dim, per):
    """Gates of one row, of a few (a walker has several gates), and of many (several walkers have a gate's rows; the last gate has fewer, so
    that some have none)."""
    t = make(n, dt, n, dim, per)
    check_backward(dt, t, backward(pkg, gpu, dt, t, per), per)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,dim,per", [(3, 77, 0), (40, 4096, 0), (1500, 72, 50), (9, 20001, 2)])
def test_backward_in_place(pkg, gpu, dt, n, dim, per):
    t = make(3, dt, n, dim, per)
    want = backward(pkg, gpu, dt, t, per)
    for places in ({"db": "b", "dx": "s"}, {"db": "dy", "dx": "ds"}, {"db": "s", "dx": "b"}, {"db": "ds", "dx": "dy"}):
        got = backward(pkg, gpu, dt, t, per, places=places)
        assert all(torch.equal(got[k], v) for k, v in want.items()), places


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("dim", [40, 1000, 5000, 20000])
def test_backward_parts_of_the_arguments(pkg, gpu, dt, dim):
    n = 33
    for per in (0, 4):
        t = make(4, dt, n, dim, per)
        want = backward(pkg, gpu, dt, t, per)
        got = backward(pkg, gpu, dt, t, per, skip_wg=1)
        assert all((got[k] == 7).all() for k in ("dw1", "dw2", "dgate")) and all(torch.equal(got[k], want[k]) for k in ("db", "dx"))
        got = backward(pkg, gpu, dt, t, per, skip_ig=1)
        assert all((got[k] == 7).all() for k in ("db", "dx"))
        check_backward(dt, t, got, per, only=("dw1", "dw2", "dgate"))
        t["ds"] = None  # no gradient along the residual
        check_backward(dt, t, backward(pkg, gpu, dt, t, per), per)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_backward_values(pkg, gpu, dt):
    """NaN stays in its row; rows of zeros with eps 0 take part with the residual only."""
    n, dim = 6, 130
    t = make(5, dt, n, dim)
    t["ds"][2, 3], t["b"][4] = float("nan"), 0
    got = backward(pkg, gpu, dt, t, skip_wg=1)
    assert torch.isnan(got["dx"][2, 3]) and torch.isnan(got["db"][2]).all()
    good = [0, 1, 3, 5]
    cut = {k: v if v is None or v.shape[0] != n else v[good] for k, v in t.items()}
    check_backward(dt, cut, {k: got[k][good] for k in ("db", "dx")}, only=("db", "dx"))
    t = make(6, dt, n, dim)
    t["b"][1], t["s"][3] = 0, 0
    got = backward(pkg, gpu, dt, t, eps=0.0)
    assert (got["db"][1] == 0).all() and all(torch.isfinite(got[k]).all() for k in got)
    assert torch.equal(got["dx"][3].cpu(), (t["ds"][3].double() * ALPHA).to(t["ds"].dtype))


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,dim,per", [(10, 333, 0), (700, 129, 100), (3, 5001, 1)])
def test_unaligned_tensors(pkg, gpu, dt, n, dim, per):
    t = make(7, dt, n, dim, per)

    def off(v, fill=False):
        if v is None:
            return None
        buf = torch.full((v.numel() + 2,), 7, dtype=v.dtype, device="cuda")
        o = buf[1:-1].view(v.shape)
        return o if fill else o.copy_(v)

    d = {k: off(v) for k, v in t.items()}
    s, y = off(t["s"], True), off(t["s"], True)
    a, keep = tn.join_args(pkg, dim, b=d["b"], x=d["x"], gate=d["gate"], w1=d["w1"], w2=d["w2"], s=s, y=y, alpha=ALPHA, per=per)
    pkg.call("ptl_norm_join_%s_fw_batched" % dt, a, n)
    check_forward(dt, t, s, y, per)
    out = {"db": off(t["b"], True), "dx": off(t["b"], True), "dw1": off(t["w1"], True), "dw2": off(t["w2"], True), "dgate": off(t["gate"], True)}
    a, keep = tn.join_args(pkg, dim, alpha=ALPHA, per=per, **{k: d[k] for k in ("b", "s", "w1", "w2", "gate", "dy", "ds")}, **out)
    pkg.call("ptl_norm_join_%s_bw_batched" % dt, a, n)
    check_backward(dt, t, out, per)


@pytest.mark.parametrize("per", [0, 2])
def test_gradients_against_differences(pkg, gpu, per):
    n, dim, h = 3, 5, 1e-5
    t = make(8, "fp32", n, dim, per)
    d = {k: t[k].double() for k in ("b", "x", "gate", "w1", "w2")}
    s, _ = tn.join64(d["b"], d["x"], d["gate"], d["w1"], d["w2"], ALPHA, EPS, per or n)
    t["s"] = s.float()
    got = backward(pkg, gpu, "fp32", t, per)

    def f(v):
        s, y = tn.join64(v["b"], v["x"], v["gate"], v["w1"], v["w2"], ALPHA, EPS, per or n)
        return (s * t["ds"].double()).sum() + (y * t["dy"].double()).sum()

    for k, name in (("b", "db"), ("x", "dx"), ("gate", "dgate"), ("w1", "dw1"), ("w2", "dw2")):
        for i in range(d[k].numel()):
            up, down = {**d, k: d[k].clone()}, {**d, k: d[k].clone()}
            up[k].view(-1)[i] += h
            down[k].view(-1)[i] -= h
            assert abs(float(f(up) - f(down)) / (2 * h) - float(got[name].view(-1)[i])) < 2e-5, (k, i)


def test_host_arrays(pkg, gpu):
    n, dim, per = 7, 50, 3
    t = make(9, "fp16", n, dim, per)
    s, y = forward(pkg, gpu, "fp16", t, per)
    h = {k: v.numpy() for k, v in t.items()}
    z = lambda v: torch.zeros_like(v).numpy()  # noqa: E731
    hs, hy = z(t["s"]), z(t["s"])
    a, keep = tn.join_args(pkg, dim, b=h["b"], x=h["x"], gate=h["gate"], w1=h["w1"], w2=h["w2"], s=hs, y=hy, alpha=ALPHA, per=per)
    pkg.call("ptl_norm_join_fp16_fw_batched", a, n)
    assert torch.equal(torch.from_numpy(hs), s.cpu()) and torch.equal(torch.from_numpy(hy), y.cpu())
    want = backward(pkg, gpu, "fp16", t, per)
    out = {"db": z(t["b"]), "dx": z(t["b"]), "dw1": z(t["w1"]), "dw2": z(t["w2"]), "dgate": z(t["gate"])}
    a, keep = tn.join_args(pkg, dim, alpha=ALPHA, per=per, **{k: h[k] for k in ("b", "s", "w1", "w2", "gate", "dy", "ds")}, **out)
    pkg.call("ptl_norm_join_fp16_bw_batched", a, n)
    assert all(torch.equal(torch.from_numpy(out[k]), want[k].cpu()) for k in out)


def test_many_gates_of_the_longest_rows(pkg, gpu, monkeypatch):
    """Rows of 2^24 values with six gates: more columns of gates than one launch has threads to add up in parts.  The rows repeat 1024 values, so
    that means are those of 1024, and every column's results are those of the first 1024; the sums are as long as the rows."""
    n, dim, per = 12, 1024, 2
    t = make(11, "fp16", n, dim, per)
    long = {k: None if v is None else v.cuda().repeat(*([1] * (v.dim() - 1)), 1 << 14) for k, v in t.items()}
    got = backward(pkg, gpu, "fp16", long, per=per)
    for k, v in got.items():
        blocks = v.view(-1, 1 << 14, dim)
        assert (blocks == blocks[:, :1]).all(), k
    reach = chain(1 << 24)
    monkeypatch.setitem(globals(), "chain", lambda d: reach)
    check_backward("fp16", t, {k: v[..., :dim] for k, v in got.items()}, per=per)
