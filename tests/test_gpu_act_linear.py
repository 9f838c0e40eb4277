"""Dense layers with bias, activation and residual against their formula in 64 bits.  u = 2^-24; a sum of n products is at most n u of
the sum of their magnitudes off, however it is formed."""
import ctypes

import pytest
import torch

import transformer as tr
import tuning as tn

pytestmark = pytest.mark.gpu
U = tr.U


def inputs(seed, dt, n, n_in, n_out, bias=1, skip=1):
    x, w = tr.rand(seed, n, n_in, dt=dt), tr.rand(seed + 1, n_out, n_in, scale=1.5 / n_in ** 0.5, dt=dt)
    return x, w, tr.rand(seed + 2, n_out, scale=0.3, dt=dt) if bias else None, tr.rand(seed + 3, n, n_out, dt=dt) if skip else None


def forward(pkg, gpu, dt, act, x, w, b, skip, keep=True, over=False):
    n, n_in, n_out = x.shape[0], x.shape[1], w.shape[0]
    X, W, B = tr.dev(x), tr.dev(w), None if b is None else tr.dev(b)
    y = torch.full((n + 1, n_out), 7, dtype=X.dtype, device="cuda")
    h = torch.full((n + 1, n_out), 7, dtype=X.dtype, device="cuda") if keep else None
    S = None if skip is None else tr.dev(skip)
    if over:  # the output in the residual's place
        y[:n] = S
        S = y
    a, held = tn.act_args(pkg, n_in, n_out, tn.ACTS[act], x=X, w=W, b=B, h=h, skip=S, y=y)
    pkg.call("ptl_act_linear_%s_fw_batched" % dt, a, n)
    assert gpu.ptl_sync() == 0
    assert (y[n] == 7).all() and (h is None or (h[n] == 7).all())  # behind the last sample
    return y[:n], None if h is None else h[:n]


def check_forward(dt, act, x, w, b, skip, y, h):
    n_in = x.shape[1]
    x, w = x.double(), w.double()
    ref = x @ w.t() + (0 if b is None else b.double())
    off = U * ((n_in + 2) * (x.abs() @ w.abs().t()) + 2 * ref.abs())
    if h is not None:
        tr.within(h, ref, off + tr.step(ref, dt), "h")
    f, _ = tn.act64(ref, act)
    steps = torch.zeros_like(ref) if act == "none" else tr.act_steps(ref, act)
    out = f if skip is None else f + skip.double()
    # slopes of the activations are at most 1.13
    tr.within(y, out, 1.13 * off + f.abs() * U * steps + 2 * U * out.abs() + tr.step(out, dt), "y")


SHAPES = [(1, 1, 1), (1, 5, 3), (2, 7, 16), (3, 64, 17), (5, 785, 33), (8, 128, 40), (9, 100, 31), (33, 64, 64), (64, 33, 96), (65, 129, 65),
          (130, 200, 130), (257, 72, 150)]


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,n_in,n_out", SHAPES)
def test_forward(pkg, gpu, dt, n, n_in, n_out):
    for act, bias, keep, skip in (("silu", 0, 1, 1), ("gelu", 1, 0, 1), ("relu", 1, 1, 0), ("sigmoid", 0, 0, 1), ("none", 1, 1, 1), ("none", 0, 0, 0)):
        x, w, b, s = inputs(n + n_in, dt, n, n_in, n_out, bias, skip)
        check_forward(dt, act, x, w, b, s, *forward(pkg, gpu, dt, act, x, w, b, s, keep))


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,n_in,n_out", [(1, 4096, 700), (4, 2048, 1001), (12, 1024, 600), (16, 3000, 1000), (391, 785, 333), (300, 1024, 512), (600, 512, 1000),
                                          (1024, 256, 2112), (520, 1040, 2051), (2000, 264, 1999)])
def test_forward_larger(pkg, gpu, dt, n, n_in, n_out):
    """Tiles of every size, rows that are copied, k in parts."""
    for act, skip, keep in (("gelu", 1, 1), ("none", 1, 0)):
        x, w, b, s = inputs(n, dt, n, n_in, n_out, n % 2, skip)
        check_forward(dt, act, x, w, b, s, *forward(pkg, gpu, dt, act, x, w, b, s, keep))


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,n_in,n_out", [(1, 40, 33), (20, 300, 77), (300, 1024, 512), (1500, 512, 1000)])
def test_output_in_the_residuals_place(pkg, gpu, dt, n, n_in, n_out):
    x, w, b, s = inputs(n, dt, n, n_in, n_out)
    y, _ = forward(pkg, gpu, dt, "silu", x, w, b, s, keep=False)
    z, _ = forward(pkg, gpu, dt, "silu", x, w, b, s, keep=False, over=True)
    assert torch.equal(y, z)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n", [1, 3, 70])
def test_forward_values(pkg, gpu, dt, n):
    """What is no number stays in its sample or its output, also next to the end of a row that ends inside a piece; far
    pre-activations take their limits."""
    n_in, n_out = 37, 20
    x, w, _, s = inputs(3, dt, n, n_in, n_out)
    w[4, 36], s[0, 19], s[n - 1, 7] = float("nan"), float("inf"), float("nan")
    y, h = forward(pkg, gpu, dt, "gelu", x, w, None, s)
    good = torch.ones(n, n_out, dtype=torch.bool)
    good[:, 4] = good[0, 19] = good[n - 1, 7] = False
    assert torch.isnan(h[:, 4]).all() and torch.isfinite(h.cpu()[:, [i for i in range(n_out) if i != 4]]).all()
    assert torch.equal(torch.isfinite(y.cpu()), good)
    x = torch.zeros(n, 3, dtype=tr.t_dtype(dt))
    x[:, 0] = 1000
    w = torch.zeros(3, 3, dtype=tr.t_dtype(dt))
    w[0, 0], w[1, 0] = 1, -1
    for act, want in (("silu", (1000, 0, 0)), ("gelu", (1000, 0, 0)), ("sigmoid", (1, 0, 0.5)), ("relu", (1000, 0, 0)), ("none", (1000, -1000, 0))):
        y, _ = forward(pkg, gpu, dt, act, x, w, None, None)
        assert torch.equal(y.double().cpu(), torch.tensor([want], dtype=torch.float64).expand(n, 3)), act


def backward(pkg, gpu, dt, act, x, w, h, dy, bias, over=None, **more):
    n, n_in, n_out = x.shape[0], x.shape[1], w.shape[0]
    X, W, H, DY = (None if t is None else tr.dev(t) for t in (x, w, h, dy))
    dx, dw = torch.full_like(X, 7), torch.full_like(W, 7)
    dh = None if h is None else H if over == "h" else DY if over == "dy" else torch.full_like(H, 7)
    db = torch.full((n_out,), 7, dtype=X.dtype, device="cuda") if bias else None
    a, keep = tn.act_args(pkg, n_in, n_out, tn.ACTS[act], x=X, dx=dx, w=W, dw=dw, db=db, h=H, dh=dh, dy=DY, **more)
    pkg.call("ptl_act_linear_%s_bw_batched" % dt, a, n)
    assert gpu.ptl_sync() == 0
    if over != "dy":
        assert torch.equal(DY.cpu(), dy)
    return dh, dx, dw, db


def check_backward(dt, act, x, w, h, dy, dh, dx, dw, db):
    n, n_out = dy.shape
    d = dy.double()
    if act == "none":
        ref, tol, got = d, torch.zeros_like(d), d
    else:
        g = h.double()
        f, df = tn.act64(g, act)
        ref = d * df
        # the slope is a sum of two terms: act / g (gate 1: its limit) and the rest
        first = torch.where(g != 0, f / g, torch.ones_like(g)).abs() if act in ("silu", "gelu") else torch.zeros_like(g)
        tol = d.abs() * U * (tr.act_steps(g, act) + 8) * (2 * first + df.abs())
        tr.within(dh, ref, tol + tr.step(ref, dt), "dh")
        got = dh.double().cpu()  # what the products read
    off = torch.zeros_like(got)
    if act != "none" and dt == "fp16" and (n <= 2 or n * n_out < 16384):  # ... few of them: before they are rounded, in two halves of 11 bits
        got, off = ref, tol + ref.abs() * 2.0 ** -22 + 2.0 ** -36
    x, w = x.double(), w.double()
    if dx is not None:
        ref = got @ w
        tr.within(dx, ref, U * (2 * n_out + 8) * (got.abs() @ w.abs()) + off @ w.abs() + tr.step(ref, dt), "dx")
    if dw is not None:
        ref = got.t() @ x
        tr.within(dw, ref, U * (2 * n + 8) * (got.abs().t() @ x.abs()) + off.t() @ x.abs() + tr.step(ref, dt), "dw")
    if db is not None:
        ref = got.sum(0)
        tr.within(db, ref, U * (n + 4) * got.abs().sum(0) + off.sum(0) + tr.step(ref, dt), "db")


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,n_in,n_out", SHAPES + [(391, 785, 333), (512, 1024, 704), (700, 520, 1001), (1024, 512, 1024)])
def test_backward(pkg, gpu, dt, n, n_in, n_out):
    for act, bias in (("silu", 0), ("gelu", 1), ("relu", 0), ("sigmoid", 1), ("none", 0), ("none", 1)):
        x, w, _, _ = inputs(n, dt, n, n_in, n_out)
        h = None if act == "none" else tr.rand(n + 5, n, n_out, scale=1.5, dt=dt)
        dy = tr.rand(n + 6, n, n_out, scale=0.5, dt=dt)
        check_backward(dt, act, x, w, h, dy, *backward(pkg, gpu, dt, act, x, w, h, dy, bias))


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,n_in,n_out", [(2, 70, 50), (20, 50, 30), (64, 512, 1408), (300, 1024, 1024)])
def test_backward_skips_and_in_place(pkg, gpu, dt, n, n_in, n_out):
    x, w, _, _ = inputs(1, dt, n, n_in, n_out)
    h, dy = tr.rand(5, n, n_out, dt=dt), tr.rand(6, n, n_out, dt=dt)
    full = backward(pkg, gpu, dt, "silu", x, w, h, dy, 1)
    for over in ("h", "dy"):
        again = backward(pkg, gpu, dt, "silu", x, w, h, dy, 1, over=over)
        assert all(torch.equal(a, b) for a, b in zip(full, again)), over
    for act in ("silu", "none"):
        H = h if act != "none" else None
        full = backward(pkg, gpu, dt, act, x, w, H, dy, 1)
        dh, dx, dw, db = backward(pkg, gpu, dt, act, x, w, H, dy, 1, skip_wg=1)
        assert (H is None or torch.equal(dh, full[0])) and (dw == 7).all() and (db == 7).all()
        check_backward(dt, act, x, w, H, dy, dh, dx, None, None)
        dh, dx, dw, db = backward(pkg, gpu, dt, act, x, w, H, dy, 1, skip_ig=1)
        assert (H is None or torch.equal(dh, full[0])) and (dx == 7).all()
        check_backward(dt, act, x, w, H, dy, dh, None, dw, db)
        dh, dx, dw, db = backward(pkg, gpu, dt, act, x, w, H, dy, 1, skip_ig=1, skip_wg=1)
        assert (H is None or torch.equal(dh, full[0])) and (dx == 7).all() and (dw == 7).all()


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_unaligned_tensors(pkg, gpu, dt):
    """Tensors that start inside a 16-byte piece: views one element into a buffer."""
    for n, n_in, n_out in ((3, 65, 40), (70, 128, 96), (400, 512, 640)):
        x, w, b, s = inputs(n, dt, n, n_in, n_out)
        h, dy = tr.rand(n + 5, n, n_out, dt=dt), tr.rand(n + 6, n, n_out, dt=dt)

        def off(t, fill=None):
            buf = torch.full((t.numel() + 2,), 7, dtype=t.dtype, device="cuda")
            v = buf[1:-1].view(t.shape)
            if fill is None:
                v.copy_(t)
            return v

        X, W, B, S, H, DY = (off(t) for t in (x, w, b, s, h, dy))
        y, hid, dx, dw, db, dh = (off(t, 7) for t in (s, s, x, w, b, h))
        a, keep = tn.act_args(pkg, n_in, n_out, 2, x=X, w=W, b=B, h=hid, skip=S, y=y)
        pkg.call("ptl_act_linear_%s_fw_batched" % dt, a, n)
        check_forward(dt, "gelu", x, w, b, s, y, hid)
        a, keep = tn.act_args(pkg, n_in, n_out, 2, x=X, dx=dx, w=W, dw=dw, db=db, h=H, dh=dh, dy=DY)
        pkg.call("ptl_act_linear_%s_bw_batched" % dt, a, n)
        check_backward(dt, "gelu", x, w, h, dy, dh, dx, dw, db)


def test_gradients_against_differences(pkg, gpu):
    n, n_in, n_out, h = 2, 5, 4, 1e-5
    x, w, b, s = inputs(7, "fp32", n, n_in, n_out)
    dy = tr.rand(8, n, n_out)
    for act in ("silu", "gelu", "sigmoid", "none"):
        _, hidden = forward(pkg, gpu, "fp32", act, x, w, b, s)
        _, dx, dw, db = backward(pkg, gpu, "fp32", act, x, w, None if act == "none" else hidden.cpu(), dy, 1)

        def f(x_, w_, b_):
            return ((tn.act64(x_ @ w_.t() + b_, act)[0] + s.double()) * dy.double()).sum()

        at = [x.double(), w.double(), b.double()]
        for k, got in enumerate((dx, dw, db)):
            for i in range(got.numel()):
                e = [torch.zeros_like(t) for t in at]
                e[k].view(-1)[i] = h
                up, down = (f(*(t + sg * d for t, d in zip(at, e))) for sg in (1, -1))
                assert abs((up - down) / (2 * h) - float(got.view(-1)[i])) < 1e-5


@pytest.mark.parametrize("act", ["silu", "none"])
def test_host_arrays(pkg, gpu, act):
    n, n_in, n_out = 5, 33, 12
    x, w, b, s = inputs(9, "fp16", n, n_in, n_out)
    dy = tr.rand(10, n, n_out, dt="fp16")
    y, h = forward(pkg, gpu, "fp16", act, x, w, b, s)
    z = lambda *sh: torch.zeros(*sh, dtype=torch.float16).numpy()  # noqa: E731
    hy, hh = z(n, n_out), z(n, n_out)
    a, keep = tn.act_args(pkg, n_in, n_out, tn.ACTS[act], x=x.numpy(), w=w.numpy(), b=b.numpy(), h=hh, skip=s.numpy(), y=hy)
    pkg.call("ptl_act_linear_fp16_fw_batched", a, n)
    assert torch.equal(torch.from_numpy(hy), y.cpu()) and torch.equal(torch.from_numpy(hh), h.cpu())
    want = backward(pkg, gpu, "fp16", act, x, w, None if act == "none" else h.cpu(), dy, 1)
    dh, dx, dw, db = z(n, n_out), z(n, n_in), z(n_out, n_in), z(n_out)
    a, keep = tn.act_args(pkg, n_in, n_out, tn.ACTS[act], x=x.numpy(), dx=dx, w=w.numpy(), dw=dw, db=db, h=hh, dh=dh, dy=dy.numpy())
    pkg.call("ptl_act_linear_fp16_bw_batched", a, n)
    for got, ref in zip((dh, dx, dw, db), want):
        assert ref is None or torch.equal(torch.from_numpy(got), ref.cpu())


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_same_as_a_dense_layer(pkg, gpu, dt):
    """Without activation and residual: within both calls' roundings of what the framework's dense layer gives."""
    n, n_in, n_out = 50, 96, 40
    x, w, b, _ = inputs(4, dt, n, n_in, n_out)
    y, _ = forward(pkg, gpu, dt, "none", x, w, b, None)
    keep, l = [], (pkg.LinearArgs if dt == "fp32" else pkg.LinearArgs)()
    out = torch.empty_like(y)
    l.input, l.coeff, l.bias = tr.ptr(keep, pkg, tr.dev(x), None, n_in), tr.ptr(keep, pkg, tr.dev(w), None, n_in, n_out), tr.ptr(keep, pkg, tr.dev(b), None, n_out)
    l.output, l.use_biases = tr.ptr(keep, pkg, out, None, n_out), 1
    pkg.call("ptl_linear_%s_fw_batched" % dt, l, n)
    ref = x.double() @ w.double().t() + b.double()
    tr.within(y, out.double().cpu(), 2 * (U * (n_in + 4) * (x.double().abs() @ w.double().abs().t()) + U * 2 * ref.abs() + tr.step(ref, dt)))


@pytest.mark.parametrize("n,n_in,n_out", [(1000, 1500, 4100), (4096, 1000, 1100), (1500, 2056, 4000), (4000, 1000, 2100), (2500, 776, 3001)])
def test_forward_large_tiles(pkg, gpu, n, n_in, n_out):
    """fp16 tiles of 256 x 128, 256 x 256 and 128 x 128 whose last rows, tokens and values of k are no whole tiles, slabs or pieces."""
    for act, skip, keep in (("gelu", 1, 1), ("none", 1, 0)):
        x, w, b, s = inputs(n, "fp16", n, n_in, n_out, 1, skip)
        check_forward("fp16", act, x, w, b, s, *forward(pkg, gpu, "fp16", act, x, w, b, s, keep))


@pytest.mark.parametrize("n,n_in,n_out", [(2100, 1000, 2003), (2048, 1032, 2048), (2000, 1001, 2100), (8300, 300, 1700)])
def test_backward_large_tiles(pkg, gpu, n, n_in, n_out):
    """Gradients of 16 GFLOP and more in fp16: tiles of 256 x 128, both products and each alone."""
    x, w, _, _ = inputs(n, "fp16", n, n_in, n_out)
    h, dy = tr.rand(n + 5, n, n_out, scale=1.5, dt="fp16"), tr.rand(n + 6, n, n_out, scale=0.5, dt="fp16")
    check_backward("fp16", "gelu", x, w, h, dy, *backward(pkg, gpu, "fp16", "gelu", x, w, h, dy, 1))


@pytest.mark.parametrize("n,n_in,n_out", [(4100, 1000, 2003), (2100, 2050, 2000)])
def test_backward_large_tiles_alone(pkg, gpu, n, n_in, n_out):
    x, w, _, _ = inputs(n, "fp16", n, n_in, n_out)
    h, dy = tr.rand(n + 5, n, n_out, scale=1.5, dt="fp16"), tr.rand(n + 6, n, n_out, scale=0.5, dt="fp16")
    dh, dx, dw, db = backward(pkg, gpu, "fp16", "silu", x, w, h, dy, 1, skip_wg=1)
    check_backward("fp16", "silu", x, w, h, dy, dh, dx, None, None)
    dh, dx, dw, db = backward(pkg, gpu, "fp16", "silu", x, w, h, dy, 1, skip_ig=1)
    check_backward("fp16", "silu", x, w, h, dy, dh, None, dw, db)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
@pytest.mark.parametrize("n", [1, 40])
def test_backward_far_values(pkg, gpu, dt, act, n):
    """Derivatives of far and infinite pre-activations take their limits; what is no number stays where it is."""
    top = torch.finfo(tr.t_dtype(dt)).max
    far = [0.0, -0.0, 200.0, -200.0, 300.0, -300.0, top, -top, float("inf"), -float("inf"), float("nan"), 1.0]
    h = torch.tensor([far] * n, dtype=tr.t_dtype(dt))
    dy = torch.ones_like(h)
    x, w = torch.zeros(n, 5, dtype=h.dtype), torch.zeros(len(far), 5, dtype=h.dtype)
    dh, _, _, _ = backward(pkg, gpu, dt, act, x, w, h, dy, 0)
    at0 = {"silu": 0.5, "gelu": 0.5, "relu": 0.0, "sigmoid": 0.25}[act]
    hi = 0.0 if act == "sigmoid" else 1.0
    want = torch.tensor([at0, at0] + [hi, 0.0] * 4, dtype=torch.float64).expand(n, 10)
    assert torch.equal(dh[:, :10].double().cpu(), want)
    assert torch.isnan(dh[:, 10]).all() and torch.isfinite(dh[:, 11]).all()


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n_in,n_out", [(1, 2050), (1000, 3001), (3001, 2111), (6100, 2048), (6200, 2049)])
def test_one_token_many_outputs(pkg, gpu, dt, n_in, n_out):
    for act, skip, keep in (("silu", 1, 1), ("none", 0, 0)):
        x, w, b, s = inputs(n_in, dt, 1, n_in, n_out, 1, skip)
        check_forward(dt, act, x, w, b, s, *forward(pkg, gpu, dt, act, x, w, b, s, keep))


@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("bias", [0, 1])
@pytest.mark.parametrize("n,n_in,n_out", [(1200, 80, 2564), (4000, 100, 2001), (2500, 600, 515), (530, 1031, 2500), (3100, 512, 500), (340, 1801, 2050)])
def test_backward_with_and_without_copies(pkg, gpu, act, bias, n, n_in, n_out):
    """fp16 rows of which some or all are no whole 16-byte pieces, on both sides of the sizes from which they are copied."""
    x, w, _, _ = inputs(n, "fp16", n, n_in, n_out)
    h, dy = None if act == "none" else tr.rand(n + 5, n, n_out, scale=1.5, dt="fp16"), tr.rand(n + 6, n, n_out, scale=0.5, dt="fp16")
    check_backward("fp16", act, x, w, h, dy, *backward(pkg, gpu, "fp16", act, x, w, h, dy, bias))


@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("n,n_in,n_out", [(10, 2048, 1640), (16, 1504, 1400), (33, 1024, 2000), (100, 2056, 1000), (9, 2048, 1824), (17, 8192, 256)])
def test_backward_few_tokens_and_large_weights(pkg, gpu, act, n, n_in, n_out):
    x, w, _, _ = inputs(n, "fp16", n, n_in, n_out)
    h, dy = None if act == "none" else tr.rand(n + 5, n, n_out, scale=1.5, dt="fp16"), tr.rand(n + 6, n, n_out, scale=0.5, dt="fp16")
    check_backward("fp16", act, x, w, h, dy, *backward(pkg, gpu, "fp16", act, x, w, h, dy, 1))
