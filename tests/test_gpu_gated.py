"""Gated dense layers against their formula in 64 bits.  u = 2^-24; a sum of n products is at most n u of the sum of their
magnitudes off, however it is formed."""
import ctypes

import pytest
import torch

import transformer as tr

pytestmark = pytest.mark.gpu
U = tr.U


def inputs(seed, dt, n, n_in, n_out, bias):
    x, w = tr.rand(seed, n, n_in, dt=dt), tr.rand(seed + 1, 2 * n_out, n_in, scale=1.5 / n_in ** 0.5, dt=dt)
    return x, w, tr.rand(seed + 2, 2 * n_out, scale=0.3, dt=dt) if bias else None


def forward(pkg, gpu, dt, act, x, w, b, keep=True):
    n, n_in, n_out = x.shape[0], x.shape[1], w.shape[0] // 2
    X, W, B = tr.dev(x), tr.dev(w), None if b is None else tr.dev(b)
    y = torch.full((n + 1, n_out), 7, dtype=X.dtype, device="cuda")
    h = torch.full((n + 1, 2 * n_out), 7, dtype=X.dtype, device="cuda") if keep else None
    a, held = tr.gated_args(pkg, n_in, n_out, tr.ACTS[act], x=X, w=W, b=B, h=h, y=y)
    pkg.call("ptl_gated_linear_%s_fw_batched" % dt, a, n)
    assert gpu.ptl_sync() == 0
    assert (y[n] == 7).all() and (h is None or (h[n] == 7).all())  # behind the last sample
    return y[:n], None if h is None else h[:n]


def check_forward(dt, act, x, w, b, y, h):
    n_in, n_out = x.shape[1], w.shape[0] // 2
    x, w = x.double(), w.double()
    ref = x @ w.t() + (0 if b is None else b.double())
    off = U * ((n_in + 2) * (x.abs() @ w.abs().t()) + 2 * ref.abs())
    if h is not None:
        tr.within(h, ref, off + tr.step(ref, dt), "h")
    g, up, og, ou = ref[:, :n_out], ref[:, n_out:], off[:, :n_out], off[:, n_out:]
    f, _ = tr.act64(g, act)
    # slopes of the activations are at most 1.13
    of = 1.13 * og + f.abs() * U * tr.act_steps(g, act)
    tr.within(y, f * up, of * up.abs() + (f.abs() + of) * ou + (f * up).abs() * U * 2 + tr.step(f * up, dt), "y")


SHAPES = [(1, 1, 1), (1, 5, 3), (2, 7, 16), (3, 64, 17), (5, 785, 33), (8, 128, 40), (9, 100, 31), (33, 64, 64), (64, 33, 96), (65, 129, 65),
          (130, 200, 130), (257, 72, 150)]


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,n_in,n_out", SHAPES)
def test_forward(pkg, gpu, dt, n, n_in, n_out):
    for act, bias, keep in (("silu", 0, 1), ("gelu", 1, 0), ("relu", 1, 1), ("sigmoid", 0, 0)):
        x, w, b = inputs(n + n_in, dt, n, n_in, n_out, bias)
        check_forward(dt, act, x, w, b, *forward(pkg, gpu, dt, act, x, w, b, keep))


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,n_in,n_out", [(1, 4096, 700), (4, 2048, 1001), (12, 1024, 600), (391, 785, 333), (300, 1024, 512), (600, 512, 1000),
                                          (1024, 256, 2112), (520, 1040, 2051)])
def test_forward_larger(pkg, gpu, dt, n, n_in, n_out):
    x, w, b = inputs(n, dt, n, n_in, n_out, n % 2)
    check_forward(dt, "silu", x, w, b, *forward(pkg, gpu, dt, "silu", x, w, b))


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n", [1, 3, 70])
def test_forward_values(pkg, gpu, dt, n):
    """What is no number stays in its sample or its output, also next to the end of a row that ends inside a piece; far values of
    the gate take their limits."""
    n_in, n_out = 37, 20
    x, w, _ = inputs(3, dt, n, n_in, n_out, 0)
    w[4, 36], w[n_out + 7, 0] = float("nan"), float("inf")
    y, h = forward(pkg, gpu, dt, "silu", x, w, None)
    good = [i for i in range(n_out) if i not in (4, 7)]
    assert torch.isnan(h[:, 4]).all() and not torch.isfinite(h[:, n_out + 7]).any() and torch.isfinite(h[:, good]).all()
    assert torch.isnan(y[:, 4]).all() and torch.isfinite(y[:, good]).all()
    # gates of +-1000 and 0
    x = torch.zeros(n, 3, dtype=tr.t_dtype(dt))
    x[:, 0], x[:, 1] = 1000, 1
    w = torch.zeros(6, 3, dtype=tr.t_dtype(dt))
    w[0, 0], w[1, 0] = 1, -1
    w[3:, 1] = 2
    for act, want in (("silu", (2000, 0, 0)), ("gelu", (2000, 0, 0)), ("sigmoid", (2, 0, 1)), ("relu", (2000, 0, 0))):
        y, _ = forward(pkg, gpu, dt, act, x, w, None)
        assert torch.equal(y.double().cpu(), torch.tensor([want], dtype=torch.float64).expand(n, 3)), act


def backward(pkg, gpu, dt, act, x, w, h, dy, bias, **more):
    n, n_in, n_out = x.shape[0], x.shape[1], w.shape[0] // 2
    X, W, H, DY = (tr.dev(t) for t in (x, w, h, dy))
    dx, dw, dh = torch.full_like(X, 7), torch.full_like(W, 7), H if more.pop("over", 0) else torch.full_like(H, 7)
    db = torch.full((2 * n_out,), 7, dtype=X.dtype, device="cuda") if bias else None
    a, keep = tr.gated_args(pkg, n_in, n_out, tr.ACTS[act], x=X, dx=dx, w=W, dw=dw, db=db, h=H, dh=dh, dy=DY, **more)
    pkg.call("ptl_gated_linear_%s_bw_batched" % dt, a, n)
    assert gpu.ptl_sync() == 0
    return dh, dx, dw, db


def check_backward(dt, act, x, w, h, dy, dh, dx, dw, db):
    n, n_out = x.shape[0], w.shape[0] // 2
    g, up, d = h[:, :n_out].double(), h[:, n_out:].double(), dy.double()
    f, df = tr.act64(g, act)
    ref = torch.cat([d * up * df, d * f], 1)
    # the slope is a sum of two terms: act / g (gate 1: its limit) and the rest
    first = torch.where(g != 0, f / g, torch.ones_like(g)).abs() if act in ("silu", "gelu") else torch.zeros_like(g)
    slope = U * (tr.act_steps(g, act) + 8) * (2 * first + df.abs())
    tol = torch.cat([(d * up).abs() * slope, (d * f).abs() * U * (tr.act_steps(g, act) + 2)], 1)
    tr.within(dh, ref, tol + tr.step(ref, dt), "dh")
    got = dh.double().cpu()  # what the products read
    off = torch.zeros_like(got)
    if dt == "fp16" and (n <= 2 or 2 * n * n_out < 16384):  # ... few of them: before they are rounded, in two halves of 11 bits; the second in steps of 2^-24 / 2048
        got, off = ref, tol + ref.abs() * 2.0 ** -22 + 2.0 ** -36
    x, w = x.double(), w.double()
    if dx is not None:
        ref = got @ w
        tr.within(dx, ref, U * (4 * n_out + 8) * (got.abs() @ w.abs()) + off @ w.abs() + tr.step(ref, dt), "dx")
    if dw is not None:
        ref = got.t() @ x
        tr.within(dw, ref, U * (2 * n + 8) * (got.abs().t() @ x.abs()) + off.t() @ x.abs() + tr.step(ref, dt), "dw")
    if db is not None:
        ref = got.sum(0)
        tr.within(db, ref, U * (n + 4) * got.abs().sum(0) + off.sum(0) + tr.step(ref, dt), "db")


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,n_in,n_out", SHAPES + [(391, 785, 333), (512, 1024, 704)])
def test_backward(pkg, gpu, dt, n, n_in, n_out):
    for act, bias in (("silu", 0), ("gelu", 1), ("relu", 0), ("sigmoid", 1)):
        x, w, _ = inputs(n, dt, n, n_in, n_out, 0)
        h, dy = tr.rand(n + 5, n, 2 * n_out, scale=1.5, dt=dt), tr.rand(n + 6, n, n_out, scale=0.5, dt=dt)
        check_backward(dt, act, x, w, h, dy, *backward(pkg, gpu, dt, act, x, w, h, dy, bias))


def test_backward_skips_and_in_place(pkg, gpu):
    n, n_in, n_out = 20, 50, 30
    x, w, _ = inputs(1, "fp32", n, n_in, n_out, 0)
    h, dy = tr.rand(5, n, 2 * n_out), tr.rand(6, n, n_out)
    full = backward(pkg, gpu, "fp32", "silu", x, w, h, dy, 1)
    dh, dx, dw, db = backward(pkg, gpu, "fp32", "silu", x, w, h, dy, 1, over=1)
    assert all(torch.equal(a, b) for a, b in zip(full, (dh, dx, dw, db)))
    dh, dx, dw, db = backward(pkg, gpu, "fp32", "silu", x, w, h, dy, 1, skip_wg=1)
    assert torch.equal(dh, full[0]) and (dw == 7).all() and (db == 7).all()
    check_backward("fp32", "silu", x, w, h, dy, dh, dx, None, None)
    dh, dx, dw, db = backward(pkg, gpu, "fp32", "silu", x, w, h, dy, 1, skip_ig=1)
    assert torch.equal(dh, full[0]) and (dx == 7).all()
    check_backward("fp32", "silu", x, w, h, dy, dh, None, dw, db)
    dh, dx, dw, db = backward(pkg, gpu, "fp32", "silu", x, w, h, dy, 1, skip_ig=1, skip_wg=1)
    assert torch.equal(dh, full[0]) and (dx == 7).all() and (dw == 7).all()


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
def test_backward_far_gates(pkg, gpu, act):
    """Gates far from 0, where the slope is 0 or 1 and squares overflow."""
    g = torch.tensor([-3e38, -1e20, -2e4, -90.0, -20.0, 0.0, 20.0, 90.0, 2e4, 1e20, 3e38])
    n_out = g.numel()
    h, dy = torch.cat([g, torch.ones(n_out)])[None], torch.full((1, n_out), 0.5)
    x, w = torch.ones(1, 2), torch.zeros(2 * n_out, 2)
    dh = backward(pkg, gpu, "fp32", act, x, w, h, dy, 0)[0].double().cpu()
    f, df = tr.act64(g.double(), act)
    df = torch.where(g.abs() >= 90, (g > 0).double() * (0 if act == "sigmoid" else 1), df)
    want = torch.cat([0.5 * df, 0.5 * f])[None]
    assert torch.allclose(dh, want, rtol=1e-5, atol=1e-7), (dh, want)


def test_gradients_against_differences(pkg, gpu):
    n, n_in, n_out, h = 2, 5, 4, 1e-5
    x, w, b = inputs(7, "fp32", n, n_in, n_out, 1)
    dy = tr.rand(8, n, n_out)
    for act in ("silu", "gelu", "sigmoid"):
        _, hidden = forward(pkg, gpu, "fp32", act, x, w, b)
        _, dx, dw, db = backward(pkg, gpu, "fp32", act, x, w, hidden.cpu(), dy, 1)

        def f(x_, w_, b_):
            p = x_ @ w_.t() + b_
            return (tr.act64(p[:, :n_out], act)[0] * p[:, n_out:] * dy.double()).sum()

        at = [x.double(), w.double(), b.double()]
        for k, got in enumerate((dx, dw, db)):
            for i in range(got.numel()):
                e = [torch.zeros_like(t) for t in at]
                e[k].view(-1)[i] = h
                up, down = (f(*(t + s * d for t, d in zip(at, e))) for s in (1, -1))
                assert abs((up - down) / (2 * h) - float(got.view(-1)[i])) < 1e-5


def test_host_arrays(pkg, gpu):
    n, n_in, n_out = 5, 33, 12
    x, w, b = inputs(9, "fp16", n, n_in, n_out, 1)
    dy = tr.rand(10, n, n_out, dt="fp16")
    y, h = forward(pkg, gpu, "fp16", "silu", x, w, b)
    z = lambda *s: torch.zeros(*s, dtype=torch.float16).numpy()  # noqa: E731
    hy, hh = z(n, n_out), z(n, 2 * n_out)
    a, keep = tr.gated_args(pkg, n_in, n_out, 1, x=x.numpy(), w=w.numpy(), b=b.numpy(), h=hh, y=hy)
    pkg.call("ptl_gated_linear_fp16_fw_batched", a, n)
    assert torch.equal(torch.from_numpy(hy), y.cpu()) and torch.equal(torch.from_numpy(hh), h.cpu())
    want = backward(pkg, gpu, "fp16", "silu", x, w, h.cpu(), dy, 1)
    dh, dx, dw, db = z(n, 2 * n_out), z(n, n_in), z(2 * n_out, n_in), z(2 * n_out)
    a, keep = tr.gated_args(pkg, n_in, n_out, 1, x=x.numpy(), dx=dx, w=w.numpy(), dw=dw, db=db, h=hh, dh=dh, dy=dy.numpy())
    pkg.call("ptl_gated_linear_fp16_bw_batched", a, n)
    for got, ref in zip((dh, dx, dw, db), want):
        assert torch.equal(torch.from_numpy(got), ref.cpu())


@pytest.mark.parametrize("dt,n,n_in,n_out,tile", [("fp16", 2, 1000, 300, 0), ("fp16", 3, 1000, 300, 32032), ("fp16", 40, 1024, 300, 32032), ("fp16", 40, 1025, 300, 32032),
                                                  ("fp16", 40, 1026, 300, 32032), ("fp16", 700, 512, 600, 64064), ("fp16", 700, 511, 600, 64064),
                                                  ("fp16", 700, 510, 600, 64064), ("fp16", 1500, 1024, 1100, 128128), ("fp16", 2100, 1025, 1500, 128128),
                                                  ("fp16", 2048, 1024, 2100, 256256), ("fp16", 2048, 1021, 2100, 256256), ("fp32", 4, 600, 300, 0),
                                                  ("fp32", 40, 1024, 100, 32032), ("fp32", 40, 1023, 1000, 32032), ("fp32", 900, 256, 900, 32064),
                                                  ("fp32", 900, 255, 900, 32064), ("fp32", 2000, 600, 900, 64128), ("fp32", 2001, 601, 901, 64128)])
def test_every_kernel(pkg, gpu, dt, n, n_in, n_out, tile):
    """Each kernel on sizes that it is chosen for, the ones that copy rows first among them (1021 and 1025 inputs)."""
    x, w, b = inputs(n, dt, n, n_in, n_out, 1)
    check_forward(dt, "gelu", x, w, b, *forward(pkg, gpu, dt, "gelu", x, w, b))
    assert gpu.ptl_last_gemm_tile() == tile


@pytest.mark.parametrize("n,n_in,n_out,bias", [(64, 2048, 800, 1), (70, 1032, 2500, 0), (1000, 256, 804, 1), (2056, 520, 260, 1), (520, 1024, 1024, 0),
                                               (1300, 384, 1000, 1), (2500, 136, 900, 0)])
def test_backward_own_products(pkg, gpu, n, n_in, n_out, bias):
    """Layers from 1.5 GFLOP on, whose products are made in one launch: in parts and not, ends of k and of rows inside a tile."""
    x, w, _ = inputs(n, "fp16", n, n_in, n_out, 0)
    h, dy = tr.rand(n + 5, n, 2 * n_out, scale=1.5, dt="fp16"), tr.rand(n + 6, n, n_out, scale=0.5, dt="fp16")
    full = backward(pkg, gpu, "fp16", "silu", x, w, h, dy, bias)
    check_backward("fp16", "silu", x, w, h, dy, *full)
    dh, dx, dw, db = backward(pkg, gpu, "fp16", "silu", x, w, h, dy, bias, skip_ig=1)
    check_backward("fp16", "silu", x, w, h, dy, dh, None, dw, db)
    assert (dx == 7).all()
    dh, dx, dw, db = backward(pkg, gpu, "fp16", "silu", x, w, h, dy, bias, skip_wg=1)
    check_backward("fp16", "silu", x, w, h, dy, dh, dx, None, None)
    assert (dw == 7).all() and (db is None or (db == 7).all())


def test_bias_gradients_are_sums_of_what_is_stored(pkg, gpu):
    """64 tokens, so that a single value rounded another way than it is stored shows in the sum."""
    n, n_in, n_out = 64, 2048, 1600
    x, w, _ = inputs(n, "fp16", n, n_in, n_out, 0)
    h, dy = tr.rand(n + 5, n, 2 * n_out, scale=1.5, dt="fp16"), tr.rand(n + 6, n, n_out, scale=0.5, dt="fp16")
    for act in ("silu", "gelu", "sigmoid", "relu"):
        check_backward("fp16", act, x, w, h, dy, *backward(pkg, gpu, "fp16", act, x, w, h, dy, 1))


@pytest.mark.parametrize("n,n_in,n_out,bias", [(500, 1100, 2050, 1), (701, 1001, 1003, 1), (3001, 83, 1701, 0), (64, 2045, 3001, 1), (9000, 130, 321, 1)])
def test_backward_own_products_of_odd_sizes(pkg, gpu, n, n_in, n_out, bias):
    """Layers from 3 GFLOP on whose rows are no whole 16-byte pieces: the operands as copies, each gradient alone, in place."""
    x, w, _ = inputs(n, "fp16", n, n_in, n_out, 0)
    h, dy = tr.rand(n + 5, n, 2 * n_out, scale=1.5, dt="fp16"), tr.rand(n + 6, n, n_out, scale=0.5, dt="fp16")
    full = backward(pkg, gpu, "fp16", "silu", x, w, h, dy, bias)
    check_backward("fp16", "silu", x, w, h, dy, *full)
    dh, dx, dw, db = backward(pkg, gpu, "fp16", "silu", x, w, h, dy, bias, over=1)
    assert all(a is None or torch.equal(a, b) for a, b in zip((dh, dx, dw, db), full))
    dh, dx, dw, _ = backward(pkg, gpu, "fp16", "silu", x, w, h, dy, bias, skip_wg=1)
    check_backward("fp16", "silu", x, w, h, dy, dh, dx, None, None)
    assert (dw == 7).all()
    dh, dx, dw, db = backward(pkg, gpu, "fp16", "silu", x, w, h, dy, bias, skip_ig=1)
    check_backward("fp16", "silu", x, w, h, dy, dh, None, dw, db)
    assert (dx == 7).all()


def test_backward_own_products_of_unaligned_tensors(pkg, gpu):
    """Whole pieces that do not start on 16 bytes; what lies behind the gradients stays as it is."""
    n, n_in, n_out = 600, 1024, 1024
    x, w, _ = inputs(n, "fp16", n, n_in, n_out, 0)
    h, dy = tr.rand(n + 5, n, 2 * n_out, scale=1.5, dt="fp16"), tr.rand(n + 6, n, n_out, scale=0.5, dt="fp16")

    def off(t, fill=None):
        b = torch.full((t.numel() + 2,), 7, dtype=torch.float16, device="cuda")
        if fill is None:
            b[1:-1] = t.flatten().cuda()
        return b, b[1:-1].view(t.shape)
    (_, X), (_, W), (_, H), (_, DY) = off(x), off(w), off(h), off(dy)
    (bx, dx), (bw, dw), (bh, dh) = off(x, 7), off(w, 7), off(h, 7)
    a, keep = tr.gated_args(pkg, n_in, n_out, 1, x=X, dx=dx, w=W, dw=dw, h=H, dh=dh, dy=DY)
    pkg.call("ptl_gated_linear_fp16_bw_batched", a, n)
    assert gpu.ptl_sync() == 0
    check_backward("fp16", "silu", x, w, h, dy, dh, dx, dw, None)
    assert all(b[0] == 7 and b[-1] == 7 for b in (bx, bw, bh))


@pytest.mark.parametrize("dt,n,n_in,n_out", [("fp32", 16, 3000, 1000), ("fp32", 70, 2001, 35), ("fp32", 500, 4096, 64), ("fp32", 8, 8193, 16), ("fp16", 20, 4097, 300),
                                             ("fp16", 64, 8192, 1024), ("fp16", 33, 8001, 70)])
def test_few_outputs_of_long_rows(pkg, gpu, dt, n, n_in, n_out):
    """k in parts of several workgroups each, with sums that another launch adds up; the same bits in every call."""
    x, w, b = inputs(n, dt, n, n_in, n_out, 1)
    y, h = forward(pkg, gpu, dt, "silu", x, w, b)
    check_forward(dt, "silu", x, w, b, y, h)
    again, none = forward(pkg, gpu, dt, "silu", x, w, b, keep=0)
    assert torch.equal(again, y) and none is None
    y, h = forward(pkg, gpu, dt, "gelu", x, w, None)
    check_forward(dt, "gelu", x, w, None, y, h)


@pytest.mark.parametrize("n,n_in,n_out,bias", [(16, 1600, 1600, 1), (33, 1601, 1601, 1), (153, 1134, 3135, 0), (1024, 640, 960, 1), (5000, 130, 999, 1), (6200, 64, 1700, 0),
                                               (511, 1027, 1190, 1)])
def test_backward_own_products_fp32(pkg, gpu, n, n_in, n_out, bias):
    """fp32 layers with large weights, or from 5 GFLOP on: in parts and not, as they are and as copies, each gradient alone, in place."""
    x, w, _ = inputs(n, "fp32", n, n_in, n_out, 0)
    h, dy = tr.rand(n + 5, n, 2 * n_out, scale=1.5), tr.rand(n + 6, n, n_out, scale=0.5)
    full = backward(pkg, gpu, "fp32", "silu", x, w, h, dy, bias)
    check_backward("fp32", "silu", x, w, h, dy, *full)
    over = backward(pkg, gpu, "fp32", "silu", x, w, h, dy, bias, over=1)
    assert all(a is None or torch.equal(a, b) for a, b in zip(over, full))
    dh, dx, dw, _ = backward(pkg, gpu, "fp32", "silu", x, w, h, dy, bias, skip_wg=1)
    check_backward("fp32", "silu", x, w, h, dy, dh, dx, None, None)
    assert (dw == 7).all()
    dh, dx, dw, db = backward(pkg, gpu, "fp32", "silu", x, w, h, dy, bias, skip_ig=1)
    check_backward("fp32", "silu", x, w, h, dy, dh, None, dw, db)
    assert (dx == 7).all()


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,n_in,n_out", [(1, 1, 1), (1, 3, 5), (1, 9, 700), (2, 2954, 67), (3, 64, 64), (4, 1001, 333), (5, 130, 257), (7, 515, 40), (8, 600, 1000),
                                          (1, 2000, 9000), (2, 4101, 2000), (12, 333, 600), (100, 77, 50)])
def test_backward_of_few_tokens(pkg, gpu, dt, n, n_in, n_out):
    """Layers whose whole backward pass is one kernel and its sums, and small ones in two halves: all parts, each gradient alone, in place."""
    x, w, _ = inputs(n, dt, n, n_in, n_out, 0)
    h, dy = tr.rand(n + 5, n, 2 * n_out, scale=1.5, dt=dt), tr.rand(n + 6, n, n_out, scale=0.5, dt=dt)
    for act in ("silu", "gelu", "sigmoid", "relu"):
        full = backward(pkg, gpu, dt, act, x, w, h, dy, 1)
        check_backward(dt, act, x, w, h, dy, *full)
    over = backward(pkg, gpu, dt, act, x, w, h, dy, 1, over=1)
    assert all(torch.equal(a, b) for a, b in zip(over, full))
    dh, dx, dw, _ = backward(pkg, gpu, dt, act, x, w, h, dy, 1, skip_wg=1)
    check_backward(dt, act, x, w, h, dy, dh, dx, None, None)
    assert (dw == 7).all()
    dh, dx, dw, db = backward(pkg, gpu, dt, act, x, w, h, dy, 1, skip_ig=1)
    check_backward(dt, act, x, w, h, dy, dh, None, dw, db)
    assert (dx == 7).all()


def test_backward_of_few_tokens_with_infinities(pkg, gpu):
    """A gradient beyond the largest half number is infinite in hidden->diff and in what depends on it, nowhere else."""
    for n in (1, 20):
        n_in, n_out = 40, 30
        x, w, _ = inputs(n, "fp16", n, n_in, n_out, 0)
        h, dy = torch.ones(n, 2 * n_out, dtype=torch.float16), torch.ones(n, n_out, dtype=torch.float16)
        h[0, n_out + 3], dy[0, 3] = 60000, 60000
        dh, dx, dw, db = backward(pkg, gpu, "fp16", "relu", x, w, h, dy, 1)
        assert torch.isinf(dh[0, 3]) and torch.isfinite(dh[0, :3]).all() and torch.isinf(db[3])
        assert not torch.isfinite(dw[3]).any() and torch.isfinite(dw[:3]).all() and not torch.isfinite(dx[0]).any()
        assert n == 1 or torch.isfinite(dx[1:]).all()


def test_backward_of_few_tokens_is_the_same_in_every_call(pkg, gpu):
    """The piece that ends a row is another workgroup's and shares values with the one before: they are the same values."""
    n, n_in, n_out = 2, 2561, 3000
    x, w, _ = inputs(n, "fp16", n, n_in, n_out, 0)
    h, dy = tr.rand(n + 5, n, 2 * n_out, scale=1.5, dt="fp16"), tr.rand(n + 6, n, n_out, scale=0.5, dt="fp16")
    X, W, H, DY = (tr.dev(t) for t in (x, w, h, dy))
    dx, dw, dh = torch.empty_like(X), torch.empty_like(W), torch.empty_like(H)
    a, keep = tr.gated_args(pkg, n_in, n_out, 1, x=X, dx=dx, w=W, dw=dw, h=H, dh=dh, dy=DY)
    first = None
    for _ in range(100):
        dw.fill_(7)
        pkg.call("ptl_gated_linear_fp16_bw_batched", a, n)
        assert gpu.ptl_sync() == 0
        first = first or [t.clone() for t in (dh, dx, dw)]
        assert all(torch.equal(p, q) for p, q in zip(first, (dh, dx, dw)))


LIMITS = {"silu": (float("inf"), 0.0), "gelu": (float("inf"), 0.0), "relu": (float("inf"), 0.0), "sigmoid": (1.0, 0.0)}  # at +inf, at -inf


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n", [1, 3, 70, 700])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
def test_infinite_gates(pkg, gpu, dt, n, act):
    """A gate of +-inf (of a bias, forward; as an overflow of fp16 is kept, backward) takes the activation's limit and the slope's, and
    a NaN stays one."""
    n_in, n_out = 33, 40
    x, w, b = inputs(5, dt, n, n_in, n_out, 1)
    b[3], b[4], b[5] = float("inf"), -float("inf"), float("nan")
    y, h = forward(pkg, gpu, dt, act, x, w, b)
    up = (x.double() @ w.double().t() + b.double())[:, n_out:]
    high, low = LIMITS[act]
    got = y.double().cpu()
    if high == 1:
        off = U * (n_in + 2) * (x.double().abs() @ w.double().abs().t() + b.double().abs())[:, n_out + 3] + tr.step(up[:, 3], dt) + 4 * U * up[:, 3].abs()
        tr.within(got[:, 3], up[:, 3], off)
    else:
        assert torch.equal(got[:, 3], torch.sign(up[:, 3]) * high)
    assert (got[:, 4] == low).all() and torch.isnan(got[:, 5]).all() and torch.isfinite(torch.cat([got[:, :3], got[:, 6:]], 1)).all()
    dy = tr.rand(6, n, n_out, scale=0.5, dt=dt)
    hidden = h.cpu()
    dh = backward(pkg, gpu, dt, act, x, w, hidden, dy, 1)[0].double().cpu()
    d, u = dy.double(), hidden[:, n_out:].double()
    slope = 0.0 if act == "sigmoid" else 1.0
    want = d[:, 3] * u[:, 3] * slope
    tr.within(dh[:, 3], want, tr.step(want, dt) + 4 * U * want.abs())
    assert (dh[:, 4] == 0).all()
    if high == 1:
        tr.within(dh[:, n_out + 3], d[:, 3], tr.step(d[:, 3], dt) + 4 * U * d[:, 3].abs())
    else:
        assert torch.equal(dh[:, n_out + 3], torch.sign(d[:, 3]) * high)
    assert (dh[:, n_out + 4] == 0).all() and torch.isnan(dh[:, [5, n_out + 5]]).all()


@pytest.mark.parametrize("dt,n,n_in,n_out,path", [("fp32", 1000, 512, 1000, 0), ("fp16", 2000, 512, 1000, 1), ("fp32", 1001, 513, 999, 1)])
def test_backward_in_place_with_gradients_of_their_own(pkg, gpu, dt, n, n_in, n_out, path):
    """Layers whose gradients are a dense layer's call that could ask for more than 64 MB: it reads the pre-activations' gradients from a
    place of their own, and they take the pre-activations' place behind it.  Tensors of the device and of the host, each gradient alone."""
    x, w, _ = inputs(n, dt, n, n_in, n_out, 0)
    h, dy = tr.rand(n + 5, n, 2 * n_out, scale=1.5, dt=dt), tr.rand(n + 6, n, n_out, scale=0.5, dt=dt)
    gpu.ptl_set_gemm_path(path)
    try:
        for more in ({}, {"skip_wg": 1}, {"skip_ig": 1}):
            full = backward(pkg, gpu, dt, "silu", x, w, h, dy, 1, **more)
            over = backward(pkg, gpu, dt, "silu", x, w, h, dy, 1, over=1, **more)
            assert all(torch.equal(a, b) for a, b in zip(over, full)), more
        want = backward(pkg, gpu, dt, "silu", x, w, h, dy, 1)
        z = lambda *s: torch.full(s, 7, dtype=x.dtype).numpy()  # noqa: E731
        dx, dw, db, hh = z(n, n_in), z(2 * n_out, n_in), z(2 * n_out), h.numpy().copy()
        a, keep = tr.gated_args(pkg, n_in, n_out, 1, x=x.numpy(), dx=dx, w=w.numpy(), dw=dw, db=db, h=hh, dh=hh, dy=dy.numpy())
        pkg.call("ptl_gated_linear_%s_bw_batched" % dt, a, n)
        for got, ref in zip((hh, dx, dw, db), want):
            assert torch.equal(torch.from_numpy(got), ref.cpu())
    finally:
        gpu.ptl_set_gemm_path(0)
