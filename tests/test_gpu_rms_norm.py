"""RMS norm behind a residual against its formula in 64 bits.  u = 2^-24.  A sum of n positive terms that is formed in chains of at
most c additions is at most c u of itself off; a row's sums are formed in chains of 8 values a piece, up to 8 pieces a thread (long
rows: dim / 1024 a thread), 6 folds of a wave and 15 of its workgroup."""
import ctypes

import pytest
import torch

import transformer as tr

pytestmark = pytest.mark.gpu
U = tr.U
EPS = 1e-5


def chain(dim):
    return 64 + 21 + dim / 1024


def forward(pkg, gpu, dt, x, skip, w, y=True, q=True, eps=EPS, keep_sum=None, keep_y=None):
    n, dim = x.shape
    X, S, W = tr.dev(x), None if skip is None else tr.dev(skip), tr.dev(w)
    Y = keep_y if keep_y is not None else torch.full_like(X, 7) if y else None
    T = None if skip is None else keep_sum if keep_sum is not None else torch.full_like(X, 7)
    Q = torch.full((n, dim), 77, dtype=torch.int8, device="cuda") if q else None
    C = torch.full((n,), 7.0, device="cuda") if q else None
    a, keep = tr.norm_args(pkg, dim, x=X, skip=S, total=T, w=W, y=Y, q=Q, scale=C, eps=eps)
    pkg.call("ptl_rms_norm_%s_fw_batched" % dt, a, n)
    assert gpu.ptl_sync() == 0
    return T, Y, Q, C


def check_forward(dt, x, skip, w, T, Y, Q, C, eps=EPS):
    dim = x.shape[1]
    s = x.double() if skip is None else x.double() + skip.double()
    ref = tr.norm64(s, w.double(), eps)
    if T is not None:
        tr.within(T, s, tr.step(s, dt) + s.abs() * 2 * U)
    if Y is not None:  # s and three products round, the root and the quotient, half of the sum's error
        tr.within(Y, ref, tr.step(ref, dt) + ref.abs() * U * (chain(dim) / 2 + 8))
    if Q is not None:
        amax = ref.abs().amax(1)
        tr.within(C, amax / 127, amax / 127 * U * (chain(dim) / 2 + 10) + 2.0 ** -149)
        unit = torch.where(amax > 0, 127 / amax, torch.zeros_like(amax))[:, None]
        off = (Q.cpu().double() - ref * unit).abs()
        assert float(off.max()) <= 0.5 + 127 * 6 * U  # a value within its own rounding of a border may fall on either side


DIMS = [1, 3, 4, 7, 8, 9, 63, 64, 257, 512, 785, 1000, 1024, 2056, 4095, 4096, 4100, 8200, 16384]


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("dim", DIMS)
def test_forward(pkg, gpu, dt, dim):
    for n, residual in ((1, 1), (5, 0), (67, 1)):
        x, w = tr.rand(dim + n, n, dim, scale=2.0, dt=dt), 1 + tr.rand(dim, dim, scale=0.2, dt=dt)
        skip = tr.rand(dim + 1, n, dim, dt=dt) if residual else None
        check_forward(dt, x, skip, w, *forward(pkg, gpu, dt, x, skip, w))


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,dim", [(1500, 64), (1030, 500), (1100, 1001), (1025, 4096), (3, 33000), (2, 70001)])
def test_forward_many_rows_and_long_rows(pkg, gpu, dt, n, dim):
    x, w, skip = tr.rand(dim, n, dim, dt=dt), 1 + tr.rand(dim + 1, dim, scale=0.2, dt=dt), tr.rand(dim + 2, n, dim, dt=dt)
    check_forward(dt, x, skip, w, *forward(pkg, gpu, dt, x, skip, w))
    # one output alone, without a residual
    check_forward(dt, x, None, w, *forward(pkg, gpu, dt, x, None, w, y=False))
    check_forward(dt, x, None, w, *forward(pkg, gpu, dt, x, None, w, q=False))


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_forward_values(pkg, gpu, dt):
    """A row of zeros (with and without eps), infinities, NaN, tiny and large values; rows around them are not touched."""
    dim = 100
    x, w = tr.rand(1, 8, dim, dt=dt), 1 + tr.rand(2, dim, scale=0.2, dt=dt)
    x[1] = 0
    x[2, 5], x[3, 7], x[4, 99] = float("inf"), float("nan"), -float("inf")
    x[5] *= 1e-4
    x[6] *= 3e3
    T, Y, Q, C = forward(pkg, gpu, dt, x, None, w)
    good = [0, 1, 5, 6, 7]
    check_forward(dt, x[good], None, w, None, Y[good], Q[good], C[good])
    assert not torch.isfinite(C[[2, 3, 4]]).any()
    assert torch.isnan(Y[3]).all() and torch.isnan(Y[2, 5]) and torch.isnan(Y[4, 99])
    assert (Y[1] == 0).all() and (Q[1] == 0).all() and C[1] == 0


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_forward_in_place(pkg, gpu, dt):
    for n, dim in ((3, 77), (2, 4096), (1100, 200)):
        x, w, skip = tr.rand(3, n, dim, dt=dt), 1 + tr.rand(4, dim, scale=0.2, dt=dt), tr.rand(5, n, dim, dt=dt)
        T, Y, _, _ = forward(pkg, gpu, dt, x, skip, w, q=False)
        X, S, W = tr.dev(x), tr.dev(skip), tr.dev(w)
        a, keep = tr.norm_args(pkg, dim, x=X, skip=S, total=S, w=W, y=X)
        pkg.call("ptl_rms_norm_%s_fw_batched" % dt, a, n)
        assert torch.equal(S, T) and torch.equal(X, Y)


def backward(pkg, gpu, dt, s, dy, add, w, residual, name="bw", **skips):
    n, dim = s.shape
    S, DY, W = tr.dev(s), tr.dev(dy), tr.dev(w)
    A = None if add is None else tr.dev(add)
    DX, DW = torch.full_like(S, 7), torch.full_like(W, 7)
    DK = torch.full_like(S, 7) if residual else None
    a, keep = tr.norm_args(pkg, dim, x=None if residual else S, dx=DX, dskip=DK, total=S if residual else None, dtotal=A, w=W, dw=DW,
                           dy=DY, **skips)
    pkg.call("ptl_rms_norm_%s_bw_batched" % dt, a, n)
    assert gpu.ptl_sync() == 0
    return DX, DK, DW


def check_backward(dt, s, dy, add, w, DX, DK, DW):
    n, dim = s.shape
    s, dy, w = s.double(), dy.double(), w.double()
    r = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + EPS)
    g = dy * w
    m = r ** 3 * (g * s).mean(1, keepdim=True)
    ref = r * g - m * s + (0 if add is None else add.double())
    # each term as far off as its sums and a dozen roundings may take it; signs differ within the second sum
    c = U * (chain(dim) + 16)
    tol = c * ((r * g).abs() + r ** 3 * (g * s).abs().mean(1, keepdim=True) * s.abs()) + 2 * U * ref.abs()
    if add is not None:
        tol = tol + 2 * U * add.double().abs()
    if DX is not None:
        tr.within(DX, ref, tol + tr.step(ref, dt), "dx")
    if DK is not None:
        assert torch.equal(DK, DX)
    if DW is not None:
        t = dy * s * r
        tr.within(DW, t.sum(0), t.abs().sum(0) * U * (chain(dim) / 2 + 8 + n) + tr.step(t.sum(0), dt), "dw")


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("dim", DIMS)
def test_backward(pkg, gpu, dt, dim):
    for n, residual in ((1, 1), (7, 0), (67, 1)):
        s, dy, w = tr.rand(dim + n, n, dim, dt=dt), tr.rand(dim + 1, n, dim, scale=0.5, dt=dt), 1 + tr.rand(dim, dim, scale=0.2, dt=dt)
        add = tr.rand(dim + 2, n, dim, dt=dt) if residual else None
        check_backward(dt, s, dy, add, w, *backward(pkg, gpu, dt, s, dy, add, w, residual))


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,dim", [(5000, 64), (4099, 100), (1100, 1001), (2050, 1024), (3, 20001), (70, 17000), (2, 33001)])
def test_backward_many_rows_and_long_rows(pkg, gpu, dt, n, dim):
    s, dy, w, add = (tr.rand(dim, n, dim, dt=dt), tr.rand(dim + 1, n, dim, scale=0.5, dt=dt), 1 + tr.rand(dim, dim, scale=0.2, dt=dt),
                     tr.rand(dim + 2, n, dim, dt=dt))
    check_backward(dt, s, dy, add, w, *backward(pkg, gpu, dt, s, dy, add, w, 1))


def test_backward_skips_and_shared_buffers(pkg, gpu):
    for n, dim in ((9, 77), (300, 512), (2, 17000)):
        s, dy, w, add = tr.rand(1, n, dim), tr.rand(2, n, dim), 1 + tr.rand(3, dim, scale=0.2), tr.rand(4, n, dim)
        DX, DK, DW = backward(pkg, gpu, "fp32", s, dy, add, w, 1)
        a, _, b = backward(pkg, gpu, "fp32", s, dy, add, w, 1, skip_wg=1)
        assert torch.equal(a, DX) and (b == 7).all()
        a, c, b = backward(pkg, gpu, "fp32", s, dy, add, w, 1, skip_ig=1)
        assert (a == 7).all() and (c == 7).all() and torch.equal(b, DW)
        for which in ("dy", "add", "s", "both"):  # the gradient in the place of a tensor that is read
            S, DY, W, A = tr.dev(s), tr.dev(dy), tr.dev(w), tr.dev(add)
            out = {"dy": DY, "add": A, "s": S, "both": torch.empty_like(S)}[which]
            dw = torch.empty_like(W)
            a, keep = tr.norm_args(pkg, dim, dx=out, dskip=out, total=S, dtotal=A, w=W, dw=dw, dy=DY)
            pkg.call("ptl_rms_norm_fp32_bw_batched", a, n)
            assert torch.equal(out, DX) and torch.equal(dw, DW), which


def test_backward_against_differences(pkg, gpu):
    """The gradient against central differences of the forward formula in 64 bits, whose own error is of the order of h^2."""
    n, dim, h = 3, 24, 1e-4
    s, dy, w = tr.rand(1, n, dim), tr.rand(2, n, dim), 1 + tr.rand(3, dim, scale=0.2)
    DX, _, DW = backward(pkg, gpu, "fp32", s, dy, None, w, 0)

    def f(s_, w_):
        return (tr.norm64(s_, w_, EPS) * dy.double()).sum()

    s64, w64 = s.double(), w.double()
    for i in range(n):
        for j in range(dim):
            e = torch.zeros_like(s64)
            e[i, j] = h
            assert abs((f(s64 + e, w64) - f(s64 - e, w64)) / (2 * h) - float(DX[i, j])) < 1e-5
    for j in range(dim):
        e = torch.zeros_like(w64)
        e[j] = h
        assert abs((f(s64, w64 + e) - f(s64, w64 - e)) / (2 * h) - float(DW[j])) < 1e-5


def test_host_arrays(pkg, gpu):
    n, dim = 6, 50
    x, w, skip, dy = tr.rand(1, n, dim, dt="fp16"), 1 + tr.rand(2, dim, dt="fp16"), tr.rand(3, n, dim, dt="fp16"), tr.rand(4, n, dim, dt="fp16")
    want = forward(pkg, gpu, "fp16", x, skip, w)
    total, y, q, scale = torch.zeros(n, dim, dtype=torch.float16).numpy(), torch.zeros(n, dim, dtype=torch.float16).numpy(), \
        torch.zeros(n, dim, dtype=torch.int8).numpy(), torch.zeros(n).numpy()
    a, keep = tr.norm_args(pkg, dim, x=x.numpy(), skip=skip.numpy(), total=total, w=w.numpy(), y=y, q=q, scale=scale)
    pkg.call("ptl_rms_norm_fp16_fw_batched", a, n)
    for got, ref in zip((total, y, q, scale), want):
        assert torch.equal(torch.from_numpy(got), ref.cpu())
    dx, _, dw = backward(pkg, gpu, "fp16", x, dy, None, w, 0)
    hx, hw = y.copy(), w.numpy().copy()
    a, keep = tr.norm_args(pkg, dim, x=x.numpy(), dx=hx, w=w.numpy(), dw=hw, dy=dy.numpy())
    pkg.call("ptl_rms_norm_fp16_bw_batched", a, n)
    assert torch.equal(torch.from_numpy(hx), dx.cpu()) and torch.equal(torch.from_numpy(hw), dw.cpu())


def test_unaligned_tensors(pkg, gpu):
    """Tensors that start one element behind a 16-byte border."""
    n, dim = 5, 260
    for dt in ("fp32", "fp16"):
        def off(t):
            b = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
            b[1:] = t.flatten().cuda()
            return b[1:].view(t.shape)
        x, w, skip = tr.rand(1, n, dim, dt=dt), 1 + tr.rand(2, dim, scale=0.2, dt=dt), tr.rand(3, n, dim, dt=dt)
        X, W, S, T, Y = off(x), off(w), off(skip), off(x * 0 + 7), off(x * 0 + 7)
        Q = torch.zeros(n * dim + 1, dtype=torch.int8, device="cuda")[1:].view(n, dim)
        C = torch.zeros(n, device="cuda")
        a, keep = tr.norm_args(pkg, dim, x=X, skip=S, total=T, w=W, y=Y, q=Q, scale=C)
        pkg.call("ptl_rms_norm_%s_fw_batched" % dt, a, n)
        for got, ref in zip((T, Y, Q, C), forward(pkg, gpu, dt, x, skip, w)):
            assert torch.equal(got, ref)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,dim", [(2, 130), (3, 1001), (13, 515), (2, 2051), (4, 4099), (300, 9001), (5, 10001), (3, 12291), (1, 16383)])
def test_rows_that_end_inside_a_piece(pkg, gpu, dt, n, dim):
    """Up to a few rows (one workgroup has the weights' gradient) and many, forward and backward, also in the place of what is read."""
    x, w, skip = tr.rand(dim, n, dim, dt=dt), 1 + tr.rand(dim + 1, dim, scale=0.2, dt=dt), tr.rand(dim + 2, n, dim, dt=dt)
    T, Y, Q, C = forward(pkg, gpu, dt, x, skip, w)
    check_forward(dt, x, skip, w, T, Y, Q, C)
    X, S, W = tr.dev(x), tr.dev(skip), tr.dev(w)
    a, keep = tr.norm_args(pkg, dim, x=X, skip=S, total=S, w=W, y=X)
    pkg.call("ptl_rms_norm_%s_fw_batched" % dt, a, n)
    assert torch.equal(S, T) and torch.equal(X, Y)
    dy = tr.rand(dim + 3, n, dim, scale=0.5, dt=dt)
    DX, DK, DW = backward(pkg, gpu, dt, x, dy, skip, w, 1)
    check_backward(dt, x, dy, skip, w, DX, DK, DW)
    for which in ("dy", "add", "s"):
        S, DY, A = tr.dev(x), tr.dev(dy), tr.dev(skip)
        out, dw = {"dy": DY, "add": A, "s": S}[which], torch.empty_like(W)
        a, keep = tr.norm_args(pkg, dim, dx=out, dskip=out, total=S, dtotal=A, w=W, dw=dw, dy=DY)
        pkg.call("ptl_rms_norm_%s_bw_batched" % dt, a, n)
        assert torch.equal(out, DX) and torch.equal(dw, DW), which
    # without the gradient along the residual, rows around the batch as they were
    big = torch.full((n + 2, dim), 7.0, dtype=W.dtype, device="cuda")
    a, keep = tr.norm_args(pkg, dim, x=tr.dev(x), dx=big[1:n + 1], w=W, dw=torch.empty_like(W), dy=tr.dev(dy))
    pkg.call("ptl_rms_norm_%s_bw_batched" % dt, a, n)
    check_backward(dt, x, dy, None, w, big[1:n + 1], None, None)
    assert (big[0] == 7).all() and (big[n + 1] == 7).all()


# rows of a wave, of a workgroup with one and several pieces a thread, and rows that are walked
VARIANTS = [5, 100, 1001, 4096, 9001, 40001]


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("dim", VARIANTS)
def test_no_numbers_among_the_weights_in_8_bits(pkg, gpu, dt, dim):
    """NaN or an infinity in coeff, also one that meets a 0: every row has a value that is no finite number, and so is its scale."""
    x = tr.rand(1, 6, dim, dt=dt)
    x[3, dim // 2] = 0
    for bad in ("nan", "inf", "-inf"):
        w = 1 + tr.rand(2, dim, scale=0.2, dt=dt)
        w[dim // 2] = float(bad)
        _, Y, _, C = forward(pkg, gpu, dt, x, None, w)
        assert not torch.isfinite(Y[:, dim // 2]).any() and not torch.isfinite(C).any(), bad
        assert torch.isfinite(torch.cat([Y[:, : dim // 2], Y[:, dim // 2 + 1:]], 1)).all()


@pytest.mark.parametrize("dim", VARIANTS)
def test_tiny_rows_in_8_bits(pkg, gpu, dim):
    """Rows whose largest |s w| is at the end of fp32's range: zeros stay zeros and the largest value becomes 127.  A value that is no
    normal number is off by up to 2^-150, which is 127 * 2^-150 / max|y| of the unit."""
    x, w = tr.rand(1, 5, dim).double(), 1 + tr.rand(2, dim, scale=0.2)
    x[:, ::3] = 0
    x = (x * torch.tensor([1.0, 1e-36, 2e-38, 1e-40, 1e-42], dtype=torch.float64)[:, None]).float()
    _, _, Q, C = forward(pkg, gpu, "fp32", x, None, w, y=False)
    v = x.double() * w.double()
    ref = tr.norm64(x.double(), w.double(), EPS)
    amax = v.abs().amax(1, keepdim=True)
    off = (Q.cpu().double() - v * 127 / amax).abs()
    assert (off <= 0.5 + 127 * (6 * U + 2.0 ** -149 / amax)).all()
    assert (Q.cpu()[x == 0] == 0).all() and (Q.abs().amax(1) == 127).all()
    amax = ref.abs().amax(1)
    tr.within(C, amax / 127, amax / 127 * U * (chain(dim) / 2 + 10) + 2.0 ** -148 * (1 + amax / v.abs().amax(1)))


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("dim", VARIANTS)
def test_rows_of_zeros_without_eps(pkg, gpu, dt, dim):
    """eps = 0: a row of zeros has zeros, the scale 0 and no gradient but the one along the residual; the other rows are as always."""
    x, w = tr.rand(1, 4, dim, dt=dt), 1 + tr.rand(2, dim, scale=0.2, dt=dt)
    x[1] = 0
    _, Y, Q, C = forward(pkg, gpu, dt, x, None, w, eps=0.0)
    assert (Y[1] == 0).all() and (Q[1] == 0).all() and C[1] == 0
    check_forward(dt, x[[0, 2, 3]], None, w, None, Y[[0, 2, 3]], Q[[0, 2, 3]], C[[0, 2, 3]], eps=0.0)
    dy, add = tr.rand(3, 4, dim, scale=0.5, dt=dt), tr.rand(4, 4, dim, dt=dt)
    DX, _, DW = backward(pkg, gpu, dt, x, dy, add, w, 1, eps=0.0)
    assert torch.equal(DX[1].cpu(), add[1])
    rest = [0, 2, 3]
    A, _, B = backward(pkg, gpu, dt, x[rest], dy[rest], add[rest], w, 1, eps=0.0)
    assert torch.equal(DX[rest], A)
    t = (dy.double() * x.double() / torch.sqrt((x.double() ** 2).mean(1, keepdim=True)))[rest]
    tr.within(DW, t.sum(0), t.abs().sum(0) * U * (chain(dim) / 2 + 12) + tr.step(t.sum(0), dt), "dw")


@pytest.mark.parametrize("dim", VARIANTS)
def test_backward_of_very_small_and_very_large_rows(pkg, gpu, dim):
    """Gradients of the size of 1 / rms, which fp32 holds where (1 / rms)^3 is infinite or subnormal."""
    n = 5
    for size, eps in ((1e14, EPS), (3e14, EPS), (1e-14, 0.0), (1e-16, 0.0)):
        s = (tr.rand(1, n, dim).double() * size).float()
        dy, w = tr.rand(2, n, dim, scale=0.5), 1 + tr.rand(3, dim, scale=0.2)
        DX, _, DW = backward(pkg, gpu, "fp32", s, dy, None, w, 0, eps=eps)
        s64, g = s.double(), dy.double() * w.double()
        r = 1 / torch.sqrt((s64 * s64).mean(1, keepdim=True) + eps)
        ref = r * (g - s64 * r * r * (g * s64).mean(1, keepdim=True))
        c = U * (chain(dim) + 16)
        tol = c * ((r * g).abs() + r ** 3 * (g * s64).abs().mean(1, keepdim=True) * s64.abs()) + 2 * U * ref.abs() + 2.0 ** -149
        tr.within(DX, ref, tol, "dx of rows of %g" % size)
        t = dy.double() * s64 * r
        tr.within(DW, t.sum(0), t.abs().sum(0) * U * (chain(dim) / 2 + 8 + n), "dw")
