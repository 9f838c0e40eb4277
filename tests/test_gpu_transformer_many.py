"""More rows than one launch takes (2^25 by the wave), and products of more outputs than one call forms."""
import ctypes

import pytest
import torch

import transformer as tr

pytestmark = pytest.mark.gpu
N = 2 ** 25 + 5


def test_norm(pkg, gpu):
    """Rows of two values: y = s w / sqrt(mean s^2 + eps), against float64 on the device."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = torch.randn(N, 2, dtype=torch.float16, device="cuda", generator=g), torch.tensor([1.5, -0.75], dtype=torch.float16, device="cuda")
    y, dx = torch.full_like(x, 7), torch.full_like(x, 7)
    a, keep = tr.norm_args(pkg, 2, x=x, w=w, y=y, eps=1e-5)
    pkg.call("ptl_rms_norm_fp16_fw_batched", a, N)
    assert gpu.ptl_sync() == 0
    for part in (slice(0, 100000), slice(N - 100000, N)):
        s = x[part].double()
        ref = s * w.double() / torch.sqrt((s * s).mean(1, keepdim=True) + 1e-5)
        tr.within(y[part], ref.cpu(), tr.step(ref.cpu(), "fp16") + ref.cpu().abs() * 16 * tr.U)
    # the way back, on which workgroups walk over the rows: a thousandth of the bytes would show rows left out
    a, keep = tr.norm_args(pkg, 2, x=x, dx=dx, w=w, dy=y, skip_wg=1, eps=1e-5)
    pkg.call("ptl_rms_norm_fp16_bw_batched", a, N)
    assert gpu.ptl_sync() == 0 and int((dx == 7).all(1).sum()) == 0


def test_distillation(pkg, gpu):
    """Two classes, one of them named: loss = -log q, gradient q - p."""
    g = torch.Generator(device="cuda").manual_seed(2)
    z = torch.randn(N, 2, dtype=torch.float16, device="cuda", generator=g)
    grad, loss = torch.full_like(z, 7), torch.full((N,), 7.0, device="cuda")
    a, keep = tr.distill_args(pkg, z, grad, torch.zeros(N, 1, dtype=torch.float16, device="cuda"), torch.ones(N, 1, dtype=torch.int32, device="cuda"),
                              loss, 1.0, 1.0)
    assert gpu.ptl_distill_fp16_batched(ctypes.byref(a), N, 2) == 0 and gpu.ptl_sync() == 0
    for part in (slice(0, 100000), slice(N - 100000, N)):
        lq = torch.log_softmax(z[part].double().cpu(), 1)
        tr.within(loss[part], -lq[:, 1], tr.U * 64 * (1 + lq[:, 1].abs() + z[part].abs().amax(1).double().cpu()))
        ref = lq.exp() - torch.tensor([0.0, 1.0], dtype=torch.float64)
        tr.within(grad[part], ref, tr.step(ref, "fp16") + 64 * tr.U)
    assert int((loss == 7).sum()) == 0


def test_more_outputs_than_a_call_forms(pkg, gpu):
    n = 2 ** 30
    A, B = torch.ones(n, 1, dtype=torch.int8, device="cuda"), torch.ones(1, 1, dtype=torch.int8, device="cuda")
    C = torch.full((n, 1), 7, dtype=torch.float16, device="cuda")
    a, keep = tr.int8_args(pkg, A, B, C)
    assert gpu.ptl_mm_int8_fp16(ctypes.byref(a)) == 1 and "more outputs" in gpu.ptl_last_error().decode()
    assert gpu.ptl_sync() == 0 and bool((C == 7).all())
    a.N = 2 ** 24 + 3
    assert gpu.ptl_mm_int8_fp16(ctypes.byref(a)) == 0 and gpu.ptl_sync() == 0
    assert bool((C[:a.N] == 1).all()) and bool((C[a.N:] == 7).all())


def test_norm_backward(pkg, gpu):
    """The gradients of all rows, of two values each, and the weights' gradient, a sum over all rows, against the sum in 64 bits (formed on the device, in parts)."""
    g = torch.Generator(device="cuda").manual_seed(3)
    for dt in ("fp16", "fp32"):
        t = tr.t_dtype(dt)
        s, dy = (torch.randn(N, 2, dtype=t, device="cuda", generator=g) for _ in range(2))
        dy = (s + dy * 0.3) * 5e-4  # (so that the weights' gradient is as large as its terms' sum, and no infinity in fp16)
        w = torch.tensor([1.5, -0.75], dtype=t, device="cuda")
        dx, dw = torch.full_like(s, 7), torch.full_like(w, 7)
        a, keep = tr.norm_args(pkg, 2, x=s, dx=dx, w=w, dw=dw, dy=dy, eps=1e-5)
        pkg.call("ptl_rms_norm_%s_bw_batched" % dt, a, N)
        assert gpu.ptl_sync() == 0
        total, size, off = torch.zeros(2, dtype=torch.float64), torch.zeros(2, dtype=torch.float64), 0.0
        for at in range(0, N, 1 << 22):
            part = slice(at, min(at + (1 << 22), N))
            x, d = s[part].double(), dy[part].double()
            r = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-5)
            v = d * x * r
            total += v.sum(0).cpu()
            size += v.abs().sum(0).cpu()
            h = d * w.double()
            ref = r * (h - x * r * r * (h * x).mean(1, keepdim=True))
            # sums of two terms and a dozen roundings of either term, and the result's own
            tol = 32 * tr.U * ((r * h).abs() + (x * r).abs() * r * (h * x * r).abs().mean(1, keepdim=True)) + (ref.abs() * 2.0 ** -11 + 2.0 ** -25 if dt == "fp16" else 0)
            off = max(off, float(((dx[part].double() - ref).abs() - tol).max()))
        assert off <= 0, dt
        # a wave's chain: N rows over the waves of at most sqrt(72 N sizeof) workgroups of four; fp16: the workgroups' sums in 32 chains
        groups = int((72.0 * N * s.element_size()) ** 0.5)
        c = N / (4 * groups) + 16 + (groups / 32 + 32 if dt == "fp16" else 0)
        tr.within(dw, total, size * tr.U * c + tr.step(total, dt), "dw " + dt)
