"""Products of 8-bit integers with scales against exact integers and 64 bits.  The sum is exact; it takes one rounding to fp32, one
with each scale, one with the bias and one to the tensor type."""
import ctypes

import pytest
import torch

import transformer as tr

pytestmark = pytest.mark.gpu
U = tr.U


def ints(seed, *shape, most=127):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g).to(torch.int8)


def check(pkg, gpu, dt, A, B, sa, sb, bias, place=lambda t: t.cuda()):
    n, m = A.shape[0], B.shape[0]
    C = torch.full((n + 1, m), 7, dtype=tr.t_dtype(dt), device="cuda")
    a, keep = tr.int8_args(pkg, place(A), place(B), C, *(None if t is None else t.cuda() for t in (sa, sb, bias)))
    assert getattr(gpu, "ptl_mm_int8_" + dt)(ctypes.byref(a)) == 0, gpu.ptl_last_error()
    assert gpu.ptl_sync() == 0
    ref = A.double() @ B.double().t()
    if sa is not None:
        ref = ref * sa.double()[:, None]
    if sb is not None:
        ref = ref * sb.double()
    tol = ref.abs() * 4 * U
    if bias is not None:
        ref = ref + bias.double()
    tr.within(C[:n], ref, tol + ref.abs() * 2 * U + tr.step(ref, dt))
    assert (C[n] == 7).all()
    return C[:n]


SHAPES = [(1, 1, 1), (1, 3, 15), (1, 65, 16), (2, 17, 17), (3, 100, 33), (4, 33, 127), (5, 64, 128), (8, 200, 129), (9, 31, 785), (17, 40, 300),
          (33, 32, 64), (64, 129, 1000), (65, 65, 65), (130, 257, 192), (257, 130, 144)]


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,m,k", SHAPES)
def test_product(pkg, gpu, dt, n, m, k):
    A, B = ints(n + k, n, k), ints(m + k, m, k)
    sa, sb = tr.rand(1, n).abs() * 0.01 + 0.001, tr.rand(2, m).abs() * 0.02 + 0.001
    check(pkg, gpu, dt, A, B, sa, sb, tr.rand(3, m, dt=dt))
    check(pkg, gpu, dt, A, B, sa * 0.1, None, None)
    check(pkg, gpu, dt, A, B, None, sb * 0.1, None)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,m,k", [(1, 4096, 4096), (2, 1000, 8192), (7, 512, 2000), (12, 700, 1024), (300, 600, 512), (520, 1030, 1040),
                                   (1024, 2048, 256), (391, 333, 785), (1030, 2050, 100)])
def test_larger_products(pkg, gpu, dt, n, m, k):
    A, B = ints(n, n, k), ints(m, m, k)
    sa, sb = tr.rand(1, n).abs() * 0.001 + 0.0001, tr.rand(2, m).abs() * 0.02 + 0.001
    check(pkg, gpu, dt, A, B, sa, sb, tr.rand(3, m, dt=dt))


def test_sums_are_exact(pkg, gpu):
    """The largest sums there are, and sums that fp32 could not form: without scales the output is the integer, rounded once."""
    k = 131071
    for n, m in ((1, 3), (3, 5), (20, 40)):
        A, B = torch.full((n, k), -128, dtype=torch.int8), torch.full((m, k), -128, dtype=torch.int8)
        B[0] = 127
        C = check(pkg, gpu, "fp32", A, B, None, None, None)
        exact = (A.long() @ B.long().t()).float()
        assert torch.equal(C.cpu(), exact)
    # a small difference of large sums
    k = 4096
    for n in (1, 40):
        A, B = torch.full((n, k), 127, dtype=torch.int8), torch.full((33, k), 127, dtype=torch.int8)
        B[:, k // 2:] = -127
        B[:, 0] = torch.arange(33).to(torch.int8)
        C = check(pkg, gpu, "fp32", A, B, None, None, None)
        assert torch.equal(C[0].cpu(), (127 * (torch.arange(33) - 127)).float())


def test_scales_that_are_no_numbers(pkg, gpu):
    """They stay in their row or column."""
    for n in (3, 70):
        A, B = ints(1, n, 40), ints(2, 50, 40)
        sa, sb = torch.ones(n), torch.ones(50)
        sa[1], sb[7] = float("nan"), float("inf")
        A[:, 0], B[7] = 1, 0
        B[7, 0] = 1  # (a sum that is not 0)
        C = check(pkg, gpu, "fp32", A, B, sa, sb, None)
        assert torch.isnan(C[1]).all() and torch.isinf(C[0, 7]) and torch.isfinite(C[0, :7]).all()


def test_unaligned_operands_and_host_arrays(pkg, gpu):
    def off(t):
        b = torch.empty(t.numel() + 3, dtype=t.dtype, device="cuda")
        b[3:] = t.flatten().cuda()
        return b[3:].view(t.shape)
    for n, m, k in ((2, 40, 64), (70, 90, 256)):
        A, B, sa, sb = ints(1, n, k), ints(2, m, k), torch.rand(n) * 0.1, torch.rand(m)
        C = check(pkg, gpu, "fp16", A, B, sa, sb, None)
        assert torch.equal(C, check(pkg, gpu, "fp16", A, B, sa, sb, None, place=off))
        H = torch.zeros(n, m, dtype=torch.float16).numpy()
        a, keep = tr.int8_args(pkg, A.numpy(), B.numpy(), H, sa.numpy(), sb.numpy())
        assert gpu.ptl_mm_int8_fp16(ctypes.byref(a)) == 0
        assert torch.equal(torch.from_numpy(H), C.cpu())


@pytest.mark.parametrize("n,m,k,tile", [(4, 300, 1000, 0), (30, 500, 2048, 32032), (30, 500, 2049, 32032), (900, 1000, 1024, 64064),
                                        (900, 1000, 1022, 64064), (900, 1000, 1025, 64064), (900, 1000, 1028, 64064), (2048, 2048, 1024, 128128), (4096, 2048, 2045, 128128),
                                        (2300, 4100, 2048, 256256), (2048, 4100, 2045, 256256)])
def test_every_kernel(pkg, gpu, n, m, k, tile):
    """Each kernel on sizes that it is chosen for, the ones that copy rows first among them (their rows do not start on 16 bytes)."""
    A, B = ints(n, n, k), ints(m, m, k)
    sa, sb = tr.rand(1, n).abs() * 0.001 + 0.0001, tr.rand(2, m).abs() * 0.02 + 0.001
    check(pkg, gpu, "fp16", A, B, sa, sb, tr.rand(3, m, dt="fp16"))
    assert gpu.ptl_last_gemm_tile() == tile


@pytest.mark.parametrize("n,m,k", [(64, 2048, 8193), (20, 100, 65537), (8, 256, 131071), (500, 64, 30000)])
def test_few_outputs_of_long_rows(pkg, gpu, n, m, k):
    """k in parts of several workgroups each: the sums stay exact."""
    A, B = ints(n, n, k), ints(m, m, k)
    check(pkg, gpu, "fp16", A, B, tr.rand(1, n).abs() * 1e-4 + 1e-5, tr.rand(2, m).abs() * 0.02 + 0.001, tr.rand(3, m, dt="fp16"))
    if n < 100:
        A, B = torch.full((n, k), -128, dtype=torch.int8), torch.full((m, k), -128, dtype=torch.int8)
        B[::3, : k // 2] = 127
        C = check(pkg, gpu, "fp32", A, B, None, None, None)
        # rows alike: two sums, each formed by hand
        whole, half = 16384 * k, -128 * 127 * (k // 2) + 16384 * (k - k // 2)
        assert (C[:, 1::3] == float(torch.tensor(whole).float())).all() and (C[:, ::3] == float(torch.tensor(half).float())).all()
