"""Distillation from top logits against its definition in 64 bits.  u = 2^-24."""
import ctypes
import math

import pytest
import torch

import transformer as tr

pytestmark = pytest.mark.gpu
U = tr.U


def run(pkg, gpu, dt, z, teacher, classes, temperature=2.0, weight=3.0, step=2, in_place=False):
    Z, T, C = tr.dev(z), tr.dev(teacher), classes.cuda()
    grad = Z if in_place else torch.full_like(Z, 7)
    loss = torch.full((z.shape[0],), 7.0, device="cuda")
    a, keep = tr.distill_args(pkg, Z, grad, T, C, loss, temperature, weight)
    rc = getattr(gpu, "ptl_distill_%s_batched" % dt)(ctypes.byref(a), z.shape[0], step)
    assert rc == 0 and gpu.ptl_sync() == 0, gpu.ptl_last_error()
    return loss, grad


def check(dt, z, teacher, classes, loss, grad, temperature=2.0, weight=3.0):
    """An exponential is off by the rounding of its exponent, at most 4 u |z - m| / T of itself, and an ulp of its own; a sum of
    them by its longest chain, 128 additions in a thread (long rows: dim / 1024) and 21 folds."""
    ref_loss, ref_grad, target = tr.distill64(z, teacher, classes, temperature, weight)
    v = z.shape[1]
    there = (classes >= 0) & (classes < v)
    fin = torch.where(torch.isfinite(z), z.double(), torch.zeros((), dtype=torch.float64))
    c = 128 + 21 + v / 1024 + 16
    if loss is not None:
        # log p and log q: differences of at most `far` from the largest, and logs of sums that are c u (and the exponents') off
        u = torch.where(there & torch.isfinite(teacher), teacher.double(), torch.zeros((), dtype=torch.float64))
        far = (u.abs().amax(1) * 2 + fin.abs().amax(1) * 2) / temperature + math.log(v) + math.log(classes.shape[1] + 1)
        tr.within(loss, ref_loss, abs(weight) * U * (far * (classes.shape[1] + 40) + c), "loss")
    if grad is not None:
        zz = (z.double().amax(1, keepdim=True) - fin) / temperature
        q = torch.softmax(z.double() / temperature, 1).nan_to_num()
        tol = abs(weight) / temperature * U * (q * (c + 4 * zz + 16) + target * (classes.shape[1] + 64 + 8 * 40)) + ref_grad.abs() * 4 * U
        tr.within(grad, ref_grad, tol + tr.step(ref_grad, dt) + abs(weight) / temperature * 2.0 ** -120, "grad")


def case(seed, n, v, k, dt, empty=True):
    g = torch.Generator().manual_seed(seed)
    z = tr.rand(seed, n, v, scale=2.0, dt=dt)
    classes = torch.stack([torch.randperm(v, generator=g)[:k] if k <= v else torch.randint(0, v, (k,), generator=g) for _ in range(n)])
    teacher = tr.rand(seed + 1, n, k, scale=2.0, dt=dt)
    classes = classes.to(torch.int32)
    if empty:
        sent = torch.randint(0, 2 * k + 1, (n, 1), generator=g)
        classes[torch.arange(k)[None] >= sent] = -1
    return z, teacher, classes


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("v", [1, 2, 3, 7, 8, 9, 255, 1000, 1024, 2049, 4097, 8192, 10001, 16390, 32000, 32770, 65544])
def test_both_steps(pkg, gpu, dt, v):
    for n, k in ((1, 1), (3, 5), (150 if v < 20000 else 130, 64 if v >= 64 else 2)):
        z, teacher, classes = case(v + n, n, v, min(k, v), dt)
        check(dt, z, teacher, classes, *run(pkg, gpu, dt, z, teacher, classes))


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,v,k", [(1, 131072, 128), (2, 131073, 7), (4, 262147, 2048), (140, 66001, 33)])
def test_large_vocabularies(pkg, gpu, dt, n, v, k):
    z, teacher, classes = case(n, n, v, k, dt)
    check(dt, z, teacher, classes, *run(pkg, gpu, dt, z, teacher, classes))


@pytest.mark.parametrize("n,v", [(2, 500), (2, 30000), (140, 9000)])
def test_single_steps_and_in_place(pkg, gpu, n, v):
    for dt in ("fp32", "fp16"):
        z, teacher, classes = case(5, n, v, 20, dt)
        loss, grad = run(pkg, gpu, dt, z, teacher, classes)
        only, none = run(pkg, gpu, dt, z, teacher, classes, step=0)
        assert torch.equal(only, loss) and (none == 7).all()
        none, only = run(pkg, gpu, dt, z, teacher, classes, step=1)
        assert torch.equal(only, grad) and (none == 7).all()
        again, over = run(pkg, gpu, dt, z, teacher, classes, in_place=True)
        assert torch.equal(again, loss) and torch.equal(over, grad)


@pytest.mark.parametrize("n,v", [(6, 300), (6, 20000)])
def test_entries(pkg, gpu, n, v):
    """Rows that name nothing, one class many times, classes out of range, and teachers of -inf; students of -inf."""
    for dt in ("fp32", "fp16"):
        z, teacher, classes = case(9, n, v, 12, dt, empty=False)
        classes[0] = -1
        classes[1] = 17
        classes[2, ::2] = torch.tensor([v, v + 1, 2 ** 31 - 1, -2 ** 31, -1, v], dtype=torch.int32)
        teacher[3, :6] = -float("inf")
        teacher[4] = -float("inf")
        z[5, 100:] = -float("inf")
        classes[5] = torch.arange(12, dtype=torch.int32) * 3
        loss, grad = run(pkg, gpu, dt, z, teacher, classes)
        check(dt, z, teacher, classes, loss, grad)
        assert loss[0] == 0 and (grad[0] == 0).all() and loss[4] == 0 and (grad[4] == 0).all() and (grad[5, 100:] == 0).all()
        # a named class that the student rules out: the loss is infinite, the gradient is not
        z[5, 3] = -float("inf")
        loss, grad = run(pkg, gpu, dt, z, teacher, classes)
        check(dt, z, teacher, classes, loss, grad)
        assert loss[5] == float("inf") and torch.isfinite(grad[5]).all()


@pytest.mark.parametrize("n,v", [(4, 300), (4, 20000)])
def test_no_numbers(pkg, gpu, n, v):
    """A NaN or an infinity of the student or the teacher stays in its row."""
    z, teacher, classes = case(11, n, v, 6, "fp32", empty=False)
    z[1, v // 2], teacher[2, 3] = float("nan"), float("nan")
    loss, grad = run(pkg, gpu, "fp32", z, teacher, classes)
    assert torch.isnan(loss[[1, 2]]).all() and torch.isnan(grad[1]).all() and torch.isnan(grad[2, classes[2, 0].item()])
    keep = [0, 3]
    check("fp32", z[keep], teacher[keep], classes[keep], loss[keep], grad[keep])


def test_temperatures_and_weights(pkg, gpu):
    for temperature, weight in ((0.05, 1.0), (1.0, -2.0), (30.0, 900.0), (1.0, 0.0)):
        z, teacher, classes = case(13, 3, 3000, 40, "fp32")
        loss, grad = run(pkg, gpu, "fp32", z, teacher, classes, temperature, weight)
        check("fp32", z, teacher, classes, loss, grad, temperature, weight)


def test_gradient_against_differences(pkg, gpu):
    n, v, h = 2, 40, 1e-4
    z, teacher, classes = case(15, n, v, 6, "fp32", empty=False)
    _, grad = run(pkg, gpu, "fp32", z, teacher, classes)
    for i in range(n):
        for j in range(v):
            e = torch.zeros(n, v, dtype=torch.float64)
            e[i, j] = h
            up, down = (tr.distill64(z.double() + s * e, teacher, classes, 2.0, 3.0)[0].sum() for s in (1, -1))
            assert abs((up - down) / (2 * h) - float(grad[i, j])) < 1e-5


def test_host_arrays(pkg, gpu):
    z, teacher, classes = case(17, 3, 700, 9, "fp16")
    loss, grad = run(pkg, gpu, "fp16", z, teacher, classes)
    hl, hg = torch.zeros(3).numpy(), torch.zeros(3, 700, dtype=torch.float16).numpy()
    a, keep = tr.distill_args(pkg, z.numpy(), hg, teacher.numpy(), classes.numpy(), hl, 2.0, 3.0)
    assert gpu.ptl_distill_fp16_batched(ctypes.byref(a), 3, 2) == 0
    assert torch.equal(torch.from_numpy(hl), loss.cpu()) and torch.equal(torch.from_numpy(hg), grad.cpu())


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,v,k", [(1027, 300, 5), (1030, 500, 250), (1025, 1500, 64), (1025, 2000, 70), (4100, 4000, 9), (1100, 9, 12)])
def test_rows_by_the_wave(pkg, gpu, dt, n, v, k):
    """Rows enough that each has one wave; some name a class twice, among them classes far apart in the row of entries."""
    z, teacher, classes = case(n, n, v, k, dt)
    classes[5, -1] = classes[5, 0] = 3
    classes[7] = 4
    check(dt, z, teacher, classes, *run(pkg, gpu, dt, z, teacher, classes))


@pytest.mark.parametrize("n,v,k", [(3, 5000, 2048), (3, 100000, 2048), (200, 3000, 1000), (1030, 300, 700), (1030, 300, 512), (1030, 2000, 2048)])
def test_many_entries_named_twice(pkg, gpu, n, v, k):
    g = torch.Generator().manual_seed(n)
    z, teacher, _ = case(n, n, v, k, "fp32")
    classes = torch.randint(0, v, (n, k), generator=g, dtype=torch.int32)
    check("fp32", z, teacher, classes, *run(pkg, gpu, "fp32", z, teacher, classes))


@pytest.mark.parametrize("dt,n,v", [("fp16", 5, 40001), ("fp32", 130, 70001), ("fp16", 130, 131075)])
def test_values_in_rows_that_no_workgroup_holds(pkg, gpu, dt, n, v):
    """Few rows in parts, many that are walked: stretches of -inf at either end, one class left, a NaN; in the place of the logits."""
    z, teacher, classes = case(v, n, v, 20, dt, empty=False)
    z[0, :33000], z[1, 20000:] = -float("inf"), -float("inf")
    z[2], z[2, v - 1] = -float("inf"), 1.5
    classes[0] = torch.arange(20, dtype=torch.int32) + 34000
    classes[1], classes[2] = torch.arange(20, dtype=torch.int32), v - 1
    z[3, 9] = float("nan")
    loss, grad = run(pkg, gpu, dt, z, teacher, classes)
    keep = [i for i in range(n) if i != 3]
    check(dt, z[keep], teacher[keep], classes[keep], loss[keep], grad[keep])
    assert torch.isnan(loss[3]) and torch.isnan(grad[3]).all()
    again, over = run(pkg, gpu, dt, z, teacher, classes, in_place=True)
    assert torch.equal(again[keep], loss[keep]) and torch.equal(over[keep], grad[keep])


def case_at(seed, n, v, k, dt, temperature, far, spread):
    """Logits around `far`, a teacher whose logits differ by some temperatures."""
    z, _, classes = case(seed, n, v, k, dt)
    z = (z.double() * spread / 2 + far).to(z.dtype)
    top = z.float().topk(min(k, 3), dim=1).indices  # the first entries name the largest classes
    classes[:, : top.shape[1]] = top.to(torch.int32)
    return z, tr.rand(seed + 1, n, k, scale=2.0 * temperature, dt=dt), classes


def check_at(dt, z, teacher, classes, loss, grad, temperature, weight):
    """Temperature and weight are fp32 numbers here.  log p and log q are differences from the row's largest logit, 4 u of themselves off
    (the difference, 1 / T, the product), less the log of a sum, which is c u off, and rounded; p and the terms follow from them."""
    ref_loss, _, _ = tr.distill64(z, teacher, classes, temperature, weight)
    v, k = z.shape[1], classes.shape[1]
    at = torch.where((classes >= 0) & (classes < v), classes, torch.zeros_like(classes)).long()
    there = (classes >= 0) & (classes < v)
    zz = (z.double().amax(1, keepdim=True) - z.double().gather(1, at)) / temperature
    u = torch.where(there, teacher.double() / temperature, torch.tensor(-math.inf, dtype=torch.float64))
    uu = torch.where(there, u.amax(1, keepdim=True) - u, torch.zeros_like(u))
    log_q = torch.log_softmax(z.double() / temperature, 1).gather(1, at)
    log_p = torch.where(there, torch.log_softmax(torch.where(there, u, torch.full_like(u, -1e300)), 1), torch.zeros_like(u))
    p = torch.where(there, log_p.exp(), torch.zeros_like(u))
    c = 128 + 21 + v / 1024 + 16
    off = p * (4 * zz + 4 * uu + 2 * c + (log_p.abs() + log_q.abs()) * (c + 4 * uu + k + 30))
    tr.within(loss, ref_loss, abs(weight) * U * off.sum(1) + 2.0 ** -140, "loss")
    check(dt, z, teacher, classes, None, grad, temperature, weight)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,v,k", [(3, 3000, 40), (1030, 300, 9), (3, 40001, 40), (130, 131075, 20)])
def test_low_temperatures_and_far_logits(pkg, gpu, dt, n, v, k):
    """Rows by the workgroup, by the wave, in parts and walked.  A class' probability follows from its distance from the largest logit,
    however far from 0 both lie in units of the temperature."""
    cases = ((0.05, 0, 2), (0.05, 1000, 2), (0.01, 100, 1), (1e-3, 5, 5), (1e-3, -1, 0.01), (1e-4, 0, 100), (1e-5, 100, 1), (1e-6, 0, 5), (1e-6, 0, 2000),
             (1.0, 30000, 20), (2.0, -60000, 40))
    for temperature, far, spread in cases if n < 100 else cases[1::3]:
        temperature = float(torch.tensor(temperature, dtype=torch.float32))
        weight = float(torch.tensor(3 * temperature, dtype=torch.float32))
        z, teacher, classes = case_at(n + v, n, v, k, dt, temperature, far, spread)
        loss, grad = run(pkg, gpu, dt, z, teacher, classes, temperature, weight)
        check_at(dt, z, teacher, classes, loss, grad, temperature, weight)
