"""The clipped policy loss against its formula in 64 bits.  u = 2^-24.  A row's sum of exponentials is formed in chains of 8 values a piece, up
to 16 pieces a thread (longer rows: dim / 1024 a thread), 6 folds of a wave and 4 of the waves' sums; the exponent of a term is off
by a few u of itself, and of the maximum's where it is formed from the logit as it was read."""
import ctypes
import math

import pytest
import torch

import transformer as tr
import tuning as tn

pytestmark = pytest.mark.gpu
U = tr.U
LOW, HIGH, BETA, T = 0.25, 0.25, 0.125, 0.75


def make(seed, dt, n, v, ref=True, row_weight=True, temperature=T, low=LOW, high=HIGH):
    """Logits and rows' data; no ratio within 1e-4 of a border, where the fp32 sum may fall on either side."""
    z = tr.rand(seed, n, v, scale=2.0, dt=dt)
    g = torch.Generator().manual_seed(seed)
    a = torch.randint(0, v, (n,), generator=g)
    a[::2] = z[::2].double().argmax(1)
    lp = torch.log_softmax(z.double() / temperature, 1).gather(1, a[:, None])[:, 0]
    moved = torch.randn(n, generator=g, dtype=torch.float64) * 0.3
    for border in (math.log(1 - low), math.log(1 + high)):
        moved = torch.where((moved - border).abs() < 1e-3, moved + 0.01, moved)
    t = {"z": z, "action": a.to(torch.int32), "old": (lp - moved).float(), "adv": torch.randn(n, generator=g),
         "ref": (lp + torch.randn(n, generator=g, dtype=torch.float64) * 0.4).float() if ref else None,
         "row_weight": torch.rand(n, generator=g) + 0.5 if row_weight else None}
    t["action"][3::8] = -1  # padding
    if n > 5:
        t["action"][5] = v
    return t


def run(pkg, gpu, dt, t, step=2, over=False, temperature=T, weight=None, low=LOW, high=HIGH, beta=BETA):
    n, v = t["z"].shape
    weight = (1024.0 if dt == "fp16" else 1.0) if weight is None else weight
    d = {k: None if x is None else x.cuda() for k, x in t.items()}
    grad = d["z"] if over else torch.full((n + 1, v), 7, dtype=d["z"].dtype, device="cuda")
    loss, logp = (torch.full((n + 1,), 7.0, device="cuda") for _ in range(2))
    a, keep = tn.policy_args(pkg, d["z"], grad, d["action"], d["old"], d["adv"], d["ref"], d["row_weight"], loss, logp, low, high, beta, temperature, weight)
    assert getattr(gpu, "ptl_policy_loss_%s_batched" % dt)(ctypes.byref(a), n, step) == 0, gpu.ptl_last_error()
    assert gpu.ptl_sync() == 0
    assert loss[n] == 7 and logp[n] == 7 and (over or (grad[n] == 7).all())
    return loss[:n], logp[:n], grad[:n]


def check(dt, t, loss, logp, grad, temperature=T, weight=None, low=LOW, high=HIGH, beta=BETA):
    n, v = t["z"].shape
    weight = (1024.0 if dt == "fp16" else 1.0) if weight is None else weight
    z = t["z"].double().requires_grad_(True)
    old, adv = t["old"].double(), t["adv"].double()
    ref = None if t["ref"] is None else t["ref"].double()
    rw = None if t["row_weight"] is None else t["row_weight"].double()
    want, lp = tn.policy64(z, t["action"], old, adv, ref, rw, low, high, beta, temperature, weight)
    z = z.detach()
    there = (t["action"] >= 0) & (t["action"] < v)
    at = torch.where(there, t["action"], torch.zeros_like(t["action"])).long()[:, None]
    y = (z - z.amax(1, keepdim=True)) / temperature
    masked = y == -math.inf
    e = torch.exp(y)
    y = torch.where(masked, torch.zeros_like(y), y.abs())
    S = e.sum(1)
    far = z.amax(1, keepdim=True).abs() / temperature if dt == "fp16" else 0.0
    own = U * (6 + 6 * y + 2 * far)  # of an exponential: the instruction, and its exponent
    rel_s = (e * own).sum(1) / S + U * (128 + 16 + 10 + v / 1024)
    e_lp = 4 * U * y.gather(1, at)[:, 0] + rel_s + 3 * U * torch.log(S).abs() + 2 * U * lp.detach().abs()
    lp = lp.detach()
    tr.within(logp, lp, torch.where(there, e_lp, torch.zeros_like(e_lp)), "logp")
    ratio = torch.exp(lp - old)
    w = weight * (1.0 if rw is None else rw) * torch.ones(n, dtype=torch.float64)
    e_r = e_lp + 4 * U * (lp - old).abs() + 6 * U  # of the ratio
    tol, tol_slope = (ratio * adv).abs() * e_r, (ratio * adv).abs() * e_r
    whole, clipped = ratio * adv, ratio.clamp(1 - low, 1 + high) * adv
    slope = torch.where(whole <= clipped, -whole, torch.zeros_like(whole))
    if ref is not None:
        d = ref - lp
        e_d = e_lp + U * d.abs()
        tol = tol + beta * (torch.expm1(d).abs() * e_d + 8 * U * (torch.expm1(d).abs() + d.abs()))
        tol_slope = tol_slope + beta * (torch.exp(d) * e_d + 4 * U * torch.expm1(d).abs())
        slope = slope - beta * torch.expm1(d)
    if loss is not None:
        tr.within(loss, want.detach(), torch.where(there, w * tol + 6 * U * want.detach().abs(), torch.zeros_like(tol)), "loss")
    if grad is None:
        return
    q, hot = e / S[:, None], torch.zeros_like(z).scatter_(1, at, 1.0)
    c = torch.where(there, w / temperature * slope, torch.zeros_like(w))[:, None]
    dz = torch.where(there[:, None], c * (hot - q), torch.zeros_like(q))
    e_c = torch.where(there, w / temperature * tol_slope + 6 * U * c[:, 0].abs(), torch.zeros_like(w))[:, None]
    tol = e_c * (hot - q).abs() + c.abs() * (q * (own + rel_s[:, None] + 6 * U) + 2 * U * hot)
    tol = tol + tr.step(dz, dt)
    if dt == "fp16":  # from 65520 on the nearest number is infinity
        dz = torch.where(dz.abs() >= 65520, math.inf * dz.sign(), dz)
    tr.within(grad, dz, tol, "grad")


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,v", [(1, 1), (7, 2), (9, 3), (30, 5), (17, 8), (40, 63), (12, 100), (20, 257), (33, 1000), (9, 2050), (300, 1001), (6, 4100),
                                 (5, 9999), (4, 17000), (70, 20001), (60, 33000), (50, 50000), (3, 65537), (2, 131072), (50, 66000), (140, 70001)])
def test_both(pkg, gpu, dt, n, v):
    t = make(n + v, dt, n, v)
    check(dt, t, *run(pkg, gpu, dt, t))


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,v", [(1100, 60), (1101, 700), (1030, 1500), (4200, 2049), (4100, 4000)])
def test_rows_by_the_wave(pkg, gpu, dt, n, v):
    t = make(n, dt, n, v)
    check(dt, t, *run(pkg, gpu, dt, t))


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_longest_rows(pkg, gpu, dt):
    """Rows that no workgroup holds, enough of them not to be cut into parts."""
    t = make(3, dt, 130, 135001)
    check(dt, t, *run(pkg, gpu, dt, t))
    loss, logp, grad = run(pkg, gpu, dt, t)
    assert torch.equal(run(pkg, gpu, dt, t, over=True)[2], grad)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,v", [(10, 300), (1200, 300), (20, 40000), (3, 140000)])
def test_steps_places_and_what_may_be_missing(pkg, gpu, dt, n, v):
    t = make(5, dt, n, v)
    loss, logp, grad = run(pkg, gpu, dt, t)
    only_loss, lp, g = run(pkg, gpu, dt, t, step=0)
    assert torch.equal(only_loss, loss) and torch.equal(lp, logp) and (g == 7).all()
    l, lp, g = run(pkg, gpu, dt, t, step=1)
    assert (l == 7).all() and torch.equal(lp, logp) and torch.equal(g, grad)
    l, lp, g = run(pkg, gpu, dt, t, over=True)
    assert torch.equal(l, loss) and torch.equal(lp, logp) and torch.equal(g, grad)
    t = make(6, dt, n, v, ref=False, row_weight=False, temperature=1.5, low=0.1, high=0.5)
    k = dict(temperature=1.5, low=0.1, high=0.5, weight=64.0)
    check(dt, t, *run(pkg, gpu, dt, t, **k), **k)
    t["ref"] = torch.full((n,), -math.inf)  # not read without a factor
    check(dt, {**t, "ref": None}, *run(pkg, gpu, dt, t, beta=0.0, **k), **k)
    k = dict(low=0.5, high=math.inf)
    t = make(7, dt, n, v, low=0.5, high=0.25)
    check(dt, t, *run(pkg, gpu, dt, t, **k), **k)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,v", [(8, 100), (8, 30001), (8, 140000)])
def test_values(pkg, gpu, dt, n, v):
    """Classes that are masked out, an action among them, a row of nothing else, NaN and infinities in rows that are left out, no advantage."""
    t = make(8, dt, n, v)
    t["action"] = torch.arange(n, dtype=torch.int32) % v
    ninf = float("-inf")
    t["z"][0, 50:] = ninf
    t["z"][1, 1] = ninf  # the action
    t["z"][2] = ninf
    t["z"][3, 5], t["z"][4, 7], t["z"][5, 9] = float("nan"), float("nan"), float("inf")
    t["action"][3], t["action"][5] = -1, 2 ** 31 - 1
    t["adv"][6] = 0
    t["ref"][1] = ninf  # (a reference that masks it too: the difference is none)
    loss, logp, grad = run(pkg, gpu, dt, t)
    good = [0, 6, 7]
    cut = {k: x[good] for k, x in t.items()}
    check(dt, cut, loss[good], logp[good], grad[good])
    assert logp[1] == ninf and torch.isnan(logp[2]) and torch.isnan(loss[2]) and torch.isnan(grad[2]).all()
    for row in (3, 5):
        assert loss[row] == 0 and logp[row] == 0 and (grad[row] == 0).all()
    assert torch.isnan(loss[4]) and torch.isnan(grad[4]).all()
    t["ref"] = None  # without a reference a masked action has ratio 0
    loss, logp, grad = run(pkg, gpu, dt, t)
    assert loss[1] == 0 if t["adv"][1] > 0 else torch.isfinite(loss[1])
    assert (grad[1] == 0).all()


def test_small_differences_from_the_reference(pkg, gpu):
    """exp(d) - 1 - d is half of d squared near 0, where the difference of two floats would be nothing but their roundings."""
    n, v = 6, 4
    z = torch.zeros(n, v)
    lp = torch.full((n,), -math.log(4.0), dtype=torch.float64)
    d = torch.tensor([0.0, 1e-3, -1e-3, 0.05, -0.2, 0.3], dtype=torch.float64)
    t = {"z": z, "action": torch.zeros(n, dtype=torch.int32), "old": lp.float(), "adv": torch.zeros(n), "ref": (lp + d).float(), "row_weight": None}
    loss, logp, _ = run(pkg, gpu, "fp32", t, temperature=1.0, beta=1.0)
    away = t["ref"].double() - logp.double().cpu()
    want = torch.expm1(away) - away
    assert ((loss.double().cpu() - want).abs() <= 8 * U * want + 2.0 ** -24 * away.abs() * away.abs() + 1e-16).all()


def test_gradient_against_differences(pkg, gpu):
    n, v, h = 6, 7, 1e-5
    t = make(9, "fp32", n, v)
    t["action"] = torch.arange(n, dtype=torch.int32)
    lp = torch.log_softmax(t["z"].double() / T, 1).gather(1, t["action"].long()[:, None])[:, 0]
    t["old"] = (lp - torch.tensor([0.1, -0.1, 0.4, 0.4, -0.5, -0.5], dtype=torch.float64)).float()  # both sides of both borders
    t["adv"] = torch.tensor([1.0, -1.0, 1.0, -1.0, 1.0, -1.0])
    _, _, grad = run(pkg, gpu, "fp32", t)

    def f(z):
        return tn.policy64(z, t["action"], t["old"].double(), t["adv"].double(), t["ref"].double(), t["row_weight"].double(), LOW, HIGH, BETA, T, 1.0)[0].sum()

    for i in range(n * v):
        up, down = t["z"].double(), t["z"].double()
        up.view(-1)[i] += h
        down.view(-1)[i] -= h
        # (the references here are up to 6 away: exp(d) times what the logarithm is off, some 16 u, is at most 1e-5 of a gradient)
        want = float(f(up) - f(down)) / (2 * h)
        assert abs(want - float(grad.reshape(-1)[i])) < 1e-5 * max(1.0, abs(want))


def test_host_arrays(pkg, gpu):
    t = make(10, "fp16", 9, 77)
    loss, logp, grad = run(pkg, gpu, "fp16", t)
    h = {k: x.numpy() for k, x in t.items()}
    g, l, p = torch.zeros(9, 77, dtype=torch.float16).numpy(), torch.zeros(9).numpy(), torch.zeros(9).numpy()
    a, keep = tn.policy_args(pkg, h["z"], g, h["action"], h["old"], h["adv"], h["ref"], h["row_weight"], l, p, LOW, HIGH, BETA, T, 1024.0)
    assert gpu.ptl_policy_loss_fp16_batched(ctypes.byref(a), 9, 2) == 0
    assert torch.equal(torch.from_numpy(g), grad.cpu()) and torch.equal(torch.from_numpy(l), loss.cpu()) and torch.equal(torch.from_numpy(p), logp.cpu())
