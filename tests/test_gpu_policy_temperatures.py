"""The clipped policy loss over the whole range of temperatures, with rows whose logits lie far from 0, in every way a row is taken: by a wave, by a
workgroup, read twice, in parts.  What a row's classes have in common changes nothing, so that no bound here grows with it.  u = 2^-24."""
import math

import pytest
import torch

import test_gpu_policy as pol
import transformer as tr
import tuning as tn

pytestmark = pytest.mark.gpu
U = tr.U
PEAKS = [100.0, -100.0, 2000.0, 4999.0, 20000.0, -20000.0, 30000.0, 60000.0, -60000.0, 65504.0]
# 2^-7 and its neighbours; the others span what is accepted
TEMPERATURES = [1e-6, 1e-5, 2e-5, 1e-3, 0.0078, 0.0078125, 0.0079, 0.05, 30.0, 1e6]


def make(seed, dt, n, v, temperature):
    """Rows with their largest logit at PEAKS.  A third of the classes lies within some temperatures of it, as far as the type can tell them
    from it, the others below; the largest is there twice where a row has two classes.  Actions are classes near the largest."""
    g = torch.Generator().manual_seed(seed)
    peak = torch.tensor([PEAKS[i % len(PEAKS)] for i in range(n)], dtype=torch.float64).to(tr.t_dtype(dt)).double()[:, None]
    down = torch.rand(n, v, generator=g, dtype=torch.float64)
    near = torch.rand(n, v, generator=g) < 0.3
    z = (peak - torch.where(near, down * 4 * temperature, 1 + down * 90)).clamp(min=-65504).to(tr.t_dtype(dt))
    z = torch.minimum(z, peak.to(z.dtype))
    at = torch.randint(0, v, (n, 2), generator=g)
    z.scatter_(1, at, peak.to(z.dtype).expand(n, 2))
    a = at[:, 0].clone()
    y = (z.double() - peak) / temperature
    for i in range(0, n, 3):  # every third another class, the first that is not far below
        a[i] = torch.nonzero(y[i] >= -4)[0, 0]
    lp = torch.log_softmax(y, 1).gather(1, a[:, None])[:, 0]
    moved = torch.randn(n, generator=g, dtype=torch.float64) * 0.3
    for border in (math.log(1 - pol.LOW), math.log(1 + pol.HIGH)):
        moved = torch.where((moved - border).abs() < 1e-3, moved + 0.01, moved)
    return {"z": z, "action": a.to(torch.int32), "old": (lp - moved).float(), "adv": torch.randn(n, generator=g),
            "ref": (lp + torch.randn(n, generator=g, dtype=torch.float64) * 0.4).float(), "row_weight": torch.rand(n, generator=g) + 0.5}


def check(dt, t, loss, logp, grad, temperature, weight):
    """As the other tests', but for the maximum's share: exponents are within u of themselves and of what a common factor of the row adds to them,
    1/2 at most; a logarithm is of a sum times that factor."""
    n, v = t["z"].shape
    temperature = tn.f32(temperature)
    z, old, adv, ref, rw = (t[k].double() for k in ("z", "old", "adv", "ref", "row_weight"))
    at = t["action"].long()[:, None]
    y = (z - z.amax(1, keepdim=True)) / temperature
    e = torch.exp(y)
    S = e.sum(1)
    lp = y.gather(1, at)[:, 0] - torch.log(S)
    y = torch.where(y == -math.inf, torch.zeros_like(y), y.abs())
    own = U * (8 + 6 * y)
    rel_s = (e * own).sum(1) / S + U * (128 + 16 + 10 + v / 1024)
    e_lp = 4 * U * y.gather(1, at)[:, 0] + rel_s + 3 * U * (torch.log(S) + 1) + 2 * U * lp.abs()
    tr.within(logp, lp, e_lp, "logp")
    ratio, d, w = torch.exp(lp - old), ref - lp, weight * rw
    e_r, e_d = e_lp + 4 * U * (lp - old).abs() + 6 * U, e_lp + U * d.abs()
    whole, clipped = ratio * adv, ratio.clamp(1 - pol.LOW, 1 + pol.HIGH) * adv
    want = w * (-torch.minimum(whole, clipped) + pol.BETA * (torch.expm1(d) - d))
    tol = whole.abs() * e_r + pol.BETA * (torch.expm1(d).abs() * e_d + 8 * U * (torch.expm1(d).abs() + d.abs()))
    tr.within(loss, want, w * tol + 6 * U * want.abs(), "loss")
    slope = torch.where(whole <= clipped, -whole, torch.zeros_like(whole)) - pol.BETA * torch.expm1(d)
    tol = whole.abs() * e_r + pol.BETA * (torch.exp(d) * e_d + 4 * U * torch.expm1(d).abs())
    c, e_c = (w / temperature * slope)[:, None], (w / temperature * tol)[:, None]
    e_c = e_c + 6 * U * c.abs()
    q, hot = e / S[:, None], torch.zeros_like(z).scatter_(1, at, 1.0)
    dz = c * (hot - q)
    # (the instruction has no subnormal results: an exponential below 2^-126, with a row's factor of up to 2^(1/2) below 2^-125, is 0, of a sum of 1 at
    # least, which times c is all that is lost)
    tol = e_c * (hot - q).abs() + c.abs() * (q * (own + rel_s[:, None] + 6 * U) + 2 * U * hot + 2.0 ** -125)
    tr.within(grad, dz, tol + tr.step(dz, dt), "grad")


# a workgroup's classes in one piece a thread, in several; a wave's; parts of rows; read twice
SIZES = [(30, 2), (30, 300), (12, 9999), (1100, 60), (1030, 1500), (4100, 4000), (4, 140000), (130, 135001)]


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,v", SIZES)
def test_temperatures(pkg, gpu, dt, n, v):
    every = TEMPERATURES if n * v < 2000000 else [1e-6, 0.0079]
    for temperature in every:
        t = make(n + v, dt, n, v, temperature)
        weight = tn.f32(min(1024.0, 1024.0 * temperature))  # (the gradients' size is that of weight / temperature)
        loss, logp, grad = pol.run(pkg, gpu, dt, t, temperature=temperature, weight=weight)
        assert torch.isfinite(loss).all() and torch.isfinite(logp).all() and torch.isfinite(grad).all(), temperature
        check(dt, t, loss, logp, grad, temperature, weight)


@pytest.mark.parametrize("n,v", [(10, 50), (1200, 50), (20, 40000), (10, 140000)])
def test_one_class_is_all(pkg, gpu, n, v):
    """fp16, the smallest temperature: the largest logit's log-probability is 0, its loss that of its ratio, the gradients 0."""
    t = make(1, "fp16", n, v, 1e-6)
    peak = t["z"].amax(1, keepdim=True)
    t["z"] = torch.where(t["z"] == peak, torch.full_like(peak, -65504), t["z"])
    t["action"] = (torch.arange(n) % v).to(torch.int32)
    t["z"].scatter_(1, t["action"].long()[:, None], (peak.float().abs() + 50).clamp(max=65504).half())
    t["old"], t["ref"], t["adv"] = torch.zeros(n), None, torch.ones(n)
    loss, logp, grad = pol.run(pkg, gpu, "fp16", t, temperature=1e-6, weight=1.0)
    assert (logp == 0).all() and torch.equal(loss.cpu(), -t["row_weight"]) and (grad == 0).all()


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("n,v", [(10, 100), (1100, 100), (10, 30001), (10, 140000)])
def test_masked_classes(pkg, gpu, dt, n, v):
    """Logits of -inf, an action among them, a row of nothing else, NaN in rows that are left out and in others, at a small temperature."""
    temperature, ninf = 1e-4, -math.inf
    t = make(2, dt, n, v, temperature)
    t["z"][0] = torch.where(torch.arange(v) == t["action"][0], t["z"][0], torch.full_like(t["z"][0], ninf))
    t["old"][0], t["ref"][0] = 0.125, -0.25  # (the only class that is left: its log-probability is 0)
    t["z"][1, t["action"][1].long()] = ninf
    t["z"][2] = ninf
    t["z"][3, 5], t["z"][4, 7] = math.nan, math.nan
    t["action"][3] = -1
    weight = tn.f32(1024 * temperature)
    loss, logp, grad = pol.run(pkg, gpu, dt, t, temperature=temperature, weight=weight)
    good = [0] + list(range(5, n))
    check(dt, {k: x[good] for k, x in t.items()}, loss[good], logp[good], grad[good], temperature, weight)
    assert logp[1] == ninf and torch.isnan(logp[2]) and torch.isnan(grad[2]).all()
    assert loss[3] == 0 and logp[3] == 0 and (grad[3] == 0).all() and torch.isnan(loss[4]) and torch.isnan(grad[4]).all()
