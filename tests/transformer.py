"""Argument structs over torch tensors or numpy arrays, tolerances and 64-bit forms for the operators of
include/ptl_transformer.h."""
import ctypes
import math

import numpy as np
import torch

U = 2.0 ** -24  # half a step of fp32, relative to the value


def t_dtype(dt):
    return torch.float32 if dt == "fp32" else torch.float16


def step(ref, dt):
    """Half a step of the tensor type at `ref`, subnormals included."""
    ref = ref.abs()
    return ref * U + 2.0 ** -150 if dt == "fp32" else ref * 2.0 ** -11 + 2.0 ** -25


def dev(t, dt=None):
    return t.to(t_dtype(dt) if dt else t.dtype).cuda()


def rand(seed, *shape, scale=1.0, dt="fp32"):
    """Normal values of the tensor type, on the CPU, from the seed alone."""
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale).to(t_dtype(dt))


def ptr(keep, pkg, data, diff, dim, rows=1):
    b = pkg.blob(data, diff, 1, rows, dim, rows * dim)
    keep += [b, data, diff]
    return ctypes.pointer(b)


def norm_args(pkg, dim, x=None, dx=None, skip=None, dskip=None, total=None, dtotal=None, w=None, dw=None, y=None, dy=None, q=None,
              scale=None, eps=1e-5, skip_wg=0, skip_ig=0, has_skip=None, has_sum=None):
    keep, a = [], pkg.RmsNormArgs()
    a.input, a.coeff, a.output = ptr(keep, pkg, x, dx, dim), ptr(keep, pkg, w, dw, dim), ptr(keep, pkg, y, dy, dim)
    if has_skip or (has_skip is None and (skip is not None or dskip is not None)):
        a.skip = ptr(keep, pkg, skip, dskip, dim)
    if has_sum or (has_sum is None and (total is not None or dtotal is not None)):
        a.sum = ptr(keep, pkg, total, dtotal, dim)
    a.q_data, a.q_scale, a.eps, a.skip_wg_grad, a.skip_in_grad = pkg.addr(q), pkg.addr(scale), eps, skip_wg, skip_ig
    keep += [q, scale]
    return a, keep


def gated_args(pkg, n_in, n_out, act, x=None, dx=None, w=None, dw=None, b=None, db=None, h=None, dh=None, y=None, dy=None, skip_wg=0,
               skip_ig=0):
    keep, a = [], pkg.GatedLinearArgs()
    a.input, a.coeff = ptr(keep, pkg, x, dx, n_in), ptr(keep, pkg, w, dw, n_in, 2 * n_out)
    a.output = ptr(keep, pkg, y, dy, n_out)
    if b is not None or db is not None:
        a.bias, a.use_biases = ptr(keep, pkg, b, db, 2 * n_out), 1
    if h is not None or dh is not None:
        a.hidden = ptr(keep, pkg, h, dh, 2 * n_out)
    a.activation, a.skip_wg_grad, a.skip_in_grad = act, skip_wg, skip_ig
    return a, keep


def int8_args(pkg, A, B, C, sa=None, sb=None, bias=None):
    a = pkg.MatMulInt8Args()
    a.A, a.B, a.C, a.A_scale, a.B_scale, a.bias = (pkg.addr(t) for t in (A, B, C, sa, sb, bias))
    a.N, a.K, a.M, a.USE_BIASES = A.shape[0], A.shape[1], B.shape[0], int(bias is not None)
    return a, [A, B, C, sa, sb, bias]


def distill_args(pkg, z, grad, teacher, classes, loss, temperature, weight):
    keep, a = [], pkg.DistillArgs()
    a.output = ptr(keep, pkg, z, grad, z.shape[-1])
    a.teacher, a.classes, a.n_top = pkg.addr(teacher), pkg.addr(classes), classes.shape[-1]
    a.temperature, a.weight, a.wr_loss = temperature, weight, pkg.addr(loss)
    return a, keep + [teacher, classes, loss]


def within(got, ref, tol, what=""):
    """Every value of `got` within `tol` of `ref`; no number where there is none, infinities alike."""
    got, ref = got.detach().double().cpu(), ref.double()
    tol = tol.double() if isinstance(tol, torch.Tensor) else torch.full_like(ref, tol)
    assert got.shape == ref.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]), what
    fine = torch.isfinite(ref)
    off = (got[fine] - ref[fine]).abs() - tol[fine]
    if off.numel():
        i = int(off.argmax())
        assert off[i] <= 0, (what, float(got[fine][i]), float(ref[fine][i]), float(tol[fine][i]))


ACTS = {"sigmoid": 0, "silu": 1, "gelu": 2, "relu": 3}


def act64(g, act):
    """The activation and its derivative in 64 bits."""
    if act == "relu":
        return g.clamp(min=0), (g > 0).double()
    if act == "gelu":  # (1 + tanh(u)) / 2 = sigmoid(2 u): without the difference, which leaves 64 bits five digits at g = -6
        c = math.sqrt(2 / math.pi)
        u = c * (g + 0.044715 * g ** 3)
        s = torch.sigmoid(2 * u)
        return g * s, s + g * s * torch.sigmoid(-2 * u) * 2 * c * (1 + 3 * 0.044715 * g * g)
    s = torch.sigmoid(g)
    if act == "sigmoid":
        return s, s * torch.sigmoid(-g)
    return g * s, s + g * s * torch.sigmoid(-g)


def act_steps(g, act):
    """Roundings of an activation in fp32, in u of itself: a dozen operations, and the exponent of exp, which four roundings form."""
    if act == "relu":
        return torch.zeros_like(g)
    return 16 + 6 * (1.6 * g.abs() * (1 + 0.044715 * g * g) if act == "gelu" else g.abs())


def norm64(s, w, eps):
    return s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * w


def distill64(z, teacher, classes, temperature, weight):
    """Losses and gradients in 64 bits, from the definition; also p of every class and the logs that the losses are made of."""
    n, v = z.shape
    z = z.double() / temperature
    log_q = torch.log_softmax(z, 1)
    there = (classes >= 0) & (classes < v)
    u = torch.where(there, teacher.double() / temperature, torch.tensor(-math.inf, dtype=torch.float64))
    some = (u.amax(1) > -math.inf) | torch.isnan(u).any(1)
    log_p = torch.where(some[:, None], torch.log_softmax(u, 1), torch.zeros_like(u))
    p = torch.where(some[:, None], torch.exp(log_p), torch.zeros_like(u))
    at = torch.where(there, classes.long(), torch.zeros_like(classes).long())
    terms = torch.where((p != 0) & some[:, None], p * (log_p - log_q.gather(1, at)), torch.zeros_like(p))
    target = torch.zeros(n, v, dtype=torch.float64).scatter_add_(1, at, torch.where(there, p, torch.zeros_like(p)))
    grad = torch.where(some[:, None], weight / temperature * (torch.exp(log_q) - target), torch.zeros_like(target))
    return weight * terms.sum(1), grad, target
