"""Argument structs over torch tensors or numpy arrays and 64-bit forms for the operators of include/ptl_tuning.h."""
import ctypes

import torch

import transformer as tr

ACTS = dict(tr.ACTS, none=4)


def act64(h, act):
    return (h, torch.ones_like(h)) if act == "none" else tr.act64(h, act)


def act_args(pkg, n_in, n_out, act, x=None, dx=None, w=None, dw=None, b=None, db=None, h=None, dh=None, skip=None, y=None, dy=None,
             skip_wg=0, skip_ig=0):
    keep, a = [], pkg.ActLinearArgs()
    a.input, a.coeff = tr.ptr(keep, pkg, x, dx, n_in), tr.ptr(keep, pkg, w, dw, n_in, n_out)
    a.output = tr.ptr(keep, pkg, y, dy, n_out)
    if b is not None or db is not None:
        a.bias, a.use_biases = tr.ptr(keep, pkg, b, db, n_out), 1
    if h is not None or dh is not None:
        a.hidden = tr.ptr(keep, pkg, h, dh, n_out)
    if skip is not None:
        a.skip = tr.ptr(keep, pkg, skip, None, n_out)
    a.activation, a.skip_wg_grad, a.skip_in_grad = act, skip_wg, skip_ig
    return a, keep


def join_args(pkg, dim, b=None, db=None, x=None, dx=None, gate=None, dgate=None, w1=None, dw1=None, w2=None, dw2=None, s=None, ds=None, y=None,
              dy=None, alpha=0.75, eps=1e-5, per=0, skip_wg=0, skip_ig=0):
    keep, a = [], pkg.NormJoinArgs()
    a.input, a.skip, a.sum = tr.ptr(keep, pkg, b, db, dim), tr.ptr(keep, pkg, x, dx, dim), tr.ptr(keep, pkg, s, ds, dim)
    a.coeff_post = tr.ptr(keep, pkg, w1, dw1, dim)
    if w2 is not None or dw2 is not None:
        a.coeff_pre = tr.ptr(keep, pkg, w2, dw2, dim)
        a.output = tr.ptr(keep, pkg, y, dy, dim)
    if gate is not None or dgate is not None:
        a.gate = tr.ptr(keep, pkg, gate, dgate, dim)
    a.skip_scale, a.eps, a.rows_per_gate, a.skip_wg_grad, a.skip_in_grad = alpha, eps, per, skip_wg, skip_ig
    return a, keep


def policy_args(pkg, z, grad, actions, old, adv, ref=None, row_weight=None, loss=None, logp=None, low=0.25, high=0.25, beta=0.125, temperature=1.0,
                weight=1.0):
    keep, a = [], pkg.PolicyLossArgs()
    a.output = tr.ptr(keep, pkg, z, grad, z.shape[-1])
    a.actions, a.old_logp, a.ref_logp, a.advantages, a.row_weight = (pkg.addr(t) for t in (actions, old, ref, adv, row_weight))
    a.clip_low, a.clip_high, a.beta, a.temperature, a.weight = low, high, beta, temperature, weight
    a.wr_loss, a.wr_logp = pkg.addr(loss), pkg.addr(logp)
    return a, keep + [actions, old, ref, adv, row_weight, loss, logp]


def state(pkg, keep, **t):
    s = pkg.AdamwState()
    for k, v in t.items():
        setattr(s, k, pkg.addr(v))
    keep += [s, t]
    return ctypes.pointer(s)


def adamw_step(pkg, t=1, beta1=0.9, beta2=0.999, eps=1e-8, step_data=None, factor=None):
    h = pkg.AdamwStep()
    h.beta1, h.beta2, h.eps, h.step, h.step_data, h.grad_factor = beta1, beta2, eps, t, pkg.addr(step_data), pkg.addr(factor)
    return h


def f32(v):
    return ctypes.c_float(v).value


def adamw64(w, g, m, v, t, lr, decay, beta1=0.9, beta2=0.999, eps=1e-8):
    """The step in 64 bits with the fp32 values of the constants: weights, moments, and the part of the step that Adam has."""
    lr, decay, beta1, beta2, eps = (f32(c) for c in (lr, decay, beta1, beta2, eps))
    m, v = beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g
    up = m / (1 - beta1 ** t) / ((v / (1 - beta2 ** t)).sqrt() + eps)
    return w - lr * (up + decay * w), m, v, lr * up


def join64(b, x, gate, w1, w2, alpha, eps, per):
    """s and y (or None) in 64 bits, differentiable."""
    n = b.shape[0]
    u = b / torch.sqrt((b * b).mean(1, keepdim=True) + eps) * w1
    if gate is not None:
        u = u * (gate if gate.shape[0] == 1 else gate[torch.arange(n) // per])
    s = alpha * x + u
    return s, None if w2 is None else s / torch.sqrt((s * s).mean(1, keepdim=True) + eps) * w2


def policy64(z, action, old, adv, ref, row_weight, low, high, beta, temperature, weight):
    """Losses (differentiable to z) and log-probabilities in 64 bits; rows without an action have 0."""
    there = (action >= 0) & (action < z.shape[1])
    at = torch.where(there, action, torch.zeros_like(action)).long()[:, None]
    lp = torch.log_softmax(z / temperature, 1).gather(1, at)[:, 0]
    ratio = torch.exp(lp - old)
    loss = -torch.minimum(ratio * adv, ratio.clamp(1 - low, 1 + high) * adv)
    if ref is not None:
        loss = loss + beta * (torch.exp(ref - lp) - (ref - lp) - 1)
    loss = loss * weight * (1 if row_weight is None else row_weight)
    zero = torch.zeros_like(loss)
    return torch.where(there, loss, zero), torch.where(there, lp, zero)
