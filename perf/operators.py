"""The operators of a transformer's feed-forward half and of its training by a teacher, as passes of a user's program.

Four of them: the root-mean-square normalisation behind a residual's addition (forward, with an output in 8 bits,
backward), the gated dense layer (forward, backward), the product of 8-bit integers with scales, and the loss against a
teacher's top logits with its gradient.  The ranges of `draw` cover single tokens (latency) to large batches, sizes that
fill whole vectors and tiles and sizes that do not, fp32 and fp16, with and without biases and residuals.
"""
import ctypes
import importlib
import math

import torch

own = False

# At most this much work in a drawn case (the largest listed ones move 340 MB and form 190 GFLOP); fp32 products run at a
# sixteenth of the fp16 matrix rate.
MOST_FLOPS = {"fp16": 180e9, "fp32": 12e9}
MOST_BYTES = 320e6
EPS = 1e-5


def listed():
    return [
        # one token between two layers of a decoder: the latency of a launch
        {"name": "norm_token", "kind": "norm", "step": "fw", "dtype": "fp16", "n": 1, "dim": 4096, "residual": 1},
        # a small model's batch, no size a multiple of anything
        {"name": "norm_ragged", "kind": "norm", "step": "fw", "dtype": "fp32", "n": 391, "dim": 785, "residual": 1},
        # a prompt in front of a frozen layer that runs in 8 bits
        {"name": "norm_8bit", "kind": "norm", "step": "8bit", "dtype": "fp16", "n": 2048, "dim": 4096, "residual": 1},
        # a training batch on the way back, with the gradient that comes along the residual
        {"name": "norm_backward", "kind": "norm", "step": "bw", "dtype": "fp16", "n": 8192, "dim": 4096, "residual": 1},
        # one token through both projections
        {"name": "gated_token", "kind": "gated", "step": "fw", "dtype": "fp16", "n": 1, "n_in": 1024, "n_out": 2816,
         "act": "silu", "keep": 0, "bias": 0},
        # a training batch, pre-activations kept for the way back
        {"name": "gated_batch", "kind": "gated", "step": "fw", "dtype": "fp16", "n": 4096, "n_in": 2048, "n_out": 5632,
         "act": "silu", "keep": 1, "bias": 0},
        # ... and back: gradients of the pre-activations, the input and both weights
        {"name": "gated_backward", "kind": "gated", "step": "bw", "dtype": "fp16", "n": 2048, "n_in": 2048, "n_out": 5632,
         "act": "silu", "keep": 1, "bias": 0},
        # a small fp32 layer with biases, no size a multiple of anything
        {"name": "gated_ragged", "kind": "gated", "step": "fw", "dtype": "fp32", "n": 391, "n_in": 785, "n_out": 333,
         "act": "gelu", "keep": 1, "bias": 1},
        # one token through a frozen 8-bit layer: its weights from memory
        {"name": "int8_token", "kind": "int8", "dtype": "fp16", "n": 1, "n_in": 4096, "n_out": 4096, "bias": 0},
        # a prompt through the same layer
        {"name": "int8_prompt", "kind": "int8", "dtype": "fp16", "n": 4096, "n_in": 4096, "n_out": 4096, "bias": 0},
        # a training batch over a vocabulary of ordinary size
        {"name": "distill_batch", "kind": "distill", "step": "both", "dtype": "fp16", "n": 2048, "classes": 32000, "top": 64},
        # a few tokens over a large vocabulary
        {"name": "distill_few", "kind": "distill", "step": "both", "dtype": "fp32", "n": 4, "classes": 131072, "top": 128},
    ]


# ---- drawn cases -------------------------------------------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size between lo and hi: as drawn (often odd), or, half of the time, whole vectors as layers mostly have them."""
    v = _log(rng, lo, hi)
    if rng.random() < 0.5:
        step = 64 if v >= 96 else 16 if v >= 24 else 8
        v = max(step, (v + step // 2) // step * step)
    return max(lo, min(hi, v))


def _draw_one(rng):
    kind = rng.choice(["norm", "norm", "gated", "gated", "int8", "distill"])
    dtype = rng.choice(["fp16", "fp16", "fp32"])
    n = 1 if rng.random() < 0.15 else _log(rng, 2, 8192)
    if kind == "norm":
        return {"kind": kind, "step": rng.choice(["fw", "fw", "8bit", "bw", "bw"]), "dtype": dtype, "n": n,
                "dim": _size(rng, 64, 16384), "residual": rng.choice([0, 1, 1])}
    if kind == "gated":
        step = rng.choice(["fw", "bw"])
        return {"kind": kind, "step": step, "dtype": dtype, "n": n, "n_in": _size(rng, 64, 4096),
                "n_out": _size(rng, 64, 8192), "act": rng.choice(["silu", "gelu"]),
                "keep": 1 if step == "bw" else rng.randint(0, 1), "bias": rng.choice([0, 0, 1])}
    if kind == "int8":
        return {"kind": kind, "dtype": dtype, "n": n, "n_in": _size(rng, 64, 8192), "n_out": _size(rng, 64, 8192),
                "bias": rng.choice([0, 0, 1])}
    return {"kind": kind, "step": rng.choice(["both", "both", "loss"]), "dtype": dtype, "n": n,
            "classes": _size(rng, 256, 131072), "top": _log(rng, 1, 256)}


def draw(rng):
    while True:
        case = _draw_one(rng)
        w = work(case)
        matrix = "fp16" if case["kind"] == "int8" else case["dtype"]
        if w["flops"] <= MOST_FLOPS[matrix] and w["bytes"] <= MOST_BYTES:
            return case


def work(case):
    """Each input of a pass read once and each of its outputs written once."""
    e = 4 if case["dtype"] == "fp32" else 2
    n, kind = float(case["n"]), case["kind"]
    if kind == "norm":
        c, res = case["dim"], case["residual"]
        if case["step"] == "bw":  # the sum, dy and, with a residual, its gradient; dx
            return {"bytes": e * (n * c * (3 + res) + 2.0 * c), "flops": 10.0 * n * c}
        if case["step"] == "8bit":  # x (and the residual); the sum, the 8 bits and the scales
            return {"bytes": n * c * (e * (1 + 2 * res) + 1) + e * c + 4.0 * n, "flops": 8.0 * n * c}
        return {"bytes": e * (n * c * (2 + 2 * res) + c), "flops": 5.0 * n * c}
    if kind == "gated":
        i, o = case["n_in"], case["n_out"]
        w, b = 2.0 * o * i, 2.0 * o * case["bias"]
        if case["step"] == "bw":  # x, the pre-activations, dy, weights; gradients of pre-activations, input, weights
            return {"bytes": e * (2 * n * i + 5 * n * o + 2 * w + b), "flops": 8.0 * n * i * o + 20.0 * n * o}
        return {"bytes": e * (n * i + w + b + n * o * (1 + 2 * case["keep"])), "flops": 4.0 * n * i * o + 10.0 * n * o}
    if kind == "int8":
        i, o = case["n_in"], case["n_out"]
        return {"bytes": n * i + 1.0 * o * i + 4.0 * (n + o) + e * (n * o + o * case["bias"]), "flops": 2.0 * n * i * o}
    v, k = case["classes"], case["top"]
    both = case["step"] == "both"
    return {"bytes": e * n * v * (2 if both else 1) + n * k * (e + 4) + 4.0 * n, "flops": n * v * (6.0 if both else 4.0)}


# ---- inputs ------------------------------------------------------------------------------------------------------

TEMPERATURE = 2.0


def _weight(case):
    """Of a row's loss: the mean over rows, times T^2 so that gradients keep their size, times the loss scale of an fp16 run."""
    scale = min(65536.0, 1024.0 * case["n"]) if case["dtype"] == "fp16" else 1.0
    return TEMPERATURE ** 2 * scale / case["n"]


def _inputs(case, seed):
    """The tensors of a pass, on the GPU, from the seed alone."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    t = torch.float32 if case["dtype"] == "fp32" else torch.float16

    def normal(*shape, scale=1.0, to=t):
        return torch.randn(shape, generator=gen, device="cuda").mul_(scale).to(to)

    n, x = case["n"], {}
    if case["kind"] == "norm":
        c = case["dim"]
        # activations with a few channels far larger than the others, as transformers have them
        loud = 1 + 9 * (torch.rand(c, generator=gen, device="cuda") < 0.01)
        x["x"] = (torch.randn((n, c), generator=gen, device="cuda") * loud).to(t)
        x["w"] = (1 + 0.1 * torch.randn(c, generator=gen, device="cuda")).to(t)
        if case["step"] == "bw":
            x["dy"] = normal(n, c, scale=0.1)
            if case["residual"]:
                x["dsum"] = normal(n, c, scale=0.1)
        elif case["residual"]:
            x["skip"] = normal(n, c)
    elif case["kind"] == "gated":
        i, o = case["n_in"], case["n_out"]
        x["x"], x["w"] = normal(n, i), normal(2 * o, i, scale=1.5 / math.sqrt(i))
        if case["bias"] and case["step"] == "fw":
            x["bias"] = normal(2 * o, scale=0.1)
        if case["step"] == "bw":
            x["hidden"], x["dy"] = normal(n, 2 * o, scale=1.5), normal(n, o, scale=0.1)
    elif case["kind"] == "int8":
        i, o = case["n_in"], case["n_out"]
        x["a"] = normal(n, i, scale=40.0, to=torch.float32).round_().clamp_(-127, 127).to(torch.int8)
        x["b"] = normal(o, i, scale=40.0, to=torch.float32).round_().clamp_(-127, 127).to(torch.int8)
        x["a_scale"] = torch.rand(n, generator=gen, device="cuda").mul_(0.02).add_(0.01)
        x["b_scale"] = torch.rand(o, generator=gen, device="cuda").add_(0.5).mul_(0.025 / math.sqrt(i))
        if case["bias"]:
            x["bias"] = normal(o, scale=0.1)
    else:
        v, k = case["classes"], case["top"]
        x["z"] = normal(n, v, scale=2.0)
        teacher = x["z"].float() * 0.5 + torch.randn((n, v), generator=gen, device="cuda") * 1.5
        top, at = teacher.topk(k, dim=1)
        # rows of teachers that sent fewer entries, one in 16 of which sent none
        sent = (torch.rand((n, 1), generator=gen, device="cuda") * 4 * k).long()
        sent[torch.rand((n, 1), generator=gen, device="cuda") < 1 / 16] = 0
        x["teacher"] = top.to(t)
        x["top"] = torch.where(torch.arange(k, device="cuda") < sent, at, -1).to(torch.int32)
    return x


class State:
    """What a program has in hand before a pass: its tensors and the buffers for results."""

    def __init__(self, case, x):
        self.case, self.x, self.calls = case, x, None
        t = torch.float32 if case["dtype"] == "fp32" else torch.float16
        n, y = case["n"], {}

        def out(name, *shape, of=t):
            y[name] = torch.empty(shape, dtype=of, device="cuda")

        if case["kind"] == "norm":
            c = case["dim"]
            if case["step"] == "bw":
                out("dx", n, c)
                out("dw", c)
            else:
                if case["residual"]:
                    out("sum", n, c)
                if case["step"] == "8bit":
                    out("q", n, c, of=torch.int8)
                    out("scale", n, of=torch.float32)
                    out("value", n, c, of=torch.float16)
                else:
                    out("y", n, c)
        elif case["kind"] == "gated":
            i, o = case["n_in"], case["n_out"]
            if case["step"] == "bw":
                out("dhidden", n, 2 * o)
                out("dx", n, i)
                out("dw", 2 * o, i)
                if case["bias"]:
                    out("dbias", 2 * o)
            else:
                out("y", n, o)
                if case["keep"]:
                    out("hidden", n, 2 * o)
        elif case["kind"] == "int8":
            out("y", n, case["n_out"])
        else:
            out("loss", n, of=torch.float32)
            if case["step"] == "both":
                out("grad", n, case["classes"])
        self.y = y


def prepare(case, seed):
    return State(case, _inputs(case, seed))


# ---- the framework's calls ---------------------------------------------------------------------------------------

_ACT = {"silu": 1, "gelu": 2}


def _build(s):
    """The argument structs that a program keeps, and its calls."""
    pkg = importlib.import_module("pulp-trainlib_amd")
    lib, case, x, y, n, keep = pkg.load(), s.case, s.x, s.y, s.case["n"], []

    def blob(data, diff, dim, rows=1):
        b = pkg.blob(data, diff, 1, rows, dim, rows * dim)
        keep.append(b)
        return ctypes.pointer(b)

    kind, dt = case["kind"], case["dtype"]
    if kind == "norm":
        a, c = pkg.RmsNormArgs(), case["dim"]
        a.eps = EPS
        if case["step"] == "bw":
            a.input, a.output = blob(x["x"], y["dx"], c), blob(None, x["dy"], c)
            if case["residual"]:  # x holds the sum; its gradient goes to both branches, in one buffer
                a.skip, a.sum = blob(None, y["dx"], c), blob(x["x"], x["dsum"], c)
            a.coeff = blob(x["w"], y["dw"], c)
            call = ("ptl_rms_norm_%s_bw_batched" % dt, (a, n))
        else:
            a.input, a.coeff, a.output = blob(x["x"], None, c), blob(x["w"], None, c), blob(y.get("y"), None, c)
            if case["residual"]:
                a.skip, a.sum = blob(x["skip"], None, c), blob(y["sum"], None, c)
            if case["step"] == "8bit":
                a.q_data, a.q_scale = pkg.addr(y["q"]), pkg.addr(y["scale"])
            call = ("ptl_rms_norm_%s_fw_batched" % dt, (a, n))
    elif kind == "gated":
        a, i, o = pkg.GatedLinearArgs(), case["n_in"], case["n_out"]
        a.activation = _ACT[case["act"]]
        back = case["step"] == "bw"
        a.input = blob(x["x"], y.get("dx"), i)
        a.coeff = blob(x["w"], y.get("dw"), i, 2 * o)
        if case["bias"]:
            a.bias, a.use_biases = blob(x.get("bias"), y.get("dbias"), 2 * o), 1
        if back or case["keep"]:
            a.hidden = blob(x["hidden"] if back else y["hidden"], y.get("dhidden"), 2 * o)
        a.output = blob(y.get("y"), x.get("dy"), o)
        call = ("ptl_gated_linear_%s_%s_batched" % (dt, case["step"]), (a, n))
    elif kind == "int8":
        a = pkg.MatMulInt8Args()
        a.A, a.B, a.C = pkg.addr(x["a"]), pkg.addr(x["b"]), pkg.addr(y["y"])
        a.A_scale, a.B_scale, a.bias = pkg.addr(x["a_scale"]), pkg.addr(x["b_scale"]), pkg.addr(x.get("bias"))
        a.N, a.M, a.K, a.USE_BIASES = n, case["n_out"], case["n_in"], case["bias"]
        call = ("ptl_mm_int8_%s" % dt, (a,))
    else:
        a = pkg.DistillArgs()
        a.output = blob(x["z"], y.get("grad"), case["classes"])
        a.teacher, a.classes, a.n_top = pkg.addr(x["teacher"]), pkg.addr(x["top"]), case["top"]
        a.temperature, a.weight = TEMPERATURE, _weight(case)
        a.wr_loss = pkg.addr(y["loss"])
        call = ("ptl_distill_%s_batched" % dt, (a, n, 2 if case["step"] == "both" else 0))
    keep.append(a)
    s.keep, s.lib = keep, lib
    s.calls = (getattr(lib, call[0]), (ctypes.byref(a),) + call[1][1:])


def _run_own(s):
    if s.calls is None:
        _build(s)
    f, args = s.calls
    if f(*args):
        raise RuntimeError("%s: %s" % (f.__name__, s.lib.ptl_last_error().decode()))
    y = s.y
    if "q" in y:  # the values that the 8 bits stand for
        torch.mul(y["q"], y["scale"][:, None], out=y["value"])
        return {"value": y["value"], "sum": y["sum"]} if "sum" in y else {"value": y["value"]}
    return y


# ---- the same in elementary operations ---------------------------------------------------------------------------

def _plain_norm(case, x):
    t = x["x"].dtype
    if case["step"] == "bw":
        s, w, dy = x["x"].float(), x["w"].float(), x["dy"].float()
        r = torch.rsqrt(s.square().mean(1, keepdim=True) + EPS)
        g = dy * w
        dx = r * (g - s * r.square() * (g * s).mean(1, keepdim=True))
        if case["residual"]:
            dx = dx + x["dsum"].float()
        return {"dx": dx.to(t), "dw": (dy * s * r).sum(0).to(t)}
    s, got = x["x"].float(), {}
    if case["residual"]:
        s = s + x["skip"].float()
        got["sum"] = s.to(t)
    v = s * torch.rsqrt(s.square().mean(1, keepdim=True) + EPS) * x["w"].float()
    if case["step"] == "8bit":
        scale = v.abs().amax(1, keepdim=True) / 127
        got["value"] = ((v / scale).round() * scale).to(torch.float16)
    else:
        got["y"] = v.to(t)
    return got


def _gate(g, act):
    """The activation and its derivative."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    c = math.sqrt(2 / math.pi)
    s = torch.sigmoid(2 * c * (g + 0.044715 * g ** 3))  # (1 + tanh(u)) / 2
    return g * s, s + g * s * (1 - s) * 2 * c * (1 + 3 * 0.044715 * g * g)


def _plain_gated(case, x):
    t, o = x["x"].dtype, case["n_out"]
    if case["step"] == "fw":
        h = x["x"].float() @ x["w"].float().t()
        if case["bias"]:
            h = h + x["bias"].float()
        y = _gate(h[:, :o], case["act"])[0] * h[:, o:]
        return {"y": y.to(t), "hidden": h.to(t)} if case["keep"] else {"y": y.to(t)}
    h, dy = x["hidden"].float(), x["dy"].float()
    f, df = _gate(h[:, :o], case["act"])
    dh = torch.cat([dy * h[:, o:] * df, dy * f], 1)
    got = {"dhidden": dh.to(t), "dx": (dh @ x["w"].float()).to(t), "dw": (dh.t() @ x["x"].float()).to(t)}
    if case["bias"]:
        got["dbias"] = dh.sum(0).to(t)
    return got


def _plain_int8(case, x):
    y = x["a"].float() @ x["b"].float().t()  # (sums of such values stay below 2^24, so they are exact)
    y = y * x["a_scale"][:, None] * x["b_scale"]
    if case["bias"]:
        y = y + x["bias"].float()
    return {"y": y.to(torch.float32 if case["dtype"] == "fp32" else torch.float16)}


def _plain_distill(case, x):
    at, there = x["top"].long().clamp(min=0), x["top"] >= 0
    z = x["z"].float() / TEMPERATURE
    e = z - z.amax(1, keepdim=True)
    log_q = e - torch.log(torch.exp(e).sum(1, keepdim=True))
    u = torch.where(there, x["teacher"].float() / TEMPERATURE, -math.inf)
    u = u - u.amax(1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(u)
    total = p.sum(1, keepdim=True)
    some = (total > 0).float()
    p = p / total.clamp(min=1e-30)
    log_p = u - torch.log(total.clamp(min=1e-30))
    weight = _weight(case)
    terms = torch.where(there, p * (log_p - torch.gather(log_q, 1, at)), 0.0)
    got = {"loss": terms.sum(1) * weight}
    if case["step"] == "both":
        grad = (torch.exp(log_q) * some).scatter_add_(1, at, torch.where(there, -p, 0.0))
        got["grad"] = (grad * (weight / TEMPERATURE)).to(x["z"].dtype)
    return got


_PLAIN = {"norm": _plain_norm, "gated": _plain_gated, "int8": _plain_int8, "distill": _plain_distill}


def run(state):
    if own:
        return _run_own(state)
    return _PLAIN[state.case["kind"]](state.case, state.x)


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------

def exact(case, seed):
    x = _inputs(case, seed)
    d = {k: v.double() for k, v in x.items()}
    kind, step = case["kind"], case.get("step")
    if kind == "norm":
        s = d["x"] + d["skip"] if "skip" in d else d["x"]
        rms = (s.pow(2).sum(1, keepdim=True) / case["dim"] + EPS).sqrt()
        hat = s / rms
        if step == "bw":
            g = d["dy"] * d["w"]
            dx = (g - hat * (g * hat).sum(1, keepdim=True) / case["dim"]) / rms
            return {"dx": dx + d["dsum"] if "dsum" in d else dx, "dw": (d["dy"] * hat).sum(0)}
        y = hat * d["w"]
        got = {"sum": s} if "skip" in d else {}
        if step == "8bit":
            unit = y.abs().max(1, keepdim=True).values / 127
            got["value"] = torch.round(y / unit) * unit
        else:
            got["y"] = y
        return got
    if kind == "gated":
        o = case["n_out"]
        if step == "fw":
            h = torch.mm(d["x"], d["w"].t().contiguous()) + (d["bias"] if "bias" in d else 0.0)
        else:
            h = d["hidden"]
        gate, up = h[:, :o], h[:, o:]
        if case["act"] == "silu":
            f = gate / (1 + torch.exp(-gate))
            df = f / gate.where(gate != 0, torch.ones_like(gate)) * (1 + gate - f)
            df = torch.where(gate != 0, df, torch.full_like(df, 0.5))
        else:
            th = torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate.pow(3)))
            f = 0.5 * gate * (1 + th)
            df = 0.5 * (1 + th) + 0.5 * gate * (1 - th * th) * math.sqrt(2 / math.pi) * (1 + 0.134145 * gate * gate)
        if step == "fw":
            return {"y": f * up, "hidden": h} if case["keep"] else {"y": f * up}
        dh = torch.cat((d["dy"] * up * df, d["dy"] * f), dim=1)
        got = {"dhidden": dh, "dx": torch.mm(dh, d["w"]), "dw": torch.mm(dh.t().contiguous(), d["x"])}
        if case["bias"]:
            got["dbias"] = dh.sum(0)
        return got
    if kind == "int8":
        y = torch.mm(d["a"], d["b"].t().contiguous()) * torch.outer(d["a_scale"], d["b_scale"])
        return {"y": y + d["bias"] if "bias" in d else y}
    n, v = case["n"], case["classes"]
    weight = _weight(case)
    log_q = d["z"] / TEMPERATURE
    log_q = log_q - torch.logsumexp(log_q, 1, keepdim=True)
    left_out = x["top"] < 0
    u = (d["teacher"] / TEMPERATURE).masked_fill(left_out, -math.inf)
    none = left_out.all(1, keepdim=True)
    log_p = (u - torch.logsumexp(u, 1, keepdim=True)).masked_fill(left_out, 0.0)
    p = torch.exp(log_p).masked_fill(left_out, 0.0)
    at = x["top"].long().masked_fill(left_out, 0)
    got = {"loss": weight * (p * (log_p - log_q.gather(1, at))).sum(1)}
    if step == "both":
        target = torch.zeros((n, v), dtype=torch.float64, device="cuda").scatter_add_(1, at, p)
        got["grad"] = weight / TEMPERATURE * (torch.exp(log_q) - target).masked_fill(none, 0.0)
    return got
