"""The 8-bit codes of AdamW's second moments at the bottom of their range: each is the nearest integer, but that a root below half a step that is not
0 has code 1.  u = 2^-24."""
import pytest
import torch

import test_gpu_adamw as ad
import transformer as tr
import tuning as tn

pytestmark = pytest.mark.gpu
U = tr.U


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_codes_of_small_second_moments(pkg, gpu, dt):
    """Gradients whose fourth roots of squares are spread evenly from 0 to 4 steps behind one of 255, in every block of 256."""
    n = 256 * 40 + 77
    c = ad.Case(pkg, dt, [n], lambda i: True, fresh=True)
    at = torch.arange(n)
    root = (at * 0.6180339887) % 4.0
    root[at % 256 == 5] = 255.0
    root[at % 256 == 9] = 0.0
    g = (root.double() ** 2 * 2.0 ** -10).to(tr.t_dtype(dt))  # (the root of a square's root: fp16 holds 2^-24 and above)
    c.host[0]["g"] = g
    c.dev[0]["g"][:] = g.cuda()
    o = c.run(t=1)[0]
    v = (1 - tn.f32(0.999)) * g.double() ** 2
    want = v ** 0.25
    top = torch.nn.functional.pad(want, (0, -n % 256)).view(-1, 256).amax(1)
    want = want * (255 / top).repeat_interleave(256)[:n]
    code = o["vq"].cpu().double()
    # (of a code of k, k times what the roots, the square's product and sum, the unit and the product with it are off: some 12 u)
    slack = want * 16 * U
    nearest = (code - want).abs() <= 0.5 + slack
    raised = (code == 1) & (want > 0) & (want < 0.5 + slack)
    assert (nearest | raised).all()
    assert ((code == 0) == (v == 0)).all() and int(((want > 1.45) & (want < 1.5)).sum()) > 50
    c.check([o], t=1)
