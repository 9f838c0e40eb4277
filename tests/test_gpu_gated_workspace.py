"""What workspace a gated layer's backward call can do with where it cannot grow: its shares of the biases' sums and its products' sums in one
place, one behind the other (the same bits as with more of it); products in fewer parts.  Each case in a process of its own, whose workspace is as
small as it is reserved, in a capture."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import transformer as tr

pytestmark = pytest.mark.gpu
# tokens, inputs, outputs, biases, workspace, whether the sums are in the same order: 16 MB of shares and 16 MB of sums; sums of 30 MB or none; 30 MB
# of shares and 30 MB of sums
CASES = [(1024, 256, 2048, 1, 16 << 20, True), (7385, 256, 3752, 0, 1, False), (7385, 256, 3752, 1, 31 << 20, True)]


def in_a_process(n, n_in, n_out, bias, room, same):
    import __graft_entry__ as ge
    pkg = ge.load_package()
    gpu = pkg.load()
    assert gpu.ptl_init(0) == 0 and gpu.ptl_reserve(room, 0) == 0
    r = lambda s, *sh: tr.dev(tr.rand(s, *sh, dt="fp16"))  # noqa: E731
    x, w, h, dy = r(1, n, n_in), r(2, 2 * n_out, n_in), r(3, n, 2 * n_out), r(4, n, n_out)
    out = [torch.full_like(t, 7) for t in (x, w, h) + ((w[:, 0],) if bias else ())]
    dx, dw, dh = out[:3]
    a, keep = tr.gated_args(pkg, n_in, n_out, 1, x=x, dx=dx, w=w, dw=dw, db=out[3] if bias else None, h=h, dh=dh, dy=dy)
    call = lambda: gpu.ptl_gated_linear_fp16_bw_batched(ctypes.byref(a), n)  # noqa: E731
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    gpu.ptl_set_stream(ctypes.c_void_p(side.cuda_stream))
    with torch.cuda.graph(graph, stream=side):
        rc = call()
    assert (rc, gpu.ptl_last_error()) == (0, b""), (rc, gpu.ptl_last_error())
    got = []
    for _ in range(3):
        for t in out:
            t.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got.append([t.clone() for t in out])
    gpu.ptl_set_stream(None)
    assert all(torch.equal(g, t) for step in got for g, t in zip(step, out))
    if same:
        assert gpu.ptl_reserve(256 << 20, 0) == 0 and call() == 0 and gpu.ptl_sync() == 0
        assert all(torch.equal(g, t) for g, t in zip(got[0], out))
    d, u, g = dy.double(), h[:, n_out:].double(), h[:, :n_out].double()  # and they are the gradients
    s = torch.sigmoid(g)
    ref = torch.cat([d * u * s * (1 + g * (1 - s)), d * g * s], 1)
    rel = lambda v, want: float((v.double() - want).norm() / want.norm())  # noqa: E731
    assert rel(dh, ref) < 1e-3 and rel(dx, ref @ w.double()) < 1e-3 and rel(dw, ref.t().contiguous() @ x.double()) < 1e-3
    assert not bias or rel(out[3], ref.sum(0)) < 1e-3
    print("finished", flush=True)


@pytest.mark.parametrize("case", CASES)
def test_captured_with_little_workspace(gpu, case):
    here = os.path.dirname(os.path.abspath(__file__))
    code = "import sys; sys.path[:0] = [%r, %r]; import test_gpu_gated_workspace as t; t.in_a_process(*%r)" % (here, os.path.dirname(here), case)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "finished" in r.stdout, r.stdout + r.stderr
