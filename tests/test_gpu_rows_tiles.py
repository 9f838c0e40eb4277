"""The large tiles of the products of rows at every number of slabs of k that their loop tells apart - one and two, as many as lie in LDS, one
more, many -, with last slabs that are whole and that are not."""
import pytest
import torch

import test_gpu_act_linear as dense
import test_gpu_gated as gated
import test_gpu_mm_int8 as int8
import transformer as tr

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,m,k,tile", [(4100, 4100, 64, 128128), (4100, 4100, 128, 128128), (2050, 2050, 2000, 128128)] +
                         [(4100, 2050, k, 256256) for k in (144, 256, 272, 384, 400, 512, 640, 1040)])
def test_integers(pkg, gpu, n, m, k, tile):
    A, B = int8.ints(n, n, k), int8.ints(m, m, k)
    sa, sb = tr.rand(1, n).abs() * 0.001 + 0.0001, tr.rand(2, m).abs() * 0.02 + 0.001
    int8.check(pkg, gpu, "fp16", A, B, sa, sb, tr.rand(3, m, dt="fp16"))
    assert gpu.ptl_last_gemm_tile() == tile


@pytest.mark.parametrize("n,n_in,n_out,tile", [(4100, 136, 2050, 128128), (4100, 192, 2050, 128128), (4100, 200, 2050, 128128), (4100, 256, 2050, 128128),
                                               (4100, 328, 2050, 256256), (4100, 512, 2050, 256256), (4100, 520, 2050, 256256)])
def test_gated(pkg, gpu, n, n_in, n_out, tile):
    x, w, b = gated.inputs(n, "fp16", n, n_in, n_out, 1)
    gated.check_forward("fp16", "silu", x, w, b, *gated.forward(pkg, gpu, "fp16", "silu", x, w, b))
    assert gpu.ptl_last_gemm_tile() == tile


@pytest.mark.parametrize("n,n_in,n_out,tile", [(2050, 1000, 2050, 128256), (2050, 1024, 2050, 128256), (4100, 1000, 2050, 256256), (4100, 960, 2050, 256256),
                                               (3000, 1000, 1500, 128256)])
def test_dense(pkg, gpu, n, n_in, n_out, tile):
    x, w, b, s = dense.inputs(n, "fp16", n, n_in, n_out)
    dense.check_forward("fp16", "silu", x, w, b, s, *dense.forward(pkg, gpu, "fp16", "silu", x, w, b, s))
    assert gpu.ptl_last_gemm_tile() == tile


@pytest.mark.parametrize("n,n_in,n_out", [(64, 8008, 8001), (100, 8200, 5000), (128, 6200, 5200), (129, 8200, 4000), (191, 8200, 3400)])
def test_dense_gradients_of_few_slabs(pkg, gpu, n, n_in, n_out):
    """Tiles of 256 x 128 whose k is one, two or three slabs."""
    x, w, _, _ = dense.inputs(n, "fp16", n, n_in, n_out)
    h, dy = tr.rand(n + 5, n, n_out, scale=1.5, dt="fp16"), tr.rand(n + 6, n, n_out, scale=0.5, dt="fp16")
    dense.check_backward("fp16", "relu", x, w, h, dy, *dense.backward(pkg, gpu, "fp16", "relu", x, w, h, dy, 1))
    torch.cuda.empty_cache()
