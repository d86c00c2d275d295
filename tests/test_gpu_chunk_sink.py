"""Small weights beside a dominating one in chunk attention (csrc/paged_chunk_attention.hip): a key of value zero takes nearly
all of the softmax, and the result is what the many small weights of the others give.

Tolerance.  The kernels round P to fp16 with the largest P at 2^8 or above, so a P off by more than 2^-11 of its value is a
subnormal half, off by at most 2^-25, which is 2^-33 of the largest P.  With A = sum_k P |V| / sum_k P as in
test_gpu_paged_chunk.py the result is off by at most (2 * 2^-11 + 2e-5) A + n 2^-33 max|V| for n keys (the 2e-5 is the scores'
and the sums' fp32).  Weights of 2^-25.2 of the largest: the second term is 2^-7.8 of the result."""
import numpy as np
import pytest
import torch

from test_gpu_chunk_nan import _run
from test_gpu_paged_chunk import _problem, _reference, dev  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [14.5, 20.0, 22.3, 24.3, 25.2, 29.0, 31.5])
@pytest.mark.parametrize("d,lens,ctx", [(64, [2], [2000]), (64, [300], [2000]), (128, [2], [2000]), (128, [150], [2000]),
                                        (256, [2], [1500]), (256, [80], [1500]), (512, [2], [1000]), (512, [40], [1000])])
def test_many_small_weights_beside_a_large_one(dev, orc, d, lens, ctx, bits):
    """Every weight but one is 2^-bits of the largest, whose V is zero; the large one is the first key, or one in the middle."""
    for at in (0, ctx[0] // 2 - 3):
        P = _problem(orc, 5, lens, ctx, 4, 2, d, 16, "E5M2")
        P["q"][:] = orc.pack_fp8(np.full(4, 1.0, np.float16), "E5M2")[0]
        P["kc"][:] = orc.pack_fp8(np.full(4, 0.5, np.float16), "E5M2")[0]
        blk, slot = P["bt"][0, at // 16], at % 16
        P["kc"][blk, :, slot] = orc.pack_fp8(np.full(4, 1.0, np.float16), "E5M2")[0]
        vc = P["vc"].view(np.uint8)
        vc[...] = np.minimum(vc & 0x7F, 0x40)                  # positive, at most 2: the result is a sum without cancellation
        P["vc"][P["bt"][0, 0], :, 1, 0] = 0x40404040           # both heads have that largest value
        P["vc"][blk, :, slot] = 0
        scale = bits * np.log(2.0) / (d / 2)
        y, tol = _reference(P, orc, True, scale=scale)
        tol = tol + ctx[0] * (2.0 ** -33 - 2.0 ** -25) * 2.0
        for size in (0, None):
            got, _ = _run(P, dev, size, 0, scale=scale)
            worst = ((got - y).abs() / tol).max().item()
            print(d, lens, bits, at, size, "error over bound", worst, "relative", ((got - y).abs() / y.abs()).max().item())
            assert worst <= 1


@pytest.mark.parametrize("scale", [1e-30, 1e-38, 3e-41])
@pytest.mark.parametrize("d,lens,ctx", [(64, [2], [1500]), (64, [300], [900]), (128, [150], [900]), (256, [3], [1500]), (256, [80], [1500]), (512, [40], [1000])])
def test_scales_that_leave_all_weights_equal(dev, orc, d, lens, ctx, scale):
    """Down to subnormal scales the result is the mean of the visible values, in one key range and in several."""
    P = _problem(orc, 6, lens, ctx, 4, 2, d, 16, "E5M2")
    y, tol = _reference(P, orc, True, scale=scale)
    for size in (0, None):
        got, _ = _run(P, dev, size, 0, scale=scale)
        assert ((got - y).abs() <= tol).all(), f"workspace of {size} bytes"
