"""Scores far beyond what fp32 resolves to a fraction of a step in the exponent (csrc/paged_chunk_attention.hip): up to the
largest finite codes in q and K the result is finite and the softmax of the scores.

The keys are built so that the scores' own fp32 rounding does not decide: all keys with the same codes have the same score
bit for bit, and the others are smaller by far more than their rounding.  The weights are then 1 / n for the n largest and 0
(below 2^-100) for the rest, whatever the score; what remains is the fp16 rounding of equal P, which the quotient takes out,
and fp32 sums of n values: (n + 2) 2^-24 max|V|, n <= 2000."""
import numpy as np
import pytest
import torch

from test_gpu_chunk_nan import _run
from test_gpu_paged_chunk import _call, _problem, dev  # noqa: F401

pytestmark = pytest.mark.gpu

SHAPES = [(64, [2], [1500]), (64, [300], [900]), (128, [2], [1500]), (128, [150], [900]), (256, [3], [1500]), (256, [80], [900]),
          (512, [2], [700]), (512, [40], [700])]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"d{s[0]}_rows{s[1][0]}")
@pytest.mark.parametrize("mode,code", [("E5M2", 0x50), ("E5M2", 0x5C), ("E5M2", 0x64), ("E5M2", 0x6B), ("E5M2", 0x73), ("E5M2", 0x7B),
                                       ("E4M3", 0x60), ("E4M3", 0x6D), ("E4M3", 0x7E)])   # 2^5, 2^8 .. 57344; 2^5, 104, 448
@pytest.mark.parametrize("sign", [1, -1])
def test_equal_large_scores(dev, orc, shape, mode, code, sign):
    """Keys of the row's own code (times `sign`); every seventh has half of it from the middle on."""
    d, lens, ctx = shape
    P = _problem(orc, 8, lens, ctx, 4, 2, d, 16, mode)
    half = code - (4 if mode == "E5M2" else 8)
    n, c = lens[0], ctx[0]
    P["q"].view(np.uint8)[...] = code
    P["kc"].view(np.uint8)[...] = code if sign > 0 else code | 0x80
    small = np.zeros(c, bool)
    small[c // 2::7] = True
    for pos in np.flatnonzero(small):
        P["kc"].view(np.uint8).reshape(-1, 2, 16, d)[P["bt"][0, pos // 16], :, pos % 16] = half | (0x80 if sign < 0 else 0)
    table = orc.dec_table(mode).astype(np.float64)
    pos = np.arange(c)
    V = table[P["vc"][P["bt"][0, pos // 16], :, pos % 16].view(np.uint8)].reshape(c, 2, d)
    best = ~small if sign > 0 else small                     # the weights of the others vanish
    y = np.zeros((n, 4, d))
    for i in range(n):
        seen = pos <= c - n + i
        pick = seen & best if (seen & best).any() else seen
        y[i] = np.repeat(V[pick].mean(0), 2, axis=0)
    lim = (c + 2) * 2.0 ** -24 * np.abs(V).max()
    assert d ** 0.5 * 512 * 1.44 > 100                        # the least gap, codes of 2^5: d * 2^9 / sqrt(d)
    runs = [_run(P, dev, size, 0)[0] for size in (0, None)] if mode == "E5M2" else [_call(P, dev, True).double().cpu()]
    for got in runs:
        got = got.numpy()
        assert np.isfinite(got).all()
        assert np.abs(got - y).max() <= lim, f"{np.abs(got - y).max()} beyond {lim}"
