"""Chunk attention of more sequences than a wave looks at per step (64), against the float64 restatement of
test_gpu_paged_chunk.py: tiles through LDS, streamed columns, key ranges, empty sequences across the borders."""
import numpy as np
import pytest

from test_gpu_paged_chunk import _call, _check, _problem, _reference, dev  # noqa: F401

pytestmark = pytest.mark.gpu


def _lens(n, long, empty, rng, most):
    lens = rng.integers(1, most + 1, n)
    lens[list(empty)] = 0
    for s, rows in long.items():
        lens[s] = rows
    return lens.tolist()


# sequences, long runs, empty sequences, rows of the others, query heads, KV heads, head dim, page, longest context
CASES = [
    (65, {64: 200}, (0, 31, 63), 1, 8, 2, 64, 16, 700),
    (65, {}, (63,), 4, 4, 1, 64, 16, 1500),
    (128, {63: 150, 64: 90}, range(60, 63), 3, 4, 1, 64, 12, 400),
    (128, {127: 300}, range(62, 67), 1, 4, 1, 128, 16, 900),
    (130, {2: 130, 65: 77, 129: 140}, range(64, 65), 5, 4, 1, 64, 16, 1500),
    (130, {64: 100}, (), 2, 2, 1, 128, 16, 1300),
    (129, {128: 70}, range(63, 128, 2), 2, 2, 1, 256, 16, 600),
    (66, {65: 50}, (64,), 2, 2, 1, 512, 16, 600),
    (193, {}, range(128, 192), 3, 8, 1, 64, 16, 1200),
    (1100, {}, (), 1, 4, 1, 64, 16, 40),
    (1100, {1050: 260}, range(1020, 1030), 1, 4, 1, 64, 16, 300),
]


@pytest.mark.parametrize("mode", ["E4M3", "E5M2"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"n{c[0]}_d{c[6]}_long{len(c[1])}_ctx{c[8]}")
def test_many_sequences(dev, orc, case, mode):
    n, long, empty, most, Hq, Hkv, d, bs, top = case
    print(f"many sequences {case} {mode}", flush=True)
    rng = np.random.default_rng(n + d)
    lens = _lens(n, long, empty, rng, most)
    ctx = [max(a, int(rng.integers(1, top + 1))) for a in lens]
    ctx[n // 2] = top
    P = _problem(orc, 3, lens, ctx, Hq, Hkv, d, bs, mode, head=1, tailrows=2)
    for causal in (True, False):
        y, tol = _reference(P, orc, causal)
        for hint in (None, max(lens)):
            got = _call(P, dev, causal, max_q_len=hint)
            _check(got, y, tol)
            assert not got[:1].any() and not got[-2:].any()
