"""NaN in the operands of chunk attention (csrc/paged_chunk_attention.hip), E5M2: a row that sees a NaN score is NaN,
every other row is what the float64 restatement of test_gpu_paged_chunk.py gives, and neither depends on how many key
ranges the workspace allows."""
import numpy as np
import pytest
import torch

from test_gpu_paged_chunk import _problem, _reference, dev  # noqa: F401

pytestmark = pytest.mark.gpu

NAN = 0x7F


def _run(P, dev, size, kind, scale=None):
    """Through the C ABI with a workspace of `size` bytes (None: as many as the call asks for); fp32 or fp16 results."""
    from feather_amd import _native as N
    t = [torch.from_numpy(np.ascontiguousarray(P[k]).view(np.int32).copy()).to(dev) for k in ("q", "kc", "vc", "bt", "cu", "ctx")]
    shape = (len(P["ctx"]), P["total"], P["Hq"], P["Hkv"], P["d"])
    L, mb = N.lib(), P["bt"].shape[1]
    need = L.feather_paged_chunk_attn_scratch_bytes(*shape, mb * P["bs"], 0)
    size = need if size is None else min(size, need)
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device=dev)
    out = torch.full((P["total"], P["Hq"], P["d"]), 7.0, device=dev, dtype=torch.float32 if kind == N.CHUNK_OUT_F32 else torch.float16)
    N.check(L.feather_paged_chunk_attn_fp8(*[x.data_ptr() for x in t], out.data_ptr(), kind, 0, ws.data_ptr() if size else None, size,
                                           *shape, P["bs"], mb, P["kc"].shape[0], 0, 1, N.E5M2, P["d"] ** -0.5 if scale is None else float(scale),
                                           N.stream_ptr(dev)))
    torch.cuda.synchronize()
    return out.double().cpu(), need


def _agree(P, dev, orc, ranges=True):
    y, tol = _reference(P, orc, True)
    nan = torch.isnan(y)
    assert nan.any() and not nan.all()
    part = P["total"] * P["Hq"] * (P["d"] + 2) * 4
    for size in (None, 0, 2 * part + 16, 3 * part + 16):
        for kind in (0, 1):
            got, need = _run(P, dev, size, kind)
            assert (need > 0) == ranges
            assert torch.equal(torch.isnan(got), nan), f"workspace of {size} bytes"
            err = (got - y).abs()[~nan] - (tol + (2.0 ** -11 * y.abs() + 2.0 ** -25 if kind else 0))[~nan]
            assert err.max().item() <= 0


# lens, ctx, Hq, Hkv, d, bs, whether the call cuts its keys into ranges
SHAPES = [([3], [1538], 8, 2, 64, 16, True), ([3], [1538], 8, 2, 64, 12, True), ([2, 1], [1537, 40], 4, 2, 128, 16, True),
          ([3], [1538], 2, 2, 256, 16, True), ([2], [1537], 2, 1, 512, 16, True), ([5], [300], 8, 2, 64, 16, False),
          ([700], [900], 8, 2, 64, 16, True), ([700, 1], [900, 1030], 4, 2, 128, 16, True), ([700], [900], 4, 2, 256, 16, True),
          ([700], [900], 2, 1, 512, 6, True)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"d{s[4]}_bs{s[5]}_rows{sum(s[0])}_ctx{max(s[1])}")
def test_nan_in_a_query(dev, orc, shape):
    P = _problem(orc, 31, *shape[:6], "E5M2")
    P["q"].view(np.uint8).reshape(P["total"], P["Hq"], P["d"])[P["total"] // 2, P["Hq"] - 1, 5] = NAN
    _agree(P, dev, orc, shape[6])


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"d{s[4]}_bs{s[5]}_rows{sum(s[0])}_ctx{max(s[1])}")
def test_nan_in_a_key(dev, orc, shape):
    """Also where it is the only key of its range that a row sees (position 256 or 1536, the first of a range)."""
    lens, ctx, Hq, Hkv, d, bs = shape[:6]
    n, c = lens[0], ctx[0]
    for at in sorted({x for x in (256, 512, 768, 1536, c - 1, c - n + n // 2) if c - n < x < c}):
        P = _problem(orc, 32, *shape[:6], "E5M2")
        P["kc"].view(np.uint8).reshape(-1, Hkv, bs, d)[P["bt"][0, at // bs], 0, at % bs, 7] = NAN
        _agree(P, dev, orc, shape[6])


@pytest.mark.parametrize("code", [0x7C, 0xFC])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"d{s[4]}_bs{s[5]}_rows{sum(s[0])}_ctx{max(s[1])}")
def test_infinite_key(dev, orc, shape, code):
    """A score of +inf makes the row NaN (inf - inf), one of -inf a weight of zero, also where a range has no other."""
    lens, ctx, Hq, Hkv, d, bs = shape[:6]
    n, c = lens[0], ctx[0]
    for at in sorted({x for x in (256, 1536, c - n + n // 2) if c - n <= x < c}):
        P = _problem(orc, 33, *shape[:6], "E5M2")
        P["kc"].view(np.uint8).reshape(-1, Hkv, bs, d)[P["bt"][0, at // bs], 0, at % bs, 7] = code
        P["q"].view(np.uint8).reshape(P["total"], Hq, d)[0, 0, 7] = 0x3C          # both signs of scores, whatever the draw
        P["q"].view(np.uint8).reshape(P["total"], Hq, d)[lens[0] - 1, 0, 7] = 0x3C if code == 0x7C else 0xBC
        P["q"].view(np.uint8).reshape(P["total"], Hq, d)[lens[0] - 1, (Hq // Hkv) - 1, 7] = 0xBC if code == 0x7C else 0x3C
        if Hq // Hkv > 1:
            _agree(P, dev, orc, shape[6])
        else:                                              # one head per KV head: the last row has a score of -inf
            y, tol = _reference(P, orc, True)
            nan = torch.isnan(y)
            for size in (None, 0):
                got, _ = _run(P, dev, size, 0)
                assert torch.equal(torch.isnan(got), nan) and ((got - y).abs()[~nan] <= tol[~nan]).all()
