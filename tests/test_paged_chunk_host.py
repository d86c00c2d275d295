"""Host-side checks of the chunk operators (no GPU): argument checks of the C ABI and of the wrappers, and CPU models of
the device's index arithmetic."""
import ctypes
import math

import numpy as np
import pytest
import torch


def test_chunk_attention_argument_checks():
    from feather_amd import _native as N
    L = N.lib()

    def call(n_seq=1, total=4, Hq=8, Hkv=4, d=64, bs=16, mb=4, nb=8, maxq=0, causal=1, mode=N.E5M2, scale=0.1, kind=0, fill=1,
             ptrs=(None,) * 7, scratch=None, nbytes=0):
        return L.feather_paged_chunk_attn_fp8(*ptrs, kind, fill, scratch, nbytes, n_seq, total, Hq, Hkv, d, bs, mb, nb, maxq,
                                              causal, mode, scale, None)
    assert call(mode=5) == N.EMODE
    assert call(total=0) == N.OK and call(n_seq=0, fill=0) == N.OK
    for bad in (dict(n_seq=-1), dict(total=-1), dict(Hq=0), dict(Hkv=0), dict(bs=0), dict(mb=-1), dict(nb=0), dict(maxq=-1),
                dict(causal=2), dict(fill=2), dict(kind=3), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
                dict(scale=math.inf), dict(nbytes=-1), dict()):
        assert call(**bad) == N.EINVAL, bad                                # the last: null pointers
    for bad in (dict(Hq=6), dict(d=32), dict(d=96), dict(mb=1 << 29, bs=4), dict(total=1 << 30), dict(total=1 << 27, Hq=64),
                dict(nb=(1 << 31) - 1, bs=16)):
        assert call(**bad) == N.ESHAPE, bad
    assert call(ptrs=(4, 16, 16, 4, 4, 4, 16)) == N.EINVAL and b"misaligned" in L.feather_last_error()
    assert call(ptrs=(16, 8, 16, 4, 4, 4, 16)) == N.EINVAL
    assert call(ptrs=(16, 16, 16, 4, 4, 4, 8)) == N.EINVAL
    assert call(ptrs=(16, 16, 16, 4, 4, 4, 16), scratch=8, nbytes=64) == N.EINVAL
    size = L.feather_paged_chunk_attn_scratch_bytes
    assert size(0, 4, 8, 4, 64, 100, 0) == 0 and size(1, 4, 8, 4, 64, 100, 0) == 0 and size(-1, 4, 8, 4, 64, 100, 0) == 0
    z, rest = divmod(size(1, 4, 8, 4, 64, 100000, 4), 4 * 8 * 66 * 4)      # whole ranges of (d + 2) floats per row and head
    assert rest == 16 and z > 1
    assert size(1, 1 << 20, 8, 4, 64, 100000, 0) == 0                       # enough tiles to fill the chip
    for n_seq in (1, 3, 100, 5000):                                         # never out of proportion, whatever the lengths
        for rows in (n_seq, 10 * n_seq, 1000 * n_seq, 1 << 20):
            for d in (64, 128, 256, 512):
                for hint in (0, 1, 64, rows):
                    assert size(n_seq, rows, 32, 4, d, 1 << 20, hint) < 1 << 30
    for d in (64, 128, 256, 512):                                           # a row of more columns than a narrow tile has: no
        assert size(16, 4111, 64, 1, d, 1 << 20, 4096) < 1 << 30            # sequence is short, none gets room for one


def test_rope_chunk_argument_checks():
    from feather_amd import _native as N
    L = N.lib()

    def call(f16=0, stride=None, rot=64, layout=0, fill=1, n_seq=1, total=4, nq=4, nkv=2, d=64, bs=16, mb=4, nb=8, mode=N.E4M3,
             p=(None,) * 11):
        return L.feather_rope_append_chunk(p[0], f16, (nq + 2 * nkv) * d if stride is None else stride, p[1], p[2], p[3], p[4],
                                           1.0, rot, layout, p[5], p[6], p[7], p[8], p[9], p[10], fill, n_seq, total, nq, nkv,
                                           d, bs, mb, nb, mode, None)
    assert call(mode=3) == N.EMODE
    for bad in (dict(f16=2), dict(layout=2), dict(fill=3), dict(n_seq=-1), dict(total=-1), dict(nq=-1), dict(nkv=0), dict(bs=0),
                dict(mb=-1), dict(nb=0), dict()):
        assert call(**bad) == N.EINVAL, bad
    for bad in (dict(d=60), dict(rot=72), dict(rot=12), dict(rot=-8), dict(d=1024, rot=520), dict(stride=511), dict(stride=514),
                dict(mb=1 << 30, bs=4), dict(total=1 << 30)):
        assert call(**bad) == N.ESHAPE, bad
    assert call(n_seq=0, total=0) == N.OK
    assert call(p=(8, 4, 4, 4, 8, 8, 8, 8, 4, 4, 16)) == N.EINVAL and b"misaligned" in L.feather_last_error()


    assert call(p=(16, 4, 4, 4, 8, 8, 8, 4, 4, 4, 16)) == N.EINVAL                   # words of a row are stored in pairs


def test_cache_pool_argument_checks():
    from feather_amd import _native as N
    L = N.lib()
    arr = (ctypes.c_void_p * 2)(16, 32)
    odd = (ctypes.c_void_p * 2)(16, 8)

    def fork(caches=arr, n=2, block=64, n_seq=1, mb=2, bs=16, nb=8, p=(4, 4, 4, 4, None, 8, 8, 8, None, 4)):
        return L.feather_paged_cache_fork(ctypes.addressof(caches) if caches is not None else None, n, block, *p, n_seq, mb, bs, nb, None)
    assert fork(caches=None) == N.EINVAL and fork(caches=odd) == N.EINVAL and fork(n=-1) == N.EINVAL
    assert fork(block=24) == N.ESHAPE and fork(block=0) == N.ESHAPE and fork(nb=0) == N.ESHAPE and fork(nb=(1 << 22) + 1) == N.ESHAPE
    assert fork(n_seq=-1) == N.EINVAL and fork(bs=0) == N.EINVAL and fork(n_seq=8193) == N.ESHAPE and fork(mb=1 << 28, bs=64) == N.ESHAPE
    assert fork(p=(None, 4, 4, 4, None, 8, 8, 8, None, 4)) == N.EINVAL
    assert fork(p=(4, 4, 4, 4, None, 4, 8, 8, None, 4)) == N.EINVAL and b"tables_out is block_tables" in L.feather_last_error()
    assert fork(p=(4, 4, 4, 4, None, 8, 4, 8, None, 4)) == N.EINVAL and fork(p=(4, 4, 4, 4, None, 8, 8, 4, None, 4)) == N.EINVAL
    assert fork(p=(4, 4, 4, 4, 2, 8, 8, 8, None, 4)) == N.EINVAL

    def compact(caches=arr, n=2, block=64, entries=4, nb=8, p=(4, 4, 8, 8, 8, 8, 4)):
        return L.feather_paged_cache_compact(ctypes.addressof(caches) if caches is not None else None, n, block, *p, entries, nb, None)
    assert compact(caches=odd) == N.EINVAL and compact(block=8) == N.ESHAPE and compact(nb=0) == N.ESHAPE
    assert compact(entries=-1) == N.EINVAL and compact(p=(None, 4, 8, 8, 8, 8, 4)) == N.EINVAL
    assert compact(p=(4, 4, 8, 4, 8, 8, 4)) == N.EINVAL and compact(p=(4, 4, 8, 8, 8, 8, 2)) == N.EINVAL
    assert L.feather_paged_cache_fork_scratch_bytes(-1, 4) == 0 and L.feather_paged_cache_compact_scratch_bytes(-1) == 0


def test_wrappers_refuse_before_any_launch():
    from feather_amd.routines.paged_attention import paged_chunk_attention_fp8_acc_fp32_gpu
    from feather_amd.routines.paged_cache import paged_cache_compact, paged_cache_fork
    from feather_amd.routines.producers import rope_append_chunk, rotary_frequencies
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    kc = i32(4, 2, 16, 16)
    with pytest.raises(ValueError):                          # host tensors
        paged_chunk_attention_fp8_acc_fp32_gpu(i32(3, 4, 16), kc, kc, i32(1, 2), i32(2), i32(1))
    with pytest.raises(NotImplementedError):
        paged_chunk_attention_fp8_acc_fp32_gpu(i32(3, 4, 16), kc, kc, i32(1, 2), i32(2), i32(1), mode="E3M4")
    with pytest.raises(ValueError):
        rope_append_chunk(torch.zeros(3, 8 * 64), i32(2), i32(1), i32(1, 2), kc, kc, n_q_heads=4,
                          freq=rotary_frequencies(64, device="cpu"))
    with pytest.raises(ValueError):
        paged_cache_fork([kc], i32(1, 2), i32(1), i32(4), i32(1))
    with pytest.raises(ValueError):
        paged_cache_compact([kc], i32(1, 2), i32(4))
    for kw in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=8, theta=0.0), dict(rot_dim=8, factor=-1.0),
               dict(rot_dim=8, scaling="more"), dict(rot_dim=8, scaling="by_parts"), dict(rot_dim=2, scaling="base"),
               dict(rot_dim=8, scaling="by_parts", original_context=100, low=4.0, high=4.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(device="cpu", **kw)


def test_rotary_frequencies():
    from feather_amd.routines.producers import rotary_frequencies
    j = np.arange(32)
    plain = 10000.0 ** (-2 * j / 64) / (2 * np.pi)
    f = lambda **kw: rotary_frequencies(64, device="cpu", **kw).numpy()
    assert np.allclose(f(), plain, rtol=1e-14, atol=0)
    assert np.allclose(f(scaling="linear", factor=4.0), plain / 4, rtol=1e-14, atol=0)
    base = f(scaling="base", factor=8.0)
    assert base[0] == plain[0] and abs(base[-1] * 8 / plain[-1] - 1) < 1e-12      # the slowest pair by the whole factor
    parts = f(scaling="by_parts", factor=8.0, original_context=4096, low=1.0, high=32.0)
    turns = 4096 * plain
    assert np.array_equal(parts[turns >= 32], f()[turns >= 32])
    assert np.allclose(parts[turns <= 1], plain[turns <= 1] / 8, rtol=1e-14, atol=0)
    assert (np.diff(parts) < 0).all()


def test_division_by_the_block_size():
    """pos / block_size as the kernels compute it: umulhi(2 pos, m) >> s with m = floor(2^(31 + s) / size) + 1."""
    rng = np.random.default_rng(0)
    for size in [1, 2, 3, 5, 6, 7, 12, 16, 20, 31, 32, 33, 100, 255, 1000, 65535, 65537, (1 << 29) - 1, 1 << 29]:
        s = 0
        while (1 << s) < size:
            s += 1
        m = (1 << (31 + s)) // size + 1
        assert m < 1 << 32
        pos = np.unique(np.concatenate([rng.integers(0, 1 << 30, 2000), np.arange(300), (1 << 30) - 1 - np.arange(300)] +
                                       [k * size + np.array([-1, 0, 1]) for k in range(1, 50) if k * size + 1 < 1 << 30]))
        got = [((2 * int(p)) * m >> 32) >> s for p in pos]
        assert got == [int(p) // size for p in pos]


def test_tile_slots_cover_every_column_once():
    """Tile slots of the chunk attention: slot -> (sequence, tile) without lengths on the host."""
    rng = np.random.default_rng(1)
    for _ in range(200):
        n_seq, group, qt = int(rng.integers(1, 90)), int(rng.integers(1, 25)), int(rng.choice([16, 32, 64, 128, 256]))
        lens = rng.integers(0, rng.choice([2, 9, 200]), n_seq)
        cu = np.concatenate([[0], np.cumsum(lens)]) + int(rng.integers(0, 5))
        total = int(cu[-1]) + int(rng.integers(0, 4))
        slots = total * group // qt + n_seq
        first = [int(cu[s]) * group // qt + s for s in range(n_seq)]
        seen = set()
        for slot in range(slots):
            below = sum(f <= slot for f in first)
            if below == 0:
                continue
            s = below - 1
            tile = slot - first[s]
            if tile < -(-int(lens[s]) * group // qt):
                seen.add((s, tile))
        want = {(s, t) for s in range(n_seq) for t in range(-(-int(lens[s]) * group // qt))}
        assert seen == want
