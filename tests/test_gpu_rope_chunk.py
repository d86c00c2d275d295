"""Rotary positions, quantisation and append of a chunk (csrc/rope_chunk.hip).  The rotated values against float64; the
codes exactly as quant_codes of the kernel's own fp32 values; the placement exactly, every other cache word untouched.

Tolerance of the rotated values.  cos and sin carry the angle's rounding to 32 bits (an angle of at most pi/4: 2^-25) and
the polynomials' 2^-23; two products, one sum and the amplitude's product round once each: below 2^-21 (|a| + |b|) *
amplitude, whatever the position."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    return torch.device("cuda:0")


def _words(t):
    return t.view(torch.int32).cpu().numpy().view(np.uint32)


def _rotate(x, pos, freq, amp, layout):
    """x [heads, d] float64 at one position; returns (rotated, bound)."""
    half = freq.size
    y, tol = x.copy(), np.zeros_like(x)
    if half:
        turns = np.longdouble(pos) * freq.astype(np.longdouble)
        t = 2 * np.pi * (turns - np.round(turns)).astype(np.float64)
        i = np.arange(half)
        a, b = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
        y[:, a] = amp * (x[:, a] * np.cos(t) - x[:, b] * np.sin(t))
        y[:, b] = amp * (x[:, b] * np.cos(t) + x[:, a] * np.sin(t))
        # the product position * freq in 64 bits is off by 2^-53 of the turns, the angle by 2 pi as much
        lim = (2.0 ** -21 + 2 * np.pi * np.abs(turns.astype(np.float64)) * 2.0 ** -52) * abs(amp) * (np.abs(x[:, a]) + np.abs(x[:, b])) + 1e-30
        tol[:, a], tol[:, b] = lim, lim
    return y, tol


CASES = [  # lens, start, nq, nkv, d, rot, bs
    ([1, 1, 1], [0, 5, 40], 4, 2, 64, 64, 16),
    ([3, 0, 17], [0, 9, 13], 5, 1, 64, 32, 4),
    ([40], [131000], 8, 2, 128, 128, 16),
    ([9, 2], [1000000, 7], 2, 2, 128, 64, 20),
    ([2, 5], [30, 1], 32, 8, 256, 96, 16),
    ([6], [11], 1, 1, 512, 512, 3),
    ([4], [3], 3, 1, 72, 8, 16),
    ([4], [3], 0, 2, 64, 16, 16),                       # no query heads: K and V only
    ([5], [2], 2, 1, 64, 0, 16),                        # nothing is rotated
    ([1] * 70, list(range(70)), 2, 1, 64, 64, 8),
]


@pytest.mark.parametrize("mode,src", [("E4M3", torch.float32), ("E5M2", torch.float16)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"d{c[4]}_rot{c[5]}_h{c[2]}x{c[3]}_bs{c[6]}_rows{sum(c[0])}")
def test_values_codes_and_placement(dev, orc, case, layout, mode, src):
    from feather_amd.routines.producers import rope_append_chunk, rotary_frequencies
    from oracle import decode_ref
    lens, start, nq, nkv, d, rot, bs = case
    print(f"rope chunk {case} {layout} {mode} {src}", flush=True)
    rng = np.random.default_rng(d + rot)
    n_seq, total, heads, dw = len(lens), sum(lens) + 3, nq + 2 * nkv, d // 4
    cu = (np.concatenate([[0], np.cumsum(lens)]) + 2).astype(np.int32)      # two rows in front, one behind
    freq = rotary_frequencies(rot, scaling="by_parts", factor=4.0, original_context=2048, device=dev) if rot else \
        torch.empty(0, dtype=torch.float64, device=dev)
    amp = 1.1386
    first = [s // bs for s in start]
    mb = max((s + n + bs - 1) // bs for s, n in zip(start, lens)) + 1
    need = [(s + n + bs - 1) // bs - f for s, n, f in zip(start, lens, first)]
    n_blocks = sum(need) + 3
    perm = rng.permutation(n_blocks)
    bt = np.full((n_seq, mb), -1, dtype=np.int32)
    at = 0
    for s in range(n_seq):
        bt[s, first[s]:first[s] + need[s]] = perm[at:at + need[s]]
        at += need[s]
    x = torch.from_numpy(rng.standard_normal((total, heads * d)).astype(np.float32)).to(src)
    kc0 = rng.integers(0, 2 ** 32, (n_blocks, nkv, bs, dw), dtype=np.uint64).astype(np.uint32)
    vc0 = rng.integers(0, 2 ** 32, (n_blocks, nkv, bs, dw), dtype=np.uint64).astype(np.uint32)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.int32).copy()).to(dev)
    kc, vc = t(kc0), t(vc0)
    args = (t(cu), t(np.array(start, np.int32)), t(bt))
    qp, after, status, f32 = rope_append_chunk(x.to(dev), *args, kc, vc, n_q_heads=nq, freq=freq, amplitude=amp, layout=layout,
                                               mode=mode, return_f32=True)
    assert status.cpu().tolist() == [0] * n_seq
    assert after.cpu().tolist() == [s + n for s, n in zip(start, lens)]
    f32 = f32.cpu().numpy()
    xd, fq = x.double().numpy().reshape(total, heads, d), freq.cpu().numpy()
    kw, vw = kc0.copy(), vc0.copy()
    for s in range(n_seq):
        for i in range(lens[s]):
            r, pos = int(cu[s]) + i, start[s] + i
            want, tol = _rotate(xd[r, :nq + nkv], pos, fq, amp, layout)
            assert (np.abs(f32[r, :nq + nkv] - want) <= tol).all()
            assert np.array_equal(f32[r, nq + nkv:], xd[r, nq + nkv:].astype(np.float32))
            blk, slot = bt[s, pos // bs], pos % bs
            kw[blk, :, slot] = decode_ref.quant_codes(f32[r, nq:nq + nkv], mode).reshape(nkv, dw)
            vw[blk, :, slot] = decode_ref.quant_codes(f32[r, nq + nkv:], mode).reshape(nkv, dw)
    assert np.array_equal(_words(kc), kw) and np.array_equal(_words(vc), vw)
    inner = slice(2, total - 1)
    if nq:
        assert np.array_equal(_words(qp)[inner].reshape(-1), decode_ref.quant_codes(f32[inner, :nq], mode))
        assert not _words(qp)[:2].any() and not _words(qp)[-1].any()
    # rows that are slices of a wider projection give the same words
    wide = torch.zeros((total, heads * d + 8), dtype=src)
    wide[:, 4:-4] = x
    k2, v2 = t(kc0), t(vc0)
    q2, _, _ = rope_append_chunk(wide.to(dev)[:, 4:-4], *args, k2, v2, n_q_heads=nq, freq=freq, amplitude=amp, layout=layout, mode=mode)
    assert np.array_equal(_words(q2), _words(qp)) and torch.equal(k2, kc) and torch.equal(v2, vc)


def test_positions_without_a_slot(dev, orc):
    """Rows before position 0, past the table and in entries that are not blocks are dropped one by one and reported."""
    from feather_amd.routines.producers import rope_append_chunk, rotary_frequencies
    rng = np.random.default_rng(2)
    lens, start, bs, mb, n_blocks, d = [4, 4, 4, 4, 4, 0, 3, 2], [-2, 14, 2, 0, 16, 7, -9, 15], 4, 4, 20, 64
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    bt = rng.permutation(20)[:32 % 21].astype(np.int32)
    bt = np.resize(rng.permutation(n_blocks), (8, mb)).astype(np.int32)
    perm = iter(rng.permutation(n_blocks))
    bt = np.full((8, mb), -1, np.int32)
    for s, e in [(0, 0), (1, 3), (2, 0), (3, 0), (7, 3)]:
        bt[s, e] = next(perm)
    bt[2, 1] = n_blocks                                    # one past the cache
    i32 = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(dev)
    kc0 = torch.from_numpy(rng.integers(-2 ** 31, 2 ** 31, (n_blocks, 1, bs, d // 4)).astype(np.int32)).to(dev)
    kc, vc = kc0.clone(), kc0.clone()
    qkv = torch.randn(int(cu[-1]), 3 * d, device=dev)
    qp, after, status, f32 = rope_append_chunk(qkv, i32(cu), i32(start), i32(bt), kc, vc, n_q_heads=1, freq=rotary_frequencies(64),
                                               return_f32=True)
    assert status.cpu().tolist() == [1, 1, 2, 0, 1, 0, 1, 1]
    assert after.cpu().tolist() == [0, 16, 4, 4, 16, 7, 0, 16]
    from oracle import decode_ref
    want = _words(kc0).copy()
    f = f32.cpu().numpy()
    for s in range(8):
        for i in range(lens[s]):
            pos = start[s] + i
            if 0 <= pos < mb * bs and 0 <= bt[s, pos // bs] < n_blocks:
                want[bt[s, pos // bs], 0, pos % bs] = decode_ref.quant_codes(f[cu[s] + i, 2], "E4M3")
    assert np.array_equal(_words(vc), want)
    assert np.array_equal(_words(qp).reshape(-1), decode_ref.quant_codes(f[:, :1], "E4M3"))


def test_one_row_is_the_decode_steps_append(dev, orc):
    """A chunk of one row at the plain frequencies writes the words of rope_append (positions whose 32-bit angle is exact
    enough that no code differs: position 0 and small ones are compared within one code step)."""
    from feather_amd.routines.producers import rope_append, rope_append_chunk, rotary_frequencies
    rng = np.random.default_rng(3)
    B, nq, nkv, d, bs = 5, 8, 2, 64, 16
    bt = torch.arange(B * 4, dtype=torch.int32, device=dev).view(B, 4)
    ctx = torch.tensor([0, 1, 17, 40, 63], dtype=torch.int32, device=dev)
    cu = torch.arange(B + 1, dtype=torch.int32, device=dev)
    qkv = torch.from_numpy(rng.standard_normal((B, (nq + 2 * nkv) * d)).astype(np.float32)).to(dev)
    z = lambda: torch.zeros((B * 4, nkv, bs, d // 4), dtype=torch.int32, device=dev)
    k1, v1, k2, v2 = z(), z(), z(), z()
    q1, a1, s1, f1 = rope_append(qkv, ctx, bt, k1, v1, n_q_heads=nq, return_f32=True)
    q2, a2, s2, f2 = rope_append_chunk(qkv, cu, ctx, bt, k2, v2, n_q_heads=nq, freq=rotary_frequencies(d), return_f32=True)
    assert torch.equal(a1, a2) and torch.equal(s1, s2) and torch.equal(v1, v2)
    assert (f1 - f2).abs().max().item() <= 2e-5 * f1.abs().max().item()
    assert np.array_equal(_words(q1)[0], _words(q2)[0])


def test_refusals(dev):
    from feather_amd.routines.producers import rope_append_chunk, rotary_frequencies
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)
    kc, f = i32(4, 2, 16, 16), rotary_frequencies(64)
    ok = dict(qkv=torch.zeros(3, 8 * 64, device=dev), cu_seqlens=i32(2), start_pos=i32(1), block_tables=i32(1, 2), k_cache=kc,
              v_cache=i32(4, 2, 16, 16), n_q_heads=4, freq=f)
    rope_append_chunk(**ok)
    for bad in (dict(qkv=torch.zeros(3, 7 * 64, device=dev)), dict(qkv=torch.zeros(3, 8 * 64, device=dev, dtype=torch.float64)),
                dict(cu_seqlens=i32(3)), dict(start_pos=i32(2)), dict(block_tables=i32(2, 2)), dict(block_tables=i32(1, 2).long()),
                dict(k_cache=i32(4, 2, 16, 32)[..., ::2]), dict(v_cache=i32(4, 2, 8, 16)), dict(freq=f.float()),
                dict(freq=f.cpu()), dict(freq=rotary_frequencies(72)), dict(freq=rotary_frequencies(12)), dict(layout="both"),
                dict(amplitude=float("nan")), dict(n_q_heads=-1)):
        with pytest.raises(ValueError):
            rope_append_chunk(**{**ok, **bad})
    with pytest.raises(NotImplementedError):
        rope_append_chunk(**ok, mode="E2M5")
    q, after, status = rope_append_chunk(**{**ok, "cu_seqlens": i32(1), "start_pos": i32(0), "block_tables": i32(0, 2)})
    assert not q.view(torch.int32).any() and after.numel() == status.numel() == 0          # rows of no sequence
    assert rope_append_chunk(**{**ok, "qkv": torch.zeros(0, 8 * 64, device=dev)})[0].shape == (0, 4, 16)
