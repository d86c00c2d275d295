"""Attention of a chunk of new rows over the paged cache (csrc/paged_chunk_attention.hip) against a float64
restatement: codes decoded by the oracle's table, visible keys gathered position by position, softmax in float64.

Tolerance.  Scores and sums are fp32; P is rounded to fp16 (half a step, 2^-11 of the value) in the numerator and in the
denominator alike, so with A = sum_k P |V| / sum_k P the result is off by at most 2 * 2^-11 A; P below 2^-14 is a
subnormal half, off by at most 2^-25 absolute where the largest P is at least 1 (each of n keys: n 2^-25 max|V|); the
fp32 score of d exact products is off by about sqrt(d) 2^-24 of the sum of their magnitudes, below 2e-5 for these inputs
(d <= 512, normal values).  A fp16 result adds half a step, 2^-11 |y| + 2^-25."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    return torch.device("cuda:0")


def _codes(rng, shape, mode, orc, spread=1.0):
    x = (rng.standard_normal(shape) * spread).astype(np.float16)
    return orc.pack_fp8(x, mode).reshape(*shape[:-1], shape[-1] // 4)


def _problem(orc, seed, lens, ctx, Hq, Hkv, d, bs, mode, head=0, tailrows=0, max_blocks=None, spread=1.0):
    """Random rows, caches and tables; every cache slot that no context covers holds the code 0x7F (NaN in E5M2, 480 in
    E4M3) and table entries past a context are no blocks."""
    rng = np.random.default_rng(seed)
    n_seq = len(lens)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32) + head
    total = int(cu[-1]) + tailrows
    need = [-(-max(c, 0) // bs) for c in ctx]
    mb = max_blocks or max(max(need, default=0), 1)
    n_blocks = sum(need) + 2
    perm = rng.permutation(n_blocks)
    bt = np.full((n_seq, mb), -1, dtype=np.int32)
    at = 0
    used = np.zeros((n_blocks, bs), dtype=bool)
    for s, n in enumerate(need):
        bt[s, :n] = perm[at:at + n]
        for i in range(n):
            used[bt[s, i], :max(0, min(bs, ctx[s] - i * bs))] = True
        at += n
    kc = _codes(rng, (n_blocks, Hkv, bs, d), mode, orc)
    vc = _codes(rng, (n_blocks, Hkv, bs, d), mode, orc)
    for c in (kc, vc):
        c.transpose(0, 2, 1, 3)[~used] = 0x7F7F7F7F
    return dict(q=_codes(rng, (total, Hq, d), mode, orc, spread), kc=kc, vc=vc, bt=bt, cu=cu,
                ctx=np.array(ctx, dtype=np.int32), Hq=Hq, Hkv=Hkv, d=d, bs=bs, mode=mode, total=total)


def _reference(P, orc, causal, scale=None):
    """(y, bound of the error) in float64, [total, Hq, d]; rows outside every sequence are zero."""
    d, bs, mode, Hkv = P["d"], P["bs"], P["mode"], P["Hkv"]
    G = P["Hq"] // Hkv
    scale = d ** -0.5 if scale is None else scale
    table = torch.from_numpy(orc.dec_table(mode).astype(np.float64))
    dec = lambda w: table[torch.from_numpy(np.ascontiguousarray(w).view(np.uint8).astype(np.int64))]
    n_blocks, mb = P["kc"].shape[0], P["bt"].shape[1]
    y = torch.zeros((P["total"], P["Hq"], d), dtype=torch.float64)
    tol = torch.zeros_like(y)
    for s in range(len(P["ctx"])):
        r0, r1 = int(P["cu"][s]), int(P["cu"][s + 1])
        n, ctx = r1 - r0, int(min(max(P["ctx"][s], 0), mb * bs))
        if n == 0 or ctx == 0:
            continue
        pos = np.arange(ctx)
        blk = P["bt"][s, pos // bs]
        blk = np.where((blk < 0) | (blk >= n_blocks), n_blocks - 1, blk)
        for h in range(Hkv):
            K, V = dec(P["kc"][blk, h, pos % bs]), dec(P["vc"][blk, h, pos % bs])
            Q = dec(P["q"][r0:r1, h * G:(h + 1) * G]).reshape(n * G, d)
            S = (Q @ K.T).view(n, G, ctx) * scale
            if causal:
                seen = torch.from_numpy(pos)[None, :] <= (ctx - n + torch.arange(n))[:, None]
            else:
                seen = torch.ones((n, ctx), dtype=torch.bool)
            S = S.masked_fill(~seen[:, None, :], -np.inf)
            m = S.amax(-1, keepdim=True)
            p = torch.exp(S - torch.where(m == -np.inf, torch.zeros_like(m), m))
            l = p.sum(-1, keepdim=True)
            l = torch.where(l == 0, torch.ones_like(l), l)
            vmax = V.abs().max()
            y[r0:r1, h * G:(h + 1) * G] = (p.view(n * G, ctx) @ V).view(n, G, d) / l
            A = (p.view(n * G, ctx) @ V.abs()).view(n, G, d) / l
            tol[r0:r1, h * G:(h + 1) * G] = (2.0 ** -10 + 2e-5) * A + ctx * 2.0 ** -25 * vmax
    return y, tol


def _call(P, dev, causal, **kw):
    from feather_amd.routines.paged_attention import paged_chunk_attention_fp8_acc_fp32_gpu
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.int32)).to(dev)
    if "dev" not in P:
        P["dev"] = [t(P[k]) for k in ("q", "kc", "vc", "bt", "cu", "ctx")]
    return paged_chunk_attention_fp8_acc_fp32_gpu(*P["dev"], mode=P["mode"], causal=causal, **kw)


def _check(got, y, tol):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    err = (got - y).abs()
    worst = (err - tol).max().item()
    assert worst <= 0, f"off by {err.max().item():.3g}, beyond the bound by {worst:.3g}"


# lens, ctx, Hq, Hkv, d, bs
SHAPES = [
    ([1], [1], 1, 1, 64, 16),
    ([1, 4, 2], [5, 4, 40], 8, 2, 64, 16),
    ([3], [300], 4, 4, 64, 1),                            # one token per page
    ([5, 0, 1, 17], [17, 9, 0, 130], 6, 2, 64, 3),        # odd pages, an empty sequence, an empty cache
    ([70, 3], [70, 515], 12, 4, 64, 20),
    ([129], [1000], 8, 1, 64, 16),
    ([6, 2], [611, 33], 24, 1, 64, 32),                   # 24 query heads on one KV head
    ([9, 1], [300, 77], 4, 2, 128, 16),
    ([33], [33], 8, 2, 128, 5),
    ([2] * 40, list(range(2, 42)), 4, 2, 128, 8),
    ([130, 1], [700, 1025], 5, 5, 128, 64),
    ([19, 4], [90, 400], 4, 2, 256, 16),
    ([65], [257], 3, 1, 256, 6),
    ([7, 20], [7, 130], 4, 2, 512, 16),
    ([40], [290], 2, 1, 512, 7),
    ([150, 3], [400, 70], 2, 1, 512, 16),                 # several tiles at the widest head
    ([210, 64], [1203, 65], 4, 2, 256, 16),
    ([41], [700], 8, 1, 64, 16),                          # few columns, more than one tile of them
    ([9, 64, 1], [9, 2050, 1100], 8, 1, 64, 12),
    ([25], [900], 4, 1, 128, 16),
    ([15], [600], 4, 1, 256, 16),
    ([9], [700], 3, 1, 512, 16),
    ([5, 8, 70, 1], [300, 1500, 900, 40], 8, 1, 64, 16),  # drafts of more than one tile beside a chunk
    ([8, 70, 7], [1100, 70, 9], 8, 1, 64, 20),
    ([10, 16, 60], [700, 90, 1300], 4, 1, 128, 16),
    ([4], [2049], 16, 1, 64, 16),                         # few columns, a long cache: ranges
    ([1, 1, 1], [3000, 1, 777], 8, 1, 128, 16),
]


@pytest.mark.parametrize("mode", ["E4M3", "E5M2"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"d{s[4]}_h{s[2]}x{s[3]}_bs{s[5]}_rows{sum(s[0])}_ctx{max(s[1])}")
def test_chunk_attention_against_float64(dev, orc, shape, causal, mode):
    print(f"chunk attention {shape} causal={causal} {mode}", flush=True)
    P = _problem(orc, 7 + len(shape[0]) + shape[4], *shape, mode)
    y, tol = _reference(P, orc, causal)
    full = _call(P, dev, causal)
    _check(full, y, tol)
    assert torch.equal(full, _call(P, dev, causal))                     # the same bits from call to call
    for hint in (1, max(shape[0]), 10 ** 6):                            # any hint, also a wrong one, gives every row
        _check(_call(P, dev, causal, max_q_len=hint), y, tol)
    half = _call(P, dev, causal, out_dtype=torch.float16)
    _check(half, y, tol + 2.0 ** -11 * y.abs() + 2.0 ** -25)
    from oracle import decode_ref
    packed = _call(P, dev, causal, out_dtype=torch.uint32)
    assert packed.dtype == torch.uint32 and packed.shape == (P["total"], P["Hq"] * P["d"] // 4)
    assert np.array_equal(packed.view(torch.int32).cpu().numpy().view(np.uint32).reshape(-1),
                          decode_ref.quant_codes(full.cpu().numpy(), mode))


@pytest.mark.parametrize("d,lens,ctx", [(64, [10, 3], [6, 0]), (128, [40], [33]), (256, [5], [2]), (512, [9], [4])])
def test_rows_that_see_nothing_are_zero(dev, orc, d, lens, ctx):
    """More new rows than cached tokens (the first rows lie before position 0) and an empty cache."""
    for mode in ("E4M3", "E5M2"):
        P = _problem(orc, 3, lens, ctx, 4, 2, d, 16, mode)
        y, tol = _reference(P, orc, True)
        got = _call(P, dev, True)
        _check(got, y, tol)
        first = lens[0] - ctx[0]
        assert not got[:first].any() and got[first:lens[0]].any()
        assert not _call(P, dev, True, out_dtype=torch.uint32).view(torch.int32)[:first].any()


@pytest.mark.parametrize("lens,ctx", [([6, 2], [90, 300]), ([200], [900]), ([3], [2000])])
def test_rows_outside_every_sequence(dev, orc, lens, ctx):
    """Rows before cu[0] and from cu[n_seq] on are zero in a new result and untouched in the caller's."""
    P = _problem(orc, 11, lens, ctx, 8, 2, 64, 16, "E4M3", head=3, tailrows=5)
    y, tol = _reference(P, orc, True)
    got = _call(P, dev, True)
    _check(got, y, tol)
    assert not got[:3].any() and not got[-5:].any()
    for dt in (torch.float32, torch.float16, torch.uint32):
        want = _call(P, dev, True, out_dtype=dt)
        out = torch.full(want.shape, 7, dtype=torch.int32, device=dev).view(torch.uint32) if dt == torch.uint32 else torch.full_like(want, 7)
        ret = _call(P, dev, True, out_dtype=dt, out=out)
        assert ret is out
        bits = (lambda x: x.view(torch.int32)) if dt == torch.uint32 else (lambda x: x)
        assert (bits(out)[:3] == 7).all() and (bits(out)[-5:] == 7).all()
        assert torch.equal(bits(out)[3:-5], bits(want)[3:-5])


def test_no_sequence_and_no_rows(dev, orc):
    from feather_amd.routines.paged_attention import paged_chunk_attention_fp8_acc_fp32_gpu as f
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)
    kc = i32(4, 2, 16, 16)
    assert f(i32(0, 4, 16), kc, kc, i32(0, 3), i32(1), i32(0)).shape == (0, 4, 64)
    assert not f(i32(5, 4, 16), kc, kc, i32(0, 3), i32(1), i32(0)).any()
    assert not f(i32(5, 4, 16), kc, kc, i32(2, 3), i32(3), i32(2)).any()          # only empty sequences
    assert not f(i32(5, 4, 16), kc, kc, i32(1, 0), i32(2) + torch.tensor([0, 5], dtype=torch.int32, device=dev), i32(1) + 9).any()   # a table without entries


@pytest.mark.parametrize("d,bs", [(64, 16), (128, 6), (256, 16), (512, 3)])
def test_bad_table_entries_read_the_last_block(dev, orc, d, bs):
    P = _problem(orc, 5, [4, 30], [50, 61], 4, 2, d, bs, "E4M3")
    P["bt"][0, 1], P["bt"][1, 0], P["bt"][1, 3] = -1, P["kc"].shape[0] + 3, 2 ** 31 - 1
    for c in (P["kc"], P["vc"]):
        c[-1] = c[0] if not (c[0] == 0x7F7F7F7F).any() else 0x38393A3B
    y, tol = _reference(P, orc, True)
    _check(_call(P, dev, True), y, tol)


def test_lengths_beyond_the_table_are_clamped(dev, orc):
    P = _problem(orc, 5, [4, 3], [48, 16], 4, 2, 64, 16, "E5M2", max_blocks=3)
    want = _call(P, dev, True)
    P2 = dict(P, ctx=np.array([1000, 16], dtype=np.int32))
    P2.pop("dev")
    assert torch.equal(_call(P2, dev, True), want)
    P3 = dict(P, ctx=np.array([48, -7], dtype=np.int32))
    P3.pop("dev")
    got = _call(P3, dev, True)
    assert torch.equal(got[:4], want[:4]) and not got[4:].any()


@pytest.mark.parametrize("d,lens,ctx,Hq,Hkv", [(64, [3], [40], 4, 1), (64, [70], [100], 8, 2), (128, [20], [20], 4, 2),
                                               (128, [200], [300], 8, 1), (256, [33], [64], 2, 1), (512, [9], [30], 2, 2)])
@pytest.mark.parametrize("bad", [0x7C, 0xFC, 0x7F])
def test_infinite_and_nan_values_of_hidden_positions(dev, orc, d, lens, ctx, Hq, Hkv, bad):
    """E5M2 codes of inf and NaN in K and V of a position change nothing for the rows in front of it; the rows that see
    it get what the sum over their own keys gives."""
    P = _problem(orc, 21, lens, ctx, Hq, Hkv, d, 16, "E5M2")
    n, c = lens[0], ctx[0]
    at = c - n + n // 2                                    # the position of the middle row
    y, tol = _reference(P, orc, True)
    blk, slot = P["bt"][0, at // 16], at % 16
    for name in ("kc", "vc"):
        P2 = dict(P, **{name: P[name].copy()})
        P2.pop("dev", None)
        P2[name][blk, :, slot, 1] = bad * 0x010101 + (0x3C << 24)
        got = _call(P2, dev, True).double().cpu()
        before = n // 2
        err = (got[:before] - y[:before]).abs() - tol[:before]
        assert err.max().item() <= 0
        if name == "vc":                                   # dims 4 .. 6 of the rows that see the position
            hit = got[before:][..., 4:7]
            assert torch.isnan(hit).all() if bad == 0x7F else (hit == (np.inf if bad == 0x7C else -np.inf)).all()
            keep = torch.cat([got[before:][..., :4], got[before:][..., 8:]], -1)
            ref = torch.cat([y[before:][..., :4], y[before:][..., 8:]], -1)
            lim = torch.cat([tol[before:][..., :4], tol[before:][..., 8:]], -1)
            assert ((keep - ref).abs() <= lim).all()


@pytest.mark.parametrize("d", [64, 128, 256, 512])
def test_scores_that_climb_along_the_keys(dev, orc, d):
    """The running reference point is raised in steps: keys whose scores grow, fall and jump along the context."""
    for mode in ("E4M3", "E5M2"):
        P = _problem(orc, 2, [40, 2], [700, 900], 4, 2, d, 16, mode)
        rng = np.random.default_rng(1)
        for shape in (np.linspace(0.05, 6.0, 900), np.linspace(6.0, 0.05, 900), np.where(np.arange(900) % 97 == 0, 12.0, 0.2)):
            direction = np.sign(rng.standard_normal(d)).astype(np.float16)
            for s in range(2):
                for pos in range(P["ctx"][s]):
                    P["kc"][P["bt"][s, pos // 16], :, pos % 16] = orc.pack_fp8((direction * shape[pos]).astype(np.float16), mode)
            P["q"][:] = orc.pack_fp8((direction * 0.5).astype(np.float16), mode)
            P.pop("dev", None)
            y, tol = _reference(P, orc, True)
            _check(_call(P, dev, True), y, tol)


def test_workspace_small_or_missing(dev, orc):
    """Through the C ABI: no workspace and a short one give the same result up to the order of the additions."""
    from feather_amd import _native as N
    P = _problem(orc, 4, [3, 5], [1900, 3000], 8, 2, 64, 16, "E4M3")
    y, tol = _reference(P, orc, True)
    _call(P, dev, True)
    L, t = N.lib(), P["dev"]
    mb = P["bt"].shape[1]
    need = L.feather_paged_chunk_attn_scratch_bytes(2, 8, 8, 2, 64, mb * 16, 0)
    assert need > 0
    per = 8 * 8 * 66 * 4
    for size in (0, per - 1, per, 2 * per, 2 * per + 16, 3 * per + 16, need):
        ws = torch.empty(max(size, 16), dtype=torch.uint8, device=dev)
        out = torch.full((8, 8, 64), float("nan"), device=dev)
        N.check(L.feather_paged_chunk_attn_fp8(*[x.data_ptr() for x in t], out.data_ptr(), N.CHUNK_OUT_F32, 0,
                                               ws.data_ptr() if size else None, size, 2, 8, 8, 2, 64, 16, mb, P["kc"].shape[0],
                                               0, 1, N.E4M3, 64 ** -0.5, N.stream_ptr(dev)))
        torch.cuda.synchronize()
        _check(out, y, tol)


def test_other_stream_and_graph_replay(dev, orc):
    P = _problem(orc, 6, [5, 1, 64], [700, 1300, 64], 8, 2, 64, 16, "E4M3")
    P2 = _problem(orc, 8, [2, 9], [90, 500], 8, 2, 64, 16, "E4M3")
    want, want2 = _call(P, dev, True, out_dtype=torch.float16), _call(P2, dev, True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _call(P, dev, True, out_dtype=torch.float16)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _call(P, dev, True, out_dtype=torch.float16)
    for _ in range(3):
        out.fill_(float("nan"))
        assert torch.equal(_call(P2, dev, True), want2)        # eager work between the replays
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_single_rows_agree_with_the_decode_kernel(dev, orc):
    """One new row per sequence is the decode step's attention."""
    from feather_amd.routines.paged_attention import paged_attention_fp8_acc_fp32_gpu
    for mode, d in (("E4M3", 64), ("E5M2", 128)):
        P = _problem(orc, 9, [1] * 6, [1, 16, 17, 600, 999, 2], 8, 2, d, 16, mode)
        y, tol = _reference(P, orc, True)
        got = _call(P, dev, True, max_q_len=1)
        _check(got, y, tol)
        q, kc, vc, bt, _, ctx = P["dev"]
        dec = paged_attention_fp8_acc_fp32_gpu(q, kc, vc, bt, ctx, mode=mode)
        assert ((got - dec).abs().cpu() <= 2 * tol).all()


def test_cross_attention_over_a_longer_and_a_shorter_state(dev, orc):
    """causal=False: the number of rows has nothing to do with the number of cached states."""
    P = _problem(orc, 10, [77, 300], [500, 21], 4, 4, 128, 16, "E4M3")
    y, tol = _reference(P, orc, False, scale=0.2)
    _check(_call(P, dev, False, scale=0.2), y, tol)


def test_out_that_overlaps_an_input_is_refused():
    from feather_amd.routines.paged_attention import paged_chunk_attention_fp8_acc_fp32_gpu
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    q, kc, cu, ctx, tables = z(3, 4, 16), z(4, 2, 16, 16), z(2), z(1), z(1, 2)
    with pytest.raises(ValueError, match="overlaps"):
        paged_chunk_attention_fp8_acc_fp32_gpu(q, kc, kc.clone(), tables, cu, ctx, out_dtype=torch.uint32,
                                               out=q.view(3, 64).view(torch.uint32))
    with pytest.raises(ValueError, match="overlaps"):
        paged_chunk_attention_fp8_acc_fp32_gpu(q, kc, kc.clone(), tables, cu, ctx, out_dtype=torch.uint32,
                                               out=kc.view(-1)[64:256].view(3, 64).view(torch.uint32))


@pytest.mark.parametrize("lens,ctx,Hq,Hkv,d", [([1, 7, 3], [2900, 611, 1500], 8, 2, 64), ([300, 1, 1], [900, 2000, 33], 8, 2, 128),
                                               ([150, 2], [1500, 900], 4, 4, 256), ([140], [777], 2, 1, 512)])
def test_results_do_not_change_from_call_to_call(dev, orc, lens, ctx, Hq, Hkv, d):
    P = _problem(orc, 9, lens, ctx, Hq, Hkv, d, 16, "E4M3")
    first = _call(P, dev, True)
    for _ in range(5):
        assert torch.equal(_call(P, dev, True).view(torch.int32), first.view(torch.int32))
