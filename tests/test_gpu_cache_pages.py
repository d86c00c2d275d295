"""Fork and compaction of a cache's pages (csrc/cache_pages.hip) against a serial loop over slots and entries: whole
numbers, so every table, count, length, status and cache word has to be equal."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    return torch.device("cuda:0")


def _fork_loop(caches, bt, ctx, ref, parents, room, bs):
    n_seq, mb = bt.shape
    nb = ref.size
    caches = [c.copy() for c in caches]
    ref = ref.astype(np.int64).copy()
    new, out_ctx, status = np.full_like(bt, -1), np.zeros_like(ctx), np.zeros_like(ctx)
    for s in range(n_seq):
        for v in bt[s]:
            if 0 <= v < nb:
                ref[v] -= 1
    fresh, taken = [], set()
    for i in range(n_seq):
        p = parents[i]
        used = 0
        if 0 <= p < n_seq:
            L = min(max(int(ctx[p]), 0), mb * bs)
            whole, used = L // bs, -(-L // bs)
            out_ctx[i] = L
            heir = p not in taken
            taken.add(int(p))
            for e in range(mb):
                v = int(bt[p, e])
                ok = 0 <= v < nb
                if e < used and not ok:
                    status[i] = 2
                if ok and (e < whole or heir):
                    new[i, e] = v
                    ref[v] += 1
                elif ok and e == whole and used > whole:
                    fresh.append((i, e, v, whole * bs))
        want = 0 if room is None else max(int(room[i]), 0)
        if want > mb * bs and status[i] == 0:
            status[i] = 1
        for e in range(used, min(-(-want // bs), mb)):
            if new[i, e] < 0:
                fresh.append((i, e, -1, 0))
    free = [b for b in range(nb) if ref[b] == 0]
    for k, (i, e, src, keep) in enumerate(fresh):
        if k < len(free):
            new[i, e] = free[k]
            ref[free[k]] = 1
            if src >= 0:
                for c in caches:
                    c[free[k]] = c[src]
        else:
            status[i] = 3
            if src >= 0:
                out_ctx[i] = keep
    return new, out_ctx, ref.astype(np.int32), status, caches


def _compact_loop(caches, bt, ref):
    nb = ref.size
    caches = [c.copy() for c in caches]
    live = int((ref > 0).sum())
    holes = [b for b in range(live) if ref[b] <= 0]
    highs = [b for b in range(nb - 1, live - 1, -1) if ref[b] > 0]
    assert len(holes) == len(highs)
    block_map = np.where(ref > 0, np.arange(nb), -1).astype(np.int32)
    new_ref = np.where((ref > 0) & (np.arange(nb) < live), ref, 0).astype(np.int32)
    for h, b in zip(holes, highs):
        block_map[b] = h
        new_ref[h] = ref[b]
        for c in caches:
            c[h] = c[b]
    ok = (bt >= 0) & (bt < nb)
    return np.where(ok, block_map[np.where(ok, bt, 0)], -1).astype(np.int32), new_ref, block_map, live, caches


def _state(rng, n_seq, mb, bs, nb, nkv=2, dw=4, layers=2, share=True, fill=0.6):
    """Consistent tables and counts: some prefixes shared, some slots empty, spare entries past the contexts."""
    perm = list(rng.permutation(nb))
    bt, ctx = np.full((n_seq, mb), -1, np.int32), np.zeros(n_seq, np.int32)
    for s in range(n_seq):
        n = min(int(rng.integers(0, int(mb * fill) + 2)), mb, len(perm))
        own = [perm.pop() for _ in range(n)]
        if share and s and rng.random() < 0.5:             # a shared prefix of whole blocks
            p = int(rng.integers(0, s))
            k = min(int(ctx[p]) // bs, n)
            k = int(rng.integers(0, k + 1))
            perm.extend(own[:k])
            own[:k] = list(bt[p, :k])
        bt[s, :n] = own
        ctx[s] = int(rng.integers(0, n * bs + 1)) if n else 0
        if share and s and n:
            ctx[s] = max(ctx[s], min(n * bs, bs * sum(b in bt[:s] for b in own)))   # shared blocks are whole blocks of the context
    ref = np.bincount(bt[bt >= 0], minlength=nb).astype(np.int32)
    caches = [rng.integers(0, 2 ** 32, (nb, nkv, bs, dw), dtype=np.uint64).astype(np.uint32) for _ in range(2 * layers)]
    return bt, ctx, ref, caches


def _dev(dev, *arrays):
    return [torch.from_numpy(np.ascontiguousarray(a).view(np.int32).copy()).to(dev) for a in arrays]


def _words(t):
    return t.view(torch.int32).cpu().numpy().view(np.uint32)


def _fork(dev, bt, ctx, ref, caches, parents, room):
    from feather_amd.routines.paged_cache import paged_cache_fork
    tb, tc, tr, tp = _dev(dev, bt, ctx, ref, parents)
    tcaches = _dev(dev, *caches)
    got = paged_cache_fork(tcaches, tb, tc, tr, tp, room=None if room is None else _dev(dev, room)[0])
    for a, b in zip((tb, tc, tr), (bt, ctx, ref)):
        assert np.array_equal(a.cpu().numpy(), b)          # the inputs stay as they were
    return [g.cpu().numpy() for g in got], [_words(c) for c in tcaches]


def _same(got, got_caches, want):
    for name, g, w in zip(("tables", "ctx", "ref", "status"), got, want):
        assert np.array_equal(g, w), name
    for g, w in zip(got_caches, want[4]):
        assert np.array_equal(g, w)


@pytest.mark.parametrize("n_seq,mb,bs,nb,layers", [(1, 1, 1, 1, 1), (4, 5, 16, 30, 2), (9, 8, 4, 100, 1), (70, 12, 3, 700, 3),
                                                    (300, 20, 16, 5000, 1), (33, 40, 8, 9001, 5), (3, 300, 2, 1000, 1)])
def test_fork_against_a_serial_loop(dev, n_seq, mb, bs, nb, layers):
    rng = np.random.default_rng(n_seq + mb)
    for trial in range(4):
        bt, ctx, ref, caches = _state(rng, n_seq, mb, bs, nb, layers=layers)
        parents = rng.integers(-1, n_seq, n_seq).astype(np.int32) if trial else np.arange(n_seq, dtype=np.int32)
        room = None if trial % 2 else rng.integers(0, mb * bs + 3, n_seq).astype(np.int32)
        print(f"fork {n_seq} {mb} {bs} {nb} trial {trial}", flush=True)
        want = _fork_loop(caches, bt, ctx, ref, parents, room, bs)
        _same(*_fork(dev, bt, ctx, ref, caches, parents, room), want)
        if trial == 0 and room is None:
            assert np.array_equal(want[0], bt)


def test_fork_keeps_pins_and_reports_holes_and_exhaustion(dev):
    rng = np.random.default_rng(5)
    bt = np.array([[0, 1, -1], [2, 9, 7], [3, -1, -1]], np.int32)       # 9: not a block of the pool of 8
    ctx = np.array([5, 12, 4], np.int32)
    ref = np.array([1, 1, 1, 1, 0, 0, 3, 1], np.int32)                    # block 6 is pinned three times by the caller
    caches = [rng.integers(0, 2 ** 32, (8, 1, 4, 4), dtype=np.uint64).astype(np.uint32) for _ in range(2)]
    for parents, room in (([0, 0, 0], [8, 12, 12]), ([1, 1, 2], [0, 0, 99]), ([-1, 7, 2], [12, 12, 12]), ([0, 0, 0], None),
                          ([-5, -1, 3], [12, 12, 12]), ([2, 2, 2], [-4, 5, 2 ** 31 - 1])):
        parents = np.array(parents, np.int32)
        room = None if room is None else np.array(room, np.int32)
        want = _fork_loop(caches, bt, ctx, ref, parents, room, 4)
        _same(*_fork(dev, bt, ctx, ref, caches, parents, room), want)
        assert want[2][6] == 3                                            # a pinned block is never handed out
    parents, room = np.array([0, 0, 0], np.int32), np.array([12, 12, 12], np.int32)
    for pins, short in (([5], [0, 0, 3]), ([4, 5, 7], [0, 3, 3]), ([2, 3, 4, 5, 7], [3, 3, 3])):   # more of the pool is pinned: it runs out
        few = ref.copy()
        few[pins] += 1
        want = _fork_loop(caches, bt, ctx, few, parents, room, 4)
        assert want[3].tolist() == short
        _same(*_fork(dev, bt, ctx, few, caches, parents, room), want)


@pytest.mark.parametrize("n_caches", [1, 3, 8, 9, 64, 65, 130])
def test_fork_and_compact_over_many_caches(dev, n_caches):
    from feather_amd.routines.paged_cache import paged_cache_compact
    rng = np.random.default_rng(n_caches)
    bt, ctx, ref, _ = _state(rng, 6, 5, 4, 40, layers=1)
    caches = [rng.integers(0, 2 ** 32, (40, 1, 4, 4), dtype=np.uint64).astype(np.uint32) for _ in range(n_caches)]
    parents = np.array([0, 0, 1, 1, 5, -1], np.int32)
    _same(*_fork(dev, bt, ctx, ref, caches, parents, None), _fork_loop(caches, bt, ctx, ref, parents, None, 4))
    tcaches = _dev(dev, *caches)
    t, r, m, live = paged_cache_compact(tcaches, *_dev(dev, bt, ref))
    want = _compact_loop(caches, bt, ref)
    assert np.array_equal(t.cpu().numpy(), want[0]) and live.item() == want[3]
    for g, w in zip(tcaches, want[4]):
        assert np.array_equal(_words(g)[:want[3]], w[:want[3]])


@pytest.mark.parametrize("nb,used", [(1, 0), (1, 1), (2, 1), (40, 0), (40, 40), (41, 17), (4096, 1000), (4097, 4000), (20000, 7777)])
def test_compact_against_a_serial_loop(dev, nb, used):
    from feather_amd.routines.paged_cache import paged_cache_compact
    rng = np.random.default_rng(nb + used)
    ref = np.zeros(nb, np.int32)
    ref[rng.permutation(nb)[:used]] = rng.integers(1, 4, used)
    if nb > 10:
        ref[np.flatnonzero(ref == 0)[:2]] = [-1, -7][:max(0, min(2, nb - used))]   # not in use either
    bt = rng.integers(-2, nb + 2, (7, 9)).astype(np.int32)
    caches = [rng.integers(0, 2 ** 32, (nb, 1, 2, 4), dtype=np.uint64).astype(np.uint32) for _ in range(3)]
    tcaches = _dev(dev, *caches)
    tb, tr = _dev(dev, bt, ref)
    t, r, m, live = paged_cache_compact(tcaches, tb, tr)
    wt, wr, wm, wl, wc = _compact_loop(caches, bt, ref)
    assert live.item() == wl and np.array_equal(t.cpu().numpy(), wt) and np.array_equal(r.cpu().numpy(), wr)
    assert np.array_equal(m.cpu().numpy(), wm)
    assert np.array_equal(tb.cpu().numpy(), bt) and np.array_equal(tr.cpu().numpy(), ref)
    for g, w, old in zip(tcaches, wc, caches):
        assert np.array_equal(_words(g), w)                # nothing above n_live is written


def test_replay_in_a_graph_and_on_another_stream(dev):
    from feather_amd.routines.paged_cache import paged_cache_compact, paged_cache_fork
    rng = np.random.default_rng(8)
    bt, ctx, ref, caches = _state(rng, 12, 9, 4, 200)
    parents = rng.integers(-1, 12, 12).astype(np.int32)
    room = rng.integers(0, 36, 12).astype(np.int32)
    tb, tc, tr, tp, tm = _dev(dev, bt, ctx, ref, parents, room)
    want = _fork_loop(caches, bt, ctx, ref, parents, room, 4)
    wantc = _compact_loop(want[4], want[0], want[2])
    tcaches, orig = _dev(dev, *caches), _dev(dev, *caches)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = paged_cache_fork(tcaches, tb, tc, tr, tp, room=tm)
        b = paged_cache_compact(tcaches, a[0], a[2])
    side.synchronize()
    assert np.array_equal(a[0].cpu().numpy(), want[0]) and np.array_equal(b[0].cpu().numpy(), wantc[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = paged_cache_fork(tcaches, tb, tc, tr, tp, room=tm)
        b = paged_cache_compact(tcaches, a[0], a[2])
    for _ in range(3):
        for c, o in zip(tcaches, orig):
            c.copy_(o)
        for x in (*a, *b):
            x.fill_(77)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for g, w in zip(a, want):
            assert np.array_equal(g.cpu().numpy(), w)
        assert np.array_equal(b[0].cpu().numpy(), wantc[0]) and np.array_equal(b[1].cpu().numpy(), wantc[1])
        assert np.array_equal(b[2].cpu().numpy(), wantc[2]) and b[3].item() == wantc[3]
        for g, w in zip(tcaches, wantc[4]):
            assert np.array_equal(_words(g), w)


def test_refusals(dev):
    from feather_amd.routines.paged_cache import paged_cache_compact, paged_cache_fork
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)
    k, v = i32(6, 1, 4, 4), i32(6, 1, 4, 4)
    ok = dict(caches=[k, v], block_tables=i32(2, 3), ctx_lens=i32(2), ref_counts=i32(6), parents=i32(2))
    for bad in (dict(caches=[]), dict(caches=[k, k]), dict(caches=[k, i32(5, 1, 4, 4)]), dict(caches=[i32(6, 1, 4, 8)[..., ::2]]),
                dict(caches=[i32(6, 16)]), dict(caches=[i32(6, 1, 1, 3)]), dict(ref_counts=i32(5)), dict(ctx_lens=i32(3)),
                dict(parents=i32(1)), dict(parents=i32(2).long()), dict(block_tables=i32(6)), dict(block_tables=i32(2, 3).cpu()),
                dict(room=i32(3))):
        with pytest.raises(ValueError):
            paged_cache_fork(**{**ok, **bad})
    with pytest.raises(ValueError):
        paged_cache_compact([k, k], i32(2, 3), i32(6))
    with pytest.raises(ValueError):
        paged_cache_compact([k], i32(2, 3), i32(7))
    t, c, r, s = paged_cache_fork([k, v], i32(0, 3), i32(0), i32(6) + 2, i32(0))       # no slots: the counts are copied
    assert t.shape == (0, 3) and r.cpu().tolist() == [2] * 6
    t, c, r, s = paged_cache_fork([k, v], i32(2, 0), i32(2), i32(6), i32(2))           # a table without entries
    assert s.cpu().tolist() == [0, 0] and c.cpu().tolist() == [0, 0]
    assert paged_cache_compact([k], i32(0, 3), i32(6))[3].item() == 0


def test_overlapping_caches_are_refused():
    from feather_amd.routines.paged_cache import paged_cache_compact
    pool = torch.zeros((9, 2, 16, 16), dtype=torch.int32, device="cuda")
    tables, ref = torch.zeros((1, 2), dtype=torch.int32, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        paged_cache_compact([pool[:8], pool[1:]], tables, ref)
    with pytest.raises(ValueError, match="overlap"):
        paged_cache_compact([pool[:8], pool[:8]], tables, ref)
    both = torch.zeros((2, 8, 2, 16, 16), dtype=torch.int32, device="cuda")
    paged_cache_compact([both[1], both[0]], tables, ref)       # side by side is fine
