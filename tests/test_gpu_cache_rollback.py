"""Forks of slots whose lengths were set back into shared blocks (rejected drafts) or whose last block is pinned
(csrc/cache_pages.hip): a block that another table entry or a pin holds when the call starts is not left in a slot's
writable part.  Against a serial loop, word for word, and through PackedDecoder against private copies."""
import numpy as np
import pytest
import torch

from test_gpu_cache_pages import _dev, _fork, _same, _state, dev  # noqa: F401
from test_gpu_extend import _decoder, _i32

pytestmark = pytest.mark.gpu


def fork_loop(caches, bt, ctx, ref, parents, room, bs):
    """The documented fork, slot by slot and entry by entry."""
    n_seq, mb = bt.shape
    nb = ref.size
    caches = [c.copy() for c in caches]
    old = [c.copy() for c in caches]
    held = ref > 1                                           # by another entry, or a pin, when the call starts
    ref = ref.astype(np.int64).copy()
    for v in bt.reshape(-1):
        if 0 <= v < nb:
            ref[v] -= 1
    new, out_ctx, status = np.full_like(bt, -1), np.zeros_like(ctx), np.zeros_like(ctx)
    fresh, taken, sources = [], set(), set()
    for i in range(n_seq):
        p, used = int(parents[i]), 0
        want = 0 if room is None else max(int(room[i]), 0)
        if 0 <= p < n_seq:
            n = min(max(int(ctx[p]), 0), mb * bs)
            whole, used = n // bs, -(-n // bs)
            out_ctx[i] = n
            heir = p not in taken
            taken.add(p)
            for e in range(mb):
                v = int(bt[p, e])
                if not 0 <= v < nb:
                    if e < used:
                        status[i] = 2
                elif e < whole or (heir and not held[v]):
                    new[i, e] = v
                    ref[v] += 1
                elif e == whole and used > whole:
                    fresh.append((i, e, v, whole * bs))
                    sources.add(v)
        if want > mb * bs and status[i] == 0:
            status[i] = 1
        for e in range(used, min(-(-want // bs), mb)):
            if new[i, e] < 0:
                fresh.append((i, e, -1, 0))
    free = [b for b in range(nb) if ref[b] == 0 and b not in sources]
    for k, (i, e, src, keep) in enumerate(fresh):
        if k < len(free):
            new[i, e] = free[k]
            ref[free[k]] = 1
            if src >= 0:
                for c, o in zip(caches, old):
                    c[free[k]] = o[src]
        else:
            status[i] = 3
            if src >= 0:
                out_ctx[i] = keep
    return new, out_ctx, ref.astype(np.int32), status, caches


def _context(cache, row, n, bs):
    return np.concatenate([cache[b] for b in row[:-(-n // bs)]], axis=1)[:, :n] if n else cache[:0]


@pytest.mark.parametrize("n_seq,mb,bs,nb,layers", [(2, 3, 4, 12, 1), (4, 5, 16, 60, 2), (9, 8, 4, 300, 1), (70, 12, 3, 2500, 2),
                                                    (300, 20, 16, 9000, 1), (33, 40, 8, 9001, 5), (3, 300, 2, 1500, 1)])
def test_fork_after_lengths_were_set_back(dev, n_seq, mb, bs, nb, layers):
    rng = np.random.default_rng(n_seq * mb)
    for trial in range(6):
        bt, ctx, ref, caches = _state(rng, n_seq, mb, bs, nb // 2, layers=layers)
        ref = np.concatenate([ref, np.zeros(nb - nb // 2, np.int32)])
        caches = [rng.integers(0, 2 ** 32, (nb,) + c.shape[1:], dtype=np.uint64).astype(np.uint32) for c in caches]
        few = np.sort(rng.integers(0, n_seq, n_seq) // 2).astype(np.int32)          # many children of few parents: much is shared
        bt, ctx, ref, _, caches = fork_loop(caches, bt, ctx, ref, few, ctx[few] + rng.integers(0, 2 * bs, n_seq), bs)
        back = rng.random(n_seq) < 0.7
        ctx = np.where(back, (ctx * rng.random(n_seq)).astype(np.int32), ctx).astype(np.int32)
        if trial % 2:
            ref[rng.integers(0, nb, nb // 8)] += 1                                  # pins
        parents = np.arange(n_seq, dtype=np.int32) if trial < 2 else rng.integers(-1, n_seq, n_seq).astype(np.int32)
        room = None if trial % 3 == 2 else (ctx[np.maximum(parents, 0)] + rng.integers(0, bs + 2, n_seq)).astype(np.int32)
        print(f"fork after rollback {n_seq} {mb} {bs} {nb} trial {trial}", flush=True)
        want = fork_loop(caches, bt, ctx, ref, parents, room, bs)
        got, got_caches = _fork(dev, bt, ctx, ref, caches, parents, room)
        _same(got, got_caches, want)
        tables, lens, counts, status = got
        for i in range(n_seq):
            p, n = parents[i], int(lens[i])
            for b in tables[i, n // bs:]:
                assert b < 0 or counts[b] == 1                  # what a slot may write is its own
            if p >= 0 and status[i] != 2:
                assert n == min(max(int(ctx[p]), 0), mb * bs) or status[i] == 3
                for c, g in zip(caches, got_caches):
                    assert np.array_equal(_context(g, tables[i], n, bs), _context(c, bt[p], n, bs))


def test_two_slots_set_back_into_one_block(dev):
    """Length 34 in blocks of 16, two children; both go back to 30, inside the block that they share."""
    rng = np.random.default_rng(1)
    bt, ctx = np.array([[4, 2, 5, -1], [-1] * 4], np.int32), np.array([34, 0], np.int32)
    ref = np.array([0, 0, 1, 0, 1, 1, 0, 0, 0], np.int32)
    caches = [rng.integers(0, 2 ** 32, (9, 2, 16, 4), dtype=np.uint64).astype(np.uint32) for _ in range(3)]
    (t, c, r, s), caches = _fork(dev, bt, ctx, ref, caches, np.array([0, 0], np.int32), None)
    assert t.tolist() == [[4, 2, 5, -1], [4, 2, 0, -1]] and r.tolist() == [1, 0, 2, 0, 2, 1, 0, 0, 0]
    back = np.array([30, 30], np.int32)
    (t, c, r, s), after = _fork(dev, t, back, r, caches, np.array([0, 1], np.int32), None)
    assert t.tolist() == [[4, 1, 5, -1], [4, 3, 0, -1]] and c.tolist() == [30, 30] and s.tolist() == [0, 0]
    assert r.tolist() == [1, 1, 0, 1, 2, 1, 0, 0, 0]           # block 2 was copied from and is free from now on, not in this call
    for a, b in zip(after, caches):
        assert np.array_equal(a[1], b[2]) and np.array_equal(a[3], b[2]) and np.array_equal(a[2], b[2])
    # one slot goes back, the other keeps the block as a whole one of its context
    (t2, c, r, s), _ = _fork(dev, np.array([[4, 2, 5, -1], [4, 2, 0, -1]], np.int32), np.array([30, 34], np.int32),
                             np.array([1, 0, 2, 0, 2, 1, 0, 0, 0], np.int32), caches, np.array([0, 1], np.int32), None)
    assert t2.tolist() == [[4, 1, 5, -1], [4, 2, 0, -1]] and r.tolist() == [1, 1, 1, 0, 2, 1, 0, 0, 0]
    # a pinned last block stays as it is; a shared block behind the context is let go
    (t3, c, r, s), _ = _fork(dev, np.array([[4, 2, 5, -1], [4, 2, 0, -1]], np.int32), np.array([34, 16], np.int32),
                             np.array([1, 0, 2, 0, 2, 2, 0, 0, 0], np.int32), caches, np.array([0, 1], np.int32), None)
    assert t3.tolist() == [[4, 2, 1, -1], [4, -1, 0, -1]] and r.tolist() == [1, 1, 1, 0, 2, 1, 0, 0, 0]
    # no block for the copy: the whole blocks remain, and the source keeps what it holds
    full = np.array([1, 1, 2, 1, 2, 1, 1, 1, 1], np.int32)
    (t4, c, r, s), after = _fork(dev, np.array([[4, 2, 5, -1], [4, 2, 0, -1]], np.int32), back, full, caches, np.array([0, 1], np.int32), None)
    assert t4.tolist() == [[4, -1, 5, -1], [4, -1, 0, -1]] and c.tolist() == [16, 16] and s.tolist() == [3, 3]
    for a, b in zip(after, caches):
        assert np.array_equal(a, b)


def test_what_a_fork_that_runs_out_leaves_of_the_old_state(dev):
    """Blocks of ended slots are handed out in the same call and may be written; what a new row holds is as it was."""
    rng = np.random.default_rng(3)
    bt = np.array([[0, 1, -1], [2, 3, -1], [4, 5, 6]], np.int32)
    ctx = np.array([6, 7, 12], np.int32)
    ref = np.ones(7, np.int32)                                 # blocks of 4 tokens, nothing free
    caches = [rng.integers(0, 2 ** 32, (7, 1, 4, 4), dtype=np.uint64).astype(np.uint32) for _ in range(2)]
    parents, room = np.array([0, 0, 2], np.int32), np.array([9, 9, 12], np.int32)
    want = fork_loop(caches, bt, ctx, ref, parents, room, 4)
    got, after = _fork(dev, bt, ctx, ref, caches, parents, room)
    _same(got, after, want)
    tables, lens, counts, status = got
    # slot 1's blocks 2 and 3 go to the spare entry of slot 0 and to the copy of block 1; then the pool is empty
    assert tables.tolist() == [[0, 1, 2], [0, 3, -1], [4, 5, 6]] and status.tolist() == [0, 3, 0] and lens.tolist() == [6, 6, 12]
    for a, c in zip(after, caches):
        assert np.array_equal(a[3], c[1]) and not np.array_equal(a[3], c[3])   # an old row of an ended slot is void
        assert all(np.array_equal(a[b], c[b]) for b in (0, 1, 2, 4, 5, 6))      # (block 2 is reserved, not written)


@pytest.mark.parametrize("mode,head_dim,block", [("E4M3", 64, 16), ("E5M2", 128, 16)])
def test_drafts_rejected_across_a_fork(mode, head_dim, block):
    """Two samples of a prompt whose tail was itself a draft: both go back behind the fork, fork again, and go on alone."""
    dev = torch.device("cuda:0")
    n_blocks, max_blocks = 24, 6
    cfg, dec = _decoder(mode, head_dim, block, n_blocks, max_blocks, dev)
    _, ref = _decoder(mode, head_dim, block, n_blocks, max_blocks, dev)
    g = torch.Generator().manual_seed(2)
    n, keep = 2 * block + 3, 2 * block - 4
    prompt = torch.randint(0, cfg.vocab, (n,), generator=g, dtype=torch.int32).to(dev)
    tables, ctx = torch.full((2, max_blocks), -1, dtype=torch.int32, device=dev), _i32([0, 0], dev)
    counts = torch.zeros(n_blocks, dtype=torch.int32, device=dev)
    tables, ctx, counts, _ = dec.fork(tables, ctx, counts, _i32([-1, -1], dev), room=_i32([n, 0], dev))
    _, ctx, status = dec.extend(prompt, _i32([0, n, n], dev), tables, ctx)
    tables, ctx, counts, status = dec.fork(tables, ctx, counts, _i32([0, 0], dev))
    assert status.tolist() == [0, 0] and tables[0, 1].item() == tables[1, 1].item()
    ctx = _i32([keep, keep], dev)
    tables, ctx, counts, status = dec.fork(tables, ctx, counts, _i32([0, 1], dev), room=_i32([keep + 7, keep + 7], dev))
    assert status.tolist() == [0, 0] and tables[0, 1].item() != tables[1, 1].item() and ctx.tolist() == [keep, keep]
    r_tables = torch.arange(2 * max_blocks, dtype=torch.int32, device=dev).view(2, max_blocks)
    for s in range(2):
        ref.extend(prompt[:keep].contiguous(), _i32([0, keep], dev), r_tables[s:s + 1].contiguous(), _i32([0], dev))
    for a, b in zip(ref.layers, dec.layers):                    # the same codes in both, whatever the split of the prompt
        for name in ("k_cache", "v_cache"):
            for s in range(2):
                a[name][r_tables[s, :2].long()] = b[name][tables[s, :2].long()]
    ids = torch.randint(0, cfg.vocab, (14,), generator=g, dtype=torch.int32).to(dev)
    rows = _i32(list(range(14)), dev)
    got, after, status = dec.extend(ids, _i32([0, 7, 14], dev), tables, ctx, rows=rows, max_q_len=7)
    want, _, _ = ref.extend(ids, _i32([0, 7, 14], dev), r_tables, ctx, rows=rows, max_q_len=7)
    assert status.tolist() == [0, 0] and after.tolist() == [keep + 7] * 2 and torch.equal(got, want)
