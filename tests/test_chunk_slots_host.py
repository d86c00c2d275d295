"""The search for a tile's sequence as chunk attention's kernels make it (no GPU): 64 sequences per step, ending with the
first step whose sequences do not all start at or before the slot."""
import numpy as np


def _find(first, slot):
    seq = -1
    for s0 in range(0, len(first), 64):
        below = sum(f <= slot for f in first[s0:s0 + 64])
        if below:
            seq = s0 + below - 1
        if below != 64:
            break
    return seq


def test_search_in_steps_of_64():
    rng = np.random.default_rng(4)
    for n_seq in (1, 63, 64, 65, 127, 128, 129, 130, 192, 300):
        for _ in range(6):
            group, qt = int(rng.integers(1, 25)), int(rng.choice([16, 32, 64, 128, 256]))
            lens = rng.integers(0, rng.choice([1, 2, 9, 100]) + 1, n_seq)
            lens[rng.random(n_seq) < 0.3] = 0
            if n_seq > 64:
                lens[62:66] = rng.choice([0, 150], 4)[:len(lens[62:66])]
            cu = np.concatenate([[0], np.cumsum(lens)]) + int(rng.integers(0, 5))
            slots = (int(cu[-1]) + int(rng.integers(0, 4))) * group // qt + n_seq
            first = [int(cu[s]) * group // qt + s for s in range(n_seq)]
            seen = []
            for slot in range(slots):
                s = _find(first, slot)
                assert s == sum(f <= slot for f in first) - 1
                if s >= 0 and slot - first[s] < -(-int(lens[s]) * group // qt):
                    seen.append((s, slot - first[s]))
            assert seen == [(s, t) for s in range(n_seq) for t in range(-(-int(lens[s]) * group // qt))]


def test_calls_with_key_ranges_have_few_sequences():
    """The merge keeps the offsets of 512 sequences: beyond 384 no call has ranges (a workspace would be asked for)."""
    from feather_amd import _native as N
    size = N.lib().feather_paged_chunk_attn_scratch_bytes
    most = 0
    for d in (64, 128, 256, 512):
        for n_q, n_kv in ((1, 1), (4, 1), (32, 1), (64, 1), (600, 1), (32, 4), (5, 5)):
            for n_seq in (1, 64, 100, 200, 256, 300, 383, 384, 385, 400, 500, 513, 700, 1024, 1025, 5000):
                for rows in (1, n_seq, 2 * n_seq, 40 * n_seq, 2000 * n_seq):
                    for hint in (0, 1, 3, 64, 5000):
                        if size(n_seq, rows, n_q, n_kv, d, 1 << 20, hint) > 0:
                            most = max(most, n_seq)
    assert 0 < most <= 384
