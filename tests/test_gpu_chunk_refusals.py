"""Refusals of the chunk operators' wrappers for tensors that overlap, and calls beside them that are fine."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _z(*s):
    return torch.zeros(s, dtype=torch.int32, device="cuda")


def test_rope_append_into_overlapping_caches():
    from feather_amd.routines.producers import rope_append_chunk, rotary_frequencies
    qkv, freq = torch.ones((3, 8 * 64), device="cuda"), rotary_frequencies(64)
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    pool = _z(9, 2, 16, 16)
    for k, v in ((pool, pool), (pool[:8], pool[1:]), (pool[1:], pool[:8])):
        with pytest.raises(ValueError, match="overlap"):
            rope_append_chunk(qkv, cu, _z(1), _z(1, 2), k, v, n_q_heads=4, freq=freq)
    assert not pool.any()
    both = _z(2, 8, 2, 16, 16)
    _, after, status = rope_append_chunk(qkv, cu, _z(1), _z(1, 2), both[1], both[0], n_q_heads=4, freq=freq)   # side by side
    assert after.tolist() == [3] and status.tolist() == [0] and both[0].any() and both[1].any()
    q, after, _ = rope_append_chunk(qkv[:0], _z(2), _z(1) + 5, _z(1, 2), pool, pool, n_q_heads=4, freq=freq)   # no rows, nothing written
    assert q.shape == (0, 4, 16) and after.tolist() == [5]
