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


def test_attention_result_over_the_tables_or_the_lengths():
    """The workgroups read them while others already write the result."""
    from feather_amd.routines.paged_attention import paged_chunk_attention_fp8_acc_fp32_gpu
    q, kc = _z(3, 4, 16), _z(4, 2, 16, 16)
    buf = _z(3 * 64 + 8)
    out = buf[:192].view(3, 64).view(torch.uint32)
    for bad in (dict(block_tables=buf[190:192].view(1, 2)), dict(cu_seqlens=buf[4:6]), dict(ctx_lens=buf[100:101])):
        with pytest.raises(ValueError, match="overlaps"):
            paged_chunk_attention_fp8_acc_fp32_gpu(q, kc, kc, **{**dict(block_tables=_z(1, 2), cu_seqlens=_z(2), ctx_lens=_z(1)), **bad},
                                                   out_dtype=torch.uint32, out=out)
    paged_chunk_attention_fp8_acc_fp32_gpu(q, kc, kc, buf[192:194].view(1, 2), buf[194:196], buf[196:197], out_dtype=torch.uint32, out=out)
