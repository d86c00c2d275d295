"""Refusals of the chunk operators at the C ABI that need no GPU, beyond those of test_paged_chunk_host.py."""


def test_scale_whose_product_with_log2_e_overflows():
    from feather_amd import _native as N
    L = N.lib()

    def call(scale):
        return L.feather_paged_chunk_attn_fp8(*(None,) * 7, 0, 1, None, 0, 1, 0, 8, 4, 64, 16, 4, 8, 0, 1, N.E5M2, scale, None)
    assert call(2.2e38) == N.OK and call(1e-45) == N.OK            # (no rows: nothing is launched)
    assert call(2.4e38) == N.EINVAL and call(3.0e38) == N.EINVAL


def test_rope_append_into_overlapping_caches():
    """Both caches are written: rows of one must not be rows of the other."""
    from feather_amd import _native as N
    L, size = N.lib(), 8 * 2 * 16 * 64                             # blocks, KV heads, tokens, bytes of a row

    def call(k, v):
        return L.feather_rope_append_chunk(16, 0, 512, 4, 4, 4, 8, 1.0, 64, 0, 8, k, v, 4, 4, 16, 1, 1, 4, 4, 2, 64, 16, 4, 8, N.E4M3, None)
    base = 1 << 20
    for k, v in ((base, base), (base, base + 64), (base + size - 8, base), (base, base + size - 8)):
        assert call(k, v) == N.EINVAL and b"overlap" in L.feather_last_error(), (k, v)
