"""Refusals of the chunk operators at the C ABI that need no GPU, beyond those of test_paged_chunk_host.py."""


def test_scale_whose_product_with_log2_e_overflows():
    from feather_amd import _native as N
    L = N.lib()

    def call(scale):
        return L.feather_paged_chunk_attn_fp8(*(None,) * 7, 0, 1, None, 0, 1, 0, 8, 4, 64, 16, 4, 8, 0, 1, N.E5M2, scale, None)
    assert call(2.2e38) == N.OK and call(1e-45) == N.OK            # (no rows: nothing is launched)
    assert call(2.4e38) == N.EINVAL and call(3.0e38) == N.EINVAL
