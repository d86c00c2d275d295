"""The chunk operators on pages whose offsets pass 2^32 bytes and 2^31 words: the same pages at low and at high block ids
give the same bits.  (Block ids are indices, so nothing else may depend on them.)"""
import pytest
import torch

pytestmark = pytest.mark.gpu

WORDS = (1 << 31) + (1 << 22)                                  # of each cache: 8 GiB and some


@pytest.fixture(scope="module")
def pools():
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GiB of free device memory")
    yield tuple(torch.zeros(WORDS, dtype=torch.int32, device="cuda") for _ in range(2))
    torch.cuda.empty_cache()


def _shaped(pool, n_kv, bs, d):
    block = n_kv * bs * d // 4
    n = WORDS // block
    return pool[:n * block].view(n, n_kv, bs, d // 4)


def _codes(g, *shape):
    """random packed words whose codes are finite in both modes: |code| below 0x60"""
    w = torch.randint(0, 0x60, shape + (4,), generator=g, dtype=torch.int32)
    sign = torch.randint(0, 2, shape + (4,), generator=g, dtype=torch.int32) << 7
    b = (w | sign).to(torch.uint8)
    return b.view(torch.int32).squeeze(-1).to("cuda")


@pytest.mark.parametrize("d,n_kv,bs", [(64, 2, 16), (64, 2, 12), (128, 2, 16), (128, 1, 7), (256, 2, 16), (256, 1, 9), (512, 1, 16), (512, 1, 5)])
@pytest.mark.parametrize("mode", ["E4M3", "E5M2"])
def test_attention_of_far_pages(pools, d, n_kv, bs, mode):
    from feather_amd.routines.paged_attention import paged_chunk_attention_fp8_acc_fp32_gpu as attend
    g = torch.Generator().manual_seed(d + bs)
    kc, vc = (_shaped(p, n_kv, bs, d) for p in pools)
    lens, ctx = [200, 1, 3], [333, 290, 70]
    width = -(-max(ctx) // bs)
    n, total = kc.shape[0], sum(lens)
    near = torch.randperm(3 * width, generator=g).to(torch.int32).view(3, width).to("cuda")
    far = n - 1 - near
    for c in (kc, vc):
        c[:3 * width] = _codes(g, 3 * width, n_kv, bs, d // 4)
        c[n - 3 * width:] = c[:3 * width].flip(0)
    q = _codes(g, total, 2 * n_kv, d // 4)
    cu = torch.tensor([0, 200, 201, 204], dtype=torch.int32, device="cuda")
    lengths = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    a, b = (attend(q, kc, vc, t.contiguous(), cu, lengths, mode=mode) for t in (near, far))
    assert a.abs().sum().item() > 0 and torch.equal(a.view(torch.int32), b.view(torch.int32))
    cu = torch.tensor([0, 2, 3, 6], dtype=torch.int32, device="cuda")      # few rows only: the other kernel
    a, b = (attend(q[:6].contiguous(), kc, vc, t.contiguous(), cu, lengths, mode=mode, max_q_len=3) for t in (near, far))
    assert a.abs().sum().item() > 0 and torch.equal(a.view(torch.int32), b.view(torch.int32))


def test_append_fork_and_compact_of_far_pages(pools):
    from feather_amd.routines.paged_cache import paged_cache_compact, paged_cache_fork
    from feather_amd.routines.producers import rope_append_chunk, rotary_frequencies
    d, n_kv, bs = 64, 4, 16                                    # 2.1 million blocks (a pool has at most 4194304)
    kc, vc = (_shaped(p, n_kv, bs, d) for p in pools)
    n = kc.shape[0]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(40, 4 * n_kv * d, generator=g).to("cuda")
    cu, start, freq = i32([0, 40]), i32([3]), rotary_frequencies(d, device="cuda")
    tables = {"near": i32([[2, 0, 1]]), "far": i32([[n - 3, n - 1, n - 2]])}
    for c in (kc, vc):
        c[:3] = 0
        c[n - 3:] = 0
    q = {}
    for name, t in tables.items():
        q[name], after, status = rope_append_chunk(qkv, cu, start, t, kc, vc, n_q_heads=2 * n_kv, freq=freq)
        assert after.tolist() == [43] and status.tolist() == [0]
    assert torch.equal(q["near"].view(torch.int32), q["far"].view(torch.int32))
    for c in (kc, vc):
        assert torch.equal(c[tables["near"][0].long()], c[tables["far"][0].long()]) and c[:3].abs().sum().item() != 0
    # fork: the only free blocks are far; the child's copy of the last block goes there
    ref = torch.ones(n, dtype=torch.int32, device="cuda")
    ref[n - 1] = ref[n - 2] = ref[n - 3] = 0
    table = torch.cat([tables["near"], torch.full((1, 3), -1, dtype=torch.int32, device="cuda")])
    for c in (kc, vc):
        c[n - 3:] = 0
    t, ctx, ref2, status = paged_cache_fork([kc, vc], table, i32([43, 0]), ref, i32([0, 0]))
    assert t.tolist() == [[2, 0, 1], [2, 0, n - 3]] and ctx.tolist() == [43, 43] and status.tolist() == [0, 0]
    assert ref2[n - 3].item() == 1 and ref2[2].item() == 2
    for c in (kc, vc):
        assert torch.equal(c[n - 3], c[1]) and c[n - 2:].abs().sum().item() == 0
    # compact: three far blocks in use, all the others free
    ref.zero_()
    ref[n - 3] = 1
    ref[n - 1] = 2
    for c in (kc, vc):
        c[n - 1] = c[2]
        c[:3] = 0
    want = [(c[n - 3].clone(), c[n - 1].clone()) for c in (kc, vc)]
    t, ref2, block_map, live = paged_cache_compact([kc, vc], i32([[n - 1, n - 3, -1]]), ref)
    assert live.item() == 2 and t.tolist() == [[0, 1, -1]] and ref2[:3].tolist() == [2, 1, 0]
    for c, (w3, w1) in zip((kc, vc), want):
        assert torch.equal(c[0], w1) and torch.equal(c[1], w3)
