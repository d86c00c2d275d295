"""Chunked prefill, verification of drafts, forking and compaction as a serving loop runs them: the operators together,
through PackedDecoder.

Bit for bit where the same numbers are computed from the same codes at other block ids (forked and compacted caches).
Against `PackedDecoder.step` (which tests/test_gpu_decode.py holds against the oracle) values differ by roundings that the
two paths place differently.  Each path rounds P to fp16, so an attention output differs by some 2^-11 relative between
them; its FP8 code then differs where a rounding boundary lies between, boundaries being 2^-3 (E4M3) or 2^-2 (E5M2) of
the value apart: in a share f = 2^-11 * 2^3 = 2^-8 (2^-9) of the codes, by one code step of at most 2^-3 (2^-2).
A product over codes of which a share f is off by a relative step e is off by sqrt(f) e of its norm: 2^-4 * 2^-3 = 2^-7
(E4M3), 2^-4.5 * 2^-2 = 2^-6.5 (E5M2).  That error in turn moves the codes of the next operand: a relative error x of a
value flips a share x / e of its codes by e, which is sqrt(x e) of the norm -- 2^-5 for x = 2^-7, e = 2^-3, and it tends to
x = e = 2^-3 (2^-2) over many operands, never beyond: then each code is one step off.  Two layers have eight operands
after the first attention; logits are therefore held to a root-mean-square error of half the bound, 2^-4 (2^-3) of the
root mean square of the logits, and the K/V codes of layer 0, which no attention precedes, to 99 % equal codes."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _decoder(mode, head_dim, block, n_blocks, max_blocks, dev):
    from feather_amd.routines.decode import DecoderConfig, PackedDecoder, random_weights
    cfg = DecoderConfig(n_layers=2, hidden=512, n_q_heads=512 // head_dim, n_kv_heads=2, head_dim=head_dim, inter=1024, vocab=1000,
                        block_size=block)
    return cfg, PackedDecoder(cfg, random_weights(cfg, seed=3), n_blocks=n_blocks, max_blocks=max_blocks, mode=mode, device=dev)


def _rms(x):
    return x.double().pow(2).mean().sqrt().item()


@pytest.mark.parametrize("mode,head_dim,block", [("E4M3", 64, 16), ("E5M2", 128, 16), ("E4M3", 128, 12)])
def test_extend_in_chunks_matches_single_steps(mode, head_dim, block):
    dev = torch.device("cuda:0")
    max_blocks = 12
    cfg, dec = _decoder(mode, head_dim, block, 2 * max_blocks, max_blocks, dev)
    _, one = _decoder(mode, head_dim, block, 2 * max_blocks, max_blocks, dev)
    g = torch.Generator().manual_seed(7)
    tables = torch.randperm(2 * max_blocks, generator=g).to(torch.int32).view(2, max_blocks).to(dev)
    lens = (100, 37)
    toks = [torch.randint(0, cfg.vocab, (n,), generator=g, dtype=torch.int32).to(dev) for n in lens]
    # sequence 0 in chunks of 70, 29 and 1; sequence 1 in one chunk beside the second, then a chunk of none
    ctx = _i32([0, 0], dev)
    plan = ((70, 0), (29, 36), (1, 1))
    at = [0, 0]
    for n0, n1 in plan:
        ids = torch.cat([toks[0][at[0]:at[0] + n0], toks[1][at[1]:at[1] + n1]])
        logits, ctx, status = dec.extend(ids, _i32([0, n0, n0 + n1], dev), tables, ctx, max_q_len=max(n0, n1))
        at = [at[0] + n0, at[1] + n1]
        assert ctx.tolist() == at and status.tolist() == [0, 0]
    assert logits.shape == (2, cfg.vocab) and at == list(lens)
    # the same tokens one at a time
    want = [None, None]
    for s in range(2):
        for i in range(lens[s]):
            want[s] = one.step(toks[s][i:i + 1], tables[s:s + 1].contiguous(), _i32([i], dev))
    bound = 2.0 ** (-4 if mode == "E4M3" else -3)
    for s in range(2):
        err = _rms(logits[s] - want[s][0]) / _rms(want[s][0])
        print(mode, head_dim, block, s, "logits", err, "of", bound)
        assert err <= bound
    for name in ("k_cache", "v_cache"):
        a, b = dec.layers[0][name].view(torch.uint8), one.layers[0][name].view(torch.uint8)
        same = (a == b).float().mean().item()
        print(name, "equal codes", same)
        assert same >= 0.99


@pytest.mark.parametrize("mode,head_dim,block", [("E4M3", 64, 16), ("E5M2", 128, 16)])
def test_prompt_fork_draft_compact(mode, head_dim, block):
    """One prompt, three samples of it, drafts verified in one call, one sample dropped, the pool moved together."""
    dev = torch.device("cuda:0")
    n_blocks, max_blocks, bs = 40, 8, block
    cfg, dec = _decoder(mode, head_dim, block, n_blocks, max_blocks, dev)
    _, ref = _decoder(mode, head_dim, block, n_blocks, max_blocks, dev)
    g = torch.Generator().manual_seed(11)
    prompt = torch.randint(0, cfg.vocab, (2 * bs + 5,), generator=g, dtype=torch.int32).to(dev)
    n = prompt.numel()
    # ---- an empty slot reserves room, the prompt runs in two chunks
    tables, ctx = torch.full((3, max_blocks), -1, dtype=torch.int32, device=dev), _i32([0, 0, 0], dev)
    counts = torch.zeros(n_blocks, dtype=torch.int32, device=dev)
    counts[1] = 1                                              # a block that the caller holds
    tables, ctx, counts, status = dec.fork(tables, ctx, counts, _i32([-1, -1, -1], dev), room=_i32([n, 0, 0], dev))
    assert status.tolist() == [0, 0, 0] and tables[0].tolist()[:4] == [0, 2, 3, -1]
    for a, b in ((0, 20), (20, n)):
        _, ctx, status = dec.extend(prompt[a:b], _i32([0, b - a, b - a, b - a], dev), tables, ctx)
        assert status.tolist() == [0, 0, 0]
    assert ctx.tolist() == [n, 0, 0]
    # ---- three samples; the plain form copies the whole prompt for each
    room = n + 4
    f_tables, f_ctx, f_counts, status = dec.fork(tables, ctx, counts, _i32([0, 0, 0], dev), room=_i32([room] * 3, dev))
    assert status.tolist() == [0, 0, 0] and f_ctx.tolist() == [n] * 3
    assert f_counts[f_tables[0, 0]].item() == 3 and len(set(f_tables[:, 2].tolist())) == 3
    r_tables = torch.arange(3 * max_blocks, dtype=torch.int32, device=dev).view(3, max_blocks)
    for a, b in zip(ref.layers, dec.layers):
        for name in ("k_cache", "v_cache"):
            for s in range(3):
                a[name][r_tables[s, :3].long()] = b[name][tables[0, :3].long()]
    # ---- each sample verifies a draft of its own length, logits of every row
    draft = torch.randint(0, cfg.vocab, (6,), generator=g, dtype=torch.int32).to(dev)
    cu, rows = _i32([0, 3, 4, 6], dev), _i32(list(range(6)), dev)
    got, f_ctx, status = dec.extend(draft, cu, f_tables, f_ctx, rows=rows, max_q_len=3)
    want, r_ctx, _ = ref.extend(draft, cu, r_tables, _i32([n] * 3, dev), rows=rows, max_q_len=3)
    assert status.tolist() == [0, 0, 0] and torch.equal(f_ctx, r_ctx) and f_ctx.tolist() == [n + 3, n + 1, n + 2]
    assert torch.equal(got, want)
    # one accepted token of the first sample, all of the others: lengths go back, no page moves
    f_ctx = _i32([n + 1, n + 1, n + 2], dev)
    # ---- drop the middle sample, swap the others, move the pool together, decode on
    f_tables, f_ctx, f_counts, status = dec.fork(f_tables, f_ctx, f_counts, _i32([2, -1, 0], dev), room=_i32([room, 0, room], dev))
    assert status.tolist() == [0, 0, 0] and f_ctx.tolist() == [n + 2, 0, n + 1]
    c_tables, c_counts, block_map, live = dec.compact(f_tables, f_counts)
    assert live.item() == int((f_counts > 0).sum()) and int((c_counts > 0).sum()) == live.item() == int((c_counts[:live.item()] > 0).sum())
    assert block_map[1].item() == 1                            # held by the caller, already low
    keep = torch.tensor([0, 2], device=dev)
    tokens = torch.randint(0, cfg.vocab, (2,), generator=g, dtype=torch.int32).to(dev)
    got = dec.step(tokens, c_tables[keep].contiguous(), f_ctx[keep].contiguous())
    want = ref.step(tokens, r_tables[torch.tensor([2, 0], device=dev)].contiguous(), _i32([n + 2, n + 1], dev))
    assert torch.equal(got, want)


def test_extend_in_a_captured_graph():
    dev = torch.device("cuda:0")
    cfg, dec = _decoder("E4M3", 64, 16, 16, 4, dev)
    tables = torch.arange(16, dtype=torch.int32, device=dev).view(4, 4)
    cu, ctx = _i32([0, 1, 4, 4, 9], dev), _i32([3, 10, 7, 0], dev)
    ids = [torch.randint(0, cfg.vocab, (9,), generator=torch.Generator().manual_seed(i), dtype=torch.int32).to(dev) for i in range(3)]
    want = [dec.extend(t, cu, tables, ctx, max_q_len=5)[0].clone() for t in ids]
    static = ids[0].clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        dec.extend(static, cu, tables, ctx, max_q_len=5)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits, after, status = dec.extend(static, cu, tables, ctx, max_q_len=5)
    keep = [0, 1, 3]                                           # sequence 2 has no rows
    for i in (0, 1, 2, 1):
        static.copy_(ids[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits[keep], want[i][keep]) and after.tolist() == [4, 13, 7, 5] and status.tolist() == [0] * 4
        torch.ones(1000, device=dev).cumsum(0)


def test_extend_refusals():
    dev = torch.device("cuda:0")
    cfg, dec = _decoder("E4M3", 64, 16, 8, 4, dev)
    tables, cu, ctx, ids = torch.zeros((1, 4), dtype=torch.int32, device=dev), _i32([0, 2], dev), _i32([0], dev), _i32([1, 2], dev)
    for bad in (dict(token_ids=ids.long()), dict(token_ids=ids.cpu()), dict(token_ids=ids[:0]), dict(cu_seqlens=cu[:1]),
                dict(block_tables=tables[:, :3].contiguous()), dict(ctx_lens=_i32([0, 0], dev)), dict(rows=ids.long()),
                dict(rows=ids.view(1, 2)), dict(max_q_len=-1)):
        args = dict(token_ids=ids, cu_seqlens=cu, block_tables=tables, ctx_lens=ctx)
        args.update(bad)
        with pytest.raises(ValueError):
            dec.extend(**args)
    # a table without room is reported, not written
    _, after, status = dec.extend(_i32([5] * 70, dev), _i32([0, 70], dev), torch.arange(4, dtype=torch.int32, device=dev).view(1, 4), ctx)
    assert after.tolist() == [64] and status.tolist() == [1]
    logits, _, _ = dec.extend(ids, cu, tables, ctx, rows=_i32([], dev))
    assert logits.shape == (0, cfg.vocab)
