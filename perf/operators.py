"""Workloads of the paged-cache operators that serve new tokens in chunks: attention of a chunk over the paged FP8
cache, rotary positions with quantisation and append of the chunk, and the fork and compaction of a cache's pages.

``run`` computes them in plain torch (32-bit products, sums and exponentials, angles in 64 bits, integer work with
sorts and prefix sums), or, with ``own`` set, through the framework's entry points.  Packed FP8 results are returned
as the FP8 values they stand for."""
import math

import numpy as np
import torch

own = False


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # two requests whose four or five drafted tokens are verified at short contexts: nothing but latency
        {"name": "verify_two", "kind": "attend", "n_seq": 2, "q_min": 4, "q_max": 5, "chunk": 0, "ctx_min": 211,
         "ctx_max": 300, "n_q": 32, "n_kv": 4, "d": 64, "block": 16, "mode": "E4M3", "causal": True, "out": "packed"},
        # a batch of 32 requests, each with up to eight drafted tokens, at the decode benchmark's contexts
        {"name": "verify_batch", "kind": "attend", "n_seq": 32, "q_min": 3, "q_max": 8, "chunk": 0, "ctx_min": 512,
         "ctx_max": 4096, "n_q": 32, "n_kv": 4, "d": 64, "block": 16, "mode": "E4M3", "causal": True, "out": "float16"},
        # a mixed step: 16 requests decode one token while a 17th prefills a chunk of 512
        {"name": "mixed_step", "kind": "attend", "n_seq": 17, "q_min": 1, "q_max": 1, "chunk": 512, "ctx_min": 700,
         "ctx_max": 4000, "n_q": 32, "n_kv": 8, "d": 128, "block": 32, "mode": "E5M2", "causal": True, "out": "float16"},
        # cross attention: three ragged decoder chunks look at all the states of encoders of another length
        {"name": "cross_wide", "kind": "attend", "n_seq": 3, "q_min": 97, "q_max": 203, "chunk": 0, "ctx_min": 750,
         "ctx_max": 1501, "n_q": 8, "n_kv": 8, "d": 256, "block": 16, "mode": "E4M3", "causal": False, "out": "float16"},
        # one request, 16 new tokens behind a context of 65537: the cache streams once, split over its length
        {"name": "long_context", "kind": "attend", "n_seq": 1, "q_min": 16, "q_max": 16, "chunk": 0, "ctx_min": 65537,
         "ctx_max": 65537, "n_q": 32, "n_kv": 8, "d": 128, "block": 16, "mode": "E4M3", "causal": True, "out": "float16"},
        # a prefill chunk of 2048 tokens behind 6144 cached ones: compute bound
        {"name": "prefill_chunk", "kind": "attend", "n_seq": 1, "q_min": 2048, "q_max": 2048, "chunk": 0, "ctx_min": 8192,
         "ctx_max": 8192, "n_q": 32, "n_kv": 4, "d": 64, "block": 16, "mode": "E5M2", "causal": True, "out": "float16"},
        # rotary positions and append of one token for each of 32 requests
        {"name": "rotate_step", "kind": "rotate", "n_seq": 32, "q_min": 1, "q_max": 1, "pos_max": 4095, "n_q": 32,
         "n_kv": 4, "d": 64, "rot": 64, "layout": "half", "factor": 1.0, "block": 16, "mode": "E4M3", "source": "float32"},
        # ragged prefill chunks of a model that rotates half of each head, interleaved, far beyond its trained context
        {"name": "rotate_chunks", "kind": "rotate", "n_seq": 9, "q_min": 301, "q_max": 700, "pos_max": 130000, "n_q": 32,
         "n_kv": 8, "d": 128, "rot": 64, "layout": "interleaved", "factor": 8.0, "block": 16, "mode": "E4M3",
         "source": "float32"},
        # a beam search over two requests of four beams reorders its beams
        {"name": "fork_beams", "kind": "fork", "groups": 2, "beams": 4, "survivors": 2, "finished": 0, "ctx": 300,
         "max_blocks": 32, "block": 16, "n_blocks": 512, "layers": 4, "n_kv": 4, "d": 64},
        # 64 requests of four samples each: a quarter of the slots ends, the rest goes on from the survivors; 22 layers
        {"name": "fork_samples", "kind": "fork", "groups": 64, "beams": 4, "survivors": 2, "finished": 64, "ctx": 1200,
         "max_blocks": 128, "block": 16, "n_blocks": 20480, "layers": 22, "n_kv": 4, "d": 64},
        # a small pool with holes is packed together
        {"name": "compact_small", "kind": "compact", "n_seq": 8, "max_blocks": 32, "live": 150, "block": 16,
         "n_blocks": 512, "layers": 4, "n_kv": 4, "d": 64},
        # a whole decoder's pool, 60 % in use, is packed together to free its upper part
        {"name": "compact_pool", "kind": "compact", "n_seq": 64, "max_blocks": 128, "live": 4915, "block": 16,
         "n_blocks": 8192, "layers": 22, "n_kv": 4, "d": 64},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "rotate", "fork", "compact"])
    block = rng.choice([8, 16, 16, 20, 32, 64])
    if kind == "attend":
        d = rng.choice([64, 64, 128, 128, 256, 512])
        n_q, n_kv = rng.choice([(32, 4), (32, 8), (8, 8), (16, 2), (5, 1), (12, 4)])
        n_seq = _log_int(rng, 1, 48)
        ctx = _log_int(rng, 40, min(65537, 120000 // n_seq))
        rows = min(rng.choice([8, 64, 2048]), ctx, int(1.1e11 / (4.0 * d * n_q * ctx * (n_seq + 4))) + 1)
        q_max = _log_int(rng, 1, rows)
        q_min = rng.randint(max(1, q_max // 2), q_max)
        chunk = rng.choice([0, 0, min(ctx, 4 * q_max + 1)])
        return {"kind": kind, "n_seq": n_seq, "q_min": q_min, "q_max": q_max, "chunk": chunk,
                "ctx_min": rng.randint(max(q_max, ctx // 4), ctx), "ctx_max": ctx, "n_q": n_q, "n_kv": n_kv, "d": d,
                "block": block, "mode": rng.choice(["E4M3", "E5M2"]), "causal": rng.random() < 0.75,
                "out": rng.choice(["float16", "packed"]) if ctx <= 400 else "float16"}   # the mean over more keys is too small for 8 bits
    if kind == "rotate":
        d = rng.choice([64, 128, 256])
        n_q, n_kv = rng.choice([(32, 4), (32, 8), (8, 8), (5, 1)])
        n_seq = _log_int(rng, 1, 64)
        q_max = _log_int(rng, 1, min(4000, 4500 // n_seq))
        return {"kind": kind, "n_seq": n_seq, "q_min": rng.randint(max(1, q_max // 2), q_max), "q_max": q_max,
                "pos_max": _log_int(rng, q_max + 1, 1000000 // n_seq), "n_q": n_q, "n_kv": n_kv, "d": d,
                "rot": d // rng.choice([1, 1, 2, 4]), "layout": rng.choice(["half", "interleaved"]),
                "factor": rng.choice([1.0, 4.0, 8.0]), "block": block, "mode": rng.choice(["E4M3", "E5M2"]),
                "source": rng.choice(["float32", "float32", "float16"])}
    n_kv, d = rng.choice([(4, 64), (8, 64), (2, 128), (1, 128)])
    if kind == "fork":
        groups, beams = _log_int(rng, 1, 64), rng.randint(2, 5)
        ctx = _log_int(rng, block + 1, 1500)
        max_blocks = -(-ctx // block) + rng.randint(2, 20)
        n_blocks = groups * beams * max_blocks + rng.randint(1, 500)
        return {"kind": kind, "groups": groups, "beams": beams, "survivors": rng.randint(1, beams - 1),
                "finished": rng.randint(0, groups), "ctx": ctx, "max_blocks": max_blocks, "block": block,
                "n_blocks": n_blocks, "layers": max(1, min(rng.randint(1, 24), 350000 * 1024 // (n_blocks * n_kv * block * d))),
                "n_kv": n_kv, "d": d}
    n_seq, max_blocks = _log_int(rng, 1, 64), _log_int(rng, 4, 128)
    live = rng.randint(max(1, n_seq * max_blocks // 3), n_seq * max_blocks)
    n_blocks = live + _log_int(rng, 1, live + 8)
    return {"kind": kind, "n_seq": n_seq, "max_blocks": max_blocks, "live": live, "block": block, "n_blocks": n_blocks,
            "layers": max(1, min(rng.randint(1, 22), 350000 * 1024 // (n_blocks * n_kv * block * d))), "n_kv": n_kv, "d": d}


def _spread(lo, hi, n):
    """n whole numbers over [lo, hi], the largest first and the others out of order, the same for every seed."""
    return [hi - ((7 * i) % n) * (hi - lo) // max(1, n - 1) for i in range(n)]


def _lengths(c):
    """New rows and context (the new rows among it) of every sequence of an attention case."""
    q = _spread(c["q_min"], c["q_max"], c["n_seq"])
    if c["chunk"]:
        q[-1] = c["chunk"]
    ctx = _spread(c["ctx_min"], c["ctx_max"], c["n_seq"])
    if c["causal"]:
        ctx = [max(a, b) for a, b in zip(q, ctx)]
    return q, ctx


def work(c):
    if c["kind"] == "attend":
        q, ctx = _lengths(c)
        rows = sum(q)
        pairs = sum(a * b - (a * (a - 1) // 2 if c["causal"] else 0) for a, b in zip(q, ctx))
        out = 2 if c["out"] == "float16" else 1
        return {"bytes": 2 * c["n_kv"] * c["d"] * sum(ctx) + rows * c["n_q"] * c["d"] * (1 + out),
                "flops": 4 * c["n_q"] * c["d"] * pairs}
    if c["kind"] == "rotate":
        rows, heads = sum(_spread(c["q_min"], c["q_max"], c["n_seq"])), c["n_q"] + 2 * c["n_kv"]
        return {"bytes": rows * heads * c["d"] * ((4 if c["source"] == "float32" else 2) + 1),
                "flops": 3 * rows * (c["n_q"] + c["n_kv"]) * c["rot"]}
    block = c["n_kv"] * c["block"] * c["d"]
    if c["kind"] == "fork":
        slots = c["groups"] * c["beams"]
        copies = slots - c["finished"] - min(c["groups"] * c["survivors"], slots - c["finished"])
        return {"bytes": 2 * 2 * c["layers"] * block * copies + 8 * slots * c["max_blocks"] + 8 * c["n_blocks"], "flops": 0}
    moves = int(c["live"] * (1 - c["live"] / c["n_blocks"]))
    return {"bytes": 2 * 2 * c["layers"] * block * moves + 8 * c["n_seq"] * c["max_blocks"] + 12 * c["n_blocks"], "flops": 0}


# ------------------------------------------------------------------------------------------------ inputs

_FP8 = {"E4M3": torch.float8_e4m3fn, "E5M2": torch.float8_e5m2}


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _packed(shape, mode, g):
    """Normal values as packed FP8 words; the last dimension counts words."""
    x = torch.randn(*shape[:-1], shape[-1] * 4, generator=g, device=g.device, dtype=torch.float16)
    return x.to(_FP8[mode]).view(torch.int32)


def _offsets(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32)


def _tables(need, max_blocks, n_blocks, g):
    """A block table whose sequences hold `need` blocks each, drawn from a shuffled pool; the rest of a row is -1."""
    ids = torch.randperm(n_blocks, generator=g, dtype=torch.int32)
    t = torch.full((len(need), max_blocks), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = ids[at:at + n]
        at += n
    return t


def prepare(case, seed):
    c, dev = case, _device()
    g, h = torch.Generator(device=dev).manual_seed(seed), torch.Generator().manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "attend":
        q, ctx = _lengths(c)
        max_blocks = -(-max(ctx) // c["block"]) + 1
        need = [-(-x // c["block"]) for x in ctx]
        n_blocks = sum(need) + 3
        dw = c["d"] // 4
        s["q"] = _packed((sum(q), c["n_q"], dw), c["mode"], g)
        s["k_cache"] = _packed((n_blocks, c["n_kv"], c["block"], dw), c["mode"], g)
        s["v_cache"] = _packed((n_blocks, c["n_kv"], c["block"], dw), c["mode"], g)
        s["tables"] = _tables(need, max_blocks, n_blocks, h).to(dev)
        s["cu"], s["ctx"] = _offsets(q).to(dev), torch.tensor(ctx, dtype=torch.int32).to(dev)
        s["max_q"] = max(q)
    elif c["kind"] == "rotate":
        q = _spread(c["q_min"], c["q_max"], c["n_seq"])
        start = [max(0, c["pos_max"] - n - i * (c["pos_max"] // (2 * c["n_seq"]))) for i, n in enumerate(q)]
        max_blocks = -(-max(a + b for a, b in zip(start, q)) // c["block"])
        heads = c["n_q"] + 2 * c["n_kv"]
        first = [a // c["block"] for a in start]
        count = [-(-(a + n) // c["block"]) - f for a, n, f in zip(start, q, first)]
        n_blocks = sum(count) + 2
        t = torch.full((c["n_seq"], max_blocks), -1, dtype=torch.int32)
        new = _tables(count, max(count), n_blocks, h)
        for i, (f, n) in enumerate(zip(first, count)):   # the blocks of earlier positions are not looked at
            t[i, f:f + n] = new[i, :n]
        s["qkv"] = torch.randn(sum(q), heads * c["d"], generator=g, device=dev).to(getattr(torch, c["source"]))
        s["k_cache"] = _packed((n_blocks, c["n_kv"], c["block"], c["d"] // 4), c["mode"], g)
        s["v_cache"] = _packed((n_blocks, c["n_kv"], c["block"], c["d"] // 4), c["mode"], g)
        s["tables"], s["cu"], s["start"] = t.to(dev), _offsets(q).to(dev), torch.tensor(start, dtype=torch.int32).to(dev)
        s["freq"], s["amplitude"] = torch.from_numpy(_frequencies(c)).to(dev), _amplitude(c)
    elif c["kind"] == "fork":
        slots = c["groups"] * c["beams"]
        ctx = [c["ctx"] - (i // c["beams"]) % (c["ctx"] // 4 + 1) for i in range(slots)]
        ctx = [x - 1 if x % c["block"] == 0 else x for x in ctx]           # every context ends inside a block
        need = [-(-x // c["block"]) for x in ctx]
        t = _tables(need, c["max_blocks"], c["n_blocks"], h)
        for i in range(slots):                                             # the beams of a group share half of their prefix
            half = (ctx[i] // c["block"]) // 2
            t[i, :half] = t[i // c["beams"] * c["beams"], :half]
        parents = torch.empty(slots, dtype=torch.int32)
        for k in range(c["groups"]):
            keep = torch.randperm(c["beams"], generator=h)[:c["survivors"]]
            pick = torch.cat([torch.arange(c["survivors"]), torch.randint(c["survivors"], (c["beams"] - c["survivors"],), generator=h)])
            parents[k * c["beams"]:(k + 1) * c["beams"]] = (k * c["beams"] + keep[pick]).to(torch.int32)
        for k in range(c["finished"]):
            parents[(k % c["groups"] + 1) * c["beams"] - 1 - k // c["groups"]] = -1
        ref = torch.bincount(t[t >= 0].long(), minlength=c["n_blocks"]).to(torch.int32)
        s["tables"], s["parents"], s["ref"] = t.to(dev), parents.to(dev), ref.to(dev)
        s["ctx"] = torch.tensor(ctx, dtype=torch.int32).to(dev)
        s["room"] = torch.where(parents >= 0, torch.tensor(ctx, dtype=torch.int32)[parents.clamp(min=0).long()] + c["block"], 0).to(torch.int32).to(dev)
        s["caches"] = _words((2 * c["layers"], c["n_blocks"], c["n_kv"], c["block"], c["d"] // 4), g)
    else:
        per = np.diff(np.linspace(0, c["live"], c["n_seq"] + 1).astype(int)).tolist()
        t = _tables(per, c["max_blocks"], c["n_blocks"], h)
        ref = torch.bincount(t[t >= 0].long(), minlength=c["n_blocks"]).to(torch.int32)
        s["tables"], s["ref"] = t.to(dev), ref.to(dev)
        s["caches"] = _words((2 * c["layers"], c["n_blocks"], c["n_kv"], c["block"], c["d"] // 4), g)
    if "caches" in s:
        s["cache_list"] = list(s["caches"].unbind(0))
    return s


def _words(shape, g):
    return torch.randint(-2 ** 31, 2 ** 31 - 1, shape, generator=g, device=g.device, dtype=torch.int32)


def _frequencies(c):
    """Turns per position of every rotated pair: theta^(-2j / rot) / (2 pi), the slow pairs stretched by `factor`
    where a pair makes fewer than `low` turns over the trained context, unchanged above `high`, a ramp between."""
    j = np.arange(c["rot"] // 2, dtype=np.float64)
    f = 10000.0 ** (-2.0 * j / c["rot"]) / (2.0 * np.pi)
    keep = np.clip((4096.0 * f - 1.0) / (32.0 - 1.0), 0.0, 1.0)
    return f * (keep + (1.0 - keep) / c["factor"])


def _amplitude(c):
    return 0.1 * math.log(c["factor"]) + 1.0


# ------------------------------------------------------------------------------------------------ one pass

def run(s):
    kind = s["case"]["kind"]
    if kind == "attend":
        return _attend(s)
    if kind == "rotate":
        return _rotate(s)
    return _fork(s) if kind == "fork" else _compact(s)


def _decode(words, mode):
    """The framework's decode of packed words in 32 bits: E5M2 as it is; E4M3 codes with a zero exponent stand for
    m 2^-17, and 0x7F for 480."""
    x = words.view(_FP8[mode]).float()
    if mode == "E4M3":
        mag = words.view(torch.uint8) & 0x7F
        x = torch.where(mag < 8, x * 2.0 ** -8, x)
        x = torch.where(mag == 0x7F, torch.where(words.view(torch.uint8) > 0x7F, -480.0, 480.0), x)
    return x


def _attend(s):
    c = s["case"]
    if own:
        from feather_amd.routines.paged_attention import paged_chunk_attention_fp8_acc_fp32_gpu
        out = paged_chunk_attention_fp8_acc_fp32_gpu(
            s["q"], s["k_cache"], s["v_cache"], s["tables"], s["cu"], s["ctx"], mode=c["mode"], causal=c["causal"],
            max_q_len=s["max_q"], out_dtype=torch.uint32 if c["out"] == "packed" else torch.float16)
        return out.view(_FP8[c["mode"]]) if c["out"] == "packed" else out
    n_seq, n_kv, group, d, dev = c["n_seq"], c["n_kv"], c["n_q"] // c["n_kv"], c["d"], s["q"].device
    total, max_q = s["q"].shape[0], s["max_q"]
    row = torch.arange(total, device=dev)
    seq = torch.searchsorted(s["cu"][1:].long(), row, right=True)
    at = row - s["cu"].long()[seq]
    q = torch.zeros((n_seq, max_q, n_kv, group, d), device=dev)
    q[seq, at] = _decode(s["q"], c["mode"]).view(total, n_kv, group, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(n_seq, n_kv, max_q * group, d)
    blocks = s["tables"].clamp(min=0).long()
    keys = blocks.shape[1] * c["block"]
    gather = lambda cache: _decode(cache[blocks], c["mode"]).permute(0, 2, 1, 3, 4).reshape(n_seq, n_kv, keys, d)
    scores = (q @ gather(s["k_cache"]).transpose(2, 3)).view(n_seq, n_kv, max_q, group, keys) * (1.0 / math.sqrt(d))
    key = torch.arange(keys, device=dev)
    last = s["ctx"].long()[:, None].expand(n_seq, max_q) - 1
    if c["causal"]:
        lens = (s["cu"][1:] - s["cu"][:-1]).long()
        last = last - (lens[:, None] - 1 - torch.arange(max_q, device=dev)[None, :])
    hidden = (key[None, None, :] > last[:, :, None])[:, None, :, None, :]
    scores = scores.masked_fill(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    sums = p.sum(-1, keepdim=True)
    o = (p.view(n_seq, n_kv, max_q * group, keys) @ gather(s["v_cache"])).view(n_seq, n_kv, max_q, group, d)
    o = (o / torch.where(sums == 0, 1.0, sums))[seq, :, at].reshape(total, n_kv * group, d)
    return o.half().to(_FP8[c["mode"]]).view(total, -1) if c["out"] == "packed" else o.half()


def _rotate(s):
    c = s["case"]
    if own:
        from feather_amd.routines.producers import rope_append_chunk
        q, after, status = rope_append_chunk(
            s["qkv"], s["cu"], s["start"], s["tables"], s["k_cache"], s["v_cache"], n_q_heads=c["n_q"], freq=s["freq"],
            amplitude=s["amplitude"], layout=c["layout"], mode=c["mode"])
        return [q.view(_FP8[c["mode"]]), s["k_cache"].view(_FP8[c["mode"]]), s["v_cache"].view(_FP8[c["mode"]]), after, status]
    total, dev, d, rot = s["qkv"].shape[0], s["qkv"].device, c["d"], c["rot"]
    row = torch.arange(total, device=dev)
    seq = torch.searchsorted(s["cu"][1:].long(), row, right=True)
    pos = s["start"].long()[seq] + row - s["cu"].long()[seq]
    turns = pos.double()[:, None] * s["freq"]
    angle = (turns - torch.round(turns)) * (2.0 * math.pi)
    cos = (torch.cos(angle) * s["amplitude"]).float()[:, None]
    sin = (torch.sin(angle) * s["amplitude"]).float()[:, None]
    x = s["qkv"].float().view(total, -1, d)
    turned = x[:, :c["n_q"] + c["n_kv"]]
    part = turned[..., :rot]
    if c["layout"] == "half":
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        part = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    turned = torch.cat([part, turned[..., rot:]], -1)
    code = lambda v: v.half().to(_FP8[c["mode"]]).view(torch.int32)
    block, slot = s["tables"].long()[seq, pos // c["block"]], pos % c["block"]
    s["k_cache"][block, :, slot] = code(turned[:, c["n_q"]:])
    s["v_cache"][block, :, slot] = code(x[:, c["n_q"] + c["n_kv"]:])
    lens = s["cu"][1:] - s["cu"][:-1]
    return [code(turned[:, :c["n_q"]]).view(_FP8[c["mode"]]), s["k_cache"].view(_FP8[c["mode"]]),
            s["v_cache"].view(_FP8[c["mode"]]), s["start"] + lens, torch.zeros_like(s["start"])]


def _counts(table, n_blocks):
    t = table[table >= 0].long()
    return torch.zeros(n_blocks, dtype=torch.int32, device=table.device).index_add_(0, t, torch.ones_like(t, dtype=torch.int32))


def _fork(s):
    c = s["case"]
    if own:
        from feather_amd.routines.paged_cache import paged_cache_fork
        t, ctx, ref, status = paged_cache_fork(s["cache_list"], s["tables"], s["ctx"], s["ref"], s["parents"], room=s["room"])
        return [t, ctx, ref, status, s["caches"]]
    dev, slots, width, block = s["tables"].device, s["tables"].shape[0], c["max_blocks"], c["block"]
    parent = s["parents"].long().clamp(min=0)
    alive = s["parents"] >= 0
    i = torch.arange(slots, device=dev)
    same = (s["parents"][:, None] == s["parents"][None, :]) & (i[None, :] < i[:, None])
    heir = alive & ~same.any(1)
    ctx = torch.where(alive, s["ctx"][parent], 0)
    full, used = (ctx // block)[:, None], ((ctx + block - 1) // block)[:, None]
    e = torch.arange(width, device=dev)[None, :]
    old = s["tables"][parent]
    table = torch.where(alive[:, None] & ((e < full) | heir[:, None]), old, -1)
    tail = (alive & ~heir)[:, None] & (e == full) & (used > full) & (old >= 0)
    want = ((s["room"] + block - 1) // block).clamp(max=width)[:, None]
    fresh = tail | ((e >= used) & (e < want) & (table < 0))
    ref = s["ref"] - _counts(s["tables"], c["n_blocks"]) + _counts(table, c["n_blocks"])
    free = torch.nonzero(ref == 0).flatten().to(torch.int32)
    rank = (torch.cumsum(fresh.flatten(), 0) - 1).view(slots, width)
    got = fresh & (rank < free.numel())
    table[got] = free[rank[got]]
    ref = ref + _counts(torch.where(got, table, -1), c["n_blocks"])
    copy = got & tail
    s["caches"][:, table[copy].long()] = s["caches"][:, old[copy].long()]
    status = (fresh & ~got).any(1).to(torch.int32) * 3
    ctx = torch.where((tail & ~got).any(1), full[:, 0] * block, ctx)
    return [table, ctx, ref, status, s["caches"]]


def _compact(s):
    c = s["case"]
    if own:
        from feather_amd.routines.paged_cache import paged_cache_compact
        t, ref, moved, live = paged_cache_compact(s["cache_list"], s["tables"], s["ref"])
        return [t, ref, moved, live, s["caches"]]
    b = torch.arange(c["n_blocks"], device=s["ref"].device)
    used = s["ref"] > 0
    live = used.sum()
    to = torch.nonzero(~used & (b < live)).flatten()
    frm = torch.nonzero(used & (b >= live)).flatten().flip(0)
    moved = torch.where(used, b, -1).to(torch.int32)
    moved[frm] = to.to(torch.int32)
    ref = torch.where(b < live, s["ref"], 0)
    ref[to] = s["ref"][frm]
    s["caches"][:, to] = s["caches"][:, frm]
    table = torch.where(s["tables"] >= 0, moved[s["tables"].clamp(min=0).long()], -1)
    return [table, ref, moved, live.to(torch.int32).view(1), s["caches"]]


# ------------------------------------------------------------------------------------------------ 64 bits

def _values(mode):
    """The 256 values of a packed code, from the format: E5M2 is the upper byte of a half; E4M3 has a bias of 7, its
    zero-exponent codes are the halves with that mantissa and exponent zero, and nothing is infinite or NaN."""
    code = np.arange(256, dtype=np.uint16)
    if mode == "E5M2":
        bits = code << 8
    else:
        e, m = (code >> 3) & 15, code & 7
        bits = ((code & 128) << 8) | (np.where(e > 0, e + 8, 0) << 10).astype(np.uint16) | (m << 7)
    return torch.from_numpy(bits.astype(np.uint16).view(np.float16).astype(np.float64))


def exact(case, seed):
    if case["kind"] == "attend":
        return _attend_exact(case, seed)
    return _rotate_exact(case, seed) if case["kind"] == "rotate" else None


def _attend_exact(c, seed):
    s = prepare(c, seed)
    dev, d, group = s["q"].device, c["d"], c["n_q"] // c["n_kv"]
    value = _values(c["mode"]).to(dev)
    look = lambda w: value[w.contiguous().view(torch.uint8).int()]
    lens, ctxs = _lengths(c)
    out, at = torch.zeros((s["q"].shape[0], c["n_q"], d), dtype=torch.float64, device=dev), 0
    for i, (n, ctx) in enumerate(zip(lens, ctxs)):
        pos = torch.arange(ctx, device=dev)
        block, slot = s["tables"][i].long()[pos // c["block"]], pos % c["block"]
        for h in range(c["n_kv"]):
            k, v = look(s["k_cache"][block, h, slot]), look(s["v_cache"][block, h, slot])
            q = look(s["q"][at:at + n, h * group:(h + 1) * group]).transpose(0, 1).reshape(group * n, d)
            x = torch.mm(q, k.t()).div_(math.sqrt(d)).view(group, n, ctx)
            if c["causal"]:
                row = torch.arange(n, device=dev)
                x.masked_fill_(pos[None, :] - (ctx - n) > row[:, None], -math.inf)
            x = torch.exp_(x.sub_(x.max(dim=-1, keepdim=True).values))
            y = torch.mm(x.view(group * n, ctx), v) / x.sum(dim=-1).view(group * n, 1)
            out[at:at + n, h * group:(h + 1) * group] = y.view(group, n, d).transpose(0, 1)
        at += n
    if c["out"] == "packed":
        return out.view(at, -1) if c["mode"] == "E4M3" else None   # half a step of E5M2 is most of what a value may be off
    return out


def _rotate_exact(c, seed):
    if c["mode"] == "E5M2":
        return None                                                # as above
    s = prepare(c, seed)
    dev, d, pairs, q = s["qkv"].device, c["d"], c["rot"] // 2, c["n_q"]
    lens = _spread(c["q_min"], c["q_max"], c["n_seq"])
    start = s["start"].tolist()
    pos = torch.cat([torch.arange(a, a + n, device=dev) for a, n in zip(start, lens)]).double()
    turns = pos[:, None] * s["freq"][None, :]
    z = torch.polar(torch.full_like(turns, s["amplitude"]), 2.0 * math.pi * (turns - torch.floor(turns)))
    x = s["qkv"].double().view(-1, q + 2 * c["n_kv"], d)
    first = torch.arange(pairs, device=dev) * (1 if c["layout"] == "half" else 2)
    second = first + (pairs if c["layout"] == "half" else 1)
    w = torch.complex(x[:, :q + c["n_kv"]][..., first], x[:, :q + c["n_kv"]][..., second]) * z[:, None, :]
    y = x.clone()
    y[:, :q + c["n_kv"], first] = w.real
    y[:, :q + c["n_kv"], second] = w.imag
    caches = [t.view(_FP8[c["mode"]]).double() for t in (s["k_cache"], s["v_cache"])]
    at = 0
    for i, (a, n) in enumerate(zip(start, lens)):
        p = torch.arange(a, a + n, device=dev)
        block, slot = s["tables"][i].long()[p // c["block"]], p % c["block"]
        caches[0][block, :, slot] = y[at:at + n, q:q + c["n_kv"]]
        caches[1][block, :, slot] = y[at:at + n, q + c["n_kv"]:]
        at += n
    return [y[:, :q], caches[0], caches[1], None, None]
