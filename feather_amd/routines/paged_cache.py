"""The pages of a paged FP8 KV cache as a pool on the device (``csrc/cache_pages.hip``): fork the sequences of a batch
(beam search, samples of one prompt, reordering, ending), reserve room, and move the blocks in use together.  The
reference has no KV cache.

The state is a block table ``[n_seq, max_blocks]`` int32 (-1: no block), the lengths ``ctx_lens [n_seq]`` int32 and
``ref_counts [n_blocks]`` int32: how many table entries (and pins of the caller) hold a block, 0 = free.  Calls return new
tables, lengths and counts; the caches are updated in place, in blocks that were free or that the call releases: after a
fork the tables passed in are void.  Nothing is copied to the host.
"""
from __future__ import annotations

import array
import operator

import torch

from .. import _native as N

__all__ = ["paged_cache_fork", "paged_cache_compact"]


def _index(t: torch.Tensor, name: str, shape=None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or not t.is_cuda:
        raise ValueError(f"{name} must be an int32 tensor on the device")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t.contiguous()


_dtype, _shape = operator.attrgetter("dtype"), operator.attrgetter("shape")


def _pool(caches, ref_counts: torch.Tensor):
    """Checks the caches against the pool; returns their pointers as an array, how many, and the bytes and tokens of a
    block.  (A decoder has dozens of caches: every check is one pass in C over all of them.)"""
    caches = tuple(caches)
    if not caches:
        raise ValueError("caches must hold at least one cache tensor")
    first = N.as_words(caches[0], "caches[0]")
    try:
        devices, dtypes, shapes = set(map(torch.Tensor.get_device, caches)), set(map(_dtype, caches)), set(map(_shape, caches))
        whole, ptrs = all(map(torch.Tensor.is_contiguous, caches)), list(map(torch.Tensor.data_ptr, caches))
    except TypeError:
        raise ValueError("caches must be tensors of packed words") from None
    if len(devices) != 1 or len(shapes) != 1:
        raise ValueError("all caches must have the same shape and device")
    if not dtypes.issubset(N._WORD_DTYPES):
        raise ValueError(f"caches must be uint32/int32/float32 containers, got {dtypes}")
    if not whole or first.dim() != 4:
        raise ValueError("caches are updated in place: expected contiguous [n_blocks, n_kv_heads, block_size, d/4]")
    n_blocks, n_kv, block_size, dw = first.shape
    block_bytes = 4 * n_kv * block_size * dw
    if block_bytes == 0 or block_bytes % 16 != 0:
        raise ValueError(f"a block of {block_bytes} bytes is not a multiple of 16")
    ordered = sorted(ptrs)
    if min(map(operator.sub, ordered[1:], ordered), default=n_blocks * block_bytes) < n_blocks * block_bytes:
        raise ValueError("caches overlap (or the same tensor is there twice)")
    if ref_counts.shape != (n_blocks,) or n_blocks < 1:
        raise ValueError(f"ref_counts must be [n_blocks={n_blocks}] with at least one block")
    if ref_counts.device != first.device:
        raise ValueError("ref_counts and the caches must be on the same device")
    return array.array("Q", ptrs), len(ptrs), block_bytes, block_size


def paged_cache_fork(caches, block_tables: torch.Tensor, ctx_lens: torch.Tensor, ref_counts: torch.Tensor,
                     parents: torch.Tensor, *, room: torch.Tensor | None = None):
    """Slot ``i`` of the batch goes on as a copy of slot ``parents[i]``.

    caches      the caches that share the tables (K and V of every layer), each ``[n_blocks, n_kv_heads, block_size, d/4]``
    parents     ``[n_seq]`` int32; a value outside ``[0, n_seq)`` (-1) ends the slot and gives its blocks back
    room        optional ``[n_seq]`` int32: positions the slot's row must cover afterwards (fresh blocks are added)
    Returns ``(block_tables, ctx_lens, ref_counts, status)``.  Whole blocks of a context are shared by all children; the
    block it ends in stays with the first child of a parent and is copied for the others, because each of them writes its
    next token there; the first child gets a copy too if another entry or a pin holds that block (``ref_counts`` above 1),
    and entries behind the context that are held so are dropped.  That happens when a length was set back into blocks that
    an earlier fork shared: such a slot must go through this call (as its own parent) before the next append.  Fresh blocks
    are taken lowest id first in (slot, entry) order.  ``status``: 0; 1 ``room`` beyond the table; 2 a table entry within
    the context is not a block; 3 the pool ran out (the missing entries are -1, and a slot that lost the copy of its last
    block keeps its whole blocks as its length).  ``ref_counts`` must count the rows of ``block_tables``.  Blocks that the
    old rows let go may be handed out and written in the same call, so the tables passed in are void after it, also with
    status 3: a slot that must survive needs a child."""
    ref_counts = _index(ref_counts, "ref_counts")
    ptrs, n_caches, block_bytes, block_size = _pool(caches, ref_counts)
    block_tables = _index(block_tables, "block_tables")
    if block_tables.dim() != 2:
        raise ValueError("block_tables must be [n_seq, max_blocks]")
    n_seq, max_blocks = block_tables.shape
    ctx_lens, parents = _index(ctx_lens, "ctx_lens", (n_seq,)), _index(parents, "parents", (n_seq,))
    if room is not None:
        room = _index(room, "room", (n_seq,))
    dev, n_blocks = ref_counts.device, ref_counts.shape[0]
    if block_tables.device != dev or ctx_lens.device != dev or parents.device != dev or (room is not None and room.device != dev):
        raise ValueError("all tensors must be on the same device")
    tables_out, ctx_out, ref_out = torch.empty_like(block_tables), torch.empty_like(ctx_lens), torch.empty_like(ref_counts)
    status = torch.empty_like(ctx_lens)
    scratch = ref_counts.new_empty(N.lib().feather_paged_cache_fork_scratch_bytes(n_seq, n_blocks) // 4)
    N.call(dev, "feather_paged_cache_fork", ptrs.buffer_info()[0], n_caches, block_bytes, block_tables.data_ptr(),
           ctx_lens.data_ptr(), ref_counts.data_ptr(), parents.data_ptr(), room.data_ptr() if room is not None else None,
           tables_out.data_ptr(), ctx_out.data_ptr(), ref_out.data_ptr(), status.data_ptr(), scratch.data_ptr(), n_seq, max_blocks,
           block_size, n_blocks)
    return tables_out, ctx_out, ref_out, status


def paged_cache_compact(caches, block_tables: torch.Tensor, ref_counts: torch.Tensor):
    """Moves the blocks in use (``ref_counts > 0``) to the ids ``0 .. n_live - 1``.

    Returns ``(block_tables, ref_counts, block_map, n_live)``: ``block_map [n_blocks]`` int32 is the new id of every old
    block (-1: it was free), ``n_live [1]`` int32 stays on the device.  Blocks already below ``n_live`` stay; the highest
    of the others goes into the lowest hole, and so on.  Table entries that are not blocks in use come out as -1.  What
    the caches hold from ``n_live`` on is stale."""
    ref_counts = _index(ref_counts, "ref_counts")
    ptrs, n_caches, block_bytes, _ = _pool(caches, ref_counts)
    block_tables = _index(block_tables, "block_tables")
    dev, n_blocks = ref_counts.device, ref_counts.shape[0]
    if block_tables.device != dev:
        raise ValueError("all tensors must be on the same device")
    tables_out, ref_out, block_map = torch.empty_like(block_tables), torch.empty_like(ref_counts), torch.empty_like(ref_counts)
    n_live = ref_counts.new_empty(1)
    scratch = ref_counts.new_empty(N.lib().feather_paged_cache_compact_scratch_bytes(n_blocks) // 4)
    N.call(dev, "feather_paged_cache_compact", ptrs.buffer_info()[0], n_caches, block_bytes, block_tables.data_ptr(),
           ref_counts.data_ptr(), tables_out.data_ptr(), ref_out.data_ptr(), block_map.data_ptr(), n_live.data_ptr(), scratch.data_ptr(),
           block_tables.numel(), n_blocks)
    return tables_out, ref_out, block_map, n_live
