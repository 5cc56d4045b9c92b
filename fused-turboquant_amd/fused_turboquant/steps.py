"""The steps of a speculative decode around the slot cache's attention, each one
launch on the device where a host program would synchronise:

* ``step_tables``: block tables, slots, positions and lengths of a step's
  tokens from the requests' lengths; with a free list, the pages a request
  gains or gives back.
* ``tree_accept``: the accepted path of every drafted tree.
* ``tree_shape``: depths and mask of a tree (on the host).
* ``commit_slots``: the accepted tokens' slots moved to consecutive positions,
  in every layer's cache.

``v1.v1_tree_attention`` is the attention between them.  The slot caches are
those of ``v1_store`` and ``raw_store``: ``uint8[num_blocks, block_size,
num_kv_heads, slot]``.  The reference has no counterpart: its block tables and
slots come from vLLM's host-side metadata builder (``vllm_plugin/
v1_backend.py:777-830``), and it decodes one token a sequence.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence

import torch

from . import _lib, _ops


MAX_REQUESTS = 4096  # of one step_tables call


class StepTables(NamedTuple):
    """What ``step_tables`` returns."""
    slot_mapping: torch.Tensor   # int64 [num_tokens]; -1: padding, or no page
    positions: torch.Tensor      # int64 [num_tokens]; 0 for padding
    token_request: torch.Tensor  # int32 [num_tokens]; -1 for padding
    seq_lens: torch.Tensor       # int32 [B], the step's tokens among them
    missing: torch.Tensor        # int32 [1]: pages that the free list or the table's width lacked


class Accepted(NamedTuple):
    """What ``tree_accept`` returns."""
    path: torch.Tensor           # int32 [B, max_nodes]: accepted nodes, the root first; then -1
    counts: torch.Tensor         # int32 [B]
    tokens: torch.Tensor         # int64 [B, max_nodes]: the target's token after each of them; then -1


def _ints(name: str, t: torch.Tensor, dim: int, dtype: torch.dtype = torch.int32) -> torch.Tensor:
    if t.dtype != dtype or t.dim() != dim:
        raise ValueError(f"{name} must be {str(dtype).replace('torch.', '')} with {dim} dimension(s)")
    return t.contiguous()


def _in_place(name: str, t: torch.Tensor) -> torch.Tensor:
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of one dimension")
    return t


def tree_shape(parents: Sequence[int]) -> tuple[torch.Tensor, torch.Tensor]:
    """``(depths, mask)`` of a tree from its nodes' parents (the root's -1
    first, every parent before its children): int32 [n], and int64 [n, words]
    with bit j of a node's row set for its ancestors and itself, the
    ``tree_mask`` of ``v1.v1_tree_attention``.  Host tensors, computed once
    for a tree that is drafted again and again."""
    n = len(parents)
    if n == 0 or parents[0] != -1:
        raise ValueError("parents must start with the root's -1")
    depth, rows = [0], [1]
    for i in range(1, n):
        p = int(parents[i])
        if not 0 <= p < i:
            raise ValueError(f"parents[{i}] = {p}: a parent comes before its children, and there is one root")
        depth.append(depth[p] + 1)
        rows.append(rows[p] | 1 << i)
    low = (1 << 64) - 1
    words = [[(r >> 64 * w) & low for w in range((n + 63) // 64)] for r in rows]
    signed = [[x - (1 << 64) if x >> 63 else x for x in r] for r in words]
    return torch.tensor(depth, dtype=torch.int32), torch.tensor(signed, dtype=torch.int64)


def step_tables(query_start_loc: torch.Tensor, past_lens: torch.Tensor, block_table: torch.Tensor, block_size: int,
                num_tokens: int, depths: Optional[torch.Tensor] = None, num_blocks: Optional[torch.Tensor] = None,
                free_blocks: Optional[torch.Tensor] = None, free_count: Optional[torch.Tensor] = None) -> StepTables:
    """Slots and positions of a step whose request ``b`` has the flat tokens
    ``query_start_loc[b] .. query_start_loc[b + 1]`` (int32 [B + 1], ascending)
    after ``past_lens[b]`` (int32 [B]) stored ones.

    Token i of request b is stored at position ``past_lens[b] + i``; its
    ``positions`` entry (for the rotary embedding) is ``past_lens[b]`` plus i,
    or plus its entry of ``depths`` (int32 [num_tokens]; the nodes of a drafted
    tree).  ``num_tokens`` sizes the outputs; tokens behind the last request
    are padding.  A token whose page the row of ``block_table`` (int32 [B,
    max_blocks], rows contiguous) does not have, or has as a negative entry,
    gets slot -1, which the stores skip.

    With ``num_blocks`` (int32 [B], the pages each request holds),
    ``free_blocks`` (int32, room for every page of the pool) and
    ``free_count`` (int32 [1], how many of its entries are free) the tables are
    brought to the requests' lengths first, all in place: a request holds
    ceil(length / block_size) pages afterwards, more go back to the free list
    (a finished request: both its lengths 0), new ones are taken from its end.
    Requests come in order, so when the list runs out the last ones stay short:
    ``missing`` counts those pages, and the ones past the table's width.
    Nothing is read on the host.  At most 4096 requests.
    """
    qsl, past = _ints("query_start_loc", query_start_loc, 1), _ints("past_lens", past_lens, 1)
    B = past.numel()
    if qsl.numel() != B + 1:
        raise ValueError("query_start_loc must have one entry more than past_lens")
    if B > MAX_REQUESTS:
        raise ValueError(f"step_tables takes at most {MAX_REQUESTS} requests")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != B:
        raise ValueError("block_table must be int32 [B, max_blocks]")
    if block_table.numel() and block_table.shape[1] > 1 and block_table.stride(1) != 1 or (B > 1 and block_table.stride(0) < block_table.shape[1]):
        raise ValueError("block_table rows must be contiguous and must not overlap")
    if num_tokens < 0 or block_size < 1:
        raise ValueError("num_tokens must be >= 0 and block_size >= 1")
    if depths is not None:
        depths = _ints("depths", depths, 1)
        if depths.numel() < num_tokens:
            raise ValueError("depths must have an entry for every token")
    state = (num_blocks, free_blocks, free_count)
    if any(t is None for t in state) != all(t is None for t in state):
        raise ValueError("num_blocks, free_blocks and free_count go together")
    if num_blocks is not None:
        if _in_place("num_blocks", num_blocks).numel() != B or _in_place("free_count", free_count).numel() != 1:
            raise ValueError("num_blocks must have B entries and free_count one")
        _in_place("free_blocks", free_blocks)
    _lib.require_device(qsl, past, block_table, depths, *state)
    return StepTables(*_ops.ops().step_tables(qsl, past, depths, block_table, int(block_size), int(num_tokens), num_blocks,
                                              free_blocks, free_count))


def tree_accept(tokens: torch.Tensor, parents: torch.Tensor, targets: torch.Tensor, query_start_loc: torch.Tensor,
                max_nodes: int) -> Accepted:
    """The path that each tree's root starts and the target model agrees with.

    Flat nodes, request b's at ``query_start_loc[b] .. query_start_loc[b + 1]``
    (int32 [B + 1]), the root first: ``tokens`` (int64, the drafted tokens),
    ``parents`` (int32, the parent's index inside the request; every parent
    before its children, the root's entry is not read) and ``targets`` (int64,
    the token that the target model gives after each node: its argmax, or a
    sample, which leaves the target's distribution as it is).  From the root
    the walk goes to the child whose token is the current node's target, the
    lowest index among equals, until there is none.  A request without nodes
    has an empty path.  ``max_nodes`` (1 .. 2048) is the outputs' width; nodes
    past it are not looked at.
    """
    qsl = _ints("query_start_loc", query_start_loc, 1)
    tok, tgt = _ints("tokens", tokens, 1, torch.int64), _ints("targets", targets, 1, torch.int64)
    par = _ints("parents", parents, 1)
    if qsl.numel() < 1:
        raise ValueError("query_start_loc must have B + 1 entries")
    if not (tok.numel() == par.numel() == tgt.numel()):
        raise ValueError("tokens, parents and targets must have one entry per node")
    if not 1 <= max_nodes <= 2048:
        raise ValueError("max_nodes must be in 1..2048")
    _lib.require_device(tok, par, tgt, qsl)
    return Accepted(*_ops.ops().tree_accept(tok, par, tgt, qsl, int(max_nodes)))


def _check_caches(caches: Sequence[torch.Tensor]) -> None:
    first = caches[0]
    for c in caches:
        if c.dtype != torch.uint8 or c.dim() != 4:
            raise ValueError("kv_caches must be uint8 [num_blocks, block_size, num_kv_heads, slot]")
        if c.stride(3) != 1:
            raise ValueError("kv_cache slot bytes must be contiguous")
        if c.shape != first.shape or c.stride() != first.stride() or c.device != first.device:
            raise ValueError("kv_caches must have one shape and layout, on one device")
    if len({c.data_ptr() for c in caches}) != len(caches):
        raise ValueError("kv_caches names a cache twice")


def commit_slots(kv_caches: Sequence[torch.Tensor], block_table: torch.Tensor, past_lens: torch.Tensor,
                 path: torch.Tensor, counts: torch.Tensor) -> None:
    """Move the slots of every accepted path together, in place: in each cache
    of ``kv_caches`` (the layers' ``uint8[num_blocks, block_size, num_kv_heads,
    slot]``, all of one shape and layout, none twice) position ``past_lens[b] +
    path[b, j]`` of request b goes to position ``past_lens[b] + j``, for j <
    ``counts[b]``.  ``path`` (int32 [B, n]) and ``counts`` (int32 [B]) are
    ``tree_accept``'s; a path ascends, and an entry that does not ends it.
    Other slots stay as they are.  Positions without a page are skipped.  A
    slot's bytes do not depend on its position (keys are stored with their
    rotary embedding, and a node's depth on the path is its index there), so
    the sequences continue from ``past_lens + counts``.
    """
    caches = list(kv_caches)
    if block_table.dtype != torch.int32 or block_table.dim() != 2:
        raise ValueError("block_table must be int32 [B, max_blocks]")
    B = block_table.shape[0]
    past, cnt = _ints("past_lens", past_lens, 1), _ints("counts", counts, 1)
    pth = _ints("path", path, 2)
    if past.numel() != B or cnt.numel() != B or pth.shape[0] != B:
        raise ValueError("past_lens, counts and path must have one entry (row) per row of block_table")
    if not caches:
        return
    if not caches[0].is_cuda:  # (the operator checks the layers' caches, in less time)
        _check_caches(caches)
    _lib.require_device(caches[0], block_table, past, pth, cnt)
    _ops.ops().commit_slots(caches, block_table.contiguous(), past, pth, cnt)
