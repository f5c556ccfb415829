"""A tree of drafted tokens over a paged cache: where its nodes go and what each sees, attention of all nodes at once, and the walk
down the nodes that the model agreed with, whose cache rows move to the places they keep. With PyTorch reference statements.

Node 0 of a sequence is the anchor, the last token it has for certain; every other node names an earlier one as its parent. The
nodes of sequence s are rows ``cu[s]:cu[s+1]`` of a call. Node i is written at token place ``base + i`` of the sequence (``base``:
tokens before the anchor) and turned by position ``base + depth``, so that an agreed path, once moved together, is what writing
its tokens one after the other would have left.
"""
from __future__ import annotations

import struct

import torch

from .kv_e4m3 import attention_args, attention_rows, heads_ok, need, on_device, pool_ok, same_device
from .launcher import Kernels, i32, ptr

MAX_NODES = 256
MAX_POOLS = 128


def bf16_pool_ok(pool: torch.Tensor, hk: int, page_size: int, d: int) -> None:
    need(pool.dtype == torch.bfloat16 and pool.dim() == 5 and tuple(pool.shape[1:]) == (2, hk, page_size, d) and pool.is_contiguous(),
         f"a bf16 pool is a contiguous [pages, 2, {hk}, {page_size}, {d}] tensor")
    need(pool.shape[0] >= 1 and pool.data_ptr() % 16 == 0, "the pool has a page, and starts on 16 bytes")


def any_pool_ok(pool: torch.Tensor, hk: int, page_size: int, d: int) -> None:
    (pool_ok if pool.dtype == torch.uint8 else bf16_pool_ok)(pool, hk, page_size, d)


def tree_attention(q: torch.Tensor, pool: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, masks: torch.Tensor,
                   cu_q: torch.Tensor, hq: int, hk: int, d: int, page_size: int, *, out: torch.Tensor | None = None,
                   max_rows: int | None = None, max_len: int | None = None, scale: float | None = None) -> torch.Tensor:
    """Attention of every sequence's tree nodes over its cache, bf16 (``[pages, 2, hk, page_size, d]``) or 8-bit (`kv_e4m3`).

    Rows of sequence s are ``cu_q[s]:cu_q[s+1]``, its last R of ``seq_lens[s]`` tokens. Row i sees every token before the tree
    and node j where bit j of ``masks[row]`` (i64 ``[rows, words]``, 64 nodes to a word) is set: its ancestors and itself, as
    `tree_rows` gives them, or any other set. A node without a bit of its own (past the words) is seen by none; a row that sees
    nothing gives zeros; what a row does not see does not reach it, infinities and NaN included. Other arguments, and rows
    behind the last sequence's, as in `kv_e4m3.paged_attention_e4m3`."""
    heads_ok(hq, hk, d, page_size)
    any_pool_ok(pool, hk, page_size, d)
    need(cu_q is not None, "cu_q: i32 [seqs + 1]")
    out, max_rows, max_len, scale = attention_args(q, pool, block_table, seq_lens, cu_q, hq, hk, d, page_size, out, 1, max_rows, max_len, scale)
    need(masks.dtype == torch.int64 and masks.dim() == 2 and masks.is_contiguous() and masks.shape[0] >= q.shape[0]
         and 1 <= masks.shape[1] <= MAX_NODES // 64, f"masks: contiguous i64 [rows, words], up to {MAX_NODES // 64} words")
    same_device(q, masks)
    if block_table.shape[0] == 0 or max_rows == 0:
        return out
    with on_device(q):
        return attention_rows(q, pool, block_table, seq_lens, masks, cu_q, hq, hk, d, page_size, out, 1, max_rows, max_len, scale)


def _glue_ok(parents: torch.Tensor, cu: torch.Tensor, base: torch.Tensor, block_table: torch.Tensor, page_size: int, max_rows: int | None) -> int:
    need(parents.dtype == torch.int32 and parents.dim() == 1 and parents.is_contiguous(), "parents: i32 [nodes]")
    need(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.is_contiguous() and block_table.shape[1] >= 1,
         "block_table: contiguous i32 [seqs, pages]")
    seqs = block_table.shape[0]
    need(cu.dtype == torch.int32 and cu.numel() >= seqs + 1 and cu.is_contiguous(), "cu: i32 [seqs + 1]")
    need(base.dtype == torch.int64 and base.numel() >= seqs and base.is_contiguous(), "base: one i64 for each sequence")
    need(page_size >= 1, f"page_size {page_size}")
    most = min(MAX_NODES, parents.shape[0]) if max_rows is None else max_rows
    need(0 <= most <= MAX_NODES, f"{most} nodes: at most {MAX_NODES} in a tree")
    return most


def tree_rows(parents: torch.Tensor, cu: torch.Tensor, base: torch.Tensor, block_table: torch.Tensor, page_size: int, *,
              max_rows: int | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Of every node: its rotary position (i64), cache slot (i64) and mask (i64 ``[nodes, words]``, one word for every 64 of
    ``max_rows``); of every sequence: its context with the tree (i32). The counterpart of `spec.rows` for trees.

    ``parents`` (i32): a node's parent within its sequence, -1 for the anchor. A parent that is not an earlier node, a place past
    the page table, or more than ``max_rows`` (256) nodes set the error word: the node then has no parent, or slot -1 (nothing
    written), or is left out. A sequence of base < 0 is padding: slots -1, positions 0, masks 0, context 0."""
    most = _glue_ok(parents, cu, base, block_table, page_size, max_rows)
    same_device(parents, cu, base, block_table)
    n, dev = parents.shape[0], parents.device
    seqs, words = block_table.shape[0], max(1, -(-most // 64))
    lens = torch.empty(seqs, dtype=torch.int32, device=dev)
    if not seqs:                                  # no launch that would fill them
        return (torch.zeros(n, dtype=torch.int64, device=dev), torch.full((n,), -1, dtype=torch.int64, device=dev), lens,
                torch.zeros(n, words, dtype=torch.int64, device=dev))
    positions = torch.empty(n, dtype=torch.int64, device=dev)
    slots = torch.empty(n, dtype=torch.int64, device=dev)
    masks = torch.empty(n, words, dtype=torch.int64, device=dev)
    if n == 0:
        lens.copy_(base[:seqs].clamp(min=0))
    else:
        k = Kernels.get(dev)
        with on_device(parents):
            k.launch("tree", "kern_tree_rows", (seqs,), (256,),
                     [ptr(parents), ptr(cu), ptr(base), ptr(block_table), ptr(positions), ptr(slots), ptr(lens), ptr(masks), i32(n), i32(words),
                      i32(block_table.shape[1]), i32(page_size), ptr(k.err_word())])
    return positions, slots, lens, masks


def tree_keep(ids: torch.Tensor, parents: torch.Tensor, verify: torch.Tensor, cu: torch.Tensor, base: torch.Tensor,
              block_table: torch.Tensor, pools, hk: int, d: int, page_size: int, *,
              max_rows: int | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The walk from the anchor: while a child of the node reached carries the token that the model gave after it
    (``ids[child] == verify[node]``, the lowest such child), go there. Returns the nodes walked (i32 ``[seqs]``), their indices
    (i32 ``[nodes]``, the path of sequence s from ``cu[s]`` on, then -1) and the tokens that follow them (i64, likewise, then 0):
    ``verify`` along the path, the last of them new, as `spec.accept` counts them.

    In every pool of ``pools`` (all layers, one format, up to 128) the cache rows of path node i move from place base + path[i]
    to base + i. Places outside the table or the pool set the error word and are not touched."""
    heads_ok(hk, hk, d, page_size)
    most = _glue_ok(parents, cu, base, block_table, page_size, max_rows)
    n, seqs, dev = parents.shape[0], block_table.shape[0], parents.device
    for name, x in (("ids", ids), ("verify", verify)):
        need(x.dtype == torch.int64 and x.numel() >= n and x.is_contiguous(), f"{name}: one i64 for each node")
    pools = list(pools)
    need(len(pools) <= MAX_POOLS, f"{len(pools)} pools: at most {MAX_POOLS}")
    for p in pools:
        any_pool_ok(p, hk, page_size, d)
        need(p.dtype == pools[0].dtype and p.shape == pools[0].shape, "the pools of a call are alike")
    need(len({p.data_ptr() for p in pools}) == len(pools), "a pool is named once")
    same_device(parents, ids, verify, cu, base, block_table, *pools)
    if not seqs or not n:                         # no launch that would fill them
        return (torch.zeros(seqs, dtype=torch.int32, device=dev), torch.full((n,), -1, dtype=torch.int32, device=dev),
                torch.zeros(n, dtype=torch.int64, device=dev))
    count = torch.empty(seqs, dtype=torch.int32, device=dev)
    path = torch.empty(n, dtype=torch.int32, device=dev)
    emitted = torch.empty(n, dtype=torch.int64, device=dev)
    k = Kernels.get(dev)
    e4m3 = bool(pools) and pools[0].dtype == torch.uint8
    table = struct.pack(f"<{MAX_POOLS}Q", *[p.data_ptr() for p in pools], *[0] * (MAX_POOLS - len(pools)))
    with on_device(parents):
        k.launch("tree", "kern_tree_keep", (seqs, max(1, len(pools))), (128,),
                 [table, ptr(ids), ptr(parents), ptr(verify), ptr(cu), ptr(base), ptr(block_table), ptr(count), ptr(path), ptr(emitted),
                  i32(n), i32(len(pools)), i32(block_table.shape[1]), i32(page_size), i32(hk), i32(d), i32(int(e4m3)),
                  i32(pools[0].shape[0] if pools else 0), ptr(k.err_word())])
    return count, path, emitted


# ---- PyTorch references --------------------------------------------------------------------------------------------------------
def tree_masks_reference(parents) -> tuple[list[int], list[int]]:
    """Depths and masks (whole numbers of any width) of one sequence's nodes."""
    depth, mask = [], []
    for i, p in enumerate(parents):
        ok = 0 <= p < i
        depth.append(depth[p] + 1 if ok else 0)
        mask.append((mask[p] if ok else 0) | 1 << i)
    return depth, mask


def walk_reference(ids, parents, verify) -> list[int]:
    path = [0] if len(ids) else []
    while path:
        nxt = [j for j in range(path[-1] + 1, len(ids)) if parents[j] == path[-1] and ids[j] == verify[path[-1]]]
        if not nxt:
            break
        path.append(nxt[0])
    return path
