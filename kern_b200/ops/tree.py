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

from .kv_e4m3 import attention_args, attention_rows, heads_ok, i32_ok, on_device, pool_ok, same_device
from .launcher import Kernels

MAX_NODES = 256
MAX_POOLS = 128

# the kernels' parameter blocks, in their order (native alignment)
_ROWS = struct.Struct("8Q4iQ")
_KEEP = struct.Struct(f"{MAX_POOLS}Q9Q8iQ")


def any_pool_ok(pool: torch.Tensor, hk: int, page_size: int, d: int) -> int:
    """The pages of a pool in either format."""
    if pool.dtype == torch.uint8:
        return pool_ok(pool, hk, page_size, d)
    if pool.dtype != torch.bfloat16 or pool.dim() != 5 or tuple(pool.shape)[1:] != (2, hk, page_size, d) or not pool.is_contiguous():
        raise ValueError(f"a bf16 pool is a contiguous [pages, 2, {hk}, {page_size}, {d}] tensor")
    if pool.shape[0] < 1 or pool.data_ptr() % 16:
        raise ValueError("the pool has a page, and starts on 16 bytes")
    return pool.shape[0]


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
    pages = any_pool_ok(pool, hk, page_size, d)
    if cu_q is None:
        raise ValueError("cu_q: i32 [seqs + 1]")
    if masks.dtype != torch.int64 or masks.dim() != 2 or masks.shape[0] < q.shape[0] or not 1 <= masks.shape[1] <= MAX_NODES // 64 \
            or not masks.is_contiguous():
        raise ValueError(f"masks: contiguous i64 [rows, words], up to {MAX_NODES // 64} words")
    out, call = attention_args(q, pool, block_table, seq_lens, cu_q, masks, hq, d, page_size, out, 1, max_rows, max_len, scale)
    if block_table.shape[0] == 0 or call[7] == 0:
        return out
    return attention_rows(q, pool, pages, block_table, seq_lens, masks, cu_q, hq, hk, d, page_size, out, call)


def _glue_ok(parents, cu, base, block_table, page_size, max_rows) -> tuple[int, int, int, int]:
    """Checks of what both calls share: nodes, sequences, the table's width, the most nodes of one tree."""
    if parents.dtype != torch.int32 or parents.dim() != 1 or not parents.is_contiguous():
        raise ValueError("parents: i32 [nodes]")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or not block_table.is_contiguous():
        raise ValueError("block_table: contiguous i32 [seqs, pages]")
    seqs, width = block_table.shape
    if width < 1:
        raise ValueError("a row of block_table has a page")
    i32_ok(cu, seqs + 1, "cu")
    i32_ok(base, seqs, "base", torch.int64)
    if page_size < 1:
        raise ValueError(f"page_size {page_size}")
    n = parents.shape[0]
    most = min(MAX_NODES, n) if max_rows is None else max_rows
    if not 0 <= most <= MAX_NODES:
        raise ValueError(f"{most} nodes: at most {MAX_NODES} in a tree")
    return n, seqs, width, most


def tree_rows(parents: torch.Tensor, cu: torch.Tensor, base: torch.Tensor, block_table: torch.Tensor, page_size: int, *,
              max_rows: int | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Of every node: its rotary position (i64), cache slot (i64) and mask (i64 ``[nodes, words]``, one word for every 64 of
    ``max_rows``); of every sequence: its context with the tree (i32). The counterpart of `spec.rows` for trees.

    ``parents`` (i32): a node's parent within its sequence, -1 for the anchor. A parent that is not an earlier node, a place past
    the page table, or more than ``max_rows`` (256) nodes set the error word: the node then has no parent, or slot -1 (nothing
    written), or is left out. A sequence of base < 0 is padding: slots -1, positions 0, masks 0, context 0."""
    n, seqs, width, most = _glue_ok(parents, cu, base, block_table, page_size, max_rows)
    gpu = same_device(parents, cu, base, block_table)
    words, dev = max(1, -(-most // 64)), parents.device
    if not seqs or not n:                         # no launch that would fill them
        lens = base[:seqs].clamp(min=0).int()
        return (torch.zeros(n, dtype=torch.int64, device=dev), torch.full((n,), -1, dtype=torch.int64, device=dev), lens,
                torch.zeros(n, words, dtype=torch.int64, device=dev))
    # one allocation: positions, slots, masks, then the contexts
    out = torch.empty(n * (2 + words) + -(-seqs // 2), dtype=torch.int64, device=dev)
    positions, slots, masks, lens = out[:n], out[n:2 * n], out[2 * n:(2 + words) * n].view(n, words), out[(2 + words) * n:].view(torch.int32)[:seqs]
    k, at = Kernels.get(gpu), out.data_ptr()
    image = _ROWS.pack(parents.data_ptr(), cu.data_ptr(), base.data_ptr(), block_table.data_ptr(), at, at + 8 * n, at + 8 * (2 + words) * n,
                       at + 16 * n, n, words, width, page_size, k.err_ptr)
    with on_device(parents):
        k.launch_image("tree", "kern_tree_rows", seqs, 1, 1, 256, image)
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
    n, seqs, width, _ = _glue_ok(parents, cu, base, block_table, page_size, max_rows)
    i32_ok(ids, n, "ids", torch.int64)
    i32_ok(verify, n, "verify", torch.int64)
    if len(pools) > MAX_POOLS:
        raise ValueError(f"{len(pools)} pools: at most {MAX_POOLS}")
    pages = 0
    for p in pools:
        pages = any_pool_ok(p, hk, page_size, d)
        if p.dtype != pools[0].dtype or pages != pools[0].shape[0]:
            raise ValueError("the pools of a call are alike")
    where = [p.data_ptr() for p in pools]
    if len(set(where)) != len(where):
        raise ValueError("a pool is named once")
    gpu, dev = same_device(parents, ids, verify, cu, base, block_table, *pools), parents.device
    if not seqs or not n:                         # no launch that would fill them
        return (torch.zeros(seqs, dtype=torch.int32, device=dev), torch.full((n,), -1, dtype=torch.int32, device=dev),
                torch.zeros(n, dtype=torch.int64, device=dev))
    # one allocation: tokens, path, counts
    out = torch.empty(n + -(-(n + seqs) // 2), dtype=torch.int64, device=dev)
    emitted, half = out[:n], out[n:].view(torch.int32)
    path, count = half[:n], half[n:n + seqs]
    k, at = Kernels.get(gpu), out.data_ptr()
    where += [0] * (MAX_POOLS - len(where))
    image = _KEEP.pack(*where, ids.data_ptr(), parents.data_ptr(), verify.data_ptr(), cu.data_ptr(), base.data_ptr(), block_table.data_ptr(),
                       at + 12 * n, at + 8 * n, at, n, len(pools), width, page_size, hk, d, bool(pools) and pools[0].dtype == torch.uint8, pages,
                       k.err_ptr)
    with on_device(parents):
        k.launch_image("tree", "kern_tree_keep", seqs, max(1, len(pools)), 1, 128, image)
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
