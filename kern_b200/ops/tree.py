"""A tree of drafted tokens over a paged cache: where its nodes go and what each sees, attention of all nodes at once, and the walk
down the nodes that the model agreed with, whose cache rows move to the places they keep. With PyTorch reference statements.

Node 0 of a sequence is the anchor, the last token it has for certain; every other node names an earlier one as its parent. The
nodes of sequence s are rows ``cu[s]:cu[s+1]`` of a call. Node i is written at token place ``base + i`` of the sequence (``base``:
tokens before the anchor) and turned by position ``base + depth``, so that an agreed path, once moved together, is what writing
its tokens one after the other would have left.
"""
from __future__ import annotations

import torch

from . import host as _host

MAX_NODES = 256
MAX_POOLS = 128


def tree_attention(q: torch.Tensor, pool: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, masks: torch.Tensor,
                   cu_q: torch.Tensor, hq: int, hk: int, d: int, page_size: int, *, out: torch.Tensor | None = None,
                   max_rows: int | None = None, max_len: int | None = None, scale: float | None = None) -> torch.Tensor:
    """Attention of every sequence's tree nodes over its cache, bf16 (``[pages, 2, hk, page_size, d]``) or 8-bit (`kv_e4m3`).

    Rows of sequence s are ``cu_q[s]:cu_q[s+1]``, its last R of ``seq_lens[s]`` tokens. Row i sees every token before the tree
    and node j where bit j of ``masks[row]`` (i64 ``[rows, words]``, 64 nodes to a word) is set: its ancestors and itself, as
    `tree_rows` gives them, or any other set. A node without a bit of its own (past the words) is seen by none; a row that sees
    nothing gives zeros; what a row does not see does not reach it, infinities and NaN included. Other arguments, and rows
    behind the last sequence's, as in `kv_e4m3.paged_attention_e4m3`."""
    return _host.ops().attend(q, pool, block_table, seq_lens, masks, cu_q, hq, hk, d, page_size, out, 1, max_rows, max_len, scale)


def tree_rows(parents: torch.Tensor, cu: torch.Tensor, base: torch.Tensor, block_table: torch.Tensor, page_size: int, *,
              max_rows: int | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Of every node: its rotary position (i64), cache slot (i64) and mask (i64 ``[nodes, words]``, one word for every 64 of
    ``max_rows``); of every sequence: its context with the tree (i32). The counterpart of `spec.rows` for trees.

    ``parents`` (i32): a node's parent within its sequence, -1 for the anchor. A parent that is not an earlier node, a place past
    the page table, or more than ``max_rows`` (256) nodes set the error word: the node then has no parent, or slot -1 (nothing
    written), or is left out. So do bounds in ``cu`` that are none. A sequence of base < 0 is padding: slots -1, positions 0, masks 0,
    context 0; so are nodes before the first sequence and behind the last."""
    return _host.ops().tree_rows(parents, cu, base, block_table, page_size, max_rows)


def tree_keep(ids: torch.Tensor, parents: torch.Tensor, verify: torch.Tensor, cu: torch.Tensor, base: torch.Tensor,
              block_table: torch.Tensor, pools, hk: int, d: int, page_size: int, *,
              max_rows: int | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The walk from the anchor: while a child of the node reached carries the token that the model gave after it
    (``ids[child] == verify[node]``, the lowest such child), go there. Returns the nodes walked (i32 ``[seqs]``), their indices
    (i32 ``[nodes]``, the path of sequence s from ``cu[s]`` on, then -1) and the tokens that follow them (i64, likewise, then 0):
    ``verify`` along the path, the last of them new, as `spec.accept` counts them.

    In every pool of ``pools`` (all layers, one format, up to 128) the cache rows of path node i move from place base + path[i]
    to base + i. Places outside the table or the pool set the error word and are not touched; so do trees of more than ``max_rows``
    (256) nodes, whose further nodes are not walked to, and bounds in ``cu`` that are none."""
    return _host.ops().tree_keep(ids, parents, verify, cu, base, block_table, pools, hk, d, page_size, max_rows)


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
