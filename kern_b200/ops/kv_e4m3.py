"""A paged KV cache in 8-bit floating point: rotary positions and quantisation as rows are written, rows read back, and paged
GQA attention over it (single tokens, short causal blocks, prompt chunks), with PyTorch fp32 reference statements.

A row (one token, k or v, one kv head) is ``head_dim`` e4m3 codes and one scale byte ``e + 127``; it stands for ``code * 2**e``,
which bf16 holds exactly. ``e`` is the smallest exponent that brings the row's largest finite value to 448 or less, kept within
[-40, 119]; a value that is not finite is stored as NaN. A fresh pool's rows (all bytes 0) are rows of zeros. One layer's cache is a uint8 tensor ``[pages, page_bytes(...)]``: a
page's codes ``[2, kv_heads, page_size, head_dim]`` (k then v), then its scale bytes ``[2, kv_heads, page_size]``; slot =
page * page_size + offset, as in the bf16 cache, at 0.504 of its bytes (head_dim 128).
"""
from __future__ import annotations

import torch

from . import host as _host

HEAD_DIMS = (64, 128, 256)


# ---- the cache ---------------------------------------------------------------------------------------------------------------
def page_bytes(hk: int, page_size: int, d: int) -> int:
    return 2 * hk * page_size * (d + 1)


def new_pool(pages: int, hk: int, page_size: int, d: int, device="cuda") -> torch.Tensor:
    return torch.zeros(pages, page_bytes(hk, page_size, d), dtype=torch.uint8, device=device)


def views(pool: torch.Tensor, hk: int, page_size: int, d: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The codes ``[pages, 2, hk, page_size, d]`` (float8_e4m3fn) and scale bytes ``[pages, 2, hk, page_size]`` of a pool."""
    n = 2 * hk * page_size * d
    return pool[:, :n].view(torch.float8_e4m3fn).unflatten(1, (2, hk, page_size, d)), pool[:, n:].unflatten(1, (2, hk, page_size))


def rope_kv_append_e4m3(qkv: torch.Tensor, pool: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, cos: torch.Tensor,
                        sin: torch.Tensor, hq: int, hk: int, d: int, page_size: int, *, rot: int | None = None, pairs: str = "half",
                        q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6,
                        norm_plus_one: bool = False, tokens: int | None = None, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Norm (optional) and rotate q and k of every token, write k and v to the 8-bit cache at its slot, and q to ``q_out`` (by
    default in place in ``qkv``, whose other columns stay as they are). Returns the rotated queries ``[tokens, hq * d]``.

    ``pairs``: "half" turns value i with value i + rot / 2, "interleaved" value 2 i with value 2 i + 1; the first ``rot`` values
    of a head turn, the others pass. ``cos`` / ``sin``: f32 ``[max_pos, rot / 2]``, scaled for long contexts as the model has it
    (`attention.rope_tables`, the load programs' tables). A slot below zero (a padding row) is not written; a position or slot
    past its table sets the device's error word, and the row is not written. Two tokens may not have the same slot."""
    return _host.ops().append(qkv, pool, positions, slots, cos, sin, hq, hk, d, page_size, rot, pairs, q_norm, k_norm, eps, norm_plus_one, tokens, q_out)


def read_rows_e4m3(pool: torch.Tensor, slots: torch.Tensor, hk: int, d: int, page_size: int, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """The rows at ``slots`` (i64) as bf16 ``[tokens, 2, hk, d]``, exact; zeros for a slot below zero."""
    return _host.ops().read_rows(pool, slots, hk, d, page_size, out)


# ---- attention -----------------------------------------------------------------------------------------------------------------
def paged_attention_e4m3(q: torch.Tensor, pool: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, hq: int, hk: int, d: int,
                         page_size: int, *, out: torch.Tensor | None = None, cu_q: torch.Tensor | None = None, rows_per_seq: int = 1,
                         max_rows: int | None = None, max_len: int | None = None, scale: float | None = None) -> torch.Tensor:
    """Causal attention of this step's query rows over each sequence's 8-bit context: the counterpart of
    `attention.paged_attention`, for single tokens, short blocks and prompt chunks alike.

    ``q``: 2-D bf16 view, row t holds the ``hq`` query heads of token t (a column slice of the fused qkv buffer works).
    ``seq_lens[s]`` counts the context including this step's rows; rows of sequence s are ``cu_q[s]:cu_q[s+1]`` or
    ``s * rows_per_seq`` onward, and row i of R sees tokens 0 .. seq_lens[s] - R + i. ``max_rows``: the most rows of one sequence
    (all of q's unless given), ``max_len``: the longest context, which sets how it is shared out (the table's width unless given).
    Calls of more than 16 query rows to a kv head keep their speed where the scales of a context's keys, and of its values, are within 2^20
    of one another over 128 tokens (64 at head_dim 256; rows of zeros aside) and those of its values within 2^100 over all: 256 query
    rows that meet others are computed token by token, some 200 times slower, and as exactly.
    Scores and sums are held in 32 bits, weights as f16: a token whose weight times its values' scale is under 2^-25 of the row's largest
    adds nothing to the values, and its part of the sum alone.
    A row that sees nothing gives zeros; rows of ``out`` behind the last sequence's stay as they are. Pages
    outside the pool, contexts longer than the table, rows outside ``q`` and sequences of more rows than ``max_rows`` (which are
    left out) set the device's error word. Returns ``out[rows, hq * d]``."""
    return _host.ops().attend(q, pool, block_table, seq_lens, None, cu_q, hq, hk, d, page_size, out, rows_per_seq, max_rows, max_len, scale)


# ---- PyTorch references --------------------------------------------------------------------------------------------------------
def quantise_reference(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows ``x[..., d]`` -> e4m3 codes and scale bytes."""
    x = torch.where(torch.isfinite(x.float()), x.float(), float("nan"))
    m, e = torch.frexp(x.nan_to_num(0.0).abs().amax(-1))
    e = torch.where(m > 0, torch.clamp(e - 9 + (m > 0.875).int(), -40, 119), -40)
    # (values past 448 * 2^119 end there)
    return torch.ldexp(x, -e[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def dequantise_reference(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    return torch.ldexp(codes.float(), scales[..., None].int() - 127)
