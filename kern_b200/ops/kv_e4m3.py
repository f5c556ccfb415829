"""A paged KV cache in 8-bit floating point: rotary positions and quantisation as rows are written, rows read back, and paged
GQA attention over it (single tokens, short causal blocks, prompt chunks), with PyTorch fp32 reference statements.

A row (one token, k or v, one kv head) is ``head_dim`` e4m3 codes and one scale byte ``e + 127``; it stands for ``code * 2**e``,
which bf16 holds exactly. ``e`` is the smallest exponent that brings the row's largest finite value to 448 or less, kept within
[-40, 119]; a value that is not finite is stored as NaN. One layer's cache is a uint8 tensor ``[pages, page_bytes(...)]``: a
page's codes ``[2, kv_heads, page_size, head_dim]`` (k then v), then its scale bytes ``[2, kv_heads, page_size]``; slot =
page * page_size + offset, as in the bf16 cache, at 0.504 of its bytes (head_dim 128).
"""
from __future__ import annotations

import contextlib
import math

import torch

from .launcher import TM_BF16, TM_U8, Kernels, f32, i32, i64, ptr

TK = 64
LOG2E = 1.4426950408889634
HEAD_DIMS = (64, 128, 256)


def need(ok: bool, why: str) -> None:
    if not ok:
        raise ValueError(why)


def on_device(t: torch.Tensor):
    """The tensor's device as the current one for a call, where it is another."""
    return contextlib.nullcontext() if torch.cuda.current_device() == t.get_device() else torch.cuda.device(t.device)


def same_device(t: torch.Tensor, *others) -> None:
    need(t.is_cuda, "the tensors of this call live on a CUDA device")
    for o in others:
        need(o is None or o.device == t.device, f"tensors on {t.device} and {o.device if o is not None else None}")


def rows_ok(t: torch.Tensor, width: int, name: str) -> None:
    """A bf16 row tensor that the kernels read 16 bytes at a time."""
    need(t.dtype == torch.bfloat16 and t.dim() == 2 and t.shape[1] >= width and t.stride(1) == 1,
         f"{name} is a bf16 [rows, >= {width}] tensor whose columns are neighbours")
    need((t.shape[0] <= 1 or (t.stride(0) % 8 == 0 and t.stride(0) >= width)) and t.data_ptr() % 16 == 0,
         f"{name}: rows start on 16 bytes and do not overlap")


def heads_ok(hq: int, hk: int, d: int, page_size: int) -> None:
    need(hk >= 1 and hq >= 1 and hq % hk == 0 and hq // hk <= 16, f"{hq} query heads over {hk} kv heads: a whole group of at most 16")
    need(d in HEAD_DIMS, f"head_dim {d}: built for {HEAD_DIMS}")
    need(page_size >= 8 and (TK % page_size == 0 if page_size <= TK else page_size % TK == 0),
         f"page_size {page_size}: 8, 16, 32, or a multiple of {TK}")


# ---- the cache ---------------------------------------------------------------------------------------------------------------
def page_bytes(hk: int, page_size: int, d: int) -> int:
    return 2 * hk * page_size * (d + 1)


def new_pool(pages: int, hk: int, page_size: int, d: int, device="cuda") -> torch.Tensor:
    heads_ok(hk, hk, d, page_size)
    return torch.zeros(pages, page_bytes(hk, page_size, d), dtype=torch.uint8, device=device)


def views(pool: torch.Tensor, hk: int, page_size: int, d: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The codes ``[pages, 2, hk, page_size, d]`` (float8_e4m3fn) and scale bytes ``[pages, 2, hk, page_size]`` of a pool."""
    n = 2 * hk * page_size * d
    return pool[:, :n].view(torch.float8_e4m3fn).unflatten(1, (2, hk, page_size, d)), pool[:, n:].unflatten(1, (2, hk, page_size))


def pool_ok(pool: torch.Tensor, hk: int, page_size: int, d: int) -> None:
    need(pool.dtype == torch.uint8 and pool.dim() == 2 and pool.is_contiguous() and pool.shape[1] == page_bytes(hk, page_size, d),
         f"an 8-bit pool is a contiguous uint8 [pages, {page_bytes(hk, page_size, d)}] tensor for these heads and pages")
    need(pool.shape[0] >= 1 and pool.data_ptr() % 16 == 0, "the pool has a page, and starts on 16 bytes")


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
    heads_ok(hq, hk, d, page_size)
    pool_ok(pool, hk, page_size, d)
    rows_ok(qkv, (hq + 2 * hk) * d, "qkv")
    t = qkv.shape[0] if tokens is None else tokens
    need(0 <= t <= qkv.shape[0], f"{t} tokens of {qkv.shape[0]} rows")
    rot = d if rot is None else rot
    need(0 <= rot <= d and rot % 16 == 0, f"rot {rot}: a multiple of 16 up to the head's {d}")
    need(pairs in ("half", "interleaved"), f"pairs {pairs!r}: half or interleaved")
    for name, x in (("positions", positions), ("slots", slots)):
        need(x.dtype == torch.int64 and x.numel() >= t and x.is_contiguous(), f"{name}: one i64 for each token")
    for name, x in (("cos", cos), ("sin", sin)):
        need(x.dtype == torch.float32 and x.dim() == 2 and x.is_contiguous() and x.shape[1] == rot // 2 and x.shape == cos.shape
             and x.data_ptr() % 16 == 0, f"{name}: a contiguous f32 [max_pos, rot / 2] table")
    need(cos.shape[0] >= 1, "the tables have a position")
    for name, x in (("q_norm", q_norm), ("k_norm", k_norm)):
        need(x is None or (x.dtype == torch.bfloat16 and x.numel() == d and x.is_contiguous() and x.data_ptr() % 16 == 0), f"{name}: bf16 [{d}]")
    if q_out is None:
        q_out = qkv[:, : hq * d]
    else:
        rows_ok(q_out, hq * d, "q_out")
        need(q_out.shape[0] >= t, "q_out has a row for each token")
    same_device(qkv, pool, positions, slots, cos, sin, q_norm, k_norm, q_out)
    out = q_out[:t, : hq * d]
    if t == 0:
        return out
    k = Kernels.get(qkv.device)
    with on_device(qkv):
        k.launch("kv_e4m3", f"kern_rope_kv_append_e4m3_d{d}", (t,), (256,),
                 [ptr(qkv), ptr(q_out), ptr(pool), ptr(positions), ptr(slots), ptr(cos), ptr(sin), ptr(q_norm), ptr(k_norm), i32(t), i32(hq),
                  i32(hk), i32(rot), i32(page_size), f32(eps), i32(int(norm_plus_one)), i32(int(pairs == "interleaved")),
                  i64(pool.shape[0] * page_size), i32(cos.shape[0]), i32(qkv.stride(0)), i32(q_out.stride(0)), ptr(k.err_word())])
    return out


def read_rows_e4m3(pool: torch.Tensor, slots: torch.Tensor, hk: int, d: int, page_size: int, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """The rows at ``slots`` (i64) as bf16 ``[tokens, 2, hk, d]``, exact; zeros for a slot below zero."""
    heads_ok(hk, hk, d, page_size)
    pool_ok(pool, hk, page_size, d)
    need(slots.dtype == torch.int64 and slots.dim() == 1 and slots.is_contiguous(), "slots: i64 [tokens]")
    t = slots.numel()
    if out is None:
        out = torch.empty(t, 2, hk, d, dtype=torch.bfloat16, device=pool.device)
    need(out.dtype == torch.bfloat16 and tuple(out.shape) == (t, 2, hk, d) and out.is_contiguous() and out.data_ptr() % 16 == 0,
         f"out: contiguous bf16 [{t}, 2, {hk}, {d}]")
    same_device(pool, slots, out)
    if t == 0:
        return out
    k = Kernels.get(pool.device)
    with on_device(pool):
        k.launch("kv_e4m3", f"kern_kv_read_e4m3_d{d}", (-(-t * 2 * hk * (d // 8) // 256),), (256,),
                 [ptr(pool), ptr(slots), ptr(out), i32(t), i32(hk), i32(page_size), i64(pool.shape[0] * page_size), ptr(k.err_word())])
    return out


# ---- attention -----------------------------------------------------------------------------------------------------------------
def rows_smem(d: int, e4m3: bool) -> int:
    """Dynamic shared memory of the few-row kernel: its ring of tiles, scale bytes, Q's fragments (head_dim 256), barriers."""
    stage = 2 * TK * d * (1 if e4m3 else 2)
    stages = 3 if stage >= 65536 else min(8, 98304 // stage)
    return 1024 + stages * (stage + (2 * TK if e4m3 else 0)) + (8192 if d == 256 else 0) + 256


def rows_splits(ctas: int, max_len: int, sms: int, d: int) -> int:
    """Shares that a row's context is cut into: two waves of the CTAs that fit, no share under four tiles."""
    resident = sms * (1 if d == 256 else 2)
    if ctas >= 4 * resident:
        return 1
    tiles = -(-max_len // TK)
    return max(1, min(64, -(-2 * resident // ctas), -(-tiles // 4)))


def pool_map(k: Kernels, pool: torch.Tensor, hk: int, d: int, page_size: int) -> bytes:
    """3-D descriptor over a pool of either format: (value, row of a page's k | v x head x token, page)."""
    e4m3 = pool.dtype == torch.uint8
    es = 1 if e4m3 else 2
    stride = page_bytes(hk, page_size, d) if e4m3 else 2 * hk * page_size * d * 2
    cols = min(d * es, 128)
    return k.dev.encode_tensor_map(pool.data_ptr(), TM_U8 if e4m3 else TM_BF16, [d, 2 * hk * page_size, pool.shape[0]], [d * es, stride],
                                   [cols // es, min(page_size, TK), 1], cols, 256, False)


def attention_rows(q, pool, block_table, seq_lens, masks, cu_q, hq, hk, d, page_size, out, rows_per_seq, max_rows, max_len, scale) -> torch.Tensor:
    """The launches behind `paged_attention_e4m3` (masks None: causal) and `tree.tree_attention`."""
    e4m3 = pool.dtype == torch.uint8
    k = Kernels.get(q.device)
    seqs, width = block_table.shape
    toks = max(1, 16 // (hq // hk))
    nblk = -(-max_rows // toks)
    splits = rows_splits(hk * nblk * seqs, max_len, k.sm_count, d)
    ws_o = ws_ml = None
    if splits > 1:
        ws_o = torch.empty(q.shape[0] * hq * splits * d, dtype=torch.float32, device=q.device)
        ws_ml = torch.empty(q.shape[0] * hq * splits * 2, dtype=torch.float32, device=q.device)
    form = "causal" if masks is None else "tree"
    k.launch("attn_rows", f"kern_attn_rows_{'e4m3' if e4m3 else 'bf16'}_{form}_d{d}", (hk * nblk, seqs, splits), (160,),
             [pool_map(k, pool, hk, d, page_size), ptr(q), ptr(out), ptr(ws_o), ptr(ws_ml), ptr(pool), ptr(block_table), ptr(seq_lens),
              ptr(cu_q), ptr(masks), i32(0 if masks is None else masks.shape[1]), i32(rows_per_seq), i32(hq), i32(hk), i32(q.stride(0)),
              i32(out.stride(0)), i32(width), i32(page_size), i32(splits), i32(pool.shape[0]), f32(scale * LOG2E), ptr(k.err_word())],
             shared_mem=rows_smem(d, e4m3))
    if splits > 1:
        k.launch("attn_rows", f"kern_attn_rows_merge_{form}_d{d}", (-(-max_rows * hq // 8), seqs), (256,),
                 [ptr(ws_o), ptr(ws_ml), ptr(out), ptr(seq_lens), ptr(cu_q), i32(rows_per_seq), i32(hq), i32(hk), i32(splits),
                  i32(out.stride(0))], pdl=True)
    return out


def attention_args(q, pool, block_table, seq_lens, cu_q, hq, hk, d, page_size, out, rows_per_seq, max_rows, max_len, scale):
    """The checks that both attentions share; (out, max_rows, max_len, scale) with their defaults."""
    rows_ok(q, hq * d, "q")
    need(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.is_contiguous(), "block_table: contiguous i32 [seqs, pages]")
    seqs = block_table.shape[0]
    need(block_table.shape[1] >= 1 or seqs == 0, "a row of block_table has a page")
    need(seqs <= 65535, f"{seqs} sequences: at most 65535 in a call")
    need(seq_lens.dtype == torch.int32 and seq_lens.numel() >= seqs and seq_lens.is_contiguous(), "seq_lens: one i32 for each sequence")
    if cu_q is not None:
        need(cu_q.dtype == torch.int32 and cu_q.numel() >= seqs + 1 and cu_q.is_contiguous(), "cu_q: i32 [seqs + 1]")
        max_rows = q.shape[0] if max_rows is None else max_rows
    else:
        need(rows_per_seq >= 1 and q.shape[0] >= seqs * rows_per_seq, "q has rows_per_seq rows for each sequence")
        max_rows = rows_per_seq
    need(0 <= max_rows <= q.shape[0], f"max_rows {max_rows}: the most rows of one sequence, of {q.shape[0]}")
    if out is None:
        out = torch.empty(q.shape[0], hq * d, dtype=torch.bfloat16, device=q.device)
    else:
        rows_ok(out, hq * d, "out")
        need(out.shape[0] >= q.shape[0], "out has a row for each of q's")
    if max_len is None:
        max_len = block_table.shape[1] * page_size
    need(max_len >= 0, f"max_len {max_len}")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    same_device(q, pool, block_table, seq_lens, cu_q, out)
    return out, max_rows, max_len, scale


def paged_attention_e4m3(q: torch.Tensor, pool: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, hq: int, hk: int, d: int,
                         page_size: int, *, out: torch.Tensor | None = None, cu_q: torch.Tensor | None = None, rows_per_seq: int = 1,
                         max_rows: int | None = None, max_len: int | None = None, scale: float | None = None) -> torch.Tensor:
    """Causal attention of this step's query rows over each sequence's 8-bit context: the counterpart of
    `attention.paged_attention`, for single tokens, short blocks and prompt chunks alike.

    ``q``: 2-D bf16 view, row t holds the ``hq`` query heads of token t (a column slice of the fused qkv buffer works).
    ``seq_lens[s]`` counts the context including this step's rows; rows of sequence s are ``cu_q[s]:cu_q[s+1]`` or
    ``s * rows_per_seq`` onward, and row i of R sees tokens 0 .. seq_lens[s] - R + i. ``max_rows``: the most rows of one sequence
    (all of q's unless given), ``max_len``: the longest context, which sets how it is shared out (the table's width unless given).
    A row that sees nothing gives zeros; rows of ``out`` behind the last sequence's stay as they are. Rows that sequences leave
    out of their table's reach, and pages outside the pool, set the device's error word. Returns ``out[rows, hq * d]``."""
    heads_ok(hq, hk, d, page_size)
    pool_ok(pool, hk, page_size, d)
    out, max_rows, max_len, scale = attention_args(q, pool, block_table, seq_lens, cu_q, hq, hk, d, page_size, out, rows_per_seq, max_rows,
                                                   max_len, scale)
    if block_table.shape[0] == 0 or max_rows == 0:
        return out
    with on_device(q):
        return attention_rows(q, pool, block_table, seq_lens, None, cu_q, hq, hk, d, page_size, out, rows_per_seq, max_rows, max_len, scale)


# ---- PyTorch references --------------------------------------------------------------------------------------------------------
def quantise_reference(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows ``x[..., d]`` -> e4m3 codes and scale bytes."""
    x = torch.where(torch.isfinite(x.float()), x.float(), float("nan"))
    m, e = torch.frexp(x.nan_to_num(0.0).abs().amax(-1))
    e = torch.where(m > 0, torch.clamp(e - 9 + (m > 0.875).int(), -40, 119), -40)
    return torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def dequantise_reference(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    return torch.ldexp(codes.float(), scales[..., None].int() - 127)
