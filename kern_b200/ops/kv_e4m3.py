"""A paged KV cache in 8-bit floating point: rotary positions and quantisation as rows are written, rows read back, and paged
GQA attention over it (single tokens, short causal blocks, prompt chunks), with PyTorch fp32 reference statements.

A row (one token, k or v, one kv head) is ``head_dim`` e4m3 codes and one scale byte ``e + 127``; it stands for ``code * 2**e``,
which bf16 holds exactly. ``e`` is the smallest exponent that brings the row's largest finite value to 448 or less, kept within
[-40, 119]; a value that is not finite is stored as NaN. One layer's cache is a uint8 tensor ``[pages, page_bytes(...)]``: a
page's codes ``[2, kv_heads, page_size, head_dim]`` (k then v), then its scale bytes ``[2, kv_heads, page_size]``; slot =
page * page_size + offset, as in the bf16 cache, at 0.504 of its bytes (head_dim 128).
"""
from __future__ import annotations

import struct

import torch

from .launcher import TM_BF16, TM_U8, Kernels

TK = 64
LOG2E = 1.4426950408889634
HEAD_DIMS = (64, 128, 256)

# the kernels' parameter blocks, in their order (native alignment)
_APPEND = struct.Struct("9Q4ifiq3iQ")
_READ = struct.Struct("3Q3iqQ")
_ROWS = struct.Struct("128s9Q10ifQ")
_MERGE = struct.Struct("5Q6i")


class _Here:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def on_device(t: torch.Tensor):
    """The tensor's device as the current one for a call, where it is another."""
    return _HERE if torch._C._cuda_getDevice() == t.get_device() else torch.cuda.device(t.device)


def same_device(t: torch.Tensor, *others) -> int:
    at = t.get_device()
    if at < 0:
        raise ValueError("the tensors of this call live on a CUDA device")
    for o in others:
        if o is not None and o.get_device() != at:
            raise ValueError(f"tensors on {t.device} and {o.device}")
    return at


def rows_ok(t: torch.Tensor, width: int, name: str) -> tuple[int, int]:
    """A bf16 row tensor that the kernels read 16 bytes at a time: its rows and the elements from one to the next."""
    if t.dtype != torch.bfloat16 or t.dim() != 2:
        raise ValueError(f"{name} is a bf16 [rows, >= {width}] tensor")
    n, w = t.shape
    step, one = t.stride()
    if w < width or (one != 1 and w > 1):
        raise ValueError(f"{name} is a bf16 [rows, >= {width}] tensor whose columns are neighbours")
    if (n > 1 and (step % 8 or step < width)) or t.data_ptr() % 16:
        raise ValueError(f"{name}: rows start on 16 bytes and do not overlap")
    return n, step


def i32_ok(t: torch.Tensor, count: int, name: str, dtype=torch.int32) -> None:
    if t.dtype != dtype or t.numel() < count or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous {dtype}, {count} of them")


def heads_ok(hq: int, hk: int, d: int, page_size: int) -> None:
    if hk < 1 or hq < 1 or hq % hk or hq > 16 * hk:
        raise ValueError(f"{hq} query heads over {hk} kv heads: a whole group of at most 16")
    if d not in HEAD_DIMS:
        raise ValueError(f"head_dim {d}: built for {HEAD_DIMS}")
    if page_size < 8 or (TK % page_size if page_size <= TK else page_size % TK):
        raise ValueError(f"page_size {page_size}: 8, 16, 32, or a multiple of {TK}")


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


def pool_ok(pool: torch.Tensor, hk: int, page_size: int, d: int) -> int:
    """The pages of an 8-bit pool."""
    if pool.dtype != torch.uint8 or pool.dim() != 2 or pool.shape[1] != page_bytes(hk, page_size, d) or not pool.is_contiguous():
        raise ValueError(f"an 8-bit pool is a contiguous uint8 [pages, {page_bytes(hk, page_size, d)}] tensor for these heads and pages")
    if pool.shape[0] < 1 or pool.data_ptr() % 16:
        raise ValueError("the pool has a page, and starts on 16 bytes")
    return pool.shape[0]


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
    pages = pool_ok(pool, hk, page_size, d)
    t, qkv_step = rows_ok(qkv, (hq + 2 * hk) * d, "qkv")
    if tokens is not None:
        if not 0 <= tokens <= t:
            raise ValueError(f"{tokens} tokens of {t} rows")
        t = tokens
    rot = d if rot is None else rot
    if not 0 <= rot <= d or rot % 16:
        raise ValueError(f"rot {rot}: a multiple of 16 up to the head's {d}")
    if pairs not in ("half", "interleaved"):
        raise ValueError(f"pairs {pairs!r}: half or interleaved")
    i32_ok(positions, t, "positions", torch.int64)
    i32_ok(slots, t, "slots", torch.int64)
    for name, x in (("cos", cos), ("sin", sin)):
        if x.dtype != torch.float32 or x.dim() != 2 or not x.is_contiguous() or x.shape[1] != rot // 2 or x.data_ptr() % 16:
            raise ValueError(f"{name}: a contiguous f32 [max_pos, rot / 2] table")
    max_pos = cos.shape[0]
    if max_pos < 1 or sin.shape[0] != max_pos:
        raise ValueError("the tables have the same positions, one at least")
    for name, x in (("q_norm", q_norm), ("k_norm", k_norm)):
        if x is not None and (x.dtype != torch.bfloat16 or x.numel() != d or not x.is_contiguous() or x.data_ptr() % 16):
            raise ValueError(f"{name}: bf16 [{d}]")
    if q_out is None:
        q_out, out_step = qkv, qkv_step
    else:
        n, out_step = rows_ok(q_out, hq * d, "q_out")
        if n < t:
            raise ValueError("q_out has a row for each token")
    gpu = same_device(qkv, pool, positions, slots, cos, sin, q_norm, k_norm, q_out)
    if t:
        k = Kernels.get(gpu)
        image = _APPEND.pack(qkv.data_ptr(), q_out.data_ptr(), pool.data_ptr(), positions.data_ptr(), slots.data_ptr(), cos.data_ptr(),
                             sin.data_ptr(), 0 if q_norm is None else q_norm.data_ptr(), 0 if k_norm is None else k_norm.data_ptr(), hq, hk,
                             rot, page_size, eps, bool(norm_plus_one), pages * page_size, max_pos, qkv_step, out_step, k.err_ptr)
        norm = "" if q_norm is None and k_norm is None else "_norm"
        with on_device(qkv):
            k.launch_image("kv_e4m3", f"kern_rope_kv_append_e4m3_{pairs}{norm}_d{d}", t, 1, 1, 128, image)
    return q_out[:t, : hq * d]


def read_rows_e4m3(pool: torch.Tensor, slots: torch.Tensor, hk: int, d: int, page_size: int, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """The rows at ``slots`` (i64) as bf16 ``[tokens, 2, hk, d]``, exact; zeros for a slot below zero."""
    heads_ok(hk, hk, d, page_size)
    pages = pool_ok(pool, hk, page_size, d)
    if slots.dtype != torch.int64 or slots.dim() != 1 or not slots.is_contiguous():
        raise ValueError("slots: i64 [tokens]")
    t = slots.numel()
    if out is None:
        out = torch.empty(t, 2, hk, d, dtype=torch.bfloat16, device=pool.device)
    elif out.dtype != torch.bfloat16 or tuple(out.shape) != (t, 2, hk, d) or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"out: contiguous bf16 [{t}, 2, {hk}, {d}]")
    gpu = same_device(pool, slots, out)
    if t:
        k = Kernels.get(gpu)
        image = _READ.pack(pool.data_ptr(), slots.data_ptr(), out.data_ptr(), t, hk, page_size, pages * page_size, k.err_ptr)
        with on_device(pool):
            k.launch_image("kv_e4m3", f"kern_kv_read_e4m3_d{d}", t, 1, 1, 128, image)
    return out


# ---- attention -----------------------------------------------------------------------------------------------------------------
def rows_form(d: int, e4m3: bool, nt: int) -> tuple[int, int]:
    """Dynamic shared memory of the few-row kernel with 8 * nt query rows to a CTA, and its CTAs on an SM: a ring of tiles of 128
    tokens (64 where a row is over 128 bytes), their scale bytes, Q's fragments (head_dim 256 and 16 rows), barriers."""
    row = d * (1 if e4m3 else 2)
    tile = 128 if row <= 128 else 64
    stage, per_sm = 2 * tile * row, 1 if d == 256 or d * nt > 256 else 2
    stages = 3 if stage >= 65536 else (196608 if per_sm == 1 else 98304) // stage
    return 1024 + stages * (stage + (2 * tile if e4m3 else 0)) + (nt * d * 16 if d == 256 and nt > 1 else 0) + 256, per_sm


def rows_shares(ctas: int, max_len: int, resident: int) -> tuple[int, int]:
    """(shares that a row's context is cut into, CTAs of a cluster): as many as fill the SMs once, two where the rows alone fill
    them up to four times (a share's end then leaves less of the last wave idle), none of under 128 tokens. Up to 8 shares are one
    cluster, more are clusters of 8 and a joining launch."""
    want = min(max(1, -(-max_len // 128)), resident // ctas if ctas < resident else (2 if ctas < 4 * resident else 1), 256)
    cluster = 8 if want >= 8 else 4 if want >= 4 else 2 if want >= 2 else 1
    return want // cluster * cluster, cluster


# query rows of a sequence and kv head above which the tensor-core kernel runs (head_dim 64 and 128)
TILE_ROWS = 32


def tile_smem(d: int, e4m3: bool) -> int:
    """Dynamic shared memory of the many-row kernel: two tiles of Q, a ring of K and V halves as 16-bit values (four, or five where
    they are copied as they are), two halves of codes with their scale bytes, barriers."""
    return 768 + 2 * 128 * d * 2 + (4 if e4m3 else 5) * 128 * d * 2 + (2 * (128 * d + 256) if e4m3 else 0) + 1024 + 512


def tile_shares(ctas: int, max_len: int, sms: int) -> int:
    return max(1, min(-(-3 * sms // ctas), -(-max_len // 512), 64)) if ctas < 3 * sms else 1


def pool_map(k: Kernels, pool: torch.Tensor, e4m3: bool, pages: int, hk: int, d: int, page_size: int) -> bytes:
    """3-D descriptor over a pool of either format: (value, row of a page's k | v x head x token, page)."""
    es = 1 if e4m3 else 2
    stride = page_bytes(hk, page_size, d) if e4m3 else 2 * hk * page_size * d * 2
    cols = min(d * es, 128)
    return k.dev.encode_tensor_map(pool.data_ptr(), TM_U8 if e4m3 else TM_BF16, (d, 2 * hk * page_size, pages), (d * es, stride),
                                   (cols // es, min(page_size, TK), 1), cols, 256, False)


def attention_rows(q, pool, pages, block_table, seq_lens, masks, cu_q, hq, hk, d, page_size, out, call) -> torch.Tensor:
    """The launches behind `paged_attention_e4m3` (masks None: causal) and `tree.tree_attention`; `call` from `attention_args`."""
    gpu, n, q_step, out_step, seqs, width, rows_per_seq, max_rows, max_len, scale = call
    e4m3 = pool.dtype == torch.uint8
    k = Kernels.get(gpu)
    g = hq // hk
    tiled = g * max_rows > TILE_ROWS and d <= 128
    if tiled:
        entry, toks, cluster, threads, smem = "attn_tile", 256 // g, 1, 512, tile_smem(d, e4m3)
        nblk = min(n // toks + seqs, seqs * -(-max_rows // toks))          # blocks of all sequences, at most
        shares = tile_shares(hk * nblk, max_len, k.sm_count)
        gx, gy, last, name = hk, nblk, seqs, ""
    else:
        # query rows of a CTA: the fewest eights that hold a sequence's, up to what registers hold
        nt = 1 if g * max_rows <= 8 else 2 if g * max_rows <= 16 or d == 256 else 4
        toks, threads = 8 * nt // g, 160
        nblk = -(-max_rows // toks)
        smem, per_sm = rows_form(d, e4m3, nt)
        shares, cluster = rows_shares(hk * nblk * seqs, max_len, k.sm_count * per_sm)
        entry, gx, gy, last, name = "attn_rows", hk * nblk, seqs, cluster, f"_n{nt}"
    ws_o = ws_ml = 0
    if shares > cluster:
        parts = n * hq * (shares // cluster)
        ws = torch.empty(parts * (d + 2), dtype=torch.float32, device=q.device)
        ws_o = ws.data_ptr()
        ws_ml = ws_o + 4 * parts * d
    form = "causal" if masks is None else "tree"
    out_at, lens_at, cu_at = out.data_ptr(), seq_lens.data_ptr(), 0 if cu_q is None else cu_q.data_ptr()
    image = _ROWS.pack(pool_map(k, pool, e4m3, pages, hk, d, page_size), q.data_ptr(), out_at, ws_o, ws_ml, pool.data_ptr(),
                       block_table.data_ptr(), lens_at, cu_at, 0 if masks is None else masks.data_ptr(),
                       0 if masks is None else masks.shape[1], rows_per_seq, hq, hk, q_step, out_step, width, page_size, last, pages,
                       scale * LOG2E, k.err_ptr)
    with on_device(q):
        k.launch_image(entry, f"kern_{entry}_{'e4m3' if e4m3 else 'bf16'}_{form}_d{d}{name}", gx, gy, shares, threads, image, smem, False, cluster)
        if shares > cluster:
            image = _MERGE.pack(ws_o, ws_ml, out_at, lens_at, cu_at, rows_per_seq, hq, toks, shares, cluster, out_step)
            k.launch_image("attn_rows", f"kern_attn_rows_merge_{form}_d{d}", -(-max_rows * hq // 8), seqs, 1, 256, image, 0, True)
    return out


def attention_args(q, pool, block_table, seq_lens, cu_q, masks, hq, d, page_size, out, rows_per_seq, max_rows, max_len, scale):
    """The checks that both attentions share: the output, and the call's numbers with their defaults."""
    n, q_step = rows_ok(q, hq * d, "q")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or not block_table.is_contiguous():
        raise ValueError("block_table: contiguous i32 [seqs, pages]")
    seqs, width = block_table.shape
    if seqs > 65535 or (width < 1 and seqs):
        raise ValueError(f"block_table [{seqs}, {width}]: at most 65535 sequences, a page to a row")
    i32_ok(seq_lens, seqs, "seq_lens")
    if cu_q is not None:
        i32_ok(cu_q, seqs + 1, "cu_q")
        rows_per_seq = 1
        max_rows = n if max_rows is None else max_rows
    else:
        if rows_per_seq < 1 or n < seqs * rows_per_seq:
            raise ValueError("q has rows_per_seq rows for each sequence")
        max_rows = rows_per_seq
    if not 0 <= max_rows <= n and seqs:
        raise ValueError(f"max_rows {max_rows}: the most rows of one sequence, of {n}")
    if out is None:
        out = torch.empty(n, hq * d, dtype=torch.bfloat16, device=q.device)
        out_step = hq * d
    else:
        m, out_step = rows_ok(out, hq * d, "out")
        if m < n:
            raise ValueError("out has a row for each of q's")
    if max_len is None:
        max_len = width * page_size
    elif max_len < 0:
        raise ValueError(f"max_len {max_len}")
    if scale is not None and not scale > 0:
        raise ValueError(f"scale {scale}: above zero")
    gpu = same_device(q, pool, block_table, seq_lens, cu_q, masks, out)
    return out, (gpu, n, q_step, out_step, seqs, width, rows_per_seq, max_rows, max_len, d ** -0.5 if scale is None else float(scale))


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
    pages = pool_ok(pool, hk, page_size, d)
    out, call = attention_args(q, pool, block_table, seq_lens, cu_q, None, hq, d, page_size, out, rows_per_seq, max_rows, max_len, scale)
    if block_table.shape[0] == 0 or call[7] == 0:
        return out
    return attention_rows(q, pool, pages, block_table, seq_lens, None, cu_q, hq, hk, d, page_size, out, call)


# ---- PyTorch references --------------------------------------------------------------------------------------------------------
def quantise_reference(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows ``x[..., d]`` -> e4m3 codes and scale bytes."""
    x = torch.where(torch.isfinite(x.float()), x.float(), float("nan"))
    m, e = torch.frexp(x.nan_to_num(0.0).abs().amax(-1))
    e = torch.where(m > 0, torch.clamp(e - 9 + (m > 0.875).int(), -40, 119), -40)
    return torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def dequantise_reference(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    return torch.ldexp(codes.float(), scales[..., None].int() - 127)
