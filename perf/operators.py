"""Speculative decoding over a quantised paged cache, operator by operator: what is measured, and its plain form.

Four operators that one serving step runs in a row:

* ``append``: rotary positions of q and k (half or interleaved pairs, part of the head, with or without query / key norms), k and v
  quantised to 8-bit floating point as they are written into the pages, and the written rows read back;
* ``attend``: attention of single tokens, short blocks of rows or prompt chunks over that cache;
* ``tree``: attention of a tree of drafted tokens over a cache, bf16 or 8-bit: every node sees the context and its own ancestors;
* ``keep``: positions, slots and ancestor masks of a tree's nodes, then the walk down the nodes that the model agreed with and the
  move of their cache rows to the places they keep, over all layers.

Cache formats. bf16: ``[pages, 2, kv heads, page size, head dim]``. 8-bit: bytes ``[pages, 2 * kv heads * page size * (head dim + 1)]``:
a page's values as e4m3, ``[2, kv heads, page size, head dim]``, then one scale byte for each row, ``[2, kv heads, page size]``; a row
stands for its values times ``2 ** (byte - 127)``.
"""
import math

import torch

own = False

# ---- the cases -------------------------------------------------------------------------------------------------------------
# Head layouts (query heads, kv heads, head dim) of this repository's decoders: the smallest that its kernels take, the dense 8B, the
# routed 30B, the hybrid 27B; page sizes are those of its configurations and tests.
HEADS = [(4, 2, 64), (32, 8, 128), (32, 4, 128), (24, 4, 256), (8, 8, 128), (16, 2, 64)]


def listed():
    return [
        # a few sequences' single tokens in the smallest decoder: one launch's latency
        dict(name="append_5", op="append", tokens=5, hq=4, hk=2, d=64, page=16, rot=64, pairs="half", norm=False, max_pos=256),
        # single tokens of a full decode batch, a quarter of a wide head rotated, queries and keys normed
        dict(name="append_256_wide", op="append", tokens=256, hq=24, hk=4, d=256, page=64, rot=64, pairs="interleaved", norm=True, max_pos=32768),
        # the largest call of the dense 8B: a prompt chunk and decode rows together
        dict(name="append_8192", op="append", tokens=8192, hq=32, hk=8, d=128, page=64, rot=128, pairs="half", norm=False, max_pos=8192),
        # one user's next token
        dict(name="attend_1x1001", op="attend", seqs=1, rows=1, ragged=False, least=1001, most=1001, hq=32, hk=8, d=128, page=64),
        # an ordinary decode batch, contexts of every length
        dict(name="attend_64x4096", op="attend", seqs=64, rows=1, ragged=False, least=200, most=4096, hq=32, hk=8, d=128, page=64),
        # two long conversations, eight query heads to a kv head
        dict(name="attend_2x100003", op="attend", seqs=2, rows=1, ragged=False, least=90001, most=100003, hq=32, hk=4, d=128, page=64),
        # prompt chunks of several sequences behind what they have already
        dict(name="attend_prompts", op="attend", seqs=4, rows=2048, ragged=True, least=2048, most=6000, hq=32, hk=8, d=128, page=64),
        # one user's drafted tree
        dict(name="tree_1x17", op="tree", kind="bf16", seqs=1, nodes=17, ragged=False, least=701, most=701, hq=32, hk=8, d=128, page=64),
        # a batch of trees over an 8-bit cache
        dict(name="tree_16x64_e4m3", op="tree", kind="e4m3", seqs=16, nodes=64, ragged=True, least=500, most=4096, hq=32, hk=8, d=128, page=64),
        # the largest batch of trees over a bf16 cache
        dict(name="tree_64x32", op="tree", kind="bf16", seqs=64, nodes=32, ragged=True, least=1000, most=8192, hq=32, hk=8, d=128, page=64),
        # the end of a round: two layers of the smallest decoder
        dict(name="keep_3x9", op="keep", kind="e4m3", seqs=3, nodes=9, layers=2, hq=4, hk=2, d=64, page=16),
        # the end of a round of a large batch, several layers of the dense 8B
        dict(name="keep_128x32", op="keep", kind="bf16", seqs=128, nodes=32, layers=12, hq=32, hk=8, d=128, page=64),
    ]


def _spread(rng, lo, hi):
    """Whole numbers spread over the logarithm of a range."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "tree", "tree", "keep"])
    hq, hk, d = rng.choice(HEADS)
    page = rng.choice([16, 32, 64, 128])
    heads = dict(hq=hq, hk=hk, d=d, page=page)
    if op == "append":
        rot = rng.choice([d, d, d // 2, d // 4])
        return dict(op=op, tokens=_spread(rng, 1, min(8192, 40_000_000 // ((hq + 4 * hk) * d))), rot=rot, pairs=rng.choice(["half", "interleaved"]),
                    norm=rng.random() < 0.5, max_pos=_spread(rng, 300, 32768), **heads)
    if op == "attend":
        if rng.random() < 0.3:          # prompt chunks, ragged
            rows = _spread(rng, 17, 2048)
            return dict(op=op, seqs=rng.randint(1, 4), rows=rows, ragged=True, least=rows, most=rows + _spread(rng, 1, 4000 * 128 // d), **heads)
        rows = rng.choice([1, 1, 1, 2, 5])
        most = _spread(rng, 8, 65536)
        seqs = _spread(rng, 1, max(1, min(256, 130000 * 1024 // (hk * d) // most)))
        return dict(op=op, seqs=seqs, rows=rows, ragged=False, least=max(rows, most // rng.choice([1, 2, 16])), most=most, **heads)
    nodes = rng.randint(2, 64)
    if op == "tree":
        most = nodes + _spread(rng, 1, 16384)
        seqs = _spread(rng, 1, max(1, min(64, 120000 * 32 // hq * 128 // d * 32 // max(nodes, 32) // most)))
        return dict(op=op, kind=rng.choice(["bf16", "e4m3"]), seqs=seqs, nodes=nodes, ragged=rng.random() < 0.5, least=max(nodes, most // rng.choice([1, 4])), most=most, **heads)
    return dict(op=op, kind=rng.choice(["bf16", "e4m3"]), seqs=_spread(rng, 1, 128), nodes=nodes, layers=rng.randint(1, 12 * 1024 // max(1024, hk * d)), **heads)


# ---- inputs ----------------------------------------------------------------------------------------------------------------
def _sizes(case):
    """Row counts and context lengths of a case's sequences (a context counts its rows): the case's own, whatever the inputs' seed."""
    import random

    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n = case["seqs"]
    most_rows = case["nodes"] if "nodes" in case else case["rows"]
    rows = [most_rows] * n
    if case.get("ragged"):
        rows = [most_rows if i == 0 else rng.randint(1, most_rows) for i in range(n)]
    if "most" not in case:
        return rows, [rng.randint(1, 40) for _ in range(n)]
    lens = [case["most"] if i == 0 else rng.randint(case["least"], case["most"]) for i in range(n)]
    return rows, [max(l, r) for l, r in zip(lens, rows)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _keys_values(g, rows, hk, d):
    """k and v as a decoder makes them: rows of different size, a few large key channels; [rows, 2, hk, d] f32."""
    x = torch.randn(rows, 2, hk, d, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(rows, 2, hk, 1, generator=g, device="cuda"))
    x[:, 0, :, 3] *= 4
    x[:, 0, :, d // 2 + 5] *= 3
    return x


def _make_cache(g, kind, pages, hk, page, d):
    """A filled pool in one of the two formats, made from bf16 keys and values."""
    x = _keys_values(g, pages * page, hk, d).to(torch.bfloat16).view(pages, page, 2, hk, d).permute(0, 2, 3, 1, 4)
    if kind == "bf16":
        return x.contiguous()
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.clamp(e - 9 + (m > 0.875), -40, 119)
    v = torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn).contiguous()
    return torch.cat([v.view(torch.uint8).reshape(pages, -1), (e + 127).to(torch.uint8).reshape(pages, -1)], 1).contiguous()


def _tables(g, need, page):
    """A page table in which every sequence has `need[s]` pages, scattered over the pool; entries past those are page 0."""
    total = sum(need)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(need), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, total


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cu(rows):
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    return cu


def _parents(rng, n):
    """A drafted tree of n nodes, the anchor first: a few branches, some of them long."""
    return [-1] + [max(0, i - 1 - int(rng.expovariate(0.6))) for i in range(1, n)]


def prepare(case, seed):
    import random

    g, rng = _gen(seed), random.Random(seed * 31 + 5)
    hq, hk, d, page = case["hq"], case["hk"], case["d"], case["page"]
    st = dict(case=case)
    if case["op"] == "append":
        t, rot = case["tokens"], case["rot"]
        pages = -(-t * 5 // 4 // page) + 2
        x = torch.randn(t, hq + 2 * hk, d, generator=g, device="cuda")
        x[:, hq:] = _keys_values(g, t, hk, d).view(t, 2 * hk, d)
        st["qkv"] = x.view(t, -1).to(torch.bfloat16)
        st["q"] = torch.empty(t, hq * d, dtype=torch.bfloat16, device="cuda")
        st["pool"] = torch.zeros(pages, 2 * hk * page * (d + 1), dtype=torch.uint8, device="cuda")
        st["positions"] = torch.randint(0, case["max_pos"], (t,), generator=g, device="cuda")
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:t].clone()
        if t > 3:
            slots[t // 2] = -1                       # a padding row: rotated, not written
        st["slots"] = slots
        inv = 1e6 ** (-torch.arange(0, rot // 2, dtype=torch.float64, device="cuda") * 2 / rot)
        ang = torch.arange(case["max_pos"], dtype=torch.float64, device="cuda")[:, None] * inv
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        if case["norm"]:
            st["q_norm"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16)
            st["k_norm"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16)
        return st
    rows, lens = _sizes(case)
    cu = _cu(rows)
    st.update(max_rows=max(rows), cu=_i32(cu))
    if case["op"] == "keep":
        base, need = lens, [-(-(l + r) // page) for l, r in zip(lens, rows)]
        st["table"], pages = _tables(g, need, page)
        st["pools"] = [_make_cache(g, case["kind"], pages, hk, page, d) for _ in range(case["layers"])]
        st["base"] = torch.tensor(base, dtype=torch.int64, device="cuda")
        st["parents"] = _i32([p for r in rows for p in _parents(rng, r)])
        ids = torch.randint(0, 50000, (cu[-1],), generator=g, device="cuda")
        parents = st["parents"].long()
        at = torch.repeat_interleave(st["cu"][:-1].long(), st["cu"].long().diff())
        verify = torch.randint(0, 50000, (cu[-1],), generator=g, device="cuda")
        # four nodes of five agree with what the model says after their parent
        agree = (torch.rand(cu[-1], generator=g, device="cuda") < 0.8) & (parents >= 0)
        st["ids"] = torch.where(agree, verify[(at + parents.clamp(min=0))], ids)
        st["verify"] = verify
        return st
    st["table"], pages = _tables(g, [-(-l // page) for l in lens], page)
    st["pool"] = _make_cache(g, case.get("kind", "e4m3"), pages, hk, page, d)
    st["lens"], st["max_len"] = _i32(lens), max(lens)
    wide = torch.randn(cu[-1], (hq + 2 * hk) * d, generator=g, device="cuda").to(torch.bfloat16)
    st["q"] = wide[:, : hq * d]                      # the queries of a fused q | k | v row
    if case["op"] == "tree":
        masks = []
        for r in rows:
            m = []
            for i, p in enumerate(_parents(rng, r)):
                m.append((1 << i) | (m[p] if p >= 0 else 0))
            masks += [v - (1 << 64) if v >= 1 << 63 else v for v in m]
        st["masks"] = torch.tensor(masks, dtype=torch.int64, device="cuda").view(-1, 1)
    return st


# ---- plain forms -------------------------------------------------------------------------------------------------------------
def _rotate(x, cos, sin, rot, pairs):
    """x [tokens, heads, d] f32, cos / sin [tokens, 1, rot / 2]"""
    r = x[..., :rot]
    if pairs == "half":
        a, b = r[..., : rot // 2], r[..., rot // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([r, x[..., rot:]], -1)


def _plain_append(st):
    c = st["case"]
    hq, hk, d, page, t = c["hq"], c["hk"], c["d"], c["page"], c["tokens"]
    x = st["qkv"].float().view(t, hq + 2 * hk, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * st["q_norm"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * st["k_norm"].float()
    cos, sin = st["cos"][st["positions"]][:, None], st["sin"][st["positions"]][:, None]
    q, k = _rotate(q, cos, sin, c["rot"], c["pairs"]), _rotate(k, cos, sin, c["rot"], c["pairs"])
    st["q"][:] = q.reshape(t, -1).to(torch.bfloat16)
    kv = torch.stack([k, v], 1)
    m, e = torch.frexp(kv.abs().amax(-1))
    e = torch.clamp(e - 9 + (m > 0.875), -40, 119)
    codes = torch.ldexp(kv, -e[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    keep = st["slots"] >= 0
    pg, off = st["slots"][keep] // page, st["slots"][keep] % page
    n = 2 * hk * page * d
    st["pool"][:, :n].view(-1, 2, hk, page, d)[pg, :, :, off] = codes[keep]
    st["pool"][:, n:].view(-1, 2, hk, page)[pg, :, :, off] = (e[keep] + 127).to(torch.uint8)
    # the written rows read back
    at = st["slots"].clamp(min=0)
    back = st["pool"][:, :n].view(torch.float8_e4m3fn).view(-1, 2, hk, page, d)[at // page, :, :, at % page].float()
    size = torch.ldexp(torch.ones((), device="cuda"), st["pool"][:, n:].view(-1, 2, hk, page)[at // page, :, :, at % page].int() - 127)
    back = torch.where(keep[:, None, None, None], back * size[..., None], 0).to(torch.bfloat16)
    return st["q"], back


def _plain_context(pool, table, hk, page, d):
    """Keys and values of every sequence, f32 [seqs, 2, hk, tokens, d]."""
    if pool.dtype == torch.bfloat16:
        x = pool[table.long()].float()
    else:
        n = 2 * hk * page * d
        x = pool[:, :n].view(torch.float8_e4m3fn).view(-1, 2, hk, page, d)[table.long()].float()
        e = pool[:, n:].view(-1, 2, hk, page)[table.long()].int() - 127
        x = x * torch.ldexp(torch.ones((), device=x.device), e)[..., None]
    s, w = table.shape
    return x.permute(0, 2, 3, 1, 4, 5).reshape(s, 2, hk, w * page, d)


def _plain_attention(st):
    c = st["case"]
    hq, hk, d, page, n = c["hq"], c["hk"], c["d"], c["page"], c["seqs"]
    lens, cu, most = st["lens"].long(), st["cu"].long(), st["max_rows"]
    kv = _plain_context(st["pool"], st["table"], hk, page, d)
    at = torch.arange(kv.shape[3], device="cuda")
    rows = cu.diff()
    kv = kv.masked_fill((at >= lens[:, None])[:, None, None, :, None], 0)
    r = torch.arange(most, device="cuda")
    live = r < rows[:, None]
    take = torch.where(live, cu[:-1, None] + r, 0)
    q = st["q"].float().view(-1, hk, hq // hk, d)[take]                            # [seqs, rows, hk, group, d]
    first = lens - rows                                                            # what the sequence had before its rows
    if c["op"] == "tree":
        node = at - first[:, None]                                                 # [seqs, tokens]
        bits = (st["masks"][take][..., 0][:, :, None] >> node.clamp(0, 63)[:, None]) & 1
        seen = (node < 0)[:, None] | ((node < rows[:, None])[:, None] & (bits == 1))
    else:
        seen = at <= (first[:, None] + r)[..., None]
    x = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d) * d ** -0.5, kv[:, 0].transpose(-1, -2))
    x = x.view(n, hk, hq // hk, most, -1).masked_fill(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(torch.isinf(top), 0, top))
    o = torch.matmul(x.view(n, hk, -1, x.shape[-1]), kv[:, 1]).view(n, hk, hq // hk, most, d) / x.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(n, most, hq * d)[live].to(torch.bfloat16)


def _plain_keep(st):
    c = st["case"]
    hk, d, page, n, most = c["hk"], c["d"], c["page"], c["seqs"], st["max_rows"]
    cu, base, table = st["cu"].long(), st["base"], st["table"].long()
    r = torch.arange(most, device="cuda")
    live = r < cu.diff()[:, None]
    take = torch.where(live, cu[:-1, None] + r, 0)
    par = torch.where(live, st["parents"].long()[take], -1)
    # a node's ancestors with itself: repeated squaring of the relation
    up = torch.eye(most, device="cuda").expand(n, -1, -1) + (par[..., None] == r).float()
    for _ in range(max(1, (most - 1).bit_length())):
        up = (torch.matmul(up, up) > 0).float()
    depth = up.sum(-1).long() - 1
    at = base[:, None] + depth
    place = base[:, None] + r
    slot = torch.gather(table, 1, (place // page).clamp(max=table.shape[1] - 1)) * page + place % page
    masks = (up.long() << r).sum(-1)
    ids, verify = st["ids"][take], st["verify"][take]
    hit = live & (par >= 0) & (ids == torch.gather(verify, 1, par.clamp(min=0)))
    twin = hit[:, :, None] & hit[:, None, :] & (par[:, :, None] == par[:, None, :]) & (r[None, :] < r[:, None])
    good = (hit & ~twin.any(-1)) | (r == 0)
    on = live & ((up * (~good)[:, None, :]).sum(-1) == 0)                          # every ancestor was agreed with
    count = on.sum(-1)
    path = torch.where(r < count[:, None], torch.argsort((~on).long(), dim=1, stable=True), -1)
    emitted = torch.where(path >= 0, torch.gather(verify, 1, path.clamp(min=0)), 0)
    src = torch.gather(slot, 1, path.clamp(min=0))[path >= 0]
    dst = slot[path >= 0]
    sp, so, dp, do = src // page, src % page, dst // page, dst % page
    for pool in st["pools"]:
        if c["kind"] == "bf16":
            pool[dp, :, :, do] = pool[sp, :, :, so]
        else:
            m = 2 * hk * page * d
            vals, size = pool[:, :m].view(-1, 2, hk, page, d), pool[:, m:].view(-1, 2, hk, page)
            vals[dp, :, :, do] = vals[sp, :, :, so]
            size[dp, :, :, do] = size[sp, :, :, so]
    return (at[live], slot[live], (base + cu.diff()).int(), masks[live][:, None], count.int(), path[live].int(), emitted[live], *st["pools"])


# ---- one pass -----------------------------------------------------------------------------------------------------------------
def _own(st):
    from kern_b200.ops import kv_e4m3, tree

    c = st["case"]
    hq, hk, d, page = c["hq"], c["hk"], c["d"], c["page"]
    if c["op"] == "append":
        q = kv_e4m3.rope_kv_append_e4m3(st["qkv"], st["pool"], st["positions"], st["slots"], st["cos"], st["sin"], hq, hk, d, page,
                                        rot=c["rot"], pairs=c["pairs"], q_norm=st.get("q_norm"), k_norm=st.get("k_norm"), eps=1e-6, q_out=st["q"])
        return q, kv_e4m3.read_rows_e4m3(st["pool"], st["slots"], hk, d, page)
    if c["op"] == "attend":
        return kv_e4m3.paged_attention_e4m3(st["q"], st["pool"], st["table"], st["lens"], hq, hk, d, page, cu_q=st["cu"],
                                            max_rows=st["max_rows"], max_len=st["max_len"])
    if c["op"] == "tree":
        return tree.tree_attention(st["q"], st["pool"], st["table"], st["lens"], st["masks"], st["cu"], hq, hk, d, page,
                                   max_rows=st["max_rows"], max_len=st["max_len"])
    positions, slots, lens, masks = tree.tree_rows(st["parents"], st["cu"], st["base"], st["table"], page, max_rows=st["max_rows"])
    count, path, emitted = tree.tree_keep(st["ids"], st["parents"], st["verify"], st["cu"], st["base"], st["table"], st["pools"],
                                          hk, d, page, max_rows=st["max_rows"])
    return (positions, slots, lens, masks, count, path, emitted, *st["pools"])


def run(st):
    if own:
        return _own(st)
    op = st["case"]["op"]
    return _plain_append(st) if op == "append" else _plain_keep(st) if op == "keep" else _plain_attention(st)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------
def work(case):
    hq, hk, d = case["hq"], case["hk"], case["d"]
    if case["op"] == "append":
        t = case["tokens"]
        row = 2 * (hq + 2 * hk) * d + 2 * hq * d + 2 * 2 * hk * (d + 1) + 4 * case["rot"] + 16 + 2 * 2 * hk * d
        return dict(bytes=t * row, flops=t * (hq + 2 * hk) * d * 6)
    if case["op"] == "keep":
        nodes, size = case["seqs"] * case["nodes"], 2 * hk * (2 * d if case["kind"] == "bf16" else d + 1)
        moved = case["seqs"] * min(3.0, case["nodes"] / 2)          # rows of a round that change place, about
        return dict(bytes=nodes * (8 + 4 + 8 + 8 + 8 + 8 + 4 + 8) + 2 * moved * size * case["layers"], flops=nodes * 8)
    rows, lens = _sizes(case)
    size = 2 * hk * (2 * d if case.get("kind") == "bf16" else d + 1)
    pairs = sum(l * r - (r * (r - 1) // 2 if case["op"] == "attend" else 0) for r, l in zip(rows, lens))
    return dict(bytes=sum(lens) * size + sum(rows) * hq * d * 4, flops=4 * pairs * hq * d)


# ---- in 64 bits, from the definitions ---------------------------------------------------------------------------------------------
def _exact_row(bytes_row, scale):
    """A cache row's values in 64 bits from its e4m3 bytes: sign, four exponent bits (bias 7), three of mantissa."""
    b = bytes_row.to(torch.int64)
    e, m = (b >> 3) & 15, (b & 7).double()
    v = torch.where(e == 0, m / 512, (8 + m) * torch.exp2((e - 10).double()))
    return torch.where(b >= 128, -v, v) * torch.exp2(scale.double() - 127)[..., None]


def _exact_tokens(st, s, first, last):
    """Keys and values [2, hk, last - first, d] of tokens first .. last - 1 of sequence s, in 64 bits."""
    c = st["case"]
    hk, d, page = c["hk"], c["d"], c["page"]
    tok = torch.arange(first, last, device="cuda")
    pg = st["table"][s].long()[tok // page]
    if st["pool"].dtype == torch.bfloat16:
        return st["pool"][pg, :, :, tok % page].double().permute(1, 2, 0, 3)
    n = 2 * hk * page * d
    val = st["pool"][:, :n].view(-1, 2, hk, page, d)[pg, :, :, tok % page]
    return _exact_row(val, st["pool"][:, n:].view(-1, 2, hk, page)[pg, :, :, tok % page]).permute(1, 2, 0, 3)


def _exact_attention(case, seed):
    st = prepare(case, seed)
    hq, hk, d = case["hq"], case["hk"], case["d"]
    out = torch.zeros(st["q"].shape[0], hq, d, dtype=torch.float64, device="cuda")
    lens, cu = st["lens"].tolist(), st["cu"].tolist()
    for s, length in enumerate(lens):
        lo, hi = cu[s], cu[s + 1]
        k, v = _exact_tokens(st, s, 0, length)
        past = length - (hi - lo)
        j = torch.arange(length, device="cuda")
        for a in range(lo, hi, 128):                 # query rows in slices: a slice's scores stay small
            b = min(hi, a + 128)
            q = st["q"][a:b].double().view(b - a, hk, hq // hk, d)
            x = torch.einsum("rhgd,hld->rhgl", q, k) / math.sqrt(d)
            if case["op"] == "tree":
                bit = torch.stack([(st["masks"][a:b, 0] >> i) & 1 for i in range(hi - lo)], 1).bool()
                see = torch.cat([torch.ones(b - a, past, dtype=torch.bool, device="cuda"), bit], 1)
            else:
                see = j[None] <= past + torch.arange(a - lo, b - lo, device="cuda")[:, None]
            x = torch.where(see[:, None, None], x, torch.tensor(-torch.inf, dtype=torch.float64, device="cuda"))
            out[a:b] = torch.einsum("rhgl,hld->rhgd", torch.softmax(x, -1), v).reshape(b - a, hq, d)
    return out.view(-1, hq * d)


def _exact_append(case, seed):
    st = prepare(case, seed)
    hq, hk, d, t, rot = case["hq"], case["hk"], case["d"], case["tokens"], case["rot"]
    x = st["qkv"].double().view(t, hq + 2 * hk, d).clone()
    for lo, hi, w in ((0, hq, "q_norm"), (hq, hq + hk, "k_norm")):
        if case["norm"]:
            x[:, lo:hi] = x[:, lo:hi] / torch.sqrt((x[:, lo:hi] ** 2).sum(-1, keepdim=True) / d + 1e-6) * st[w].double()
        turn = torch.complex(st["cos"].double(), st["sin"].double())[st["positions"]][:, None]
        first = slice(0, rot // 2) if case["pairs"] == "half" else slice(0, rot, 2)
        second = slice(rot // 2, rot) if case["pairs"] == "half" else slice(1, rot, 2)
        z = torch.complex(x[:, lo:hi, first].contiguous(), x[:, lo:hi, second].contiguous()) * turn
        x[:, lo:hi, first], x[:, lo:hi, second] = z.real, z.imag
    kv = x[:, hq:].reshape(t, 2, hk, d)
    top = kv.abs().amax(-1, keepdim=True)
    # the smallest power of two that brings the row's largest value to 448 or less
    step = torch.exp2(torch.where(top > 0, torch.ceil(torch.log2(top / 448)), -40.0).clamp(-40, 119))
    u = kv.abs() / step
    ulp = torch.exp2(torch.floor(torch.log2(u.clamp(min=2.0 ** -6))) - 3)
    back = torch.sign(kv) * torch.round(u / ulp) * ulp * step                      # to nearest, ties to even
    back = back * (st["slots"] >= 0).double()[:, None, None, None]
    return x[:, :hq].reshape(t, hq * d), back


def exact(case, seed):
    if case["op"] == "append":
        return _exact_append(case, seed)
    if case["op"] == "keep":
        return None                                  # whole numbers, and rows moved as they are
    return _exact_attention(case, seed)
