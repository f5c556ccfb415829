"""The 8-bit paged cache and the attentions over it and over drafted trees, against statements in 64 bits (sm_100a)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from kern_b200.ops import kv_e4m3 as K8
from kern_b200.ops import tree as TR
from kern_b200.ops.launcher import Kernels

BF = 2.0 ** -8              # half a bf16 step, relative


@pytest.fixture(autouse=True)
def _no_device_error(cuda):
    yield
    Kernels.get(cuda).check_error()


def fill_cache(kind, lens, hk, d, page, gen, spare=3, size=1.0):
    """A pool with scattered pages holding bf16 keys and values of every sequence; (pool, table, [kv 64-bit [2, L, hk, d]])."""
    need = [-(-l // page) for l in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen)
    table = torch.zeros(len(lens), max(1, max(need)), dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n].int()
        at += n
    kv = torch.randn(pages, 2, hk, page, d, generator=gen) * torch.exp(0.5 * torch.randn(pages, 2, hk, page, 1, generator=gen)) * size
    kv = kv.bfloat16()
    if kind == "bf16":
        pool, exact = kv.cuda(), kv.double()
    else:
        codes, scales = K8.quantise_reference(kv)
        exact = torch.ldexp(codes.double(), (scales.int() - 127)[..., None])
        pool = torch.cat([codes.view(torch.uint8).reshape(pages, -1), scales.reshape(pages, -1)], 1).contiguous().cuda()
    out = []
    for s, l in enumerate(lens):
        rows = exact[table[s].long()].permute(1, 0, 3, 2, 4).reshape(2, -1, hk, d)[:, :l]
        out.append(rows)
    return pool, table.cuda(), out


def attend64(q, kv, seen, scale):
    """q [R, hq, d], kv [2, L, hk, d], seen [R, L] -> [R, hq, d], 64 bits; rows that see nothing are zeros."""
    r, hq, d = q.shape
    g = hq // kv.shape[2]
    k, v = kv[0].repeat_interleave(g, 1), kv[1].repeat_interleave(g, 1)
    x = torch.einsum("rhd,lhd->hrl", q.double(), k) * scale
    x = x.masked_fill(~seen[None], float("-inf"))
    p = torch.softmax(x, -1)
    p = torch.where(seen.any(-1)[None, :, None], p, 0.0)
    live = torch.where(seen.any(0)[:, None, None], v, 0.0)
    return torch.einsum("hrl,lhd->rhd", p, live), torch.einsum("hrl,lhd->rhd", p, live.abs())


def close(out, ref, spread, weight):
    """|out - ref| <= half a step of the output's rounding + `weight`, the relative error of a softmax weight, over sum p |v|
    + 2^-18 of the same for scores and sums in 32 bits."""
    got = out.double().cpu()
    off = (got - ref).abs()
    allow = BF * ref.abs() * 1.01 + (weight + 2.0 ** -14) * spread + 1e-30
    assert bool((off <= allow).all()), (float((off / allow).max()), int((off > allow).sum()), got.shape)


# a bf16 weight is off by 2^-8 of itself at most (p and its sum: p alone is rounded); an f16 one by 2^-11, or 2^-25 of the largest
WEIGHT = {"bf16": 2.0 ** -8, "e4m3": 2.0 ** -10}


def rotated64(x, cos, sin, rot, pairs):
    x = x.clone()
    a, b = (x[..., :rot // 2].clone(), x[..., rot // 2:rot].clone()) if pairs == "half" else (x[..., 0:rot:2].clone(), x[..., 1:rot:2].clone())
    if pairs == "half":
        x[..., :rot // 2], x[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    else:
        x[..., 0:rot:2], x[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    return x


@pytest.mark.parametrize("hq,hk,d,page,rot,pairs,norm,t", [
    (4, 2, 64, 16, 64, "half", False, 1), (32, 8, 128, 64, 128, "half", True, 77), (24, 4, 256, 64, 64, "interleaved", True, 5),
    (16, 16, 64, 8, 32, "interleaved", False, 33), (8, 1, 128, 128, 16, "half", False, 300), (3, 1, 256, 32, 256, "interleaved", False, 9),
    (5, 5, 128, 16, 0, "half", True, 4)])
def test_append_and_read_back(cuda, hq, hk, d, page, rot, pairs, norm, t):
    g = torch.Generator().manual_seed(t)
    extra = 24                                             # the row carries more than q | k | v
    qkv = (torch.randn(t, (hq + 2 * hk) * d + extra, generator=g) * 3).bfloat16()
    pages = -(-t // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:t].clone()
    if t > 2:
        slots[1] = -1
    positions = torch.randint(0, 500, (t,), generator=g)
    ang = torch.arange(500, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, max(rot // 2, 1), dtype=torch.float64) * 2 / max(rot, 1))
    cos, sin = (ang.cos().float()[:, : rot // 2].contiguous(), ang.sin().float()[:, : rot // 2].contiguous())
    qn, kn = ((1 + 0.2 * torch.randn(2, d, generator=g)).bfloat16() if norm else (None, None))
    pool = K8.new_pool(pages, hk, page, d, cuda)
    pool.fill_(0x55)
    q_out = torch.full((t + 2, hq * d), 7.0, dtype=torch.bfloat16, device=cuda)
    dev = qkv.cuda()
    args = (positions.cuda(), slots.cuda(), cos.cuda(), sin.cuda(), hq, hk, d, page)
    opts = dict(rot=rot, pairs=pairs, q_norm=qn.cuda() if norm else None, k_norm=kn.cuda() if norm else None, eps=1e-6, norm_plus_one=norm)
    got = K8.rope_kv_append_e4m3(dev, pool, *args, q_out=q_out, **opts)
    assert torch.equal(dev.cpu(), qkv) and got.shape == (t, hq * d) and bool((q_out[t:] == 7).all())
    x = qkv[:, : (hq + 2 * hk) * d].double().view(t, -1, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    if norm:
        q = q / torch.sqrt(q.pow(2).mean(-1, keepdim=True) + 1e-6) * (qn.double() + 1)
        k = k / torch.sqrt(k.pow(2).mean(-1, keepdim=True) + 1e-6) * (kn.double() + 1)
    c, s = cos[positions][:, None].double(), sin[positions][:, None].double()
    q, k = rotated64(q, c, s, rot, pairs), rotated64(k, c, s, rot, pairs)
    want = q.reshape(t, -1)
    # bf16's half step; 2^-20 of the pair's size for the arithmetic in 32 bits
    assert bool(((got.double().cpu() - want).abs() <= BF * want.abs() + 2.0 ** -20 * want.abs().max()).all())
    back = K8.read_rows_e4m3(pool, slots.cuda(), hk, d, page).double().cpu()
    kv = torch.stack([k, v], 1)
    kv[slots < 0] = 0
    top = kv.abs().amax(-1, keepdim=True)
    # e4m3's half step (2^-4), and half its smallest step under the scale: at most 2^-10 of 2^e, e <= log2(top / 448) + 1
    assert bool(((back - kv).abs() <= 2.0 ** -4 * kv.abs() * (1 + 1e-6) + 2.0 ** -10 * top / 448 * 2 + 1e-30).all())
    # the values follow the statement exactly: codes and bytes of the same rows (v has no arithmetic before it)
    codes, scales = K8.views(pool, hk, page, d)
    want_c, want_s = K8.quantise_reference(qkv[:, (hq + hk) * d:(hq + 2 * hk) * d].view(t, hk, d))
    keep = slots >= 0
    at = slots[keep].cuda()
    assert torch.equal(codes.view(torch.uint8)[at // page, 1, :, at % page].cpu(), want_c.view(torch.uint8)[keep])
    assert torch.equal(scales[at // page, 1, :, at % page].cpu(), want_s[keep])
    # nothing else was written
    mask = torch.ones(pages * page, dtype=torch.bool)
    mask[slots[keep]] = False
    rest = mask.nonzero()[:, 0].cuda()
    assert bool((codes.view(torch.uint8)[rest // page, :, :, rest % page] == 0x55).all()) and bool((scales[rest // page, :, :, rest % page] == 0x55).all())
    # in place: the same queries, and the other columns untouched
    pool2 = torch.full_like(pool, 0x55)
    q2 = K8.rope_kv_append_e4m3(dev, pool2, *args, **opts)
    assert torch.equal(q2, got) and torch.equal(pool2, pool) and torch.equal(dev[:, hq * d:].cpu(), qkv[:, hq * d:])


def test_append_of_values_at_the_edges(cuda):
    """Rows of zeros, of one huge value, at a power of two's border, tiny, infinite and NaN."""
    hk, d, page = 1, 64, 16
    rows = torch.zeros(8, d)
    rows[1, 5] = 3e38
    rows[2, 0] = 448.0
    rows[3, 0], rows[3, 1] = 450.0, 1.0
    rows[4] = 2.0 ** -60
    rows[5, 3], rows[5, 4] = float("inf"), 2.0
    rows[6, 7], rows[6, 8] = float("nan"), -2.0
    rows[7] = torch.linspace(-1, 1, d)
    qkv = torch.cat([torch.zeros(8, d), rows, rows], 1).bfloat16()
    pool = K8.new_pool(2, hk, page, d, cuda)
    zero = torch.zeros(4, 0, device=cuda)
    slots = torch.arange(8, device=cuda)
    K8.rope_kv_append_e4m3(qkv.cuda(), pool, slots % 4, slots, zero, zero, 1, hk, d, page, rot=0)
    codes, scales = K8.quantise_reference(rows.bfloat16())
    c, s = K8.views(pool, hk, page, d)
    assert torch.equal(s[0, 0, 0, :8].cpu(), scales) and torch.equal(s[0, 1, 0, :8].cpu(), scales)
    nan = torch.isnan(codes.float())
    assert torch.equal(torch.isnan(c[0, 0, 0, :8].float()).cpu(), nan) and int(nan.sum()) == 2
    assert torch.equal(c[0, 0, 0, :8].float().cpu()[~nan], codes.float()[~nan])
    assert scales[0] == 87 and scales[2] == 127 and scales[3] == 128 and scales[4] == 87
    back = K8.read_rows_e4m3(pool, slots, hk, d, page)[:, 0, 0].float().cpu()
    assert torch.equal(back[~nan], K8.dequantise_reference(codes, scales)[~nan])


@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("norm", [False, True])
def test_codes_are_those_of_the_exact_values(cuda, pairs, norm):
    """Over many rows no code differs from that of the key in 64 bits: values next to a border are decided there."""
    hq, hk, d, page, t = 8, 8, 128, 64, 4096
    g = torch.Generator().manual_seed(11)
    qkv = torch.randn(t, (hq + 2 * hk) * d, generator=g).bfloat16()
    qkv[5, hq * d:(hq + 1) * d] = 0.5                       # with a cosine of 1: ties, and a power of two's border
    qkv[6, hq * d + 3] = float("inf")
    positions = torch.randint(0, 2000, (t,), generator=g)
    positions[5] = 0
    ang = torch.arange(2000, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, d // 4, dtype=torch.float64) * 4 / d)
    cos, sin = ang.cos().float(), ang.sin().float()         # half of the head turns
    kn = (1 + 0.2 * torch.randn(d, generator=g)).bfloat16() if norm else None
    pool = K8.new_pool(t // page, hk, page, d, cuda)
    slots = torch.arange(t, device=cuda)
    K8.rope_kv_append_e4m3(qkv.cuda(), pool, positions.cuda(), slots, cos.cuda(), sin.cuda(), hq, hk, d, page, rot=d // 2, pairs=pairs,
                           k_norm=None if kn is None else kn.cuda(), eps=1e-6)
    k = qkv[:, hq * d:(hq + hk) * d].double().view(t, hk, d)
    if norm:
        k = k / torch.sqrt(k.pow(2).mean(-1, keepdim=True) + 1e-6) * kn.double()
    k = rotated64(k, cos[positions][:, None].double(), sin[positions][:, None].double(), d // 2, pairs)
    k = torch.where(torch.isfinite(k), k, float("nan"))
    top = k.nan_to_num(0.0).abs().amax(-1)
    e = torch.where(top > 0, torch.ceil(torch.log2(top / 448)), -40.0).clamp(-40, 119)
    u = (k * torch.exp2(-e)[..., None]).abs()
    ulp = torch.exp2(torch.floor(torch.log2(u.clamp(min=2.0 ** -6))) - 3)
    want = torch.sign(k) * torch.round(u / ulp) * ulp       # to nearest, ties to even
    codes, scales = K8.views(pool, hk, page, d)
    got = codes[:, 0].permute(0, 2, 1, 3).reshape(t, hk, d).float().double().cpu()
    assert torch.equal(scales[:, 0].permute(0, 2, 1).reshape(t, hk).cpu().double() - 127, e)
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fin) and torch.equal(got[fin], want[fin])


LAYOUTS = [(32, 8, 128, 64), (4, 2, 64, 16), (24, 4, 256, 64), (16, 1, 128, 8), (5, 5, 64, 128), (12, 4, 128, 32)]


@pytest.mark.parametrize("hq,hk,d,page", LAYOUTS)
@pytest.mark.parametrize("lens,rows", [([1, 0, 700, 64, 65], 1), ([3, 200, 16], 3), ([1300], 1), ([9, 2, 140], 7)])
def test_attention_of_fixed_rows(cuda, hq, hk, d, page, lens, rows):
    g = torch.Generator().manual_seed(len(lens) * 10 + rows)
    pool, table, kv = fill_cache("e4m3", lens, hk, d, page, g)
    q = torch.randn(len(lens) * rows + 2, (hq + 2 * hk) * d, generator=g).bfloat16().cuda()[:, : hq * d]
    out = torch.full((q.shape[0], hq * d), 5.0, dtype=torch.bfloat16, device=cuda)
    K8.paged_attention_e4m3(q, pool, table, torch.tensor(lens, dtype=torch.int32, device=cuda), hq, hk, d, page, out=out, rows_per_seq=rows)
    assert bool((out[len(lens) * rows:] == 5).all())
    for s, l in enumerate(lens):
        seen = torch.arange(l)[None] <= (l - rows + torch.arange(rows))[:, None]
        ref, spread = attend64(q[s * rows:(s + 1) * rows].cpu().view(rows, hq, d), kv[s], seen, d ** -0.5)
        close(out[s * rows:(s + 1) * rows].view(rows, hq, d), ref, spread, WEIGHT["e4m3"])


@pytest.mark.parametrize("hq,hk,d,page", [(32, 8, 128, 64), (16, 2, 64, 16), (24, 4, 256, 64), (16, 16, 128, 8)])
def test_attention_of_ragged_chunks(cuda, hq, hk, d, page):
    g = torch.Generator().manual_seed(3)
    rows, lens = [1, 150, 0, 33, 64, 2], [400, 150, 7, 300, 64, 1000]
    pool, table, kv = fill_cache("e4m3", lens, hk, d, page, g)
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    q = (2 * torch.randn(cu[-1], hq * d, generator=g)).bfloat16().cuda()
    out = K8.paged_attention_e4m3(q, pool, table, torch.tensor(lens, dtype=torch.int32, device=cuda), hq, hk, d, page,
                                  cu_q=torch.tensor(cu, dtype=torch.int32, device=cuda), max_rows=150, max_len=1000, scale=0.1)
    for s, l in enumerate(lens):
        r = rows[s]
        seen = torch.arange(l)[None] <= (l - r + torch.arange(r))[:, None]
        ref, spread = attend64(q[cu[s]:cu[s + 1]].cpu().view(r, hq, d), kv[s], seen, 0.1)
        close(out[cu[s]:cu[s + 1]].view(r, hq, d), ref, spread, WEIGHT["e4m3"])


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hk,d,page", LAYOUTS)
@pytest.mark.parametrize("rows,past", [([1, 5, 0, 17], [0, 300, 4, 63]), ([64, 40], [1000, 1]), ([130, 9], [77, 500])])
def test_tree_attention(cuda, kind, hq, hk, d, page, rows, past):
    g = torch.Generator().manual_seed(sum(rows))
    lens = [r + p for r, p in zip(rows, past)]
    pool, table, kv = fill_cache(kind, lens, hk, d, page, g)
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    words = -(-max(rows) // 64)
    bits = torch.rand(cu[-1], words * 64, generator=g) < 0.3
    bits[cu[-2]:cu[-2] + 2] = False                       # rows that see the context alone, or nothing
    weights = torch.tensor([1 << i if i < 63 else -(1 << 63) for i in range(64)])
    masks = (bits.view(cu[-1], words, 64).long() * weights).sum(-1)
    q = torch.randn(cu[-1], hq * d, generator=g).bfloat16().cuda()
    out = TR.tree_attention(q, pool, table, torch.tensor(lens, dtype=torch.int32, device=cuda), masks.cuda(),
                            torch.tensor(cu, dtype=torch.int32, device=cuda), hq, hk, d, page, max_rows=max(rows))
    for s, l in enumerate(lens):
        r = rows[s]
        seen = torch.ones(r, l, dtype=torch.bool)
        seen[:, l - r:] = bits[cu[s]:cu[s + 1], :r]
        ref, spread = attend64(q[cu[s]:cu[s + 1]].cpu().view(r, hq, d), kv[s], seen, d ** -0.5)
        close(out[cu[s]:cu[s + 1]].view(r, hq, d), ref, spread, WEIGHT[kind])


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("nodes", [6, 90])
@pytest.mark.parametrize("d", [128, 64, 256])
def test_what_a_row_does_not_see_does_not_reach_it(cuda, kind, nodes, d):
    """Infinities and NaN behind the sequence's end, and in nodes that some rows see and others do not."""
    hq, hk, page, past = 8, 2, 64, 100
    l = past + nodes
    g = torch.Generator().manual_seed(9)
    pool, table, kv = fill_cache(kind, [l], hk, d, page, g)
    bits = torch.rand(nodes, nodes, generator=g) < 0.4
    bad = {2: float("nan"), 4: float("inf"), 5: float("-inf")}
    for i, v in bad.items():
        bits[i, i] = True
        p, o = int(table[0, (past + i) // page]), (past + i) % page
        if kind == "bf16":
            pool[p, 1, :, o, 7] = v
            pool[p, 0, :, o, 9] = v if i == 2 else 0.5
            kv[0][0, past + i, :, 9] = v if i == 2 else 0.5
        else:
            v = float("nan")
            K8.views(pool, hk, page, d)[0].view(torch.uint8)[p, 1, :, o, 7] = 0x7F
        kv[0][1, past + i, :, 7] = v
    tail = torch.arange(l, table.shape[1] * page)
    for t in tail.tolist():                                # the rest of the last page
        p, o = int(table[0, t // page]), t % page
        if kind == "bf16":
            pool[p, :, :, o] = float("nan")
        else:
            c, s = K8.views(pool, hk, page, d)
            c.view(torch.uint8)[p, :, :, o] = 0x7F
            s[p, :, :, o] = 255
    weights = torch.tensor([1 << i if i < 63 else -(1 << 63) for i in range(64)])
    words = -(-nodes // 64)
    wide = torch.zeros(nodes, words * 64, dtype=torch.bool)
    wide[:, :nodes] = bits
    masks = (wide.view(nodes, words, 64).long() * weights).sum(-1)
    q = torch.randn(nodes, hq * d, generator=g).bfloat16().cuda()
    out = TR.tree_attention(q, pool, table, torch.tensor([l], dtype=torch.int32, device=cuda), masks.cuda(),
                            torch.tensor([0, nodes], dtype=torch.int32, device=cuda), hq, hk, d, page).double().cpu().view(nodes, hq, d)
    seen = torch.ones(nodes, l, dtype=torch.bool)
    seen[:, past:] = bits
    for r in range(nodes):                                 # row by row: the statement must not mix what others see
        keep = seen[r].nonzero()[:, 0]
        ref, spread = attend64(q[r:r + 1].cpu().view(1, hq, d), kv[0][:, keep], torch.ones(1, len(keep), dtype=torch.bool), d ** -0.5)
        fin = torch.isfinite(ref[0])
        assert torch.equal(torch.isnan(out[r]), torch.isnan(ref[0])), r
        assert torch.equal(out[r][~fin & ~torch.isnan(ref[0])], ref[0][~fin & ~torch.isnan(ref[0])]), r
        if bool(fin.any()):
            allow = BF * ref[0][fin].abs() * 1.01 + (WEIGHT[kind] + 2.0 ** -14) * spread[0][fin]
            assert bool(((out[r][fin] - ref[0][fin]).abs() <= allow).all()), r
    # the same with causal rows, over the 8-bit cache
    if kind == "e4m3":
        got = K8.paged_attention_e4m3(q, pool, table, torch.tensor([l], dtype=torch.int32, device=cuda), hq, hk, d, page,
                                      rows_per_seq=nodes).double().cpu().view(nodes, hq, d)
        assert bool(torch.isfinite(got[:2]).all()) and bool(torch.isnan(got[2:, :, 7]).all())


@pytest.mark.parametrize("size", [1e-9, 1e9])
def test_value_rows_of_very_different_sizes(cuda, size):
    """Half of the tokens have values a billion times larger or smaller: what a row attends to keeps its precision."""
    hq, hk, d, page, l = 4, 1, 128, 64, 500
    g = torch.Generator().manual_seed(1)
    k = torch.randn(l, hk, d, generator=g)
    v = torch.randn(l, hk, d, generator=g)
    v[::2] *= size
    k[::2, :, 0] += 40.0                                   # queries with a large first value look at the even tokens, negative at the odd
    qkv = torch.cat([torch.zeros(l, hq * d), k.view(l, -1), v.view(l, -1)], 1).bfloat16().cuda()
    pool = K8.new_pool(8, hk, page, d, cuda)
    none = torch.zeros(1, 0, device=cuda)
    slots = torch.arange(l, device=cuda)
    K8.rope_kv_append_e4m3(qkv, pool, slots * 0, slots, none, none, hq, hk, d, page, rot=0)
    kv = K8.read_rows_e4m3(pool, slots, hk, d, page).double().cpu().permute(1, 0, 2, 3)
    q = torch.randn(1, hq, d, generator=g)
    q[:, :2, 0], q[:, 2:, 0] = 6.0, -6.0
    q = q.bfloat16()
    table = torch.arange(8, dtype=torch.int32, device=cuda)[None]
    out = K8.paged_attention_e4m3(q.view(1, -1).cuda(), pool, table, torch.tensor([l], dtype=torch.int32, device=cuda), hq, hk, d, page)
    ref, spread = attend64(q, kv, torch.ones(1, l, dtype=torch.bool), d ** -0.5)
    close(out.view(1, hq, d), ref, spread, WEIGHT["e4m3"])
