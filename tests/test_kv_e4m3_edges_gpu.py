"""Attention over the 8-bit cache, and its append, where scales, rows and arguments are at their ends (sm_100a)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from kern_b200.ops import kv_e4m3 as K8
from kern_b200.ops import tree as TR
from kern_b200.ops.launcher import Kernels
from test_kv_e4m3_gpu import WEIGHT, attend64, close, fill_cache


@pytest.fixture(autouse=True)
def _no_device_error(cuda):
    yield
    Kernels.get(cuda).check_error()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cache_of(k, v, page):
    """A pool with the rows k and v [L, hk, d] of one sequence on scattered pages; (pool, table, 64-bit rows [2, L, hk, d])."""
    l, hk, d = k.shape
    need = -(-l // page)
    kv = torch.zeros(need * page, 2, hk, d)
    kv[:l] = torch.stack([k, v], 1)
    codes, scales = K8.quantise_reference(kv.bfloat16())
    exact = torch.ldexp(codes.double(), (scales.int() - 127)[..., None])
    table = torch.randperm(need + 2, generator=torch.Generator().manual_seed(l))[:need].int()
    pool = K8.new_pool(need + 2, hk, page, d, "cuda")
    c, s = K8.views(pool, hk, page, d)
    at = table.long().cuda()
    c.view(torch.uint8)[at] = codes.view(torch.uint8).view(need, page, 2, hk, d).permute(0, 2, 3, 1, 4).cuda()
    s[at] = scales.view(need, page, 2, hk).permute(0, 2, 3, 1).cuda()
    return pool, table.cuda()[None], exact[:l].permute(1, 0, 2, 3)


def causal(rows, l):
    return torch.arange(l)[None] <= (l - rows + torch.arange(rows))[:, None]


def bits_of(seen):
    """[rows, nodes] bool -> i64 [rows, words]"""
    rows, nodes = seen.shape
    words = -(-nodes // 64)
    wide = torch.zeros(rows, words * 64, dtype=torch.bool)
    wide[:, :nodes] = seen
    weights = torch.tensor([1 << i if i < 63 else -(1 << 63) for i in range(64)])
    return (wide.view(rows, words, 64).long() * weights).sum(-1).cuda()


def both_ways(q, pool, table, l, hq, hk, d, page, **k):
    """The rows as causal ones and as a tree that is a chain: (causal, tree), [rows, hq, d]."""
    rows = q.shape[0]
    a = K8.paged_attention_e4m3(q, pool, table, i32([l]), hq, hk, d, page, rows_per_seq=rows, **k)
    out = [a.view(rows, hq, d)]
    if rows <= TR.MAX_NODES:
        chain = bits_of(torch.ones(rows, rows).tril().bool())
        out.append(TR.tree_attention(q, pool, table, i32([l]), chain, i32([0, rows]), hq, hk, d, page, **k).view(rows, hq, d))
    return out


@pytest.mark.parametrize("d", [256, 128, 64])
def test_value_tiles_of_other_sizes(cuda, d):
    """Every 64 tokens' values have another size: a value tile's exponent taken from a neighbour's scale bytes shows at once. From idle with
    cold caches, and one behind the other."""
    hq, hk, page, l, rows = 24, 4, 64, 4000, 40
    g = torch.Generator().manual_seed(d)
    k, v = torch.randn(2, l, hk, d, generator=g)
    v *= torch.exp2(torch.randint(-8, 9, (-(-l // 64),), generator=g).float()).repeat_interleave(64)[:l, None, None]
    pool, table, kv = cache_of(k, v, page)
    q = torch.randn(rows, hq * d, generator=g).bfloat16().cuda()
    first = both_ways(q, pool, table, l, hq, hk, d, page)
    ref, spread = attend64(q.cpu().view(rows, hq, d), kv, causal(rows, l), d ** -0.5)
    for out in first:
        close(out, ref, spread, WEIGHT["e4m3"])
    cold = torch.empty(200 << 20, dtype=torch.uint8, device=cuda)
    wrong = torch.zeros((), dtype=torch.int64, device=cuda)
    for i in range(100):
        if i % 3 == 0:
            cold.fill_(i)
        if i % 3 < 2:
            torch.cuda.synchronize()
        for x, y in zip(first, both_ways(q, pool, table, l, hq, hk, d, page)):
            wrong += (x != y).any()
    assert int(wrong) == 0


def _partners(d, rot, pairs):
    """(places of a pair) that turn together"""
    return (3, 3 + rot // 2) if pairs == "half" else (6, 7)


@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (2, 1, 128), (3, 3, 64), (5, 5, 128), (2, 1, 256)])
def test_values_whose_neighbours_are_infinite_or_huge(cuda, hq, hk, d, pairs, norm):
    """Values do not turn: what stands at a rotation partner's place reaches no code but its own, whatever rows share a warp."""
    page, rot = 16, d
    a, b = _partners(d, rot, pairs)
    top = float(torch.finfo(torch.bfloat16).max)
    ends = [(float("inf"), 1.5), (1.5, float("-inf")), (float("nan"), -2.0), (top, top), (-top, 0.75 * top), (3e38, 1.0), (1.0, 2.0)]
    t = len(ends)
    g = torch.Generator().manual_seed(d)
    x = torch.randn(t, hq + 2 * hk, d, generator=g)
    for i, (u, w) in enumerate(ends):
        x[i, hq + hk:, a], x[i, hq + hk:, b] = u, w
    qkv = x.view(t, -1).bfloat16()
    ang = torch.rand(t, rot // 2, generator=g) * 6
    kn = (1 + 0.2 * torch.randn(d, generator=g)).bfloat16().cuda() if norm else None
    pool = K8.new_pool(1, hk, page, d, cuda)
    slots = torch.arange(t, device=cuda)
    K8.rope_kv_append_e4m3(qkv.cuda(), pool, slots, slots, ang.cos().cuda(), ang.sin().cuda(), hq, hk, d, page, rot=rot, pairs=pairs, k_norm=kn)
    want_c, want_s = K8.quantise_reference(qkv.view(t, -1, d)[:, hq + hk:])
    codes, scales = K8.views(pool, hk, page, d)
    got = codes[0, 1, :, :t].permute(1, 0, 2).float().cpu()
    nan = torch.isnan(want_c.float())
    assert torch.equal(torch.isnan(got), nan) and int(nan.sum()) == 3 * hk
    assert torch.equal(got[~nan], want_c.float()[~nan]) and torch.equal(scales[0, 1, :, :t].t().cpu(), want_s)


@pytest.mark.parametrize("rows", [1, 4, 100, 300])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("size", [0.0, 2.0 ** -30])
@pytest.mark.parametrize("query", [0.0, 1e-3, 1.0])
def test_caches_of_zeros_or_next_to_nothing(cuda, rows, d, size, query):
    """Keys and values of zeros give zeros; tiny ones, or queries of zeros, the mean of the values."""
    hq, hk, page, l = 8, 2, 64, 450
    g = torch.Generator().manual_seed(d)
    pool, table, kv = cache_of(*(torch.randn(2, l, hk, d, generator=g) * size), page)
    q = (torch.randn(rows, hq * d, generator=g) * query).bfloat16().cuda()
    ref, spread = attend64(q.cpu().view(rows, hq, d), kv, causal(rows, l), d ** -0.5)
    for out in both_ways(q, pool, table, l, hq, hk, d, page):
        if size:
            close(out, ref, spread, WEIGHT["e4m3"])
        else:
            assert bool((out == 0).all())


@pytest.mark.parametrize("rows", [1, 4, 100, 300])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("query", [0.0, 1e-3, 1.0])
def test_a_pool_that_nobody_has_written_to(cuda, rows, d, query):
    hq, hk, page, l = 8, 2, 64, 450
    pool, table = K8.new_pool(9, hk, page, d, cuda), torch.arange(8, dtype=torch.int32, device=cuda)[None]
    q = (torch.randn(rows, hq * d, generator=torch.Generator().manual_seed(rows)) * query).bfloat16().cuda()
    for out in both_ways(q, pool, table, l, hq, hk, d, page):
        assert bool((out == 0).all())


@pytest.mark.parametrize("rows", [1, 4, 100, 300])
@pytest.mark.parametrize("past", [100, 4000])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("first", [False, True])
def test_rows_that_nobody_has_written_to_beside_others(cuda, rows, past, d, first):
    """Every other run of 128 tokens is as `new_pool` leaves it: tokens of zeros, which count in the sum of weights."""
    hq, hk, page = 8, 2, 64
    l = past + rows
    g = torch.Generator().manual_seed(rows + past)
    empty = (torch.arange(l) // 128) % 2 == int(not first)
    k, v = torch.where(empty[:, None, None], 0.0, torch.randn(2, l, hk, d, generator=g))
    pool, table, kv = cache_of(k, v, page)
    at = empty.nonzero()[:, 0].cuda()
    K8.views(pool, hk, page, d)[1][table[0].long()[at // page], :, :, at % page] = 0
    q = torch.randn(rows, hq * d, generator=g).bfloat16().cuda()
    ref, spread = attend64(q.cpu().view(rows, hq, d), kv, causal(rows, l), d ** -0.5)
    for out in both_ways(q, pool, table, l, hq, hk, d, page):
        close(out, ref, spread, WEIGHT["e4m3"])


@pytest.mark.parametrize("rows", [1, 4, 100, 300])
@pytest.mark.parametrize("past", [100, 4000])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("low,high", [(None, 100), (-38, 100), (-30, 60), (-38, 118)])
@pytest.mark.parametrize("swap", [False, True])
def test_value_tiles_far_apart(cuda, rows, past, d, low, high, swap):
    """Runs of 128 tokens with the smallest values (or zeros) beside runs with huge ones, in either order: every token counts in the sum
    of weights. With one share of the context and with several."""
    hq, hk, page = 8, 2, 64
    l = past + rows
    g = torch.Generator().manual_seed(rows + past)
    k, v = torch.randn(2, l, hk, d, generator=g)
    small = ((torch.arange(l) // 128) % 2 == int(swap))[:, None, None]
    v = torch.where(small, v * (0.0 if low is None else 2.0 ** low), v * 2.0 ** high).clamp(-2.9e38, 2.9e38)
    pool, table, kv = cache_of(k, v, page)
    q = torch.randn(rows, hq * d, generator=g).bfloat16().cuda()
    ref, spread = attend64(q.cpu().view(rows, hq, d), kv, causal(rows, l), d ** -0.5)
    for out in both_ways(q, pool, table, l, hq, hk, d, page):
        close(out, ref, spread, WEIGHT["e4m3"])


@pytest.mark.parametrize("rows", [4, 100, 300])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("which", ["values", "keys"])
def test_rows_under_the_smallest_scale_beside_ordinary_ones(cuda, rows, d, which):
    """The first tokens' values (or keys) are under 2^-31 and share a tile with ordinary ones: rows that see them alone get them."""
    hq, hk, page, l = 8, 2, 64, rows
    g = torch.Generator().manual_seed(rows)
    k, v = torch.randn(2, l, hk, d, generator=g)
    (v if which == "values" else k)[:20] *= 2.0 ** -35
    pool, table, kv = cache_of(k, v, page)
    q = torch.randn(rows, hq * d, generator=g)
    if which == "keys":
        q *= 2.0 ** 36
        q[20:] = 0
    q = q.bfloat16().cuda()
    ref, spread = attend64(q.cpu().view(rows, hq, d), kv, causal(rows, l), d ** -0.5)
    for out in both_ways(q, pool, table, l, hq, hk, d, page):
        close(out, ref, spread, WEIGHT["e4m3"])


def failed(f):
    out = f()
    with pytest.raises(RuntimeError, match="device error"):
        Kernels.get(torch.device("cuda:0")).check_error()
    return out


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("sizes,most", [([1, 3, 1], 1), ([2, 5], 3), ([30, 90], 60), ([1, 300, 1, 200], 250), ([300], 5), ([3, 40], 0)])
def test_more_rows_than_max_rows(cuda, d, sizes, most):
    """A sequence of more rows than the call says sets the error word and is left alone; the others are as ever."""
    hq, hk, page, l = 8, 2, 64, 400
    g = torch.Generator().manual_seed(most)
    k, v = torch.randn(2, l, hk, d, generator=g)
    pool, table, kv = cache_of(k, v, page)
    n, cu = len(sizes), [0]
    for r in sizes:
        cu.append(cu[-1] + r)
    table, lens = table.expand(n, -1).contiguous(), i32([l] * n)
    q = torch.randn(cu[-1], hq * d, generator=g).bfloat16().cuda()
    masks = torch.full((cu[-1], 1), -1, dtype=torch.int64, device=cuda)
    calls = [lambda out: K8.paged_attention_e4m3(q, pool, table, lens, hq, hk, d, page, cu_q=i32(cu), max_rows=most, out=out),
             lambda out: TR.tree_attention(q, pool, table, lens, masks, i32(cu), hq, hk, d, page, max_rows=most, out=out)]
    for tree, call in enumerate(calls):
        out = failed(lambda: call(torch.full((cu[-1], hq * d), 7.0, dtype=torch.bfloat16, device=cuda)))
        for s, r in enumerate(sizes):
            mine = out[cu[s]:cu[s + 1]]
            if r > most:
                assert bool((mine == 7).all())
            elif not tree or r <= 64:
                seen = torch.ones(r, l, dtype=torch.bool) if tree else causal(r, l)
                ref, spread = attend64(q[cu[s]:cu[s + 1]].cpu().view(r, hq, d), kv, seen, d ** -0.5)
                close(mine.view(r, hq, d), ref, spread, WEIGHT["e4m3"])


@pytest.mark.parametrize("rows", [1, 40])
def test_the_workspace_is_of_the_rows_in_use(cuda, rows):
    """A few rows at the end of a buffer of 8192, over a long context in many shares."""
    hq, hk, d, page, l, all_rows = 32, 8, 128, 64, 30000, 8192
    g = torch.Generator().manual_seed(0)
    k, v = torch.randn(2, l, hk, d, generator=g)
    pool, table, kv = cache_of(k, v, page)
    q = torch.randn(all_rows, hq * d, generator=g).bfloat16().cuda()
    out = torch.zeros_like(q)
    cu, lens = i32([all_rows - rows, all_rows]), i32([l])
    call = lambda: K8.paged_attention_e4m3(q, pool, table, lens, hq, hk, d, page, cu_q=cu, max_rows=rows, out=out)
    call()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    call()
    # 256 shares at most, of d + 2 floats for every head of the rows in use
    assert torch.cuda.max_memory_allocated() - before <= rows * hq * 256 * (d + 2) * 4 + 4096
    ref, spread = attend64(q[-rows:].cpu().view(rows, hq, d), kv, causal(rows, l), d ** -0.5)
    close(out[-rows:].view(rows, hq, d), ref, spread, WEIGHT["e4m3"])
    assert bool((out[:-rows] == 0).all())


@pytest.mark.parametrize("rows", [1, 40])
def test_partials_of_some_rows_of_a_wide_buffer(cuda, rows):
    """Three sequences, one of no rows, whose rows are some of q's: each joins its own shares."""
    hq, hk, d, page, l = 8, 2, 128, 64, 9000
    g = torch.Generator().manual_seed(rows)
    k, v = torch.randn(2, l, hk, d, generator=g)
    pool, table, kv = cache_of(k, v, page)
    lens, cu = [l, 50, l - 777], [5, 5 + rows, 5 + rows, 5 + 2 * rows]
    q = torch.randn(1000, hq * d, generator=g).bfloat16().cuda()
    out = K8.paged_attention_e4m3(q, pool, table.expand(3, -1).contiguous(), i32(lens), hq, hk, d, page, cu_q=i32(cu), max_rows=rows)
    for s in (0, 2):
        ref, spread = attend64(q[cu[s]:cu[s + 1]].cpu().view(rows, hq, d), kv[:, :lens[s]], causal(rows, lens[s]), d ** -0.5)
        close(out[cu[s]:cu[s + 1]].view(rows, hq, d), ref, spread, WEIGHT["e4m3"])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_lengths_past_the_table(cuda, d, rows):
    """A length that the table has no pages for, up to the largest number there is: the error word, and no walk to its end."""
    hq, hk, page, l = 8, 2, 64, 400
    g = torch.Generator().manual_seed(rows)
    k, v = torch.randn(2, l, hk, d, generator=g)
    pool, table, kv = cache_of(k, v, page)
    table = table.expand(2, -1).contiguous()
    q = torch.randn(2 * rows, hq * d, generator=g).bfloat16().cuda()
    masks, cu = torch.ones(2 * rows, 1, dtype=torch.int64, device=cuda), i32([0, rows, 2 * rows])
    ref, spread = attend64(q[rows:].cpu().view(rows, hq, d), kv, causal(rows, l), d ** -0.5)
    for far in (l + 49, 1 << 20, (1 << 31) - 100, (1 << 31) - 1):
        lens = i32([far, l])
        for max_len in (None, 9000):                      # (in one share, and in several that are joined)
            out = failed(lambda: K8.paged_attention_e4m3(q, pool, table, lens, hq, hk, d, page, rows_per_seq=rows, max_len=max_len))
            close(out[rows:].view(rows, hq, d), ref, spread, WEIGHT["e4m3"])
            failed(lambda: TR.tree_attention(q, pool, table, lens, masks, cu, hq, hk, d, page, max_rows=rows, max_len=max_len))


def test_nodes_that_no_tree_holds(cuda):
    """Rows before the first tree, and those of a tree whose bounds are wrong: no slot, no mask, no step of a walk."""
    page = 16
    table = torch.arange(4, dtype=torch.int32, device=cuda)[None].contiguous()
    par = i32([-1, 0, 0, -1, 0, 1, 0])
    ids = torch.zeros(7, dtype=torch.int64, device=cuda)
    for cu, bad, live in (([2, 5], False, range(2, 5)), ([1, 9], True, ()), ([-3, 4], True, ()), ([4, 2], True, ())):
        for _ in range(3):                                # (places that something else has used before)
            junk = [torch.full((7,), 5, dtype=torch.int64, device=cuda) for _ in range(8)]
            del junk
            base = torch.tensor([3], device=cuda)
            flat = i32([0, 0, -1, 0, 1, 0, 0]) if live else par
            call = lambda: TR.tree_rows(flat, i32(cu), base, table, page)
            pos, slots, lens, masks = failed(call) if bad else call()
            walk = lambda: TR.tree_keep(ids, flat, ids, i32(cu), base, table, [], 2, 64, page)
            count, path, emitted = failed(walk) if bad else walk()
            rest = [i for i in range(7) if i not in live]
            assert all(int(slots[i]) == -1 and int(pos[i]) == 0 and int(masks[i]) == 0 for i in rest)
            assert all(int(path[i]) == -1 and int(emitted[i]) == 0 for i in rest)
            assert all(int(slots[i]) == 3 + i - 2 for i in live) and int(count[0]) == (3 if live else 0)


def test_places_past_32_bits(cuda):
    """A base near the largest number: no slot, and a context that no table holds, not one of some other length."""
    table = torch.arange(4, dtype=torch.int32, device=cuda)[None].contiguous()
    for base in ((1 << 32) + 3, 1 << 62, (1 << 63) - 1):
        _, slots, lens, _ = failed(lambda: TR.tree_rows(i32([-1, 0]), i32([0, 2]), torch.tensor([base], device=cuda), table, 16))
        assert slots.tolist() == [-1, -1] and lens.tolist() == [(1 << 31) - 1]


@pytest.mark.parametrize("hq,hk,d", [(32, 1, 128), (48, 2, 64), (40, 1, 256)])
def test_append_of_wide_groups(cuda, hq, hk, d):
    """More than 16 query heads to a kv head: the append has no use for the group."""
    page, t = 16, 9
    g = torch.Generator().manual_seed(hq)
    qkv = torch.randn(t, (hq + 2 * hk) * d, generator=g).bfloat16()
    ang = torch.rand(t, d // 2, generator=g) * 6
    pool = K8.new_pool(1, hk, page, d, cuda)
    slots = torch.arange(t, device=cuda)
    got = K8.rope_kv_append_e4m3(qkv.cuda(), pool, slots, slots, ang.cos().cuda(), ang.sin().cuda(), hq, hk, d, page)
    x = qkv.double().view(t, -1, d)
    c, s = ang.cos().double()[:, None], ang.sin().double()[:, None]
    q = torch.cat([x[:, :hq, : d // 2] * c - x[:, :hq, d // 2:] * s, x[:, :hq, d // 2:] * c + x[:, :hq, : d // 2] * s], -1).view(t, -1)
    assert bool(((got.double().cpu() - q).abs() <= 2.0 ** -8 * q.abs() + 2.0 ** -20 * q.abs().max()).all())
    want = K8.dequantise_reference(*K8.quantise_reference(x[:, hq + hk:].float()))
    assert torch.equal(K8.read_rows_e4m3(pool, slots, hk, d, page)[:, 1].float().cpu(), want)


@pytest.mark.parametrize("rows", [1, 4, 100])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_huge_keys_across_huge_queries(cuda, rows, d):
    """Keys and queries whose factors together pass f32's range, and whose products are 0: the mean of the values."""
    hq, hk, page, l = 8, 2, 64, 300
    g = torch.Generator().manual_seed(rows)
    k, v = torch.randn(2, l, hk, d, generator=g)
    k = torch.where(torch.arange(d) < d // 2, k * 2.0 ** 100, 0.0)
    pool, table, kv = cache_of(k, v, page)
    q = torch.where(torch.arange(d) < d // 2, 0.0, torch.randn(rows, hq, d, generator=g) * 2.0 ** 60).view(rows, -1).bfloat16().cuda()
    ref, spread = attend64(q.cpu().view(rows, hq, d), kv, causal(rows, l), d ** -0.5)
    for out in both_ways(q, pool, table, l, hq, hk, d, page):
        close(out, ref, spread, WEIGHT["e4m3"])


@pytest.mark.parametrize("heads,hk,d", [(8, 1, 128), (4, 2, 64), (2, 1, 256)])
def test_a_decoder_whose_padding_token_is_zeros(cuda, tmp_path, heads, hk, d):
    """An embedding row of zeros, as checkpoints have it for padding: its queries, keys and values are zeros, in prompts and chunks."""
    import dataclasses

    from kern_b200.engine import Engine
    from kern_b200.models import common, dense
    from kern_b200.runtime import Runtime

    cfg = dataclasses.replace(dense.TINY, kv="e4m3", heads=heads, kv_heads=hk, head_dim=d, max_context=512, max_tokens=512)
    w = dense.random_weights(cfg, seed=0, std=0.05)
    w["model.embed_tokens.weight"][3] = 0
    common.write_safetensors(tmp_path / "model.safetensors", w)
    rt = Runtime(dense.build_manifest(cfg), weights=tmp_path / "model.safetensors", tokens=cfg.page_size * 64)
    rt.once()
    eng, oracle = Engine(rt), dense.DenseOracle(cfg, w, device="cuda")
    g = torch.Generator().manual_seed(3)
    words = torch.randint(4, cfg.vocab, (60,), generator=g).tolist()
    prompts = [[3] * 200, [3] * 150 + words[:40], [3]]
    seqs, caches = [eng.open(len(p) + 40) for p in prompts], [oracle.new_cache() for _ in prompts]
    for feeds in (prompts, [[3] * 30, words[40:], [3] * 9], [[3], [3], words[:1]]):
        eng.step(list(zip(seqs, feeds)))
        logits = rt.tensor("logits")[:3].float()
        for f, c, lg in zip(feeds, caches, logits):
            ref = oracle.forward(f, c)[-1]
            # 1.3 % for codes that bf16 takes to their neighbours, as much for bf16 elsewhere; zeros exactly
            assert float((lg - ref).norm()) <= 0.05 * float(ref.norm())
    rt.check_error()


@pytest.mark.parametrize("most", [0, 1, 30, 64, 70])
def test_more_nodes_than_max_rows(cuda, most):
    """A chain of 75 nodes, all agreed with: those from `most` on have no slot and are not walked to, and the error word says so."""
    page, n = 16, 75
    table = torch.arange(8, dtype=torch.int32, device=cuda)[None].contiguous()
    par, ids = i32([i - 1 for i in range(n)]), torch.zeros(n, dtype=torch.int64, device=cuda)
    cu, base = i32([0, n]), torch.tensor([3], device=cuda)
    pos, slots, lens, masks = failed(lambda: TR.tree_rows(par, cu, base, table, page, max_rows=most))
    assert slots.tolist() == [3 + i for i in range(most)] + [-1] * (n - most) and masks.shape[1] == max(1, -(-most // 64))
    assert pos.tolist() == [3 + i for i in range(most)] + [0] * (n - most) and bool((masks[most:] == 0).all())
    pool = torch.randint(0, 255, (8, K8.page_bytes(1, page, 64)), dtype=torch.uint8, device=cuda)
    before = pool.clone()
    count, path, _ = failed(lambda: TR.tree_keep(ids, par, ids, cu, base, table, [pool], 1, 64, page, max_rows=most))
    assert count.tolist() == [most] and path.tolist() == list(range(most)) + [-1] * (n - most) and torch.equal(pool, before)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_blocks_of_up_to_128_rows(cuda, d):
    """The cases above in blocks that both tiles of the many-row kernel share, on alternate key tiles."""
    rows = 30                                              # of 4 heads
    for size in (0.0, 2.0 ** -30):
        for query in (0.0, 1.0):
            test_caches_of_zeros_or_next_to_nothing(cuda, rows, d, size, query)
    test_a_pool_that_nobody_has_written_to(cuda, rows, d, 1.0)
    for past in (100, 4000):
        for swap in (False, True):
            test_rows_that_nobody_has_written_to_beside_others(cuda, rows, past, d, swap)
            for low, high in ((None, 100), (-30, 60), (-38, 118)):
                test_value_tiles_far_apart(cuda, rows, past, d, low, high, swap)
    for which in ("values", "keys"):
        test_rows_under_the_smallest_scale_beside_ordinary_ones(cuda, rows, d, which)
    test_huge_keys_across_huge_queries(cuda, rows, d)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("kind", ["e4m3", "bf16"])
@pytest.mark.parametrize("rows", [1, 3])
def test_short_contexts_under_a_long_limit(cuda, d, kind, rows):
    """A limit that asks for many shares, each a block of its own, over contexts of one: the block that has it writes the rows, and no
    other does. From idle with cold caches, and one behind the other."""
    hq, hk, page, lens = 6, 2, 64, [3, 128, 40]
    g = torch.Generator().manual_seed(d)
    pool, table, kv = fill_cache(kind, lens, hk, d, page, g)
    table = torch.cat([table, torch.zeros(3, 2000, dtype=torch.int32, device=cuda)], 1).contiguous()
    cu, l = i32([0, rows, 2 * rows, 3 * rows]), i32(lens)
    q = torch.randn(3 * rows, hq * d, generator=g).bfloat16().cuda()
    chain = bits_of(torch.ones(rows, rows).tril().bool()).repeat(3, 1)
    if kind == "e4m3":
        call = lambda: K8.paged_attention_e4m3(q, pool, table, l, hq, hk, d, page, cu_q=cu, max_rows=rows)
    else:
        call = lambda: TR.tree_attention(q, pool, table, l, chain, cu, hq, hk, d, page, max_rows=rows)
    out, wrong = call(), torch.zeros((), dtype=torch.int64, device=cuda)
    cold = torch.empty(200 << 20, dtype=torch.uint8, device=cuda)
    for i in range(300):
        if i % 3 == 0:
            cold.fill_(i & 255)
        if i % 3 < 2:
            torch.cuda.synchronize()
        wrong += (call() != out).any()
    assert int(wrong) == 0
    for s in range(3):
        ref, spread = attend64(q[s * rows:(s + 1) * rows].cpu().view(rows, hq, d), kv[s], causal(rows, lens[s]), d ** -0.5)
        # bf16 weights are summed as rounded: 2^-8 of a weight, and of their sum
        close(out[s * rows:(s + 1) * rows].view(rows, hq, d), ref, spread, WEIGHT[kind] * (2 if kind == "bf16" else 1))
