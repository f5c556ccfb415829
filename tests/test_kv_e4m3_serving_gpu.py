"""The operators over 8-bit caches and drafted trees as a server calls them: captured, on other streams, two at once, on caches past
32 bits, and with pages and slots that do not exist (sm_100a)."""
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


def bits_of(seen):
    """[rows, nodes] bool -> i64 [rows, words]"""
    rows, nodes = seen.shape
    words = -(-nodes // 64)
    wide = torch.zeros(rows, words * 64, dtype=torch.bool)
    wide[:, :nodes] = seen
    weights = torch.tensor([1 << i if i < 63 else -(1 << 63) for i in range(64)])
    return (wide.view(rows, words, 64).long() * weights).sum(-1)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("nodes", [3, 20, 40, 90])
@pytest.mark.parametrize("d", [128, 64, 256])
def test_huge_rows_that_are_not_seen(cuda, kind, nodes, d):
    """Every third node has keys and values near the largest bf16: rows that do not see them are as if they were not there."""
    hq, hk, page, past = 8, 2, 64, 70
    l = past + nodes
    g = torch.Generator().manual_seed(nodes)
    pool, table, kv = fill_cache(kind, [l], hk, d, page, g)
    huge = torch.arange(nodes) % 3 == 1
    for i in huge.nonzero()[:, 0].tolist():
        p, o = int(table[0, (past + i) // page]), (past + i) % page
        if kind == "bf16":
            pool[p, :, :, o] = torch.finfo(torch.bfloat16).max
        else:
            c, s = K8.views(pool, hk, page, d)
            c.view(torch.uint8)[p, :, :, o], s[p, :, :, o] = 0x7E, 246      # 448 * 2^119
    seen = torch.rand(nodes, nodes, generator=g) < 0.5
    seen[:, huge] = False
    q = torch.randn(nodes, hq * d, generator=g).bfloat16().cuda()
    out = TR.tree_attention(q, pool, table, i32([l]), bits_of(seen).cuda(), i32([0, nodes]), hq, hk, d, page).view(nodes, hq, d)
    every = torch.cat([torch.ones(nodes, past, dtype=torch.bool), seen], 1)
    ref, spread = attend64(q.cpu().view(nodes, hq, d), kv[0], every, d ** -0.5)
    close(out, ref, spread, WEIGHT[kind])


@pytest.mark.parametrize("rows", [2, 100, 300])
@pytest.mark.parametrize("shared", [1, 4000])
@pytest.mark.parametrize("d", [128, 64, 256])
def test_huge_values_behind_a_causal_row(cuda, rows, shared, d):
    """The block's last token has huge values: only its own row may show it. With and without shares of the context."""
    hq, hk, page = 8, 2, 64
    l = shared + rows
    g = torch.Generator().manual_seed(rows)
    pool, table, kv = fill_cache("e4m3", [l], hk, d, page, g)
    p, o = int(table[0, (l - 1) // page]), (l - 1) % page
    c, s = K8.views(pool, hk, page, d)
    c.view(torch.uint8)[p, 1, :, o], s[p, 1, :, o] = 0x7E, 200
    kv[0][1, l - 1] = 448 * 2.0 ** 73
    q = torch.randn(rows, hq * d, generator=g).bfloat16().cuda()
    out = K8.paged_attention_e4m3(q, pool, table, i32([l]), hq, hk, d, page, rows_per_seq=rows).view(rows, hq, d)
    seen = torch.arange(l)[None] <= (l - rows + torch.arange(rows))[:, None]
    ref, spread = attend64(q[:-1].cpu().view(rows - 1, hq, d), kv[0], seen[:-1], d ** -0.5)
    close(out[:-1], ref, spread, WEIGHT["e4m3"])
    ref, spread = attend64(q[-1:].cpu().view(1, hq, d), kv[0], seen[-1:], d ** -0.5)
    close(out[-1:], ref, spread, WEIGHT["e4m3"])


def calls(cuda, seed):
    """A round's inputs, and a function that runs it: rows, append, attention over the tree, walk; then a causal call."""
    hq, hk, d, page, seqs = 8, 2, 64, 16, 3
    g = torch.Generator().manual_seed(seed)
    sizes = [5, 30, 12]
    cu = i32([0, 5, 35, 47])
    parents = torch.cat([torch.tensor([-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, n)]) for n in sizes]).int().cuda()
    pool, table, _ = fill_cache("e4m3", [200, 90, 64], hk, d, page, g)
    base = torch.tensor([150, 20, 33], device=cuda)
    ang = torch.rand(256, d // 2, generator=g) * 6
    cos, sin = ang.cos().cuda(), ang.sin().cuda()
    qkv = torch.randn(47, (hq + 2 * hk) * d, generator=g).bfloat16().cuda()
    ids, verify = torch.randint(0, 2, (2, 47), generator=g).cuda()

    def run():
        positions, slots, lens, masks = TR.tree_rows(parents, cu, base, table, page, max_rows=30)
        q = K8.rope_kv_append_e4m3(qkv, pool, positions, slots, cos, sin, hq, hk, d, page, q_out=torch.empty(47, hq * d, dtype=torch.bfloat16, device=cuda))
        a = TR.tree_attention(q, pool, table, lens, masks, cu, hq, hk, d, page, max_rows=30)
        b = K8.paged_attention_e4m3(q, pool, table, lens, hq, hk, d, page, cu_q=cu, max_rows=30)
        count, path, emitted = TR.tree_keep(ids, parents, verify, cu, base, table, [pool], hk, d, page, max_rows=30)
        return a, b, count, path, emitted
    return run, pool, (qkv, base)


def test_captured_and_replayed(cuda):
    run, pool, (qkv, base) = calls(cuda, 5)
    start = pool.clone()
    run()                                                  # (the kernels are there)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for shift in (0, 3):                                   # replayed on other numbers: nothing of the first call is kept
        base += shift
        qkv.neg_()
        pool.copy_(start)
        graph.replay()
        got, cache = [x.clone() for x in out], pool.clone()
        pool.copy_(start)
        for x, y in zip(got, run()):
            assert torch.equal(x, y)
        assert torch.equal(cache, pool)


def test_two_streams_at_once(cuda):
    (one, p1, _), (two, p2, _) = calls(cuda, 1), calls(cuda, 2)
    s1, s2 = p1.clone(), p2.clone()
    want = one(), two()
    after = p1.clone(), p2.clone()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        p1.copy_(s1), p2.copy_(s2)
        torch.cuda.synchronize()
        got = []
        for st, f in zip(streams, (one, two)):
            with torch.cuda.stream(st):
                got.append(f())
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
        assert torch.equal(p1, after[0]) and torch.equal(p2, after[1])


def test_two_graphs_with_shares_of_their_own(cuda):
    """Long contexts, whose shares go through a workspace: two captured calls in flight do not meet in it."""
    hq, hk, d, page, l = 8, 2, 128, 64, 30000
    g = torch.Generator().manual_seed(0)
    pool, table, kv = fill_cache("e4m3", [l], hk, d, page, g)
    qs = [torch.randn(1, hq * d, generator=g).bfloat16().cuda() for _ in range(2)]
    f = lambda q: K8.paged_attention_e4m3(q, pool, table, i32l, hq, hk, d, page)
    i32l = i32([l])
    f(qs[0])
    graphs, outs = [], []
    for q in qs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(f(q))
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for q, o in zip(qs, outs):
        ref, spread = attend64(q.cpu().view(1, hq, d), kv[0], torch.ones(1, l, dtype=torch.bool), d ** -0.5)
        close(o.view(1, hq, d), ref, spread, WEIGHT["e4m3"])


def test_a_cache_past_32_bits(cuda):
    hq, hk, d, page = 16, 8, 128, 64
    pages = (1 << 32) // K8.page_bytes(hk, page, d) + 64
    pool = torch.empty(pages, K8.page_bytes(hk, page, d), dtype=torch.uint8, device=cuda)
    g = torch.Generator().manual_seed(0)
    small, _, kv = fill_cache("e4m3", [300], hk, d, page, g, spare=0)
    _, t0, _ = fill_cache("e4m3", [300], hk, d, page, torch.Generator().manual_seed(0), spare=0)
    pool[pages - 5:] = small
    table = t0 + (pages - 5)
    for rows in (1, 100):
        q = torch.randn(rows, hq * d, generator=g).bfloat16().cuda()
        out = K8.paged_attention_e4m3(q, pool, table, i32([300]), hq, hk, d, page, rows_per_seq=rows)
        assert torch.equal(out, K8.paged_attention_e4m3(q, small, t0, i32([300]), hq, hk, d, page, rows_per_seq=rows))
    slots = (table[0, :2].long() * page + 7)
    assert torch.equal(K8.read_rows_e4m3(pool, slots, hk, d, page), K8.read_rows_e4m3(small, slots - (pages - 5) * page, hk, d, page))
    zero = torch.zeros(4, 0, device=cuda)
    qkv = torch.randn(2, (hq + 2 * hk) * d, generator=g).bfloat16().cuda()
    K8.rope_kv_append_e4m3(qkv, pool, slots % 4, slots, zero, zero, hq, hk, d, page, rot=0)
    K8.rope_kv_append_e4m3(qkv, small, slots % 4, slots - (pages - 5) * page, zero, zero, hq, hk, d, page, rot=0)
    assert torch.equal(pool[pages - 5:], small)
    ids = torch.zeros(3, dtype=torch.int64, device=cuda)
    for p, t in ((pool, table), (small, t0)):
        count, _, _ = TR.tree_keep(ids, i32([-1, 0, 0]), torch.tensor([1, 0, 0], device=cuda), i32([0, 3]), torch.tensor([60], device=cuda), t, [p], hk, d, page)
        count2, path, _ = TR.tree_keep(torch.tensor([0, 0, 1], device=cuda), i32([-1, 0, 0]), torch.tensor([1, 0, 0], device=cuda), i32([0, 3]),
                                       torch.tensor([62], device=cuda), t, [p], hk, d, page)
        assert count.tolist() == [1] and count2.tolist() == [2] and path.tolist() == [0, 2, -1]
    assert torch.equal(pool[pages - 5:], small)


def test_pages_slots_and_positions_that_do_not_exist(cuda):
    hq, hk, d, page = 8, 2, 64, 16
    g = torch.Generator().manual_seed(0)
    pool, table, _ = fill_cache("e4m3", [40], hk, d, page, g)
    start = pool.clone()
    err = Kernels.get(cuda)

    def failed(f):
        f()
        with pytest.raises(RuntimeError, match="device error"):
            err.check_error()
    zero, ang = torch.zeros(5, dtype=torch.int64, device=cuda), torch.zeros(9, d // 2, device=cuda)
    qkv = torch.randn(5, (hq + 2 * hk) * d, generator=g).bfloat16().cuda()
    ap = lambda pos, slots: K8.rope_kv_append_e4m3(qkv, pool, pos, slots, ang, ang, hq, hk, d, page)
    far = torch.full((5,), pool.shape[0] * page, device=cuda)
    failed(lambda: ap(zero, far))
    failed(lambda: ap(zero + 9, zero - 1))
    failed(lambda: ap(zero - 1, zero - 1))
    failed(lambda: K8.read_rows_e4m3(pool, far, hk, d, page))
    for bad in (pool.shape[0], -1, 1 << 30):
        wrong = table.clone()
        wrong[0, 1] = bad
        for rows in (1, 40):
            q = torch.randn(rows, hq * d, generator=g).bfloat16().cuda()
            failed(lambda: K8.paged_attention_e4m3(q, pool, wrong, i32([40]), hq, hk, d, page, rows_per_seq=rows))
            failed(lambda: TR.tree_attention(q, pool, wrong, i32([40]), torch.ones(rows, 1, dtype=torch.int64, device=cuda), i32([0, rows]), hq, hk, d, page))
        keep = lambda: TR.tree_keep(zero, i32([-1, 0, 1, 2, 0]), zero, i32([0, 5]), torch.tensor([14], device=cuda), wrong, [pool], hk, d, page)
        failed(lambda: TR.tree_rows(i32([-1, 0, 1, 2, 0]), i32([0, 5]), torch.tensor([14], device=cuda), torch.full_like(wrong[:, :1], bad), page)) if bad == -1 else None
        failed(keep)
    # more tokens than the table has pages for
    q = torch.randn(1, hq * d, generator=g).bfloat16().cuda()
    failed(lambda: K8.paged_attention_e4m3(q, pool, table, i32([999]), hq, hk, d, page))
    assert torch.equal(pool, start)


def test_a_batch_that_is_padded(cuda):
    """Sequences of no context, rows behind the last one: zeros, and left as they were."""
    hq, hk, d, page = 8, 2, 128, 64
    g = torch.Generator().manual_seed(0)
    lens = [0, 130, 0]
    pool, table, kv = fill_cache("e4m3", lens, hk, d, page, g)
    q = torch.randn(8, hq * d, generator=g).bfloat16().cuda()
    for rows in ([2, 1, 1], [2, 4, 0], [0, 0, 0]):
        cu = [0]
        for r in rows:
            cu.append(cu[-1] + r)
        out = torch.full((8, hq * d + 64), 3.0, dtype=torch.bfloat16, device=cuda)[:, : hq * d]
        K8.paged_attention_e4m3(q, pool, table, i32(lens), hq, hk, d, page, cu_q=i32(cu), out=out, max_rows=max(rows))
        assert bool((out[cu[-1]:] == 3).all()) and bool((out[:cu[1]] == 0).all()) and bool((out[cu[2]:cu[3]] == 0).all())
        for i in range(cu[1], cu[2]):
            n = 130 - (cu[2] - 1 - i)
            ref, spread = attend64(q[i:i + 1].cpu().view(1, hq, d), kv[1][:, :n], torch.ones(1, n, dtype=torch.bool), d ** -0.5)
            close(out[i:i + 1].view(1, hq, d), ref, spread, WEIGHT["e4m3"])


@pytest.mark.parametrize("hq,hk,d,page", [(12, 4, 128, 192), (16, 1, 64, 320), (10, 2, 128, 64), (3, 3, 256, 192), (24, 2, 64, 8)])
def test_mixed_calls_of_odd_groups_and_pages(cuda, hq, hk, d, page):
    """Single tokens, short blocks and chunks together, one longer than its context; groups of 3, 16, 5, 1 and 12, pages of 192 and 320."""
    g = torch.Generator().manual_seed(hq)
    rows, lens = [1, 90, 1, 7, 300, 0, 2], [900, 90, 0, 400, 260, 5, 129]
    pool, table, kv = fill_cache("e4m3", lens, hk, d, page, g)
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    q = torch.randn(cu[-1], hq * d, generator=g).bfloat16().cuda()
    out = K8.paged_attention_e4m3(q, pool, table, i32(lens), hq, hk, d, page, cu_q=i32(cu), max_rows=300)
    for s, l in enumerate(lens):
        r = rows[s]
        seen = torch.arange(l)[None] <= (l - r + torch.arange(r))[:, None]
        ref, spread = attend64(q[cu[s]:cu[s + 1]].cpu().view(r, hq, d), kv[s], seen, d ** -0.5)
        close(out[cu[s]:cu[s + 1]].view(r, hq, d), ref, spread, WEIGHT["e4m3"])


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_the_largest_trees(cuda, kind):
    """256 nodes, 4 words; more trees than run at once, of very different lengths."""
    hq, hk, d, page = 16, 8, 64, 16
    g = torch.Generator().manual_seed(4)
    rows = [256, 3, 255, 1] + [40] * 36
    past = [33, 2000, 0, 700] + torch.randint(0, 600, (36,), generator=g).tolist()
    lens = [r + p for r, p in zip(rows, past)]
    pool, table, kv = fill_cache(kind, lens, hk, d, page, g)
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    bits = torch.rand(cu[-1], 256, generator=g) < 0.2
    q = torch.randn(cu[-1], hq * d, generator=g).bfloat16().cuda()
    out = TR.tree_attention(q, pool, table, i32(lens), bits_of(bits).cuda(), i32(cu), hq, hk, d, page, max_rows=256)
    for s in range(0, len(rows), 3):
        r, l = rows[s], lens[s]
        seen = torch.ones(r, l, dtype=torch.bool)
        seen[:, l - r:] = bits[cu[s]:cu[s + 1], :r]
        ref, spread = attend64(q[cu[s]:cu[s + 1]].cpu().view(r, hq, d), kv[s], seen, d ** -0.5)
        close(out[cu[s]:cu[s + 1]].view(r, hq, d), ref, spread, WEIGHT[kind])


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hk,d,seqs,least,most", [(24, 4, 256, 16, 3900, 4000), (24, 4, 256, 60, 1, 900), (8, 4, 128, 16, 2000, 2100), (8, 8, 64, 30, 10, 1500)])
def test_trees_on_long_contexts(cuda, kind, hq, hk, d, seqs, least, most):
    """Many key tiles a block, in one share and in several, every place of the rings used many times."""
    page, nodes = 64, 20
    g = torch.Generator().manual_seed(seqs)
    lens = (torch.randint(least, most, (seqs,), generator=g) + nodes).tolist()
    pool, table, kv = fill_cache(kind, lens, hk, d, page, g)
    cu = [nodes * s for s in range(seqs + 1)]
    bits = torch.rand(cu[-1], nodes, generator=g) < 0.4
    q = torch.randn(cu[-1], hq * d, generator=g).bfloat16().cuda()
    out = TR.tree_attention(q, pool, table, i32(lens), bits_of(bits).cuda(), i32(cu), hq, hk, d, page, max_rows=nodes)
    args = (i32(lens), bits_of(bits).cuda(), i32(cu), hq, hk, d, page)
    cold = torch.empty(200 << 20, dtype=torch.uint8, device=cuda)
    wrong = torch.zeros((), dtype=torch.int64, device=cuda)
    for i in range(150):                                   # from idle, with cold caches, and one behind the other
        if i % 3 == 0:
            cold.fill_(i)
        if i % 3 < 2:
            torch.cuda.synchronize()
        wrong += (TR.tree_attention(q, pool, table, *args, max_rows=nodes) != out).any()
    assert int(wrong) == 0
    for s in range(0, seqs, 5):
        l = lens[s]
        seen = torch.ones(nodes, l, dtype=torch.bool)
        seen[:, l - nodes:] = bits[cu[s]:cu[s + 1]]
        ref, spread = attend64(q[cu[s]:cu[s + 1]].cpu().view(nodes, hq, d), kv[s], seen, d ** -0.5)
        close(out[cu[s]:cu[s + 1]].view(nodes, hq, d), ref, spread, WEIGHT[kind])


@pytest.mark.parametrize("seqs", [90, 200])
def test_more_single_tokens_than_run_at_once(cuda, seqs):
    hq, hk, d, page = 16, 8, 64, 16
    g = torch.Generator().manual_seed(seqs)
    lens = torch.randint(0, 400, (seqs,), generator=g).tolist()
    pool, table, kv = fill_cache("e4m3", lens, hk, d, page, g)
    q = torch.randn(seqs, hq * d, generator=g).bfloat16().cuda()
    out = K8.paged_attention_e4m3(q, pool, table, i32(lens), hq, hk, d, page).view(seqs, 1, hq, d)
    for s, l in enumerate(lens):
        ref, spread = attend64(q[s:s + 1].cpu().view(1, hq, d), kv[s], torch.ones(1, l, dtype=torch.bool), d ** -0.5)
        close(out[s], ref, spread, WEIGHT["e4m3"])


def test_a_wide_table_and_short_contexts(cuda):
    """Contexts far shorter than the table says they may be: shares that nobody has, and a joining launch with nothing to join."""
    hq, hk, d, page = 8, 2, 128, 64
    g = torch.Generator().manual_seed(0)
    lens = [70, 1]
    pool, table, kv = fill_cache("e4m3", lens, hk, d, page, g)
    table = torch.cat([table, torch.zeros(2, 2000, dtype=torch.int32, device=cuda)], 1).contiguous()
    for rows in (1, 60):
        q = torch.randn(2 * rows, hq * d, generator=g).bfloat16().cuda()
        out = K8.paged_attention_e4m3(q, pool, table, i32(lens), hq, hk, d, page, rows_per_seq=rows)
        twice = out + 0                                    # (follows both launches)
        assert torch.equal(twice, out)
        for s, l in enumerate(lens):
            seen = torch.arange(l)[None] <= (l - rows + torch.arange(rows))[:, None]
            ref, spread = attend64(q[s * rows:(s + 1) * rows].cpu().view(rows, hq, d), kv[s], seen, d ** -0.5)
            close(twice[s * rows:(s + 1) * rows].view(rows, hq, d), ref, spread, WEIGHT["e4m3"])


def test_calls_of_nothing(cuda):
    hq, hk, d, page = 8, 2, 64, 16
    pool = K8.new_pool(2, hk, page, d, cuda)
    none, some = torch.zeros(0, dtype=torch.int64, device=cuda), torch.zeros(0, hq * d, dtype=torch.bfloat16, device=cuda)
    tab = torch.zeros(4, d // 2, device=cuda)
    assert K8.rope_kv_append_e4m3(torch.zeros(0, (hq + 2 * hk) * d, dtype=torch.bfloat16, device=cuda), pool, none, none, tab, tab, hq, hk, d, page).shape == (0, hq * d)
    assert K8.read_rows_e4m3(pool, none, hk, d, page).shape == (0, 2, hk, d)
    table = torch.zeros(0, 1, dtype=torch.int32, device=cuda)
    assert K8.paged_attention_e4m3(some, pool, table, i32([]), hq, hk, d, page).shape == (0, hq * d)
    assert TR.tree_attention(some, pool, torch.zeros(1, 1, dtype=torch.int32, device=cuda), i32([3]), torch.zeros(0, 1, dtype=torch.int64, device=cuda),
                             i32([0, 0]), hq, hk, d, page).shape == (0, hq * d)
    for t, base in ((table, none), (torch.zeros(1, 1, dtype=torch.int32, device=cuda), none.new_zeros(1))):
        n = t.shape[0]
        cu = torch.zeros(n + 1, dtype=torch.int32, device=cuda)
        pos, slots, lens, masks = TR.tree_rows(i32([]), cu, base, t, page)
        assert pos.numel() == slots.numel() == masks.numel() == 0 and lens.tolist() == [0] * n
        count, path, emitted = TR.tree_keep(none, i32([]), none, cu, base, t, [pool], hk, d, page)
        assert count.tolist() == [0] * n and path.numel() == emitted.numel() == 0


def test_rows_and_parents_that_do_not_exist(cuda):
    hq, hk, d, page = 8, 2, 64, 16
    g = torch.Generator().manual_seed(0)
    pool, table, _ = fill_cache("e4m3", [40], hk, d, page, g)
    err = Kernels.get(cuda)

    def failed(f):
        out = f()
        with pytest.raises(RuntimeError, match="device error"):
            err.check_error()
        return out
    masks = torch.ones(60, 1, dtype=torch.int64, device=cuda)
    for rows, cu in ((2, [0, 3]), (2, [-1, 1]), (2, [2, 1]), (60, [0, 61]), (60, [-1, 59])):
        q = torch.randn(rows, hq * d, generator=g).bfloat16().cuda()
        out = torch.full_like(q, 3.0)
        if cu[1] >= cu[0]:                                 # (a sequence of less than no rows has none)
            failed(lambda: K8.paged_attention_e4m3(q, pool, table, i32([40]), hq, hk, d, page, cu_q=i32(cu), out=out))
            failed(lambda: TR.tree_attention(q, pool, table, i32([40]), masks, i32(cu), hq, hk, d, page, out=out))
        else:
            K8.paged_attention_e4m3(q, pool, table, i32([40]), hq, hk, d, page, cu_q=i32(cu), out=out)
        assert bool((out == 3).all())
    base, ids = torch.zeros(1, dtype=torch.int64, device=cuda), torch.zeros(4, dtype=torch.int64, device=cuda)
    failed(lambda: TR.tree_rows(i32([-1, 0, 3, 0]), i32([0, 4]), base, table, page))
    failed(lambda: TR.tree_rows(i32([-1, 0, -7, 0]), i32([0, 4]), base, table, page))
    failed(lambda: TR.tree_rows(i32([-1, 0, 0, 0]), i32([0, 5]), base, table, page))
    before = pool.clone()
    failed(lambda: TR.tree_keep(ids, i32([-1, 0, 0, 0]), ids, i32([-2, 2]), base, table, [pool], hk, d, page))
    assert torch.equal(pool, before)


@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (16, 8, 64), (24, 4, 256)])
@pytest.mark.parametrize("rows,seqs,most", [(1, 60, 900), (1, 2, 20000), (3, 20, 3000), (40, 20, 1500), (300, 2, 2500)])
def test_a_call_gives_the_same_bits_each_time(cuda, hq, hk, d, rows, seqs, most):
    """Causal calls of every kernel and way of sharing, from idle with cold caches and one behind the other."""
    page = 64
    g = torch.Generator().manual_seed(rows)
    lens = torch.randint(rows, most, (seqs,), generator=g).tolist()
    pool, table, kv = fill_cache("e4m3", lens, hk, d, page, g)
    q = torch.randn(seqs * rows, hq * d, generator=g).bfloat16().cuda()
    args = (table, i32(lens), hq, hk, d, page)
    out = K8.paged_attention_e4m3(q, pool, *args, rows_per_seq=rows)
    cold = torch.empty(200 << 20, dtype=torch.uint8, device=cuda)
    wrong = torch.zeros((), dtype=torch.int64, device=cuda)
    for i in range(60):
        if i % 3 == 0:
            cold.fill_(i)
        if i % 3 < 2:
            torch.cuda.synchronize()
        wrong += (K8.paged_attention_e4m3(q, pool, *args, rows_per_seq=rows) != out).any()
    assert int(wrong) == 0
    s = seqs - 1
    seen = torch.arange(lens[s])[None] <= (lens[s] - rows + torch.arange(rows))[:, None]
    ref, spread = attend64(q[s * rows:].cpu().view(rows, hq, d), kv[s], seen, d ** -0.5)
    close(out[s * rows:].view(rows, hq, d), ref, spread, WEIGHT["e4m3"])
