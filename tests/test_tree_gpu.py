"""Places and masks of drafted trees, the walk, the moved cache rows, and a whole round (sm_100a)."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

from kern_b200.ops import kv_e4m3 as K8
from kern_b200.ops import tree as TR
from kern_b200.ops.launcher import Kernels


@pytest.fixture(autouse=True)
def _no_device_error(cuda):
    yield
    Kernels.get(cuda).check_error()


def trees(rng, sizes, chain=False):
    return [[-1] + [i - 1 if chain else max(0, i - 1 - int(rng.expovariate(0.5))) for i in range(1, n)] if n else [] for n in sizes]


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cu_of(sizes):
    out = [0]
    for n in sizes:
        out.append(out[-1] + n)
    return out


@pytest.mark.parametrize("sizes,chain,words", [([1], False, 1), ([7, 0, 64, 3], False, 1), ([256, 65, 128, 2], False, 4), ([256, 200], True, 4), ([33, 70], True, 2)])
def test_rows(cuda, sizes, chain, words):
    rng = random.Random(len(sizes))
    page, par = 16, trees(rng, sizes, chain)
    base = [rng.randint(0, 100) for _ in sizes]
    if len(sizes) > 2:
        base[0] = -1                                       # a padding sequence
    table = torch.stack([torch.randperm(32) + 40 * s for s in range(len(sizes))]).int().cuda()
    flat = [p for t in par for p in t] + [-1, -1, -1]      # three nodes behind the last sequence
    cu = cu_of(sizes)
    pos, slots, lens, masks = TR.tree_rows(i32(flat), i32(cu), torch.tensor(base, device=cuda), table, page, max_rows=max(sizes))
    assert masks.shape == (len(flat), words)
    for s, p in enumerate(par):
        live = base[s] >= 0
        assert int(lens[s]) == (base[s] + len(p) if live else 0)
        depth, mask = TR.tree_masks_reference(p)
        for i in range(len(p)):
            at = cu[s] + i
            place = base[s] + i
            assert int(pos[at]) == (base[s] + depth[i] if live else 0)
            assert int(slots[at]) == (int(table[s, place // page]) * page + place % page if live else -1)
            assert sum((int(w) & (1 << 64) - 1) << 64 * k for k, w in enumerate(masks[at])) == (mask[i] if live else 0)
    assert bool((slots[cu[-1]:] == -1).all()) and bool((masks[cu[-1]:] == 0).all()) and bool((pos[cu[-1]:] == 0).all())


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("hk,d,page,sizes,chain,layers", [(2, 64, 16, [1, 9, 0, 40], False, 3), (8, 128, 64, [256, 64, 12], False, 2),
                                                          (1, 256, 8, [100, 30], True, 1), (3, 128, 128, [5], False, 0)])
def test_keep(cuda, kind, hk, d, page, sizes, chain, layers):
    rng = random.Random(7)
    par = trees(rng, sizes, chain)
    cu = cu_of(sizes)
    base = [rng.randint(0, 50) for _ in sizes]
    if len(sizes) > 3:
        base[1] = -1
    ids, verify = [], []
    for p in par:
        v = [rng.randint(0, 5) for _ in p]
        ids.append([v[q] if q >= 0 and rng.random() < 0.75 else rng.randint(0, 5) for q in p])
        verify.append(v)
    width = -(-(60 + max(sizes)) // page)
    pages = width * len(sizes) + 1
    table = torch.randperm(pages)[: width * len(sizes)].view(len(sizes), width).int()
    rows = 2 * hk * page
    if kind == "bf16":
        pools = [torch.randn(pages, 2, hk, page, d).bfloat16().cuda() for _ in range(layers)]
    else:
        pools = [torch.randint(0, 256, (pages, rows * (d + 1)), dtype=torch.uint8).cuda() for _ in range(layers)]
    before = [p.cpu().clone() for p in pools]
    flat = lambda x, dt: torch.tensor([v for t in x for v in t] + [3], dtype=dt, device=cuda)
    count, path, emitted = TR.tree_keep(flat(ids, torch.int64), flat(par, torch.int32), flat(verify, torch.int64), i32(cu),
                                        torch.tensor(base, device=cuda), table.cuda(), pools, hk, d, page)
    longest = 0
    for s, p in enumerate(par):
        want = TR.walk_reference(ids[s], p, verify[s]) if base[s] >= 0 else []
        longest = max(longest, len(want))
        n = len(want)
        assert int(count[s]) == n and path[cu[s]:cu[s + 1]].tolist() == want + [-1] * (len(p) - n)
        assert emitted[cu[s]:cu[s + 1]].tolist() == [verify[s][i] for i in want] + [0] * (len(p) - n)
        slot = lambda place: (int(table[s, place // page]), place % page)
        for b in before:
            old = b.clone()
            for i, node in enumerate(want):
                (dp, do), (sp, so) = slot(base[s] + i), slot(base[s] + node)
                if kind == "bf16":
                    b[dp, :, :, do] = old[sp, :, :, so]
                else:
                    for x, y in zip(K8.views(b.view(pages, -1), hk, page, d), K8.views(old, hk, page, d)):
                        x.view(torch.uint8)[dp, :, :, do] = y.view(torch.uint8)[sp, :, :, so]
    assert longest > 2 and int(path[cu[-1]]) == -1
    for p, b in zip(pools, before):
        assert torch.equal(p.cpu().view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("kind", ["e4m3", "bf16"])
def test_a_round(cuda, kind):
    """The operators as a round runs them: a tree's nodes placed, rotated and written, attended to, walked and moved; afterwards
    the cache is what writing the agreed tokens one after the other leaves, and each node's attention what they get that way."""
    from kern_b200.ops import attention as A

    hq, hk, d, page = 8, 2, 128, 16
    rng = random.Random(3)
    g = torch.Generator().manual_seed(3)
    base, sizes = [37, 0, 130], [20, 12, 31]
    par, cu = trees(rng, sizes), cu_of(sizes)
    table = torch.randperm(60)[:36].view(3, 12).int().cuda()
    cos, sin = A.rope_tables(256, d, 1e4, cuda)
    pool = K8.new_pool(60, hk, page, d, cuda) if kind == "e4m3" else torch.zeros(60, 2, hk, page, d, dtype=torch.bfloat16, device=cuda)

    def append(qkv, p, positions, slots):
        if kind == "e4m3":
            return K8.rope_kv_append_e4m3(qkv, p, positions, slots, cos, sin, hq, hk, d, page)
        A.rope_kv_append(qkv, p, positions, slots, cos, sin, hq, hk, d)
        return qkv[:, : hq * d]

    row = lambda n: torch.randn(n, (hq + 2 * hk) * d, generator=g).bfloat16().cuda()
    for s, b in enumerate(base):                           # what the sequences have
        at = torch.arange(b, device=cuda)
        if b:
            append(row(b), pool, at, table[s].long()[at // page] * page + at % page)
    start = pool.clone()
    parents, cu_d, base_d = i32([p for t in par for p in t]), i32(cu), torch.tensor(base, device=cuda)
    positions, slots, lens, masks = TR.tree_rows(parents, cu_d, base_d, table, page)
    nodes = row(cu[-1])
    kept = nodes.clone()
    q = append(nodes, pool, positions, slots)
    out = TR.tree_attention(q, pool, table, lens, masks, cu_d, hq, hk, d, page, max_rows=31)
    verify = torch.randint(0, 3, (cu[-1],), generator=g).cuda()
    ids = torch.randint(0, 3, (cu[-1],), generator=g).cuda()
    count, path, emitted = TR.tree_keep(ids, parents, verify, cu_d, base_d, table, [pool], hk, d, page)
    assert int(count.max()) > 2
    for s, b in enumerate(base):
        n = int(count[s])
        walk = path[cu[s]:cu[s] + n].long() + cu[s]
        at = b + torch.arange(n, device=cuda)
        q1 = append(kept[walk].contiguous(), start, at, table[s].long()[at // page] * page + at % page)
        assert torch.equal(q1, q[walk])
        one = (K8.paged_attention_e4m3 if kind == "e4m3" else lambda *a, **k: A.paged_attention(a[0], a[1], a[2], a[3], hq, **k))(
            q1.contiguous(), start, table[s:s + 1].contiguous(), i32([b + n]), hq, hk, d, page, rows_per_seq=n)
        # two roundings of bf16 between the two: 2^-7 of the value, and of the weights' spread
        torch.testing.assert_close(out[walk].float(), one.float(), rtol=2 ** -7, atol=2 ** -7)
        place = torch.arange(b + n, device=cuda)
        sl = table[s].long()[place // page] * page + place % page
        read = lambda p: K8.read_rows_e4m3(p, sl, hk, d, page) if kind == "e4m3" else p[sl // page, :, :, sl % page]
        assert torch.equal(read(pool), read(start))
