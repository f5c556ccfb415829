"""The 8-bit cache without a GPU: its quantisation and its refusals, and the decoders that keep one on the host-memory executor."""
import dataclasses

import pytest
import torch

from kern_b200.cpu import CpuRuntime
from kern_b200.engine import Engine
from kern_b200.models import dense, dense_dcp, dense_tp, moe, registry, spec
from kern_b200.ops import kv_e4m3 as K8
from kern_b200.ops import tree as TR
from kern_b200.runtime import verify


def test_quantisation_is_within_half_a_step_and_exact_in_bf16():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(500, 64, generator=g) * torch.exp2(torch.randint(-30, 30, (500, 1), generator=g).float())
    x[3] = 0
    codes, scales = K8.quantise_reference(x)
    back = K8.dequantise_reference(codes, scales)
    assert torch.equal(back.bfloat16().float(), back)
    e = scales.int() - 127
    assert int(e[3]) == -40 and bool(((x.abs().amax(-1) <= 448 * torch.exp2(e.float())) | (e == -40)).all())
    # half a step: 2^-4 of the value, or half of the smallest code under the scale
    assert bool(((back - x).abs() <= 2.0 ** -4 * x.abs() + 2.0 ** -10 * torch.exp2(e.float())[:, None]).all())


def test_quantisation_of_what_is_not_finite():
    x = torch.ones(2, 64)
    x[0, 3], x[1, 5] = float("inf"), float("nan")
    codes, scales = K8.quantise_reference(x)
    assert torch.equal(torch.isnan(codes.float()).nonzero(), torch.tensor([[0, 3], [1, 5]])) and scales.tolist() == [119, 119]


class Calls:
    """Valid calls on CPU tensors: what is left to refuse is the device."""

    hq, hk, d, page = 4, 2, 64, 16

    def __init__(self):
        self.pool = K8.new_pool(3, self.hk, self.page, self.d, "cpu")
        self.i = torch.zeros(5, dtype=torch.int64)
        self.tab = torch.zeros(9, 32)
        self.qkv = torch.zeros(5, 8 * 64, dtype=torch.bfloat16)
        self.table = torch.zeros(2, 3, dtype=torch.int32)
        self.lens = torch.zeros(2, dtype=torch.int32)
        self.cu = torch.tensor([0, 2, 5], dtype=torch.int32)
        self.masks = torch.zeros(5, 1, dtype=torch.int64)
        self.q = torch.zeros(5, 4 * 64, dtype=torch.bfloat16)
        self.parents = torch.zeros(5, dtype=torch.int32)

    def append(self, **k):
        a = dict(qkv=self.qkv, pool=self.pool, positions=self.i, slots=self.i, cos=self.tab, sin=self.tab, hq=self.hq, hk=self.hk, d=self.d, page_size=self.page)
        return K8.rope_kv_append_e4m3(**{**a, **k})

    def read(self, **k):
        return K8.read_rows_e4m3(**{**dict(pool=self.pool, slots=self.i, hk=self.hk, d=self.d, page_size=self.page), **k})

    def attend(self, **k):
        a = dict(q=self.q, pool=self.pool, block_table=self.table, seq_lens=self.lens, hq=self.hq, hk=self.hk, d=self.d, page_size=self.page, cu_q=self.cu)
        return K8.paged_attention_e4m3(**{**a, **k})

    def tree(self, **k):
        a = dict(q=self.q, pool=self.pool, block_table=self.table, seq_lens=self.lens, masks=self.masks, cu_q=self.cu, hq=self.hq, hk=self.hk, d=self.d, page_size=self.page)
        return TR.tree_attention(**{**a, **k})

    def rows(self, **k):
        return TR.tree_rows(**{**dict(parents=self.parents, cu=self.cu, base=self.i, block_table=self.table, page_size=self.page), **k})

    def keep(self, **k):
        a = dict(ids=self.i, parents=self.parents, verify=self.i, cu=self.cu, base=self.i, block_table=self.table, pools=[self.pool], hk=self.hk, d=self.d, page_size=self.page)
        return TR.tree_keep(**{**a, **k})


C = Calls()
BF = torch.zeros(3, 2, 2, 16, 64, dtype=torch.bfloat16)
REFUSED = [
    ("append", dict(), "CUDA device"), ("append", dict(hq=3), "whole group"), ("append", dict(d=96), "head_dim"), ("append", dict(page_size=24), "page_size"),
    ("append", dict(pool=C.pool[:, :-1]), "8-bit pool"), ("append", dict(pool=BF), "8-bit pool"), ("append", dict(rot=24), "rot"), ("append", dict(rot=80), "rot"),
    ("append", dict(rot=32), "tables"), ("append", dict(pairs="thirds"), "interleaved"), ("append", dict(positions=C.i[:4]), "positions"),
    ("append", dict(slots=C.i.int()), "slots"), ("append", dict(sin=C.tab[:8]), "same positions"), ("append", dict(cos=C.tab[:, ::2]), "tables"),
    ("append", dict(q_norm=torch.ones(64)), "q_norm"), ("append", dict(tokens=6), "tokens"), ("append", dict(qkv=C.qkv[:, :500]), "qkv"),
    ("append", dict(qkv=C.qkv.float()), "qkv"), ("append", dict(qkv=torch.zeros(5, 519, dtype=torch.bfloat16)), "16 bytes"),
    ("append", dict(q_out=C.q[:4]), "q_out"), ("append", dict(qkv=torch.zeros(5, 1024, dtype=torch.bfloat16)[:, ::2]), "neighbours"),
    ("append", dict(qkv=torch.zeros(5, 528, dtype=torch.bfloat16)[:, 1:513]), "16 bytes"),
    ("read", dict(), "CUDA device"), ("read", dict(slots=C.i.view(5, 1)), "slots"), ("read", dict(out=torch.zeros(5, 2, 2, 32, dtype=torch.bfloat16)), "out"),
    ("attend", dict(), "CUDA device"), ("attend", dict(pool=BF), "8-bit pool"), ("attend", dict(seq_lens=C.lens.long()), "seq_lens"), ("attend", dict(cu_q=C.cu[:2]), "cu_q"),
    ("attend", dict(cu_q=None, rows_per_seq=3), "rows_per_seq"), ("attend", dict(max_rows=6), "max_rows"), ("attend", dict(scale=0.0), "scale"),
    ("attend", dict(scale=float("nan")), "scale"), ("attend", dict(max_len=-1), "max_len"), ("attend", dict(block_table=C.table.t()), "block_table"),
    ("attend", dict(block_table=C.table[:, :0]), "a page to a row"), ("attend", dict(out=C.q[:3]), "out"), ("attend", dict(hq=64, hk=2), "group of at most 16"),
    ("tree", dict(), "CUDA device"), ("tree", dict(pool=BF), "CUDA device"), ("tree", dict(pool=BF.permute(0, 1, 3, 2, 4)), "bf16 pool"), ("tree", dict(pool=BF.half()), "bf16 pool"),
    ("tree", dict(masks=C.masks[:4]), "masks"), ("tree", dict(masks=torch.zeros(5, 5, dtype=torch.int64)), "masks"), ("tree", dict(cu_q=None), "cu_q"),
    ("rows", dict(), "CUDA device"), ("rows", dict(parents=C.parents.long()), "parents"), ("rows", dict(base=C.lens), "base"), ("rows", dict(max_rows=257), "at most 256"),
    ("rows", dict(page_size=0), "page_size"), ("keep", dict(), "CUDA device"), ("keep", dict(ids=C.i[:4]), "ids"), ("keep", dict(pools=[C.pool, BF]), "alike"),
    ("keep", dict(pools=[C.pool, C.pool]), "once"), ("keep", dict(pools=[BF] * 129), "at most 128"), ("keep", dict(pools=[BF[:, :1]]), "bf16 pool"),
]


@pytest.mark.parametrize("call,changed,why", REFUSED, ids=[f"{c}-{i}" for i, (c, _, _) in enumerate(REFUSED)])
def test_refusals(call, changed, why):
    with pytest.raises(ValueError, match=why):
        getattr(C, call)(**changed)


@pytest.mark.parametrize("qk_norm", [False, True])
def test_dense_decoder_with_an_8_bit_cache(qk_norm):
    cfg = dataclasses.replace(dense.TOY, kv="e4m3", qk_norm=qk_norm)
    doc = dense.build_manifest(cfg)
    m, errs = verify(doc)
    assert m is not None, errs[:5]
    assert doc["states"]["kv.l0"]["bytes_per_token"] == 2 * cfg.kv_heads * (cfg.head_dim + 1)
    w = dense.random_weights(cfg, seed=0, std=0.08)
    rt = CpuRuntime(doc, weights=w, tokens=cfg.page_size * 16)
    rt.once()
    eng, oracle = Engine(rt), dense.DenseOracle(cfg, w)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in (21, 1, 9)]
    seqs, caches = [eng.open(len(p) + 8) for p in prompts], [oracle.new_cache() for _ in prompts]
    feeds = prompts
    for _ in range(4):
        got = eng.step(list(zip(seqs, feeds)))
        logits = rt.tensor("logits")[:3].float()
        for f, c, lg in zip(feeds, caches, logits):
            ref = oracle.forward(f, c)[-1]
            # the bf16 rounding before the cache (2^-9 of a value, in the mean) takes one code in 50 to its neighbour, some 9 % away:
            # 0.09 / sqrt(50) = 1.3 % of the keys' and values' norm, and as much again for bf16 elsewhere
            assert float((lg - ref).norm() / ref.norm()) < 0.05
        feeds = [[t[0]] for t in got]


def test_what_an_8_bit_cache_does_not_go_with():
    cfg = dataclasses.replace(dense.TINY, kv="e4m3")
    for call in (lambda: spec.build_manifest(cfg), lambda: dense_dcp.build_manifest_dcp(cfg, 2), lambda: dense.build_manifest(cfg, hosted=True),
                 lambda: dense_tp.build_manifest_tp(dataclasses.replace(cfg, tp=2)), lambda: dense.build_manifest(dataclasses.replace(cfg, kv="int3"))):
        with pytest.raises(ValueError, match="e4m3"):
            call()


def test_families_take_the_cache_as_an_option():
    for name in ("tiny", "tiny-moe"):
        cfg, build, _, _ = registry.resolve(name, kv="e4m3")
        doc = build(cfg)
        entries = {l["entry"] for op in doc["ops"].values() for l in op["impl"]["launches"] if "entry" in l}
        assert any(e.startswith("kern_attn_tile_e4m3_causal") for e in entries) and any(e.startswith("kern_rope_kv_append_e4m3") for e in entries)
        assert not any("attn_decode_paged" in e for e in entries)
        assert "attn_paged" not in doc["modules"] and "attn_rows" in doc["modules"]
