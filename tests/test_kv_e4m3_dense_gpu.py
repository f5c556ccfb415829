"""The dense decoder with an 8-bit cache, manifest to engine, against its fp32 oracle (sm_100a)."""
import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,hk,d,qk_norm", [(4, 2, 64, False), (8, 1, 128, True), (2, 1, 256, False)])
def test_dense_decoder_with_an_8_bit_cache(cuda, tmp_path, heads, hk, d, qk_norm):
    from kern_b200.engine import Engine
    from kern_b200.models import common, dense
    from kern_b200.runtime import Runtime, verify

    cfg = dataclasses.replace(dense.TINY, kv="e4m3", heads=heads, kv_heads=hk, head_dim=d, qk_norm=qk_norm, max_context=512, max_tokens=512)
    w = dense.random_weights(cfg, seed=0, std=0.05)
    common.write_safetensors(tmp_path / "model.safetensors", w)
    doc = dense.build_manifest(cfg)
    m, errs = verify(doc)
    assert m is not None, errs[:5]
    rt = Runtime(doc, weights=tmp_path / "model.safetensors", tokens=cfg.page_size * 64)
    rt.once()
    eng, oracle = Engine(rt), dense.DenseOracle(cfg, w, device="cuda")
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in (300, 1, 37)]
    seqs, caches = [eng.open(len(p) + 8) for p in prompts], [oracle.new_cache() for _ in prompts]
    feeds = prompts
    for step in range(5):
        if step == 3:
            feeds[1] = torch.randint(0, cfg.vocab, (7,), generator=g).tolist()      # a chunk among single tokens
        got = eng.step(list(zip(seqs, feeds)))
        logits = rt.tensor("logits")[:3].float()
        for f, c, lg in zip(feeds, caches, logits):
            ref = oracle.forward(f, c)[-1]
            # as on the host: 1.3 % for codes that bf16 takes to their neighbours, as much for bf16 elsewhere
            assert float((lg - ref).norm() / ref.norm()) < 0.05
        feeds = [[t[0]] for t in got]
    rt.check_error()
