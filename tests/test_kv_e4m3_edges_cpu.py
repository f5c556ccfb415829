"""The 8-bit cache without a GPU: values, arguments and builds at their ends."""
import dataclasses
import subprocess
import sys
import types

import pytest
import torch

from kern_b200 import _build, cpu
from kern_b200.models import dense, moe, registry
from kern_b200.ops import host, launcher
from kern_b200.ops import kv_e4m3 as K8
from kern_b200.ops import tree as TR


def test_the_largest_bf16_values_keep_their_sign_and_size():
    """The format ends at 448 * 2^119: what is past it, and finite, becomes that."""
    top = float(torch.finfo(torch.bfloat16).max)
    x = torch.tensor([[top, -top, 2.9e38, 1.0] * 16])
    codes, scales = K8.quantise_reference(x)
    back = K8.dequantise_reference(codes, scales)[0]
    end = 448 * 2.0 ** 119
    assert scales.tolist() == [246] and back[:4].tolist() == [end, -end, end, 0.0]


def test_a_table_whose_contexts_pass_32_bits_is_refused():
    hq, hk, d, page = 4, 2, 64, 1 << 20
    pool = torch.zeros(1, K8.page_bytes(hk, page, d), dtype=torch.uint8)
    q, lens = torch.zeros(1, hq * d, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    for pages, why in ((2048, "32 bits"), (2047, "CUDA device")):
        with pytest.raises(ValueError, match=why):
            K8.paged_attention_e4m3(q, pool, torch.zeros(1, pages, dtype=torch.int32), lens, hq, hk, d, page)


@pytest.mark.parametrize("scale,why", [(1e-39, "f32 holds"), (1e-300, "f32 holds"), (3e38, "f32 holds"), (float("inf"), "f32 holds"), (-1.0, "f32 holds"),
                                       (1e-37, "CUDA device"), (2e38, "CUDA device")])
def test_scales_that_f32_does_not_hold(scale, why):
    """A scale of 0 in f32 would make NaN of scores that are not seen."""
    hq, hk, d, page = 4, 2, 64, 16
    pool, q = K8.new_pool(2, hk, page, d, "cpu"), torch.zeros(3, hq * d, dtype=torch.bfloat16)
    table, lens, cu = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32)
    with pytest.raises(ValueError, match=why):
        K8.paged_attention_e4m3(q, pool, table, lens, hq, hk, d, page, rows_per_seq=3, scale=scale)
    with pytest.raises(ValueError, match=why):
        TR.tree_attention(q, pool, table, lens, torch.zeros(3, 1, dtype=torch.int64), cu, hq, hk, d, page, scale=scale)


def test_only_attention_limits_the_group():
    """32 query heads over one kv head: written and read back as any (what is left to refuse is the device), attended by neither form."""
    hq, hk, d, page = 32, 1, 64, 16
    pool, i64 = K8.new_pool(2, hk, page, d, "cpu"), torch.zeros(3, dtype=torch.int64)
    qkv, tab = torch.zeros(3, (hq + 2 * hk) * d, dtype=torch.bfloat16), torch.zeros(9, d // 2)
    with pytest.raises(ValueError, match="CUDA device"):
        K8.rope_kv_append_e4m3(qkv, pool, i64, i64, tab, tab, hq, hk, d, page)
    with pytest.raises(ValueError, match="group of at most 16"):
        K8.paged_attention_e4m3(qkv[:, : hq * d], pool, torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), hq, hk, d, page)


@pytest.mark.parametrize("change,why", [(dict(heads=32, kv_heads=1), "group of at most 16"), (dict(page_size=48), "page_size 48"), (dict(page_size=96), "page_size 96"),
                                        (dict(page_size=4), "page_size 4"), (dict(head_dim=96), "head_dim 96"), (dict(heads=3), "whole group")])
def test_decoders_whose_layout_the_cache_does_not_have(change, why):
    cfg = dataclasses.replace(dense.TINY, kv="e4m3", **change)
    with pytest.raises(ValueError, match=why):
        dense.build_manifest(cfg)
    with pytest.raises(ValueError, match=why):
        moe.build_manifest(dataclasses.replace(moe.TINY_MOE, kv="e4m3", **change))


@pytest.mark.parametrize("page", [8, 32, 64, 192])
def test_decoders_whose_layout_it_has(page):
    assert dense.build_manifest(dataclasses.replace(dense.TINY, kv="e4m3", page_size=page))["states"]


@pytest.mark.parametrize("name", ["tiny-hybrid", "tiny-latent", "tiny-gafapel", "toy-int"])
def test_families_that_have_no_such_option(name, tmp_path):
    known = registry.families()
    name = next(n for n in known if n.startswith(name))
    for kv in ("e4m3", "bf16"):
        with pytest.raises(ValueError, match="cache of its own"):
            registry.resolve(name, kv=kv)
    assert registry.resolve(name, kv=None)
    (tmp_path / "config.json").write_text("{}")
    with pytest.raises(ValueError, match="cache of its own"):
        registry.resolve(str(tmp_path), kv="e4m3")


def test_the_host_statement_shows_nan_where_it_is_seen():
    """A NaN among the keys, or the values, reaches the rows that see it and no others, as on the device; a row that sees nothing is zeros."""
    hq, hk, d, page, rows = 2, 1, 16, 8, 5
    g = torch.Generator().manual_seed(0)
    for which, tokens in (("keys", 6), ("values", 6), ("none", 3)):
        kv = torch.randn(8, 2, hk, d, generator=g)
        if which != "none":
            kv[4, int(which == "values"), 0, 7] = float("nan")
        codes, scales = K8.quantise_reference(kv)
        pool = torch.cat([codes.view(torch.uint8).permute(1, 2, 0, 3).reshape(-1), scales.permute(1, 2, 0).reshape(-1)])
        q, out = torch.randn(rows * hq * d, generator=g).bfloat16(), torch.zeros(rows * hq * d, dtype=torch.bfloat16)
        shape = types.SimpleNamespace(_head_dim=d, _vars_seqs=1)
        cpu.CPU_KERNELS[f"kern_attn_tile_e4m3_causal_d{d}"](
            (1,), shape, q, out, 0, 0, pool, torch.zeros(1, dtype=torch.int32), torch.tensor([tokens], dtype=torch.int32), 0, 0, 0, rows, hq, hk, hq * d, hq * d, 1, page,
            1, 1, 1, rows, rows, rows, 0, 0.25 * 1.4426950408889634, torch.zeros(1, dtype=torch.int32))
        nan = torch.isnan(out.view(rows, hq, d))
        if which == "none":                                # (5 rows on 3 tokens: the first two see none)
            assert not bool(nan.any()) and bool((out.view(rows, -1)[:2] == 0).all()) and bool((out.view(rows, -1)[2:] != 0).any())
            continue
        first = 4 - (tokens - rows)                        # the row that token 4 belongs to
        assert not bool(nan[:first].any())
        assert bool(nan[first:].all()) if which == "keys" else bool(nan[first:, :, 7].all()) and int(nan.sum()) == (rows - first) * hq


# ---- what hangs on the host side's library ---------------------------------------------------------------------------------------
def test_other_operators_do_without_the_host_library():
    """Everything that was there before it imports and runs where it does not load; the operators that need it say so."""
    code = """
import sys
import kern_b200
sys.modules["kern_b200._ops_host"] = None
import torch
from kern_b200.ops import attention, basic, draft, gdn, gemm, gemm_fp8, gemm_mx, launcher, mla, moe, spec
from kern_b200 import cpu, engine, runtime
from kern_b200.models import dense
assert dense.build_manifest(dense.TOY)["programs"]
from kern_b200.ops import kv_e4m3, tree
codes, _ = kv_e4m3.quantise_reference(torch.ones(1, 64))
for call in (lambda: kv_e4m3.read_rows_e4m3(None, None, 2, 64, 16), lambda: tree.tree_rows(None, None, None, None, 16)):
    try:
        call()
    except RuntimeError as e:
        assert "_ops_host" in str(e) and "python -m kern_b200._build" in str(e), e
    else:
        raise SystemExit("no error")
print("fine")
"""
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "fine" in p.stdout, p.stderr[-2000:]


def test_a_library_built_for_another_pytorch_is_refused(monkeypatch):
    monkeypatch.setattr(host, "_ops", None)
    monkeypatch.setitem(sys.modules, "kern_b200._ops_host", types.SimpleNamespace(torch_version="1.0.0", on_missing=lambda f: None))
    with pytest.raises(RuntimeError, match="built for PyTorch 1.0.0"):
        host.ops()


@pytest.fixture
def a_build(monkeypatch, tmp_path):
    """`build_ops_host` on a tree of its own, its compiler replaced: (calls, settings)"""
    (tmp_path / "csrc" / "bindings" / "torch").mkdir(parents=True)
    (tmp_path / "csrc" / "bindings" / "torch" / "ops_host.cpp").write_text("")
    (tmp_path / "build").mkdir()
    calls, here = [], dict(version="2.0.0+cu", cuda=True, fails=False)

    def compiled(src, out):
        calls.append(here["version"])
        if here["fails"]:
            raise RuntimeError("no such function")
        out.write_text(here["version"])
    for name, value in (("PKG", tmp_path), ("CSRC", tmp_path / "csrc"), ("BUILD", tmp_path / "build"), ("_compile_ops_host", compiled),
                        ("_torch_here", lambda: (here["version"], here["cuda"]))):
        monkeypatch.setattr(_build, name, value)
    return calls, here


def test_the_library_is_built_again_for_another_pytorch(a_build):
    calls, here = a_build
    assert _build.build_ops_host().exists()
    _build.build_ops_host()
    assert calls == ["2.0.0+cu"]
    here["version"] = "2.1.0+cu"
    _build.build_ops_host(needed=False)
    _build.build_ops_host()
    assert calls == ["2.0.0+cu", "2.1.0+cu"]
    _build.ops_host_path().unlink()
    _build.build_ops_host()
    assert len(calls) == 3


def test_an_import_survives_a_library_that_cannot_be_built(a_build):
    calls, here = a_build
    here["fails"] = True
    with pytest.warns(UserWarning, match="no operators over 8-bit caches"):
        assert _build.build_ops_host(needed=False) is None
    _build.build_ops_host(needed=False)                    # (the same sources: not tried at every import)
    assert len(calls) == 1
    with pytest.raises(RuntimeError, match="no such function"):
        _build.build_ops_host()
    here.update(fails=False, cuda=False)                   # a PyTorch without CUDA has no use for it
    assert _build.build_ops_host() is None and len(calls) == 2


def test_the_pytorch_that_is_here():
    version, cuda = _build._torch_here()
    assert version == torch.__version__ and cuda == (torch.version.cuda is not None)


def test_the_count_of_launches_can_be_set(monkeypatch):
    """As it could before part of it was counted elsewhere."""
    k = object.__new__(launcher.Kernels)
    k.gpu, k._launches = 0, 5
    monkeypatch.setattr(host, "_ops", types.SimpleNamespace(launches=lambda gpu: 7))
    assert k.launches == 12
    k.launches = 0
    k._launches += 2
    assert k.launches == 2
