"""The 8-bit cache without a GPU: values, arguments and builds at their ends."""
import pytest
import torch

from kern_b200.ops import kv_e4m3 as K8


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
