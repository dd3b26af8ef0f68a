"""A prefill pool and a decode pool of which one is in 8 bits: no request could be handed over, so no pair is made."""

from types import SimpleNamespace

import pytest
import torch

from nano_infer_engine_b200.generation.pd_handoff import PDPair
from nano_infer_engine_b200.paged_cache import PagedKVCache

BF16, F8 = torch.bfloat16, torch.float8_e4m3fn


def model():
    return SimpleNamespace(embed=SimpleNamespace(weight=torch.zeros(4, 8, dtype=BF16)), decoders=[None],
                           config=SimpleNamespace(kv_head_num=2, head_dim=64))


def pool(dtype):
    return PagedKVCache(4, 16, 1, 2, 64, dtype, "cpu")


def test_pools_are_both_in_8_bits_or_neither():
    for dtype in (BF16, F8):
        PDPair.checked(model(), model(), pool(dtype), pool(dtype))
    for a, b in ((BF16, F8), (F8, BF16)):
        with pytest.raises(ValueError, match="both be 8-bit caches or neither"):
            PDPair.checked(model(), model(), pool(a), pool(b))
