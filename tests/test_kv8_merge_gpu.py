"""Decode over the 8-bit cache on tables too wide for a cluster to a request, by batch sizes that merge differently."""

import pytest
import torch
from test_kv8_gpu import BF16, F16, ops, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hd,hkv", [(64, 8), (128, 4)])
@pytest.mark.parametrize("R", [1, 3, 8, 17, 40])
def test_few_and_many_requests_on_wide_tables(cuda, R, hd, hkv, dtype):
    lens = [9000 if i == 0 else (997 * i) % 5000 for i in range(R)]
    q, (kc, vc, ks, vs), tables, sl, want = run_attention(cuda, dtype, lens, None, 32, hkv, hd, 16, seed=960 + R)
    got = ops().paged_decode_kv8(q, kc, vc, ks, vs, 1, tables, sl)
    assert torch.equal(got[:R], want[:R])  # and the same bits again


@pytest.mark.parametrize("R", [1, 5, 12])
def test_drafts_on_wide_tables(cuda, R):
    new = [4 - i % 3 for i in range(R)]
    lens = [9000 if i == 0 else (997 * i) % 5000 + 4 for i in range(R)]
    run_attention(cuda, BF16, lens, new, 32, 8, 64, 16, seed=980 + R)
