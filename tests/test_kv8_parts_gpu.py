"""Ragged attention where a processor's row tiles are nearly empty and full in turn."""

import pytest
import torch
from test_kv8_gpu import BF16, F16, ops, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hd", [64, 128])
def test_parts_without_rows_before_parts_with_rows(cuda, hd, dtype):
    """Requests of 25 tokens (100 rows: the other parts of their tile have none, for 30 key tiles) before requests
    of 200, whose parts' first factors, and the NaN of V that are kept out of the products, are the right tiles'."""
    R, G = 40, 4
    new = [25 if i % 2 == 0 else 200 for i in range(2 * R)]
    lens = [1900 + i if i % 2 == 0 else 200 + 7 * i for i in range(2 * R)]
    q, (kc, vc, ks, vs), tables, sl, clean = run_attention(cuda, dtype, lens, new, 8, 2, hd, 16, seed=950 + hd)
    starts = torch.tensor([0] + new).cumsum(0)
    T = int(starts[-1])
    bad = torch.zeros(T, 8, hd, dtype=torch.bool, device=cuda)
    v = vc.clone()
    for i in range(1, 2 * R, 6):
        at = 90 + i  # of the request's new tokens
        pos, head, dim = lens[i] - 200 + at, i % 2, i % hd
        v.view(torch.uint8)[1, tables[i, pos // 16].long(), pos % 16, head, dim] = 0x7F
        bad[int(starts[i]) + at : int(starts[i + 1]), head * G : head * G + G, dim] = True
    clean = clean.clone()
    for _ in range(3):
        got = ops().varlen_attention_kv8(q, kc, v, ks, vs, 1, tables, sl, starts.to(cuda), 200)
        assert torch.equal(got[:T].isnan(), bad)
        assert torch.equal(got[:T][~bad], clean[:T][~bad])
    ops().check_device_errors(cuda)
