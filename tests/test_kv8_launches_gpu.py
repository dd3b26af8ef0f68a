"""The package's count of launches of the 8-bit attention where the fast kernels do not take a call."""

import pytest
import torch
from test_kv8_gpu import BF16, F16, ops, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("new", [None, [40] * 6])
def test_a_call_that_falls_to_the_generic_kernel_is_one_launch(cuda, new, dtype):
    from nano_infer_engine_b200 import ops as module

    R = 6
    q, (kc, vc, ks, vs), tables, sl, _ = run_attention(cuda, dtype, [9000] * R, new, 8, 2, 64, 16, seed=810)
    qsl = torch.tensor([0] + (new or [])).cumsum(0).to(cuda)
    flat = torch.zeros(q.shape[0], 8 * 64 + 3, dtype=dtype, device=cuda)
    odd = flat.as_strided(q.shape, (8 * 64 + 3, 64, 1), 1)
    odd.copy_(q)
    counts = []
    for x in (q, odd):
        before = module.LAUNCHES
        if new is None:
            ops().paged_decode_kv8(x, kc, vc, ks, vs, 1, tables, sl)
        else:
            ops().varlen_attention_kv8(x, kc, vc, ks, vs, 1, tables, sl, qsl, 40)
        counts.append(module.LAUNCHES - before)
    ops().check_device_errors(cuda)
    assert counts == [2, 1]
