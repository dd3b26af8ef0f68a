"""Appends to the 8-bit cache whose calls are padded with thousands of tokens without a slot."""

import pytest
import torch
from test_kv8_gpu import BF16, F32, ops, run_append

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (F32, 64), (BF16, 10)])
@pytest.mark.parametrize("where", ["front", "end", "both", "inside", "far", "all"])
def test_long_stretches_without_slots(cuda, where, dtype, hd):
    """In front, behind, between tokens of one block, and where the nearest stored token lies just in or just out
    of what is looked at together (32 tokens, 256 tokens)."""
    T = 3400

    def poke(qkv, slots, total):
        first = int(slots[0])
        if where in ("front", "both"):
            slots[: T - 40] = -1
        if where in ("end", "both"):
            slots[T - 37 :] = -1
        if where == "end":
            slots[5 : T - 37] = -1
        if where == "inside":  # one block, its runs thousands of tokens apart
            slots[:] = -1
            slots[2:6] = first + torch.arange(4)
            slots[T - 9 : T - 5] = first + 4 + torch.arange(4)
        if where == "far":
            own = slots.clone()
            slots[:] = -1
            at = 0
            for i, gap in enumerate((0, 30, 31, 32, 33, 223, 224, 255, 256, 257, 300, 511, 512, 513)):
                at += gap + 1
                slots[at - 1] = own[i] if i < 11 else own[16 * (i - 10)]
        if where == "all":
            slots[:] = -1

    run_append(cuda, dtype, [T], [0], 2, 1, hd, 16, seed=930, poke=poke)
    ops().check_device_errors(cuda)


def test_padding_costs_no_more_than_tokens(cuda):
    """A call of 60000 rows of which one is a token, against one of as many tokens: it does far less work, and has to
    look at as many slots.  (Looked at one after the other they took hundreds of times as long.)"""
    T, H, D, bs = 60000, 2, 64, 16
    nb = T // bs + 1
    kc, vc = (torch.zeros(1, nb, bs, H, D, dtype=torch.float8_e4m3fn, device=cuda) for _ in range(2))
    ks, vs = (torch.zeros(1, nb, H, device=cuda) for _ in range(2))
    x = torch.randn(T, H, D, device=cuda).to(BF16)
    dense = torch.arange(T, device=cuda)
    times = []
    for slots in (dense, dense.masked_fill(dense != 0, -1), dense.masked_fill(dense != T - 1, -1)):
        best = float("inf")
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(4):
                ops().write_kv8(x, x, kc, vc, ks, vs, 0, slots)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b) / 4)
        times.append(best)
    assert max(times[1:]) <= 10 * times[0] + 0.2, times
