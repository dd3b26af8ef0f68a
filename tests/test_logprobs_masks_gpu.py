"""token_logprobs of rows that a mask leaves a handful of tokens: their answers, and that they cost what others do."""

import pytest
import torch
from test_logprobs_gpu import BF16, F16, F32, check, ops

pytestmark = pytest.mark.gpu


def masked(cuda, rows, vocab, allowed, dtype, fill, seed, where="anywhere"):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = torch.full((rows, vocab), fill, dtype=dtype, device=cuda)
    keep = torch.rand(rows, vocab, device=cuda, generator=g)
    if where == "together":
        keep = (torch.arange(vocab, device=cuda)[None] - torch.randint(0, vocab - allowed, (rows, 1), device=cuda, generator=g)) % vocab
        keep = -keep.float()
    ids = keep.topk(allowed, dim=1).indices
    x.scatter_(1, ids, (torch.randn(rows, allowed, device=cuda, generator=g) * 4).to(dtype))
    return x, ids[:, 0].clone()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("allowed", [1, 3, 10, 50, 1000])
@pytest.mark.parametrize("where", ["anywhere", "together"])
def test_few_tokens_left(cuda, where, allowed, dtype):
    for rows, vocab, top in ((1, 128256, 5), (40, 50257, 20), (200, 9001, 32), (3, 1001, 3)):
        x, tokens = masked(cuda, rows, vocab, allowed, dtype, float("-inf"), allowed + rows, where)
        check(x, tokens, top)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("allowed", [1, 4, 30])
def test_few_tokens_above_the_lowest_value(cuda, allowed, dtype):
    """Masked by the type's lowest value, by values below what the maxima know (f16 has none), by those and -inf."""
    low = torch.finfo(dtype).min
    for fill in (low, low / 2 if dtype != F16 else low):
        x, tokens = masked(cuda, 30, 50257, allowed, dtype, fill, allowed)
        check(x, tokens, 20)
        x[:, ::3] = torch.where(x[:, ::3] == fill, float("-inf"), x[:, ::3])
        check(x, tokens, 20)
        x[:, 17:-1000] = torch.where(x[:, 17:-1000] == fill, float("-inf"), x[:, 17:-1000])
        check(x, tokens, 20)


def test_sparse_masks_cost_no_more_than_none(cuda):
    """The same bytes and fewer candidates.  (Rows gone through again take three times as long and more.)"""
    for rows, top in ((1, 5), (333, 5), (333, 20)):
        times = []
        for allowed in (None, 1, 10, 100, 1000):
            if allowed is None:
                x, t = torch.randn(rows, 128256, device=cuda).to(BF16), torch.zeros(rows, dtype=torch.int64, device=cuda)
            else:
                x, t = masked(cuda, rows, 128256, allowed, BF16, float("-inf"), allowed)
            graph = torch.cuda.CUDAGraph()
            ops().token_logprobs(x, t, top=top)
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                for _ in range(4):
                    ops().token_logprobs(x, t, top=top)
            best = float("inf")
            for _ in range(6):
                a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
                a.record()
                graph.replay()
                b.record()
                torch.cuda.synchronize()
                best = min(best, a.elapsed_time(b) / 4)
            times.append(best)
        assert max(times[1:]) <= 1.6 * times[0], (rows, top, times)
        print(rows, top, [round(t * 1e3, 1) for t in times])
