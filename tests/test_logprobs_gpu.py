"""token_logprobs on the GPU against 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def ops():
    from nano_infer_engine_b200 import ops as _ops

    return _ops


def check(logits, tokens, top):
    """The sums are fp32 over at most V terms: a term is off by 2^-22 (exp), the sum of n terms in
    any order by less than log2-many roundings plus V / 512 sequential ones; x - m and log Z are one
    rounding each of values below 2^8."""
    got = ops().token_logprobs(logits, tokens, top=top)
    x = logits.double()
    R, V = x.shape
    lp = torch.log_softmax(x, dim=1)
    p = lp.exp()
    h = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
    rel = 2.0**-21 + (V / 512 + 20) * 2.0**-24
    spread = (x.amax(1) - torch.where(x.isinf(), x.amax(1, keepdim=True), x).amin(1)).clamp(min=1)
    want = lp.gather(1, tokens[:, None])[:, 0]
    fine = want.isfinite()
    assert torch.equal(got.logprobs.isneginf(), want.isneginf())
    assert ((got.logprobs.double() - want).abs()[fine] <= rel + 2.0**-22 * (want.abs()[fine] + 16)).all()
    assert ((got.entropy.double() - h).abs() <= 2 * rel * (1 + h + spread) + 2.0**-22 * 16).all()
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(got.top_ids, ids)
    t = lp.gather(1, ids)
    ok = t.isfinite()
    assert ((got.top_logprobs.double() - t).abs()[ok] <= rel + 2.0**-22 * (t.abs()[ok] + 16)).all()
    assert torch.equal(got.top_logprobs.isneginf(), t.isneginf())
    assert got.logprobs.dtype == got.entropy.dtype == got.top_logprobs.dtype == F32
    ops().check_device_errors(logits.device)
    return got


SHAPES = [(1, 1, 1), (1, 2, 2), (3, 7, 7), (5, 31, 20), (2, 128256, 20), (130, 1000, 5), (1, 50257, 32), (9, 4097, 1), (4, 33, 0),
          (700, 515, 3), (2, 300001, 8)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_logprobs_match_64_bits(cuda, shape, dtype):
    R, V, top = shape
    g = torch.Generator(device=cuda).manual_seed(R * 7 + V)
    x = (torch.randn(R, V, device=cuda, generator=g) * 4).to(dtype)
    check(x, torch.randint(0, V, (R,), device=cuda, generator=g), top)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_ties_go_to_the_lowest_index(cuda, dtype):
    x = torch.zeros(3, 5000, dtype=dtype, device=cuda)
    x[1, ::3] = 2.0
    x[2] = torch.randint(0, 3, (5000,), device=cuda).to(dtype)
    x[2, 17] = -0.0
    check(x, torch.tensor([0, 4, 4999], device=cuda), 32)


@pytest.mark.parametrize("order", ["up", "down", "late"])
def test_sorted_rows(cuda, order):
    """Rows in which the largest come last, first, or all in the last stretch."""
    V = 60000
    x = torch.arange(V, device=cuda).float()[None].repeat(2, 1) / V * 20
    if order == "down":
        x = x.flip(1).contiguous()
    if order == "late":
        x[:, :-40] = -5.0
    check(x, torch.tensor([5, V - 1], device=cuda), 32)


def test_forbidden_tokens(cuda):
    x = torch.randn(4, 3000, device=cuda).to(BF16)
    x[0, 1:] = float("-inf")  # one token left
    x[1, 10:] = float("-inf")  # fewer left than alternatives asked for
    x[2, ::2] = float("-inf")
    x[3, :2990] = float("-inf")
    got = check(x, torch.tensor([0, 11, 3, 2999], device=cuda), 20)
    assert got.logprobs[0] == 0 and got.entropy[0] == 0


def test_rows_without_a_distribution(cuda):
    x = torch.randn(5, 700, device=cuda)
    x[0] = float("-inf")
    x[1, 300] = float("nan")
    x[2, 5] = float("inf")
    x[4, 600] = float("nan")
    x[4, 100] = float("inf")
    got = ops().token_logprobs(x, torch.tensor([1, 2, 3, 4, 5], device=cuda), top=2)
    assert got.logprobs.isnan().tolist() == [True, True, True, False, True]
    assert got.entropy.isnan().tolist() == [True, True, True, False, True]
    assert got.top_logprobs.isnan().all(1).tolist() == [True, True, True, False, True]
    assert got.top_ids[0].tolist() == [0, 1] and got.top_ids[1, 0] == 300 and got.top_ids[2, 0] == 5
    assert got.top_ids[4].tolist() == [600, 100]


def test_wide_values(cuda):
    x = torch.randn(3, 2000, device=cuda)
    x[0] *= 1e30
    x[1] += 1e6
    x[2] -= 1e30
    got = ops().token_logprobs(x, x.argmax(1), top=3)
    assert got.logprobs.isfinite().all() and got.entropy.isfinite().all()
    assert got.logprobs[0] == 0 and got.entropy[0] == 0


def test_strided_rows_and_missing_tokens(cuda):
    base = torch.randn(6, 4001, device=cuda).to(BF16)
    x = base[:, 3:2004]  # rows that start at odd places
    check(x, torch.arange(6, device=cuda), 4)
    check(base[::2, :4000], torch.arange(3, device=cuda), 4)
    got = ops().token_logprobs(x, torch.tensor([0, -1, 2001, 2000, 1, 1], device=cuda), top=1)
    assert got.logprobs.isnan().tolist() == [False, True, True, False, False, False]
    assert got.entropy.isfinite().all()
    with pytest.raises(RuntimeError, match="token id outside the vocabulary"):
        ops().check_device_errors(cuda)


def test_no_rows(cuda):
    got = ops().token_logprobs(torch.empty(0, 50, device=cuda), torch.empty(0, dtype=torch.int64, device=cuda), top=3)
    assert got.logprobs.shape == (0,) and got.top_ids.shape == (0, 3)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_masks_of_the_lowest_value(cuda, dtype):
    """Rows masked by the type's lowest value, wholly and in part, some with -inf beside it."""
    low = torch.finfo(dtype).min
    x = torch.full((5, 3001), low, dtype=dtype, device=cuda)
    x[1, 7] = 3.0
    x[2, ::2] = float("-inf")
    x[3, 5:] = float("-inf")
    x[4, 2000:] = 1.0
    check(x, torch.tensor([3, 7, 11, 4, 2999], device=cuda), 8)
