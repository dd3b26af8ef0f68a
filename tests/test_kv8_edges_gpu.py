"""The 8-bit paged cache's operators where calls rarely go: NaN behind the mask, more requests than one
launch takes, captured graphs, other streams, tensors that the fast paths refuse, lists with bad entries."""

from __future__ import annotations

import kv8_plain as plain
import pytest
import torch
from test_kv8_gpu import BF16, F16, ops, run_append, run_attention, step
from test_logprobs_gpu import check as check_logprobs

pytestmark = pytest.mark.gpu


def close(got, want, dtype, slack=0.0):
    """Two results of one formula: each is off by half a step of the type and by 2^-11 of the weights' mass
    sum p |v| (kv8_plain.attention), which is 1.3 on average here and below 4 where a few keys share the weight
    (a single key's is exact): 2 * 2^-11 * 4 = 2^-8."""
    err = (got.double() - want.double()).abs()
    return bool((err <= 2 * step(dtype) * want.double().abs() + 2.0**-8 + slack).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hd,bs", [(64, 16), (128, 32)])
@pytest.mark.parametrize("ctx,new", [(0, 200), (150, 40), (37, 3), (3000, 260)])
def test_a_nan_reaches_the_rows_that_see_it_alone(cuda, dtype, hd, bs, ctx, new):
    n = ctx + new
    hkv, hq = 2, 8
    q, (kc, vc, ks, vs), tables, sl, clean = run_attention(cuda, dtype, [n], [new], hq, hkv, hd, bs, seed=400 + ctx)
    qsl = torch.tensor([0, new], device=cuda)
    clean = clean.clone()
    # V: one code of the last token, one of a token in the middle of the new ones, of different heads
    for pos, head, dim in ((n - 1, 0, 5), (ctx + new // 2, 1, hd - 1)):
        v = vc.clone()
        v.view(torch.uint8)[1, tables[0, pos // bs].long(), pos % bs, head, dim] = 0xFF if dim == 5 else 0x7F
        got = ops().varlen_attention_kv8(q, kc, v, ks, vs, 1, tables, sl, qsl, new)
        ops().check_device_errors(cuda)
        bad = torch.zeros(new, hq, hd, dtype=torch.bool, device=cuda)
        bad[pos - ctx :, head * 4 : head * 4 + 4, dim] = True
        assert torch.equal(got[:new].isnan(), bad), (pos, head)
        assert torch.equal(got[:new][~bad], clean[:new][~bad])
    # K: the score is NaN, and with it the row
    k = kc.clone()
    k.view(torch.uint8)[1, tables[0, (n - 1) // bs].long(), (n - 1) % bs, 0, 3] = 0x7F
    got = ops().varlen_attention_kv8(q, k, vc, ks, vs, 1, tables, sl, qsl, new)
    bad = torch.zeros(new, hq, hd, dtype=torch.bool, device=cuda)
    bad[new - 1, :4] = True
    assert torch.equal(got[:new].isnan(), bad)
    assert torch.equal(got[:new][~bad], clean[:new][~bad])


@pytest.mark.parametrize("lists", [False, True])
def test_decode_of_more_requests_than_a_launch_takes(cuda, lists):
    """1100 requests: three rounds, the last one short; as they come, and by lists."""
    R, hq, hkv, hd, bs = 1100, 4, 2, 64, 16
    lens = [(7 * i) % 90 for i in range(R)]
    for width in (6, 80):  # tables of few keys (one launch a round) and of more
        q, (kc, vc, ks, vs), tables, sl, want = run_attention(cuda, BF16, lens, None, hq, hkv, hd, bs, seed=500)
        tables = torch.nn.functional.pad(tables, (0, max(0, width - tables.shape[1])))
        if not lists:
            got = ops().paged_decode_kv8(q, kc, vc, ks, vs, 1, tables, sl)
            assert close(got[:R], want[:R], BF16)
            continue
        g = torch.Generator().manual_seed(1)
        order = torch.randperm(R, generator=g).to(cuda)
        shuffled = torch.empty_like(tables)
        shuffled[order] = tables
        got = ops().paged_decode_kv8(q[order.argsort()], kc, vc, ks, vs, 1, shuffled, sl, table_rows=order.int(),
                                     q_rows=order, req_list=torch.randperm(R, generator=g).int().to(cuda))
        assert close(got[order], want[:R], BF16)
    ops().check_device_errors(cuda)


@pytest.mark.parametrize("lists", [False, True])
def test_ragged_queries_of_more_requests_than_a_launch_takes(cuda, lists):
    R = 600
    new = [1 + i % 3 for i in range(R)]
    lens = [n + (5 * i) % 40 for i, n in enumerate(new)]
    q, (kc, vc, ks, vs), tables, sl, want = run_attention(cuda, F16, lens, new, 4, 2, 64, 16, seed=510)
    if lists:
        qsl = torch.tensor([0] + new).cumsum(0).to(cuda)
        pick = torch.randperm(R, generator=torch.Generator().manual_seed(2)).int().to(cuda)
        got = ops().varlen_attention_kv8(q, kc, vc, ks, vs, 1, tables, sl, qsl, 3, req_list=pick,
                                         table_rows=torch.arange(R, dtype=torch.int32, device=cuda))
        assert close(got[: sum(new)], want[: sum(new)], F16)
        ops().check_device_errors(cuda)


@pytest.mark.parametrize("new", [None, [20, 3]])
def test_lists_with_bad_entries(cuda, new):
    """A request or a table row that does not exist is flagged and passed over; the others have their answers."""
    q, (kc, vc, ks, vs), tables, sl, want = run_attention(cuda, BF16, [300, 77], new, 8, 2, 64, 16, seed=520)
    call = ops().paged_decode_kv8
    args = (q, kc, vc, ks, vs, 1, tables, sl)
    if new:
        call = ops().varlen_attention_kv8
        args += (torch.tensor([0, 20, 23], device=cuda), 20)
    rows = slice(20, 23) if new else slice(1, 2)
    for kw in (dict(req_list=torch.tensor([5, 1, -1], dtype=torch.int32, device=cuda)),
               dict(table_rows=torch.tensor([2, 1], dtype=torch.int32, device=cuda)),
               dict(table_rows=torch.tensor([-1, 1], dtype=torch.int32, device=cuda))):
        out = torch.full_like(q, 3.0)
        call(*args, out=out, **kw)
        with pytest.raises(RuntimeError):
            ops().check_device_errors(cuda)
        assert close(out[rows], want[rows], BF16)
        assert (out[: rows.start] == 3.0).all() and (out[rows.stop :] == 3.0).all()


@pytest.mark.parametrize("new", [None, [33, 5]])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_queries_that_are_not_aligned(cuda, new, dtype):
    """Rows that begin between the boundaries of wide loads, in and out."""
    q, (kc, vc, ks, vs), tables, sl, want = run_attention(cuda, dtype, [300, 77], new, 8, 2, 64, 16, seed=530)
    T = q.shape[0]
    for shift, width in ((1, 8 * 64 + 1), (2, 8 * 64 + 2), (0, 8 * 64 + 3)):
        flat = torch.zeros(T, width + shift, dtype=dtype, device=cuda)
        odd = flat.as_strided((T, 8, 64), (width + shift, 64, 1), shift)
        odd.copy_(q)
        out = torch.zeros_like(flat).as_strided((T, 8, 64), (width + shift, 64, 1), shift)
        if new is None:
            ops().paged_decode_kv8(odd, kc, vc, ks, vs, 1, tables, sl, out=out)
        else:
            ops().varlen_attention_kv8(odd, kc, vc, ks, vs, 1, tables, sl, torch.tensor([0, 33, 38], device=cuda), 33, out=out)
        n = 2 if new is None else 38
        assert close(out[:n], want[:n], dtype)
    ops().check_device_errors(cuda)


def test_two_graphs_and_two_streams(cuda):
    """Captured calls have workspaces of their own: graphs replayed on two streams at once, in any order, with
    inputs changed between replays, and eager calls beside them."""
    sets = []
    for seed in (540, 541):
        q, cache, tables, sl, _ = run_attention(cuda, BF16, [900, 2000], None, 8, 2, 64, 16, seed=seed)
        logits = torch.randn(3, 5000, device=cuda)
        tok = torch.tensor([1, 2, 3], device=cuda)
        sets.append((q, cache, tables, sl, logits, tok))

    def run(x):
        q, (kc, vc, ks, vs), tables, sl, logits, tok = x
        qsl = torch.tensor([0, 1, 2], device=cuda) if not torch.cuda.is_current_stream_capturing() else x_qsl
        a = ops().paged_decode_kv8(q, kc, vc, ks, vs, 1, tables, sl)
        b = ops().varlen_attention_kv8(q, kc, vc, ks, vs, 1, tables, sl, qsl, 1)
        k, v = ops().gather_kv8(kc, vc, ks, vs, 1, tables[0], 900)
        r = ops().token_logprobs(logits, tok, top=4)
        return a[:2], b[:2], k, v, r.logprobs, r.entropy, r.top_logprobs

    x_qsl = torch.tensor([0, 1, 2], device=cuda)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for x, s in zip(sets, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run(x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(run(x))
        graphs.append(g)
    for turn in range(6):
        for x in sets:
            x[0].mul_(0.9)
            x[4].add_(0.1 * x[4].roll(1, 1))
        torch.cuda.synchronize()
        for i in ((0, 1) if turn % 2 else (1, 0)):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        eager = [tuple(y.clone() for y in run(x)) for x in sets]
        torch.cuda.synchronize()
        for got, want in zip(outs, eager):
            for a, b in zip(got, want):
                assert torch.equal(a, b)
    ops().check_device_errors(cuda)


def test_a_cache_whose_offsets_pass_31_and_32_bits(cuda):
    """A cache of 5 GiB: blocks behind 2^32 bytes of codes in a layer, written, read and attended."""
    hkv, hd, bs = 8, 64, 16
    nb = (1 << 32) // (bs * hkv * hd) + 64
    kc = torch.empty(1, nb, bs, hkv, hd, dtype=torch.float8_e4m3fn, device=cuda)
    vc = torch.empty_like(kc)
    ks, vs = torch.zeros(1, nb, hkv, device=cuda), torch.zeros(1, nb, hkv, device=cuda)
    # the same tokens in low blocks and in high ones
    n = 100
    low = torch.tensor([3, 9, 4, 1, 0, 7, 8], dtype=torch.int32, device=cuda)
    high = torch.tensor([nb - 1, nb - 20, nb - 3, nb // 2 + 1, nb // 2, nb - 5, nb - 6], dtype=torch.int32, device=cuda)
    keys, values = torch.randn(n, hkv, hd, device=cuda).to(BF16), torch.randn(n, hkv, hd, device=cuda).to(BF16)
    pos = torch.arange(n, device=cuda)
    for table in (low, high):
        slots = table[pos // bs].long() * bs + pos % bs
        ops().write_kv8(keys, values, kc, vc, ks, vs, 0, slots)
    q = torch.randn(5, 32, hd, device=cuda).to(BF16)
    sl = torch.tensor([n], dtype=torch.int32, device=cuda)
    results = []
    for table in (low, high):
        k, v = ops().gather_kv8(kc, vc, ks, vs, 0, table, n)
        d = ops().paged_decode_kv8(q[:1], kc, vc, ks, vs, 0, table[None], sl)
        p = ops().varlen_attention_kv8(q, kc, vc, ks, vs, 0, table[None], sl, torch.tensor([0, 5], device=cuda), 5)
        results.append((k, v, d, p))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    ops().check_device_errors(cuda)


SHORT = [
    # lens, new, hq, hkv, hd, bs: few tokens to a request, at and around what one warp and the short form take
    ([2000, 2004, 5, 1], [5, 1, 5, 1], 32, 8, 64, 16),
    ([700, 16, 33], [16, 16, 2], 32, 8, 64, 16),  # 64 columns
    ([700, 17, 33], [17, 17, 2], 32, 8, 64, 16),  # one token more
    ([900, 8, 64], [8, 8, 3], 16, 4, 128, 32),
    ([900, 9, 64], [9, 9, 3], 16, 4, 128, 32),
    ([3, 0, 2, 100], [4, 2, 3, 0], 8, 2, 64, 16),  # more tokens than keys; no key; no token
    ([5000], [3], 6, 2, 128, 16),
    ([1100, 40], [7, 3], 5, 5, 64, 32),  # an odd number of column sets
    ([1100, 40], [5, 3], 24, 1, 64, 16),  # a wide group: past the short form
    ([260] * 70, [1 + i % 4 for i in range(70)], 16, 4, 64, 16),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", range(len(SHORT)))
def test_requests_of_a_few_tokens(cuda, case, dtype):
    run_attention(cuda, dtype, *SHORT[case], seed=600 + case)


def test_a_request_longer_than_the_call_says(cuda):
    q, (kc, vc, ks, vs), tables, sl, want = run_attention(cuda, BF16, [300, 77], [6, 2], 8, 2, 64, 16, seed=640)
    out = torch.full_like(q, 3.0)
    ops().varlen_attention_kv8(q, kc, vc, ks, vs, 1, tables, sl, torch.tensor([0, 6, 8], device=cuda), 2, out=out)
    with pytest.raises(RuntimeError):
        ops().check_device_errors(cuda)
    assert (out[:6] == 3.0).all() and close(out[6:8], want[6:8], BF16)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("new", [None, [5, 9], [40, 70]])
@pytest.mark.parametrize("length", [2**31 - 1, 2**31 - 70, 321])
def test_a_length_past_the_table(cuda, new, length, dtype):
    """Keys without a place in the table are flagged; those before them, and other requests, have their weight."""
    lens = [320, 77]
    q, (kc, vc, ks, vs), tables, sl, want = run_attention(cuda, dtype, lens, new, 8, 2, 64, 16, seed=700)
    tables = tables[:, :20].contiguous()  # 320 keys
    counts = new or [1, 1]
    bad = torch.tensor([length, 77], dtype=torch.int32, device=cuda)
    out = torch.zeros_like(q)
    if new is None:
        ops().paged_decode_kv8(q, kc, vc, ks, vs, 1, tables, bad, out=out)
    else:
        qsl = torch.tensor([0] + new).cumsum(0).to(cuda)
        ops().varlen_attention_kv8(q, kc, vc, ks, vs, 1, tables, bad, qsl, max(new), out=out)
    with pytest.raises(RuntimeError, match="block id outside the pool"):
        ops().check_device_errors(cuda)
    c, T = counts[0], sum(counts)
    assert close(out[c:T], want[c:T], dtype)
    seen = [min(320, length - c + 1 + j) for j in range(c)]
    for j in {0, c // 2, c - 1}:
        w, bound = plain.attention(q[j : j + 1], kc[1], vc[1], ks[1], vs[1], tables[0], seen[j], seen[j], 64**-0.5)
        assert ((out[j].double() - w[0]).abs() <= step(dtype) * (w[0].abs() + bound[0]) + bound[0] + 1e-30).all()


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_launches_are_counted(cuda, dtype):
    """The count that the package keeps, against the profiler's."""
    from nano_infer_engine_b200 import ops as module

    cases = [([100], None, 64), ([1500] * 3, None, 64), ([5000] * 40, None, 64), ([30] * 600, None, 128),
             ([2000] * 8, [5] * 8, 64), ([5000] * 40, [3] * 40, 64), ([300] * 3, [100] * 3, 128), ([40] * 300, [33] * 300, 64)]
    for lens, new, hd in cases:
        q, (kc, vc, ks, vs), tables, sl, _ = run_attention(cuda, dtype, lens, new, 8, 2, hd, 16, seed=800)
        qsl = torch.tensor([0] + (new or [])).cumsum(0).to(cuda)

        def call():
            if new is None:
                module.paged_decode_kv8(q, kc, vc, ks, vs, 1, tables, sl)
            else:
                module.varlen_attention_kv8(q, kc, vc, ks, vs, 1, tables, sl, qsl, max(new))

        before = module.LAUNCHES
        call()
        counted = module.LAUNCHES - before
        torch.cuda.synchronize()
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
            call()
            torch.cuda.synchronize()
        if not prof.key_averages():
            pytest.skip("the profiler sees no kernels here")
        seen = sum(e.count for e in prof.key_averages() if "kv8" in e.key)
        assert counted == seen, (lens[0], len(lens), new and new[0], hd)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_append_of_thousands_of_tokens(cuda, dtype):
    """More than 4096: prompts that begin anywhere in a block, one of a single token, an infinite value in between."""
    run_append(cuda, dtype, [3000, 1, 1203, 77], [5, 16, 31, 0], 4, 1, 64, 16, seed=900)

    def poke(qkv, slots, total):
        qkv[2000, ::7] = float("inf")
        qkv[4100, ::5] = float("nan")
        slots[700:703] = -1

    run_append(cuda, dtype, [4000, 300], [5, 3], 2, 2, 64, 32, seed=901, poke=poke)


def test_append_of_thousands_of_requests(cuda):
    """A token each, 600 and 4200 of them: every one in a block of its own, some where the block begins."""
    for n in (600, 4200):
        run_append(cuda, BF16, [1] * n, [i % 19 for i in range(n)], 2, 1, 64, 16, seed=910)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_logprobs_of_rows_split_in_two_and_four(cuda, dtype):
    for rows, vocab in ((100, 40001), (60, 40001), (149, 40001)):
        g = torch.Generator(device=cuda).manual_seed(rows)
        x = (torch.randn(rows, vocab, device=cuda, generator=g) * 4).to(dtype)
        x[3] = float("-inf")
        x[3, 39000] = 1.0
        check_logprobs(x, torch.randint(0, vocab, (rows,), device=cuda, generator=g), 7)
