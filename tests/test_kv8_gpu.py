"""The 8-bit paged cache on the GPU: appending, reading back and attention against plain 64-bit forms."""

import pytest
import torch

import kv8_plain as plain

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def ops():
    from nano_infer_engine_b200 import ops as _ops

    return _ops


def step(dtype):
    return torch.finfo(dtype).eps / 2  # a rounding is off by at most half a step


# ------------------------------------------------------------------ append
def run_append(cuda, dtype, new, old, hq, hkv, hd, bs, seed, poke=None, layers=2, layer=1):
    """One rope_write_kv8 call over requests with `old` cached and `new` fresh tokens; checks all of it."""
    g = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in zip(old, new)]
    nb = sum(-(-n // bs) for n in lens) + 3
    tables = plain.make_tables(lens, bs, nb, seed)
    T = sum(new)
    pos = torch.cat([torch.arange(a, a + b) for a, b in zip(old, new)])
    row = torch.cat([torch.full((b,), i) for i, b in enumerate(new)])
    slots = tables[row, pos // bs].long() * bs + pos % bs
    width = (hq + 2 * hkv) * hd
    qkv = (torch.randn(T, width + 8, generator=g) * torch.exp(torch.randn(T, 1, generator=g))).to(dtype)
    angle = pos[:, None].double() * 10000.0 ** (-torch.arange(hd // 2).double() / (hd // 2))
    sin, cos = angle.sin().to(dtype), angle.cos().to(dtype)
    codes = [plain.to_e4m3(torch.randn(layers, nb, bs, hkv, hd, generator=g) * 100) for _ in range(2)]
    scales = [torch.randint(-12, -5, (layers, nb, hkv), generator=g).float().exp2() for _ in range(2)]
    if poke is not None:
        poke(qkv, slots, nb * bs)
    q, k, v = qkv[:, : hq * hd], qkv[:, hq * hd : (hq + hkv) * hd], qkv[:, (hq + hkv) * hd : width]
    dev = qkv.to(cuda)
    dc, ds = [c.to(cuda) for c in codes], [s.to(cuda) for s in scales]
    got_q = ops().rope_write_kv8(dev[:, : hq * hd], dev[:, hq * hd : (hq + hkv) * hd], dev[:, (hq + hkv) * hd : width],
                                 sin.to(cuda), cos.to(cuda), dc[0], dc[1], ds[0], ds[1], layer, slots.to(cuda), hq)
    # queries: one rounding of the fp32 rotation, itself within three roundings of products of size |a| + |b|
    q64 = q.reshape(T, hq, hd).double()
    want = plain.rotate(q64, sin, cos)
    size = q64.abs() + q64.abs().roll(hd // 2, dims=-1)
    fine = want.abs() <= torch.finfo(dtype).max  # a rotated value past the type's largest is infinite
    slack = step(dtype) * want.abs() + 3 * 2.0**-24 * size + torch.finfo(dtype).tiny
    assert ((got_q.cpu().double() - want).abs() <= slack)[fine].all()
    # codes and scales: the same fp32 values, so bit for bit
    plain.append(plain.rotate(k.reshape(T, hkv, hd).float(), sin, cos), codes[0][layer], scales[0][layer], slots.tolist())
    plain.append(v.reshape(T, hkv, hd).float(), codes[1][layer], scales[1][layer], slots.tolist())
    for a, b in zip(dc, codes):
        x, y = a.cpu().float(), b.float()
        assert torch.equal(x.isnan(), y.isnan())
        assert torch.equal(x.nan_to_num(0.0), y.nan_to_num(0.0))
    for a, b in zip(ds, scales):
        assert torch.equal(a.cpu(), b)
    return dc, ds, tables, lens


APPENDS = [
    # new, old, hq, hkv, hd, bs
    ([1], [0], 32, 8, 64, 16),
    ([1], [15], 32, 8, 64, 16),  # the last place of a block
    ([1], [16], 32, 8, 64, 16),  # the first place of the next
    ([1] * 9, [3, 16, 47, 0, 31, 32, 5, 100, 15], 8, 2, 64, 16),
    ([70, 1, 33, 16], [5, 9, 0, 16], 32, 8, 64, 16),
    ([100, 3], [7, 30], 16, 4, 128, 32),
    ([300], [0], 4, 4, 64, 16),
    ([2100, 50], [9, 3], 8, 1, 64, 16),  # many tokens
    ([41, 2], [3, 8], 6, 3, 96, 8),
    ([10, 3], [2, 6], 2, 1, 10, 5),  # nothing aligned
    ([40], [100], 2, 2, 128, 128),
    ([5], [3], 2, 1, 256, 1),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_stores_codes_and_scales(cuda, case, dtype):
    new, old, hq, hkv, hd, bs = APPENDS[case]
    run_append(cuda, dtype, new, old, hq, hkv, hd, bs, seed=case)
    ops().check_device_errors(cuda)


def test_append_values_are_within_half_a_step(cuda):
    """Read back: within 2^-4 of the value (its 8-bit form's half step) or half the least step of the block."""
    g = torch.Generator().manual_seed(3)
    T, H, D, bs = 37, 4, 64, 16
    x = torch.randn(T, H, D, generator=g).to(BF16)
    y = (torch.randn(T, H, D, generator=g) * 1e-3).to(BF16)
    nb = 4
    kc, vc = (torch.zeros(1, nb, bs, H, D, dtype=torch.float8_e4m3fn, device=cuda) for _ in range(2))
    ks, vs = (torch.zeros(1, nb, H, device=cuda) for _ in range(2))
    ops().write_kv8(x.to(cuda), y.to(cuda), kc, vc, ks, vs, 0, torch.arange(5, 5 + T, device=cuda))
    table = torch.arange(nb, dtype=torch.int32, device=cuda)
    for dtype in (F32, BF16, F16):
        gk, gv = ops().gather_kv8(kc, vc, ks, vs, 0, table, 5 + T, dtype=dtype)
        for got, want, scale in ((gk, x, ks), (gv, y, vs)):
            s = scale[0].cpu().double().repeat_interleave(bs, 0)[5 : 5 + T][:, :, None]
            d = (got[5:].cpu().double() - want.double()).abs()
            # the output's rounding: half a step, which below its least normal value is half the least step
            # (fp16: 2^-25, for values under 2^-14; the first form of this line left that out)
            rounding = torch.maximum(step(dtype) * got[5:].cpu().double().abs(), torch.tensor(torch.finfo(dtype).smallest_normal * step(dtype)))
            assert bool((d <= torch.maximum(2.0**-4 * want.double().abs(), 2.0**-10 * s) + rounding).all())
            assert (want.double().abs() <= 448 * s).all()


def test_append_keeps_non_finite_values_out_of_the_scale(cuda):
    def poke(qkv, slots, total):
        w = qkv.shape[1]
        qkv[3, w // 2 :: 7] = float("inf")
        qkv[5, w // 2 :: 5] = float("nan")
        qkv[6, w // 2 :: 3] = float("-inf")

    run_append(cuda, BF16, [20, 1], [4, 9], 8, 4, 64, 16, seed=5, poke=poke)


def test_append_of_zeros_and_of_the_largest_values(cuda):
    def poke(qkv, slots, total):
        qkv[:4] = 0.0
        qkv[4:8] = torch.finfo(BF16).max
        qkv[8:12] = 1e-30

    run_append(cuda, BF16, [16], [0], 4, 2, 64, 4, seed=6, poke=poke)


def test_append_skips_missing_slots_and_flags_wild_ones(cuda):
    def poke(qkv, slots, total):
        slots[2] = -1  # a padded row
        slots[7] = -1

    run_append(cuda, BF16, [9, 1], [3, 20], 8, 2, 64, 16, seed=7, poke=poke)
    ops().check_device_errors(cuda)

    def wild(qkv, slots, total):
        slots[4] = total
        slots[5] = total + 1000

    run_append(cuda, BF16, [9, 1], [3, 20], 8, 2, 64, 16, seed=8, poke=wild)
    with pytest.raises(RuntimeError, match="slot outside the cache"):
        ops().check_device_errors(cuda)


def test_append_takes_the_runs_of_a_block_in_turn(cuda):
    """Neighbours of one block whose slots do not follow one another, one slot twice: as calls one after the other."""

    def poke(qkv, slots, total):
        slots[:12] = slots[:12][[4, 5, 6, 7, 0, 1, 2, 9, 9, 8, 3, 10]]

    run_append(cuda, BF16, [12, 20], [16, 3], 8, 2, 64, 16, seed=9, poke=poke)


def test_append_one_token_at_a_time_and_all_at_once_agree(cuda):
    """Steps of one token bring the block to the scale that one call gives it; codes agree where the values
    stay normal in 8 bits at each scale on the way (here all do: within 2^5 of each other)."""
    g = torch.Generator().manual_seed(11)
    T, H, D, bs = 16, 2, 64, 16
    x = (1 + torch.rand(T, H, D, generator=g)) * torch.arange(1, T + 1)[:, None, None]
    x = x * (torch.randint(0, 2, x.shape, generator=g) * 2 - 1)
    x = x.to(F32).to(cuda)
    caches = []
    for sizes in ([T], [1] * T, [3, 1, 7, 5]):
        kc, vc = (torch.zeros(1, 1, bs, H, D, dtype=torch.float8_e4m3fn, device=cuda) for _ in range(2))
        ks, vs = (torch.zeros(1, 1, H, device=cuda) for _ in range(2))
        at = 0
        for n in sizes:
            ops().write_kv8(x[at : at + n], -x[at : at + n], kc, vc, ks, vs, 0, torch.arange(at, at + n, device=cuda))
            at += n
        caches.append((kc.float(), vc.float(), ks, vs))
    for other in caches[1:]:
        for a, b in zip(caches[0], other):
            assert torch.equal(a, b)


def test_gather_flags_a_bad_block_and_zeroes_it(cuda):
    kc, vc, ks, vs = (x[None].to(cuda) for x in plain.make_cache(4, 8, 2, 32, 0))
    table = torch.tensor([1, 9, -1, 2], dtype=torch.int32, device=cuda)
    k, v = ops().gather_kv8(kc, vc, ks, vs, 0, table, 29, dtype=F32)
    assert k.shape == (29, 2, 32)
    assert (k[8:24] == 0).all() and (v[8:24] == 0).all()
    assert torch.equal(k[:8], kc[0, 1].float() * ks[0, 1][:, None])
    assert torch.equal(v[24:], (vc[0, 2].float() * vs[0, 2][:, None])[:5])
    with pytest.raises(RuntimeError, match="block id outside the pool"):
        ops().check_device_errors(cuda)


# ------------------------------------------------------------------ attention
def run_attention(cuda, dtype, lens, new, hq, hkv, hd, bs, seed, *, scale=None, layers=2, layer=1, slack_rows=3, call=None):
    """new=None: single tokens.  Checks every row, and that rows past the last request stay as they were."""
    nb = sum(-(-max(n, 0) // bs) for n in lens) + 2
    codes_k, codes_v, ks, vs = plain.make_cache(nb, bs, hkv, hd, seed, cuda)
    tables = plain.make_tables([max(n, 0) for n in lens], bs, nb, seed, width=max(1, max(-(-n // bs) for n in lens)) + 2).to(cuda)
    counts = [1] * len(lens) if new is None else new
    # what lies behind a sequence's last token in its last block is not a value
    for i, n in enumerate(lens):
        if n > 0 and n % bs:
            for c in (codes_k, codes_v):
                c.view(torch.uint8)[tables[i, n // bs].long(), n % bs :] = 0x7F

    def caches(c, s):
        c2 = torch.zeros(layers, *c.shape, dtype=c.dtype, device=cuda)
        s2 = torch.zeros(layers, *s.shape, device=cuda)
        c2[layer], s2[layer] = c, s
        return c2, s2

    (kc, ks2), (vc, vs2) = caches(codes_k, ks), caches(codes_v, vs)
    T = sum(counts)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(T + slack_rows, hq, hd, generator=g).to(dtype).to(cuda)
    out = torch.full((T + slack_rows, hq + 1, hd), 7.0, dtype=dtype, device=cuda)[:, :hq]
    sl = torch.tensor(lens, dtype=torch.int32, device=cuda)
    sc = hd**-0.5 if scale is None else scale
    if new is None:
        got = ops().paged_decode_kv8(q, kc, vc, ks2, vs2, layer, tables, sl, out=out, scale=scale)
    else:
        qsl = torch.tensor([0] + counts).cumsum(0).to(cuda)
        got = ops().varlen_attention_kv8(q, kc, vc, ks2, vs2, layer, tables, sl, qsl, max(counts), out=out, scale=scale)
    assert got is out
    ops().check_device_errors(cuda)
    at = 0
    for i, (n, c) in enumerate(zip(lens, counts)):
        want, bound = plain.attention(q[at : at + c], codes_k, codes_v, ks, vs, tables[i], max(n, 0), n - c + 1, sc)
        x = got[at : at + c].double()
        assert x.isfinite().all(), (i, n, c)
        assert ((x - want).abs() <= step(dtype) * (want.abs() + bound) + bound + torch.finfo(dtype).tiny).all(), (
            i, n, c, float(((x - want).abs() - step(dtype) * want.abs() - bound).max()))
        at += c
    assert (got[T:] == 7.0).all()
    return q, (kc, vc, ks2, vs2), tables, sl, got


DECODES = [
    # lens, hq, hkv, hd, bs
    ([1], 32, 8, 64, 16),
    ([0, 5, 0], 32, 8, 64, 16),
    ([16, 17, 15, 32, 33], 32, 8, 64, 16),
    ([700, 1, 64, 4096, 333], 32, 8, 64, 16),
    ([9000], 8, 1, 64, 16),
    ([5000, 77], 8, 8, 64, 16),  # one query head to a kv head
    ([1000, 513], 6, 2, 64, 32),  # three
    ([1000, 2], 48, 2, 128, 32),  # twenty-four
    ([2049, 130, 1], 16, 2, 128, 16),
    ([513, 40], 40, 1, 64, 64),  # forty query heads on one
    ([100, 250], 10, 5, 64, 16),  # kv heads that no power of two divides
    ([260, 31], 12, 4, 80, 16),
    ([77, 19], 4, 2, 64, 5),
    ([130] * 70, 16, 4, 64, 16),
    ([50, 3], 2, 1, 256, 16),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("case", range(len(DECODES)))
def test_decode_matches_64_bits(cuda, case, dtype):
    lens, hq, hkv, hd, bs = DECODES[case]
    run_attention(cuda, dtype, lens, None, hq, hkv, hd, bs, seed=case)


VARLENS = [
    # lens, new, hq, hkv, hd, bs
    ([1], [1], 32, 8, 64, 16),
    ([5], [5], 32, 8, 64, 16),
    ([64, 65, 63], [64, 65, 63], 8, 2, 64, 16),
    ([300, 20, 129], [2, 20, 100], 32, 8, 64, 16),
    ([1500, 700], [5, 4], 32, 8, 64, 16),
    ([600], [600], 4, 4, 64, 16),
    ([257, 1000], [257, 33], 6, 2, 64, 32),
    ([400, 130], [300, 130], 16, 2, 128, 32),
    ([200], [90], 40, 1, 64, 16),
    ([333], [333], 9, 3, 128, 16),
    ([3, 2], [5, 4], 8, 2, 64, 16),  # more rows than keys: the first rows see none
    ([120, 50], [33, 50], 4, 2, 80, 16),
    ([77, 19], [20, 19], 4, 2, 64, 5),
    ([90] * 40, [3] * 40, 16, 4, 64, 16),
    ([5000], [40], 8, 1, 64, 16),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("case", range(len(VARLENS)))
def test_varlen_matches_64_bits(cuda, case, dtype):
    lens, new, hq, hkv, hd, bs = VARLENS[case]
    run_attention(cuda, dtype, lens, new, hq, hkv, hd, bs, seed=100 + case)


@pytest.mark.parametrize("new", [None, [1, 40]])
def test_attention_with_an_own_scale(cuda, new):
    run_attention(cuda, BF16, [300, 77], new, 8, 2, 64, 16, seed=40, scale=0.3)
    run_attention(cuda, BF16, [300, 77], new, 8, 2, 64, 16, seed=41, scale=-0.1)
    run_attention(cuda, BF16, [300, 77], new, 8, 2, 64, 16, seed=42, scale=0.0)


@pytest.mark.parametrize("new", [None, [3, 60, 2]])
def test_attention_lists_and_rows(cuda, new):
    """req_list picks requests, table_rows their tables, q_rows their query rows; strided queries."""
    lens = [500, 90, 40]
    q, (kc, vc, ks, vs), tables, sl, want = run_attention(cuda, BF16, lens, new, 8, 2, 64, 16, seed=50)
    counts = new or [1, 1, 1]
    T = sum(counts)
    wide = torch.zeros(q.shape[0], 12, 64, dtype=q.dtype, device=cuda)
    wide[:, :8] = q
    order = [2, 0, 1]
    shuffled = torch.zeros_like(tables)
    for i, r in enumerate(order):
        shuffled[r] = tables[i]
    rows = torch.tensor(order, dtype=torch.int32, device=cuda)
    pick = torch.tensor([2, 0], dtype=torch.int32, device=cuda)
    out = torch.zeros_like(want)
    if new is None:
        qr = torch.tensor([1, 2, 0], device=cuda)
        out = out[:3]  # an output has the query's shape
        got = ops().paged_decode_kv8(wide[[2, 0, 1]][:, :8], kc, vc, ks, vs, 1, shuffled, sl, out=out, table_rows=rows,
                                     q_rows=qr, req_list=pick, num_requests=2)
        assert torch.equal(got[qr[2]], want[2]) and torch.equal(got[qr[0]], want[0]) and (got[qr[1]] == 0).all()
    else:
        qsl = torch.tensor([0] + counts).cumsum(0).to(cuda)
        got = ops().varlen_attention_kv8(wide[:, :8], kc, vc, ks, vs, 1, shuffled, sl, qsl, 60, out=out, table_rows=rows,
                                         req_list=pick, num_requests=2)
        assert (got[qsl[1] : qsl[2]] == 0).all() and not (got[: qsl[1]] == 0).any()
        close = (got[qsl[2] : T].double() - want[qsl[2] : T].double()).abs() <= 2 * step(BF16) * want[qsl[2] : T].double().abs() + 2.0**-9
        assert close.all()


@pytest.mark.parametrize("new", [None, [40]])
def test_a_block_outside_the_pool_is_flagged(cuda, new):
    q, (kc, vc, ks, vs), tables, sl, _ = run_attention(cuda, BF16, [200], new, 8, 2, 64, 16, seed=60)
    tables[0, 3] = kc.shape[1]
    tables[0, 5] = -1
    if new is None:
        ops().paged_decode_kv8(q, kc, vc, ks, vs, 1, tables, sl)
    else:
        ops().varlen_attention_kv8(q, kc, vc, ks, vs, 1, tables, sl, torch.tensor([0, 40], device=cuda), 40)
    with pytest.raises(RuntimeError, match="block id outside the pool"):
        ops().check_device_errors(cuda)
    # a sequence longer than its table
    if new is None:
        ops().paged_decode_kv8(q, kc, vc, ks, vs, 1, tables[:, :2].contiguous().clamp(0, 1), sl)
        with pytest.raises(RuntimeError, match="block id outside the pool"):
            ops().check_device_errors(cuda)


def test_uneven_scales(cuda):
    """Blocks whose scales are 2^40 apart: the loud block decides, the quiet ones keep their weight in the sum."""
    q, (kc, vc, ks, vs), tables, sl, _ = run_attention(cuda, BF16, [100], None, 8, 2, 64, 16, seed=70)
    for low, high in ((2.0**-45, 1.0), (1.0, 2.0**40), (2.0**-48, 2.0**-30)):
        vs2 = torch.full_like(vs, low)
        vs2[:, tables[0, 2].long()] = high
        got = ops().paged_decode_kv8(q, kc, vc, ks, vs2, 1, tables, sl)
        rows = ops().varlen_attention_kv8(q, kc, vc, ks, vs2, 1, tables, sl, torch.tensor([0, 1], device=cuda), 1)
        want, bound = plain.attention(q[:1], kc[1], vc[1], ks[1], vs2[1], tables[0], 100, 100, 64**-0.5)
        for x in (got[:1], rows[:1]):
            assert ((x.double() - want).abs() <= step(BF16) * (want.abs() + bound) + bound).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_varlen_with_many_tiles_to_a_processor(cuda, hd):
    """More row tiles than processors, whole and nearly empty ones in turn (a request's last tile has few rows)."""
    run_attention(cuda, BF16, [900, 1300, 700, 513], [257, 513, 321, 513], 16, 4, hd, 16, seed=300 + hd)
    run_attention(cuda, F16, [70] * 90, [65] * 90, 8, 2, hd, 32, seed=301 + hd)
