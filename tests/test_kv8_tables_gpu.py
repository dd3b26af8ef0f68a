"""Block tables of the 8-bit attention that are views of wider ones: they end where the view ends."""

import kv8_plain as plain
import pytest
import torch
from test_kv8_edges_gpu import close
from test_kv8_gpu import BF16, F32, ops, run_attention, step

pytestmark = pytest.mark.gpu


def view_of(tables, left):
    """The same table as the last columns of a wider one whose other entries are blocks that exist."""
    base = torch.zeros(tables.shape[0], left + tables.shape[1], dtype=torch.int32, device=tables.device)
    base[:, left:] = tables
    return base[:, left:]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("new", [None, [5, 9], [40, 70]])
@pytest.mark.parametrize("length", [2**31 - 1, 337, 321])
def test_a_length_past_a_view_of_columns(cuda, new, length, dtype):
    """The first request's table is followed in memory by blocks that are there; they are not its own."""
    q, (kc, vc, ks, vs), tables, sl, want = run_attention(cuda, dtype, [320, 77], new, 8, 2, 64, 16, seed=710)
    view = view_of(tables[:, :20], 21)  # 320 keys
    assert view.stride(0) == 41
    counts = new or [1, 1]
    c, T = counts[0], sum(counts)
    qsl = torch.tensor([0] + counts).cumsum(0).to(cuda)

    def call(table, lens, out):
        lens = torch.tensor(lens, dtype=torch.int32, device=cuda)
        if new is None:
            return ops().paged_decode_kv8(q, kc, vc, ks, vs, 1, table, lens, out=out)
        return ops().varlen_attention_kv8(q, kc, vc, ks, vs, 1, table, lens, qsl, max(new), out=out)

    got = call(view, [320, 77], torch.zeros_like(q))  # lengths that the view holds
    ops().check_device_errors(cuda)
    assert close(got[:T], want[:T], dtype)
    # the long request first, and last, where the view ends with its storage
    for lens, rows, long in (([length, 77], slice(0, c), 0), ([77, length], slice(c, T), 1)):
        table = view if long == 0 else view_of(tables[:, :20].flip(0), 21)
        got = call(table, lens, torch.zeros_like(q))
        with pytest.raises(RuntimeError, match="block id outside the pool"):
            ops().check_device_errors(cuda)
        n = counts[long]
        for j in {0, n // 2, n - 1}:
            seen = min(320, length - n + 1 + j)
            row = q[rows][j : j + 1]
            w, bound = plain.attention(row, kc[1], vc[1], ks[1], vs[1], tables[0], seen, seen, 64**-0.5)
            d = (got[rows][j].double() - w[0]).abs()
            assert (d <= step(dtype) * (w[0].abs() + bound[0]) + bound[0] + 1e-30).all(), (long, j)


def test_a_narrow_view_takes_the_form_of_its_own_width(cuda):
    """The same launches and the same bits as for a table of that width."""
    from nano_infer_engine_b200 import ops as module

    for lens, new in (([100, 60], None), ([1500] * 3, None), ([2000] * 8, [5] * 8), ([300] * 3, [100] * 3)):
        q, (kc, vc, ks, vs), tables, sl, _ = run_attention(cuda, BF16, lens, new, 8, 2, 64, 16, seed=720)
        results = []
        for table in (tables.contiguous(), view_of(tables, 4000)):
            before = module.LAUNCHES
            if new is None:
                got = module.paged_decode_kv8(q, kc, vc, ks, vs, 1, table, sl)
            else:
                qsl = torch.tensor([0] + new).cumsum(0).to(cuda)
                got = module.varlen_attention_kv8(q, kc, vc, ks, vs, 1, table, sl, qsl, max(new))
            results.append((got[: sum(new or [1] * len(lens))], module.LAUNCHES - before))
        assert torch.equal(results[0][0], results[1][0]) and results[0][1] == results[1][1], (len(lens), new)
    ops().check_device_errors(cuda)
