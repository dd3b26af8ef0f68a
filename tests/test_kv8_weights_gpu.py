"""How far below the largest a softmax weight may lie and still count in the attention over the 8-bit cache."""

import kv8_plain as plain
import pytest
import torch
from test_kv8_gpu import BF16, F16, ops, step

pytestmark = pytest.mark.gpu


def check(got, q, kc, vc, ks, vs, table, n, dtype, scale):
    """Rows of q that see the first n - len(q) + 1 ... n keys.  A weight w is off by its score's error (an fp32 sum of
    D products, D + 8 roundings of terms that sum to A), by 2^-20 for exp2, by 2^-12 for its rounding to 11 bits or,
    below 2^-23 of the largest w vs, by 2^-34 of that; the sums are fp32 sums of n terms."""
    rows, Hq, D = q.shape
    bs, H = kc.shape[1:3]
    blocks = table[: -(-n // bs)].long()
    k, v = ((c[blocks].double() * s[blocks].double()[:, None, :, None]).reshape(-1, H, D)[:n].permute(1, 0, 2)
            for c, s in ((kc, ks), (vc, vs)))  # [H, n, D]
    unit = vs[blocks].double().repeat_interleave(bs, 0)[:n].T  # [H, n]
    x = q.double().reshape(rows, H, Hq // H, D).permute(1, 2, 0, 3)  # [H, G, rows, D]
    seen = torch.arange(n, device=q.device)[None, :] < n - rows + 1 + torch.arange(rows, device=q.device)[:, None]
    s = (x @ k[:, None].transpose(2, 3) * scale).masked_fill(~seen, float("-inf"))
    size = (x.abs() @ k[:, None].abs().transpose(2, 3) * abs(scale)).masked_fill(~seen, 0.0)
    w = torch.softmax(s, dim=-1)
    want, mass = w @ v[:, None], w @ v[:, None].abs()
    top = (w * unit[:, None, None]).amax(dim=-1, keepdim=True)
    codes = (v / unit[:, :, None]).abs().sum(dim=1)[:, None, None]  # [H, 1, 1, D]
    rel = 2 * (D + 8) * 2.0**-24 * size.amax(dim=-1, keepdim=True) + 2.0**-20 + 2.0**-12 + n * 2.0**-24
    bound = rel * mass + 2.0**-34 * top * codes

    def back(y):
        return y.permute(2, 0, 1, 3).reshape(rows, Hq, D)

    want, bound = back(want), back(bound)
    # the test says something: the error it admits is far below the outputs
    assert (bound <= 2.0**-5 * want.abs()).double().mean() > 0.99
    assert ((got.double() - want).abs() <= step(dtype) * (want.abs() + bound) + bound).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [1, 3, 150])
@pytest.mark.parametrize("what", ["score", "scale"])
def test_a_long_tail_behind_keys_that_bring_nothing(cuda, what, rows, hd, dtype):
    """One key 18 nats above the others whose V is 0 (score), or 16 keys whose block of V codes 0 has a scale
    2^27 times the others' (scale): the output is the tail's, whose weights are 2^-26 or 2^-27 of the largest."""
    n, bs, H, G = 2000 + rows, 16, 2, 4
    g = torch.Generator().manual_seed(rows + hd)
    nb = -(-n // bs) + 1
    table = torch.randperm(nb, generator=g).int()
    kc = plain.to_e4m3(torch.randn(nb, bs, H, hd, generator=g) * 16)
    vc = plain.to_e4m3(50 + 300 * torch.rand(nb, bs, H, hd, generator=g))
    ks, vs = torch.full((nb, H), 1 / 64), torch.full((nb, H), 16.0)  # outputs are no subnormals of f16
    q = torch.randn(rows, H * G, hd, generator=g) * 0.5
    first = int(table[0])
    if what == "score":
        q[:, :, 0] = 64.0
        kc[:, :, :, 0] = 0.0
        kc[first, 0] = 0.0
        kc[first, 0, :, 0] = 144.0 if hd == 64 else 208.0  # 64 * 144 / 64 / 8 = 18 nats above; 64 * 208 / 64 / 128^0.5 = 18.4
        vc[first, 0] = 0.0
    else:
        vc[first] = 0.0
        vs[first] = vs[first] * 2.0**27
    q = q.to(dtype).to(cuda)
    kc, vc, ks, vs = (x[None].to(cuda) for x in (kc, vc, ks, vs))
    tables, sl = table[None].to(cuda), torch.tensor([n], dtype=torch.int32, device=cuda)
    if rows == 1:
        got = ops().paged_decode_kv8(q, kc, vc, ks, vs, 0, tables, sl)
    else:
        got = ops().varlen_attention_kv8(q, kc, vc, ks, vs, 0, tables, sl, torch.tensor([0, rows], device=cuda), rows)
    ops().check_device_errors(cuda)
    check(got, q, kc[0], vc[0], ks[0], vs[0], tables[0], n, dtype, hd**-0.5)
