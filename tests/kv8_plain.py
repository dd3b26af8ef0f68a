"""Plain implementations of the 8-bit paged cache's operators for the tests, in 64 bits."""

from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0
SCALE_MIN, SCALE_MAX = 2.0**-48, 2.0**48


def to_e4m3(x: torch.Tensor) -> torch.Tensor:
    """float8_e4m3fn codes, saturating; NaN stays NaN (torch's own conversion has no saturation)."""
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def least_scale(amax: float) -> float:
    if amax == 0:
        return SCALE_MIN
    frac, exp = math.frexp(amax)
    return min(max(math.ldexp(1.0, exp - 9 if frac <= 0.875 else exp - 8), SCALE_MIN), SCALE_MAX)


def runs_of(slots: list[int], bs: int, total: int):
    """(first token, count) of each stretch of neighbours that share a block."""
    out, t = [], 0
    while t < len(slots):
        s = slots[t]
        if s < 0 or s >= total:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and slots[t + n] == s + n and (s + n) // bs == s // bs:
            n += 1
        out.append((t, n))
        t += n
    return out


def append(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, slots: list[int]) -> None:
    """x [T, H, D] (already rotated, fp32) into codes [nb, bs, H, D] and scales [nb, H], in place, on the CPU."""
    nb, bs, H, _ = codes.shape
    x = torch.where(x.isfinite(), x, torch.full_like(x, float("nan")))
    for t, n in runs_of(slots, bs, nb * bs):
        b, off = divmod(slots[t], bs)
        for h in range(H):
            part = x[t : t + n, h]
            amax = part.nan_to_num(0.0).abs().max().item()
            s = least_scale(amax)
            if off:
                old = scales[b, h].item()
                if s > old:
                    codes[b, :off, h] = to_e4m3(codes[b, :off, h].float() * (old / s))
                else:
                    s = old
            scales[b, h] = s
            codes[b, off : off + n, h] = to_e4m3(part / s)


def rotate(x: torch.Tensor, sin: torch.Tensor, cos: torch.Tensor) -> torch.Tensor:
    """x [T, H, D] by sin/cos [T, D/2], in the type of x."""
    a, b = x.chunk(2, dim=-1)
    sin, cos = sin[:, None].to(x.dtype), cos[:, None].to(x.dtype)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def attention(q, codes_k, codes_v, ks, vs, table, n_keys, first_key_count, scale):
    """One request in 64 bits: q [n, Hq, D]; row j sees the keys [0, first_key_count + j).

    Returns the output and a bound on a kernel's error before the last rounding:
    the score is an fp32 sum of D products (D + 8 roundings of terms that sum to A at most, the
    exponent's argument included), a weight p is off by at most that, by 2^-20 for exp2 and the
    sums over the keys, and by 2^-11 for its rounding to 11 bits; a weight below 2^-14 of the
    largest p * vs is off by 2^-25 of it instead."""
    bs, H, D = codes_k.shape[1:]
    n, Hq, _ = q.shape
    G = Hq // H
    blocks = table[: -(-n_keys // bs)].long()

    def values(codes, scales):
        x = codes[blocks].double() * scales[blocks].double()[:, None, :, None]
        return x.reshape(-1, H, D)[:n_keys].permute(1, 0, 2)

    k, v = values(codes_k, ks), values(codes_v, vs)
    vscale = vs[blocks].double().repeat_interleave(bs, 0)[:n_keys].T  # [H, n_keys]
    qd = q.double().reshape(n, H, G, D).permute(1, 2, 0, 3)  # [H, G, n, D]
    s = qd @ k[:, None].transpose(2, 3) * scale
    size = qd.abs() @ k[:, None].abs().transpose(2, 3) * abs(scale)
    seen = torch.arange(n_keys, device=q.device)[None, :] < (first_key_count + torch.arange(n, device=q.device))[:, None]
    s = s.masked_fill(~seen, float("-inf"))
    some = seen.any(dim=1)
    p = torch.softmax(s, dim=-1).nan_to_num(0.0) if n_keys else s
    out = p @ v[:, None]
    size = size.masked_fill(~seen, 0.0)
    d_score = (D + 8) * 2.0**-24 * (size.amax(dim=-1, keepdim=True) if n_keys else torch.zeros_like(out[..., :1]))
    mass = p @ v[:, None].abs()
    top = (p * vscale[:, None, None]).amax(dim=-1, keepdim=True) if n_keys else torch.zeros_like(out[..., :1])
    bound = (2 * d_score + 2.0**-20 + 2.0**-11) * mass + n_keys * 2.0**-25 * E4M3_MAX * top
    out = torch.where(some[:, None], out, torch.zeros_like(out))

    def back(x):
        return x.permute(2, 0, 1, 3).reshape(n, Hq, D)

    return back(out), back(bound.expand_as(out))


def make_cache(nb, bs, H, D, seed, device="cpu"):
    """Codes of every finite value and uneven scales that are no powers of two."""
    g = torch.Generator().manual_seed(seed)
    codes, scales = [], []
    for _ in range(2):
        codes.append(to_e4m3(torch.randn(nb, bs, H, D, generator=g) * 120).to(device))
        scales.append((0.004 + 0.02 * torch.rand(nb, H, generator=g)).to(device))
    return codes[0], codes[1], scales[0], scales[1]


def make_tables(lens, bs, nb, seed, width=None):
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(nb, generator=g).tolist()
    need = [-(-n // bs) for n in lens]
    assert sum(need) <= nb
    t = torch.full((len(lens), width or max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for i, k in enumerate(need):
        t[i, :k] = torch.tensor(perm[at : at + k], dtype=torch.int32)
        at += k
    return t
