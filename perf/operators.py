"""What the operators of the 8-bit paged key/value cache and of the log probabilities cost.

Four groups of calls, as a serving program makes them:

* ``append``: keys and values of new tokens rotated, brought to 8 bits (e4m3, one scale per block and kv head)
  and stored in the paged cache; then the blocks that they went to read back as values;
* ``decode``: attention of one query token per request over that cache;
* ``varlen``: causal attention of several query tokens per request over that cache;
* ``logprobs``: log probability of a given token per row of logits, entropy, and the top alternatives.

With ``own`` false the operators are written in elementary torch operations in 32 bits; with ``own`` true
they are the calls of :mod:`nano_infer_engine_b200.ops`.
"""

from __future__ import annotations

import random

import torch

own = False

BF16, F16, F32 = "bfloat16", "float16", "float32"
E4M3_MAX = 448.0
SCALE_MIN, SCALE_MAX = 2.0**-48, 2.0**48  # what the append keeps a block's scale within
DEVICE = "cuda"


# ------------------------------------------------------------------------ cases
def listed() -> list[dict]:
    return [
        # one new token of one request: a decode step at batch 1, all latency
        dict(name="append_1", op="append", dtype=BF16, requests=1, tokens=1, context=777, hq=32, hkv=8, hd=64, bs=16, mix=1),
        # the tokens of a large prefill step, requests of uneven length starting inside a block
        dict(name="append_16384", op="append", dtype=BF16, requests=5, tokens=16384, context=100, hq=32, hkv=8, hd=64, bs=16, mix=2),
        # batch 1, a short prompt: the smallest decode call
        dict(name="decode_1x100", op="decode", dtype=BF16, requests=1, context=100, hq=32, hkv=8, hd=64, bs=16, mix=3),
        # an ordinary serving batch of uneven lengths
        dict(name="decode_16x4001", op="decode", dtype=BF16, requests=16, context=4001, hq=32, hkv=8, hd=64, bs=16, mix=4),
        # the benchmark's large ragged batch: 64 requests with contexts up to 29,600 tokens
        dict(name="decode_64x29600", op="decode", dtype=BF16, requests=64, context=29600, hq=32, hkv=8, hd=64, bs=16, mix=5),
        # one request at the configuration's longest sequence, wider heads, eight query heads on each kv head
        dict(name="decode_1x131072", op="decode", dtype=F16, requests=1, context=131072, hq=32, hkv=4, hd=128, bs=32, mix=6),
        # a few proposed tokens of each request checked at once
        dict(name="verify_8x5", op="varlen", dtype=BF16, requests=8, queries=5, context=2000, hq=32, hkv=8, hd=64, bs=16, mix=7),
        # one long prompt in one call
        dict(name="prefill_1x8192", op="varlen", dtype=BF16, requests=1, queries=8192, context=0, hq=32, hkv=8, hd=64, bs=16, mix=8),
        # chunks of several prompts, each behind its cached part
        dict(name="chunk_6x513", op="varlen", dtype=F16, requests=6, queries=513, context=4000, hq=16, hkv=4, hd=128, bs=32, mix=9),
        # the answer of one decode step: one row over the vocabulary
        dict(name="logprobs_1", op="logprobs", dtype=BF16, rows=1, vocab=128256, top=5, masked=False),
        # rows in 32 bits of which a grammar forbids about half of the tokens, an odd vocabulary
        dict(name="logprobs_333_masked", op="logprobs", dtype=F32, rows=333, vocab=50257, top=3, masked=True),
        # a scored prompt: every row of a long prefill
        dict(name="logprobs_4096", op="logprobs", dtype=BF16, rows=4096, vocab=128256, top=20, masked=False),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["append", "decode", "varlen", "logprobs"])
    mix = rng.randrange(1 << 30)
    if op == "logprobs":
        dtype = rng.choice([BF16, BF16, F16, F32])
        vocab = _log_int(rng, 1000, 256000)
        most = 4096 * 128256 * 2 // (vocab * (4 if dtype == F32 else 2))
        return dict(op=op, dtype=dtype, rows=_log_int(rng, 1, min(4096, most)), vocab=vocab, top=rng.randrange(0, 21),
                    masked=rng.random() < 0.3)
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 4, 8])
    hd = rng.choice([64, 64, 128])
    case = dict(op=op, dtype=rng.choice([BF16, BF16, F16]), hq=hkv * group, hkv=hkv, hd=hd, bs=rng.choice([16, 16, 32]), mix=mix)
    if op == "append":
        tokens = _log_int(rng, 1, 16384 * 8 * 64 // max(hkv * hd, 512) // max(1, group // 4))
        case.update(requests=rng.randint(1, min(64, tokens)), tokens=tokens, context=rng.randrange(0, 4000))
    elif op == "decode":
        requests = _log_int(rng, 1, 128)
        most = 64 * 29600 * 8 * 64 // (requests * hkv * hd)
        case.update(requests=requests, context=_log_int(rng, 1, min(131072, most)))
    else:
        requests = rng.randint(1, 16)
        queries = _log_int(rng, 2, 4096)
        room = 32 * 8192 * 8192 // (requests * case["hq"] * queries * 2)
        if room <= queries:
            queries = max(2, int((32 * 8192 * 8192 / (requests * case["hq"] * 2)) ** 0.5) - 1)
            room = queries + 1
        case.update(requests=requests, queries=queries, context=rng.randrange(0, max(1, min(16384, room - queries))))
    return case


def _contexts(case: dict) -> tuple[list[int], list[int]]:
    """Cached tokens and new tokens of each request, from the case alone."""
    r = random.Random(case["mix"])
    n = case["requests"]
    if case["op"] == "append":
        cuts = sorted(r.sample(range(1, case["tokens"]), n - 1)) if n > 1 else []
        new = [b - a for a, b in zip([0, *cuts], [*cuts, case["tokens"]])]
        return [r.randint(0, case["context"]) for _ in range(n - 1)] + [case["context"]], new
    if case["op"] == "decode":
        # the longest request has `context` tokens, the others 1 .. context
        return [case["context"] - 1] + [r.randint(1, case["context"]) - 1 for _ in range(n - 1)], [1] * n
    return (
        [case["context"]] + [r.randint(0, case["context"]) for _ in range(n - 1)],
        [case["queries"]] + [r.randint(max(1, case["queries"] // 4), case["queries"]) for _ in range(n - 1)],
    )


# ------------------------------------------------------------------------ inputs
def _paging(case: dict, old: list[int], new: list[int]):
    """Block tables over a shuffled pool that has the blocks of the sequences and no more."""
    bs = case["bs"]
    need = [-(-(a + b) // bs) for a, b in zip(old, new)]
    perm = list(range(sum(need)))
    random.Random(case["mix"] + 1).shuffle(perm)
    tables = torch.full((len(old), max(need)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = torch.tensor(perm[at : at + n], dtype=torch.int32)
        at += n
    return tables, sum(need)


def _pool(case: dict, blocks: int, g: torch.Generator):
    """One layer's codes and scales, as values of unit size with some louder channels leave them."""
    shape = (1, blocks, case["bs"], case["hkv"], case["hd"])
    codes, scales = [], []
    for _ in range(2):
        loud = 1 + 3 * (torch.rand(case["hkv"], case["hd"], device=DEVICE, generator=g) < 0.05).float()
        code = torch.empty(shape, dtype=torch.float8_e4m3fn, device=DEVICE)
        scale = torch.empty((1, blocks, case["hkv"]), device=DEVICE)
        step = max(1, (1 << 27) // (case["bs"] * case["hkv"] * case["hd"]))
        for b in range(0, blocks, step):
            x = torch.randn((min(step, blocks - b), *shape[2:]), device=DEVICE, generator=g) * loud
            s = x.abs().amax(dim=(1, 3)) / E4M3_MAX
            code[0, b : b + step] = (x / s[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
            scale[0, b : b + step] = s
        codes.append(code)
        scales.append(scale)
    return codes, scales


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    if case["op"] == "logprobs":
        logits = (torch.randn(case["rows"], case["vocab"], device=DEVICE, generator=g) * 3).to(dtype)
        tokens = torch.randint(0, case["vocab"], (case["rows"],), device=DEVICE, generator=g)
        if case["masked"]:
            shut = torch.rand(logits.shape, device=DEVICE, generator=g) < 0.5
            shut[torch.arange(case["rows"], device=DEVICE), tokens] = False
            logits.masked_fill_(shut, float("-inf"))
        return dict(case=case, logits=logits, tokens=tokens)
    old, new = _contexts(case)
    tables, blocks = _paging(case, old, new)
    hq, hkv, hd, bs = case["hq"], case["hkv"], case["hd"], case["bs"]
    total = sum(new)
    starts = torch.tensor([0] + new).cumsum(0)
    state = dict(
        case=case,
        tables=tables.to(DEVICE),
        seq_lens=torch.tensor([a + b for a, b in zip(old, new)], dtype=torch.int32, device=DEVICE),
        starts=starts.to(DEVICE),
        most_new=max(new),
        most_keys=max(a + b for a, b in zip(old, new)),
        scale=hd**-0.5,
    )
    state["q"] = torch.randn(total, hq, hd, device=DEVICE, generator=g).to(dtype)
    if case["op"] != "append":
        (state["kc"], state["vc"]), (state["ks"], state["vs"]) = _pool(case, blocks, g)
        return state
    # the projections' output: q, k and v of a token side by side
    qkv = torch.randn(total, (hq + 2 * hkv) * hd, device=DEVICE, generator=g).to(dtype)
    state["q"], state["k"], state["v"] = qkv[:, : hq * hd], qkv[:, hq * hd : (hq + hkv) * hd], qkv[:, (hq + hkv) * hd :]
    pos = torch.cat([torch.arange(a, a + b) for a, b in zip(old, new)])
    rows = torch.cat([torch.full((b,), i) for i, b in enumerate(new)])
    angle = pos[:, None].double() * 500000.0 ** (-torch.arange(hd // 2).double() / (hd // 2))
    state["sin"], state["cos"] = angle.sin().to(dtype).to(DEVICE), angle.cos().to(dtype).to(DEVICE)
    state["slots"] = (tables[rows, pos // bs].long() * bs + pos % bs).to(DEVICE)
    # blocks that earlier tokens began hold them at a power-of-two scale, the others nothing
    state["kc"], state["vc"] = (torch.zeros((1, blocks, bs, hkv, hd), dtype=torch.float8_e4m3fn, device=DEVICE) for _ in range(2))
    state["ks"], state["vs"] = (torch.full((1, blocks, hkv), SCALE_MIN, device=DEVICE) for _ in range(2))
    begun = torch.tensor([[int(tables[i, a // bs]), a % bs] for i, a in enumerate(old) if a % bs], dtype=torch.long).to(DEVICE).view(-1, 2)
    for code, scale in ((state["kc"], state["ks"]), (state["vc"], state["vs"])):
        x = torch.randn(len(begun), bs, hkv, hd, device=DEVICE, generator=g).clamp(-3.5, 3.5)
        x = x * (torch.arange(bs, device=DEVICE)[None, :] < begun[:, 1:])[:, :, None, None]
        code[0, begun[:, 0]] = (x * 128).to(torch.float8_e4m3fn)
        scale[0, begun[:, 0]] = 1 / 128
    state["filled"] = torch.cat([tables[i, a // bs : (a + b - 1) // bs + 1] for i, (a, b) in enumerate(zip(old, new))]).to(DEVICE)
    return state


# ------------------------------------------------------------------------ one pass
def run(s: dict):
    return {"append": _append, "decode": _decode, "varlen": _varlen, "logprobs": _logprobs}[s["case"]["op"]](s)


def _power_of_two_scale(amax: torch.Tensor) -> torch.Tensor:
    """The least power of two whose 448-fold is not below amax, kept within the bounds."""
    frac, exp = torch.frexp(amax)  # amax = frac * 2^exp, frac in [0.5, 1); 448 = 0.875 * 2^9
    s = torch.ldexp(torch.ones_like(amax), torch.where(frac <= 0.875, exp - 9, exp - 8))
    return torch.where(amax > 0, s, torch.full_like(s, SCALE_MIN)).clamp(SCALE_MIN, SCALE_MAX)


def _store(code, scale, x, slots, bs):
    """Bring x [T, H, D] to 8 bits in the blocks of the slots: new scales, earlier codes at the new scale, new codes."""
    blocks, hkv = scale.shape[1], scale.shape[2]
    block, off = slots // bs, slots % bs
    at = block[:, None].expand(-1, hkv)
    amax = torch.zeros((blocks, hkv), device=x.device).scatter_reduce_(0, at, x.abs().amax(dim=2), "amax")
    first = torch.full((blocks,), bs, device=x.device).scatter_reduce_(0, block, off, "amin")
    touched = first < bs
    before = torch.where((first == 0)[:, None], torch.full_like(scale[0], SCALE_MIN), scale[0])
    after = torch.where(touched[:, None], torch.maximum(_power_of_two_scale(amax), before), scale[0])
    earlier = touched[:, None] & (torch.arange(bs, device=x.device)[None, :] < first[:, None])
    b, o = earlier.nonzero(as_tuple=True)
    code[0, b, o] = (code[0, b, o].float() * (scale[0, b] / after[b])[:, :, None]).to(code.dtype)
    code[0, block, off] = (x / after[block][:, :, None]).to(code.dtype)
    scale[0] = after


def _append(s):
    c = s["case"]
    hq, hkv, hd, bs = c["hq"], c["hkv"], c["hd"], c["bs"]
    if own:
        from nano_infer_engine_b200 import ops

        q = ops.rope_write_kv8(s["q"], s["k"], s["v"], s["sin"], s["cos"], s["kc"], s["vc"], s["ks"], s["vs"], 0, s["slots"], hq)
        count = s["filled"].numel() * bs
        keys, values = ops.gather_kv8(s["kc"], s["vc"], s["ks"], s["vs"], 0, s["filled"], count, dtype=q.dtype)
        return {"q": q, "keys": keys, "values": values, "key_scales": s["ks"], "value_scales": s["vs"]}
    dtype = s["q"].dtype
    sin, cos = s["sin"].float()[:, None, :], s["cos"].float()[:, None, :]

    def rotate(x, heads):
        a, b = x.reshape(-1, heads, hd).float().split(hd // 2, dim=2)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=2)

    q = rotate(s["q"], hq).to(dtype)
    _store(s["kc"], s["ks"], rotate(s["k"], hkv), s["slots"], bs)
    _store(s["vc"], s["vs"], s["v"].reshape(-1, hkv, hd).float(), s["slots"], bs)
    b = s["filled"].long()
    keys, values = ((code[0][b].float() * scale[0][b][:, None, :, None]).to(dtype).flatten(0, 1)
                    for code, scale in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
    return {"q": q, "keys": keys, "values": values, "key_scales": s["ks"], "value_scales": s["vs"]}


def _keys_of(code, scale, tables, most):
    """The values of each request's tokens in order, [R, H, most, D]; what lies past a request's blocks is not used."""
    bs = code.shape[2]
    t = tables[:, : -(-most // bs)].clamp(min=0).long()
    x = code[0][t].float() * scale[0][t][:, :, None, :, None]
    return x.flatten(1, 2)[:, :most].transpose(1, 2)


def _decode(s):
    if own:
        from nano_infer_engine_b200 import ops

        return ops.paged_decode_kv8(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], 0, s["tables"], s["seq_lens"], scale=s["scale"])
    c = s["case"]
    most = s["most_keys"]
    q = s["q"].float().unflatten(1, (c["hkv"], -1))
    scores = q @ _keys_of(s["kc"], s["ks"], s["tables"], most).transpose(2, 3) * s["scale"]
    hidden = torch.arange(most, device=q.device)[None, :] >= s["seq_lens"][:, None]
    scores = scores.masked_fill(hidden[:, None, None, :], float("-inf"))
    p = (scores - scores.amax(dim=-1, keepdim=True)).exp()
    p = p / p.sum(dim=-1, keepdim=True)
    out = p @ _keys_of(s["vc"], s["vs"], s["tables"], most)
    return out.flatten(1, 2).to(s["q"].dtype)


def _varlen(s):
    if own:
        from nano_infer_engine_b200 import ops

        return ops.varlen_attention_kv8(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], 0, s["tables"], s["seq_lens"], s["starts"],
                                        s["most_new"], scale=s["scale"])
    c = s["case"]
    most, rows = s["most_keys"], s["most_new"]
    hkv, hd, group = c["hkv"], c["hd"], c["hq"] // c["hkv"]
    new = s["starts"][1:] - s["starts"][:-1]
    at = torch.arange(rows, device=new.device)
    real = at[None, :] < new[:, None]  # [R, rows]
    q = s["q"][(s["starts"][:-1, None] + at).clamp(max=len(s["q"]) - 1)].float()  # [R, rows, Hq, D]
    q = q.unflatten(2, (hkv, group)).permute(0, 2, 3, 1, 4).reshape(len(new), hkv, group * rows, hd)
    scores = (q @ _keys_of(s["kc"], s["ks"], s["tables"], most).transpose(2, 3)).mul_(s["scale"])
    last = (s["seq_lens"] - new)[:, None] + at  # the position of each query: it sees the keys up to there
    hidden = torch.arange(most, device=q.device) > last[:, :, None]
    scores.view(len(new), hkv, group, rows, most).masked_fill_(hidden[:, None, None], float("-inf"))
    p = scores.sub_(scores.amax(dim=-1, keepdim=True)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    out = (p @ _keys_of(s["vc"], s["vs"], s["tables"], most)) / total
    out = out.view(len(new), hkv, group, rows, hd).permute(0, 3, 1, 2, 4).reshape(len(new), rows, hkv * group, hd)
    return out[real].to(s["q"].dtype)


def _logprobs(s):
    logits, tokens, top = s["logits"], s["tokens"], s["case"]["top"]
    if own:
        from nano_infer_engine_b200 import ops

        got = ops.token_logprobs(logits, tokens, top=top)
        return [got.logprobs, got.entropy, got.top_logprobs, got.top_ids]
    x = logits.float()
    m = x.amax(dim=1, keepdim=True)
    d = x - m
    e = d.exp()
    z = e.sum(dim=1)
    log_z = z.log()
    entropy = log_z - torch.where(e > 0, d * e, torch.zeros_like(e)).sum(dim=1) / z
    lp = d.gather(1, tokens[:, None])[:, 0] - log_z
    # the largest, ties to the lowest index: one whole number per entry that sorts that way
    bits = (x + 0.0).view(torch.int32).long()
    key = (torch.where(bits < 0, -2147483648 - bits, bits) << 32) + (0x7FFFFFFF - torch.arange(x.shape[1], device=x.device))
    ids = 0x7FFFFFFF - (key.topk(top, dim=1).values & 0xFFFFFFFF)
    return [lp, entropy, d.gather(1, ids) - log_z[:, None], ids]


# ------------------------------------------------------------------------ 64 bits
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        logits, tokens, top = s["logits"], s["tokens"], case["top"]
        parts = []
        for i in range(0, len(tokens), 256):
            x = logits[i : i + 256].double()
            lse = torch.logsumexp(x, dim=1, keepdim=True)
            lp = x - lse
            p = lp.exp()
            h = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(dim=1)
            ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
            parts.append((lp.gather(1, tokens[i : i + 256, None])[:, 0], h, lp.gather(1, ids), ids))
        return [torch.cat(p) for p in zip(*parts)]
    old, new = _contexts(case)
    hq, hkv, hd, bs = case["hq"], case["hkv"], case["hd"], case["bs"]
    if case["op"] == "append":
        z = torch.complex(s["cos"].double(), s["sin"].double())[:, None, :]

        def turned(x, heads):
            x = x.reshape(-1, heads, 2, hd // 2).double()
            y = torch.complex(x[:, :, 0], x[:, :, 1]) * z
            return torch.cat([y.real, y.imag], dim=2)

        out = {"q": turned(s["q"], hq)}
        block = s["slots"] // bs
        for name, code, scale, x in (("key", s["kc"], s["ks"], turned(s["k"], hkv)),
                                     ("value", s["vc"], s["vs"], s["v"].reshape(-1, hkv, hd).double())):
            # the values of all blocks, then each block's scale from the values that are in it
            begun = torch.zeros(code.shape[1], dtype=torch.bool, device=DEVICE)
            tables = s["tables"].tolist()
            for i, a in enumerate(old):
                if a % bs:
                    begun[tables[i][a // bs]] = True
            full = code[0].double() * scale[0].double()[:, None, :, None]
            full[~begun] = 0
            full[block, s["slots"] % bs] = x
            new_max = torch.zeros(full.shape[0], hkv, dtype=torch.float64, device=DEVICE)
            new_max.scatter_reduce_(0, block[:, None].expand(-1, hkv), x.abs().amax(dim=2), "amax")
            unit = torch.exp2(torch.ceil(torch.log2(new_max / E4M3_MAX)).clamp(-48, 48))
            unit = torch.where(new_max > 0, unit, torch.full_like(unit, SCALE_MIN))
            hit = torch.zeros_like(begun)
            hit[block] = True
            kept = torch.where(begun[:, None] | ~hit[:, None], scale[0].double(), torch.full_like(unit, SCALE_MIN))
            unit = torch.where(hit[:, None], torch.maximum(unit, kept), kept)
            y = full / unit[:, None, :, None]
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)  # e4m3: 3 bits, least normal 2^-6
            out[name + "s"] = (torch.round(y / step) * step * unit[:, None, :, None])[s["filled"].long()].flatten(0, 1)
            out[name + "_scales"] = unit[None]
        return out
    got = []
    for i, (a, b) in enumerate(zip(old, new)):
        n = a + b
        t = s["tables"][i, : -(-n // bs)].long()
        k, v = ((code[0][t].double() * scale[0][t].double()[:, None, :, None]).flatten(0, 1)[:n].transpose(0, 1)
                for code, scale in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
        q0 = int(s["starts"][i])
        q = s["q"][q0 : q0 + b].double().unflatten(1, (hkv, -1))
        rows = torch.empty(b, hkv, hq // hkv, hd, dtype=torch.float64, device=DEVICE)
        seen = torch.arange(n, device=DEVICE)[None, :] <= torch.arange(a, n, device=DEVICE)[:, None]
        for h in range(hkv):
            for j in range(hq // hkv):
                w = torch.softmax((q[:, h, j] @ k[h].T * s["scale"]).masked_fill(~seen, float("-inf")), dim=1)
                rows[:, h, j] = w @ v[h]
        got.append(rows.flatten(1, 2))
    return torch.cat(got)


# ------------------------------------------------------------------------ floors
def work(case: dict) -> dict:
    size = 4 if case["dtype"] == F32 else 2
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": rows * (vocab * size + 8 + 8 + 12 * case["top"]), "flops": 5 * rows * vocab}
    old, new = _contexts(case)
    hq, hkv, hd, bs = case["hq"], case["hkv"], case["hd"], case["bs"]
    total = sum(new)
    if case["op"] == "append":
        blocks = sum((a + b - 1) // bs - a // bs + 1 for a, b in zip(old, new))
        # q, k, v, sin, cos and slots in; rotated q, codes and scales out; then the codes in and the values out
        moved = total * ((2 * hq + 2 * hkv + 1) * hd * size + 8 + 2 * hkv * hd)
        return {"bytes": moved + blocks * (bs * hkv * hd * 2 * (1 + size) + 16 * hkv), "flops": total * (3 * hq + 4 * hkv) * hd}
    codes = 2 * hkv * hd * sum(a + b for a, b in zip(old, new))
    scales = 2 * hkv * 4 * sum(-(-(a + b) // bs) for a, b in zip(old, new))
    pairs = sum(b * a + b * (b + 1) // 2 for a, b in zip(old, new))
    return {"bytes": codes + scales + 2 * total * hq * hd * size, "flops": 4 * hq * hd * pairs}
