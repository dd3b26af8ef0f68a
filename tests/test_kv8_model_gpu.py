"""A Llama-shaped model on an 8-bit cache: appending, attention, graphs, hand-over and scoring together."""

import pytest
import torch

from nano_infer_engine_b200 import ops
from nano_infer_engine_b200.generation.config import GenerationConfig
from nano_infer_engine_b200.generation.scheduler import ContinuousBatchingScheduler
from nano_infer_engine_b200.generation.score import paged_score
from nano_infer_engine_b200.models.llama import LlamaConfig, build_random_llama
from nano_infer_engine_b200.paged_cache import PagedKVCache, transfer_sequence

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


def llama(cuda, dtype=torch.bfloat16, heads=8, kv=2, hidden=512):
    cfg = LlamaConfig(vocab_size=512, hidden_size=hidden, mlp_inner_size=1024, num_layers=2, q_head_num=heads, kv_head_num=kv,
                      max_seq_len=4096)
    return build_random_llama(cfg, 0, 0.02, dtype, cuda), cfg


def cache_for(cfg, cuda, dtype=F8, blocks=256, bs=16):
    return PagedKVCache(blocks, bs, cfg.num_layers, cfg.kv_head_num, cfg.head_dim, dtype, cuda)


def prompts_for(cfg, cuda, lens, seed=5):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randint(0, cfg.vocab_size, (1, n), generator=g).to(cuda) for n in lens)


class _Exact:
    """What the model computes with the cache's values in place of the 8-bit kernels: the kernels' calls are taken
    over by plain ones on the same codes."""

    def __init__(self, monkeypatch):
        monkeypatch.setattr(ops, "paged_decode_kv8", self.decode)
        monkeypatch.setattr(ops, "varlen_attention_kv8", self.varlen)

    @staticmethod
    def _rows(q, kc, vc, ks, vs, layer, tables, sl, first, count, row, out):
        import kv8_plain as plain

        n = int(sl)
        want, _ = plain.attention(q[first : first + count], kc[layer], vc[layer], ks[layer], vs[layer], tables[row], n,
                                  n - count + 1, q.shape[2] ** -0.5)
        out[first : first + count] = want.to(out.dtype)

    def decode(self, q, kc, vc, ks, vs, layer, tables, seq_lens, *, out, table_rows, q_rows, req_list, num_requests, overlap):
        for i in req_list[:num_requests].tolist():
            self._rows(q, kc, vc, ks, vs, layer, tables, seq_lens[i], int(q_rows[i]), 1, int(table_rows[i]), out)
        return out

    def varlen(self, q, kc, vc, ks, vs, layer, tables, seq_lens, qsl, most, *, out, table_rows, req_list, num_requests):
        for i in req_list[:num_requests].tolist():
            a, b = int(qsl[i]), int(qsl[i + 1])
            self._rows(q, kc, vc, ks, vs, layer, tables, seq_lens[i], a, b - a, int(table_rows[i]), out)
        return out


def run(model, cfg, prompts, cuda, *, graphs, chunk, dtype=F8):
    model.cuda_graphs = graphs
    cache = cache_for(cfg, cuda, dtype)
    config = GenerationConfig(max_new_tokens=10, prefill_chunk_size=chunk, max_prefill_tokens_per_step=64 if chunk else None)
    sched = ContinuousBatchingScheduler(model, config, cache, 4)
    reqs = [sched.add_request(f"r{i}", p) for i, p in enumerate(prompts)]
    with torch.inference_mode():
        sched.run_until_idle()
    ops.check_device_errors(cuda)
    assert [(r.status.value, r.error) for r in reqs] == [("completed", None)] * len(reqs)
    return [r.sequence[0].tolist() for r in reqs]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_logits_match_plain_attention_on_the_same_codes(cuda, monkeypatch, dtype):
    """One ragged step of prompts, one mixed with single tokens.  The two runs differ by the attention's rounding
    alone: an output off by half a step now and then, through two layers and a head of unit-size values."""
    model, cfg = llama(cuda, dtype)
    prompts = prompts_for(cfg, cuda, (70, 33, 5))

    def logits():
        cache = cache_for(cfg, cuda)
        got = []
        ids = ("a", "b", "c")
        with torch.inference_mode():
            flat = torch.cat([p[0] for p in prompts])
            got.append(model.forward_ragged(flat, kv_cache=cache, sequence_ids=ids,
                                            query_start_loc=torch.tensor([0, 70, 103, 108], device=cuda)))
            flat = torch.tensor([3, 4, 5, 6, 7, 8], device=cuda)
            got.append(model.forward_ragged(flat, kv_cache=cache, sequence_ids=ids,
                                            query_start_loc=torch.tensor([0, 1, 5, 6], device=cuda)))
        return torch.cat(got).float()

    mine = logits()
    ops.check_device_errors(cuda)
    _Exact(monkeypatch)
    want = logits()
    rms = want.square().mean().sqrt()
    assert (mine - want).square().mean().sqrt() <= 8 * torch.finfo(dtype).eps * rms


def test_graphs_and_chunks_give_the_same_tokens(cuda):
    model, cfg = llama(cuda)
    prompts = prompts_for(cfg, cuda, (9, 33, 70, 18))
    eager = run(model, cfg, prompts, cuda, graphs=False, chunk=None)
    assert run(model, cfg, prompts, cuda, graphs=True, chunk=None) == eager
    chunked = run(model, cfg, prompts, cuda, graphs=True, chunk=16)
    assert all(a[: p.shape[1]] == p[0].tolist() and len(a) == p.shape[1] + 10 for a, p in zip(chunked, prompts))


def test_two_graphs_of_one_cache_replay_in_turn(cuda):
    """Decode graphs of two batch sizes hold workspaces of their own."""
    model, cfg = llama(cuda)
    model.cuda_graphs = True
    prompts = prompts_for(cfg, cuda, (40, 25, 33))
    with torch.inference_mode():
        def steps(graphs):
            model.cuda_graphs = graphs
            cache = cache_for(cfg, cuda)
            ids = ("a", "b", "c")
            for s, p in zip(ids, prompts):
                model(p, kv_cache=cache, sequence_id=s)
            got = []
            for i in range(6):
                who = ids if i % 2 else ids[:2]
                x = torch.full((len(who), 1), 7 + i, device=cuda)
                got.append(model(x, kv_cache=cache, sequence_ids=who)[:, 0].clone())
            return got

        for a, b in zip(steps(False), steps(True)):
            assert torch.equal(a, b)


def test_cache_write_gather_export_import_and_transfer(cuda):
    g = torch.Generator().manual_seed(0)
    a, b, c = (PagedKVCache(16, 16, 2, 2, 64, F8, cuda) for _ in range(3))
    k, v = (torch.randn(37, 2, 64, generator=g).to(torch.bfloat16).to(cuda) for _ in range(2))
    a.ensure_capacity("pad", 20)
    a.ensure_capacity("s", 40)
    for layer in range(2):
        a.write(layer, "s", 0, k[:20] * (layer + 1), v[:20])
        a.write(layer, "s", 20, k[20:] * (layer + 1), v[20:])
    a.advance("s", 37)
    b.ensure_capacity("other", 50)
    b.import_sequence("s", a.export_sequence("s"))
    transfer_sequence(a, c, "s")
    for layer in range(2):
        want = a.gather(layer, "s", 37)
        for x, y in zip(want, (k * (layer + 1), v)):
            # 8 bits: half a step of 2^-4, or of the least step of a block whose largest value is below 8
            assert ((x - y).abs() <= 2.0**-4 * y.abs() + 2.0**-10 * 2.0**-5).all()
        for other in (b, c):
            for x, y in zip(want, other.gather(layer, "s", 37)):
                assert torch.equal(x, y)
        assert a.gather(layer, "s", 5, dtype=torch.float32)[0].dtype == torch.float32
    transfer = a.export_sequence("s")
    assert (transfer.keys.view(torch.uint8)[:, 2, 5:] == 0).all()  # rows behind the sequence
    with pytest.raises(ValueError, match="scales"):
        import dataclasses

        b.import_sequence("t", dataclasses.replace(transfer, key_scales=None))
    with pytest.raises(ValueError, match="share a dtype"):
        a.write(0, "s", 0, k[:2], v[:2].float())
    with pytest.raises(TypeError):
        a.write(0, "s", 0, k[:2].double(), v[:2].double())
    ops.check_device_errors(cuda)


def test_score_matches_the_models_logits(cuda):
    model, cfg = llama(cuda)
    prompts = prompts_for(cfg, cuda, (2, 90, 33))
    for dtype in (torch.bfloat16, F8):
        cache = cache_for(cfg, cuda, dtype)
        ids = ("a", "b", "c")
        got = paged_score(model, prompts, cache, ids, top=3, chunk_size=40)
        other = cache_for(cfg, cuda, dtype)
        for s, p, r in zip(ids, prompts, got):
            n = p.shape[1]
            assert cache.get_sequence_length(s) == n and r.logprobs.shape == (n - 1,) and r.top_ids.shape == (n - 1, 3)
            with torch.inference_mode():
                logits = torch.cat([model(p[:, at : at + 40], kv_cache=other, sequence_id=s)[0] for at in range(0, n, 40)])
            want = torch.log_softmax(logits[:-1].double(), dim=1)
            picked = want.gather(1, p[0, 1:, None])[:, 0]
            assert ((r.logprobs.double() - picked).abs() <= 2.0**-20 * (16 + picked.abs())).all()
            assert torch.equal(r.top_ids, torch.sort(logits[:-1].double(), dim=1, descending=True, stable=True).indices[:, :3])
    with pytest.raises(ValueError, match="two tokens"):
        paged_score(model, (prompts[0][:, :1],), cache_for(cfg, cuda), ("a",))
    small = cache_for(cfg, cuda, blocks=2)
    with pytest.raises(ValueError, match="not enough free blocks"):
        paged_score(model, prompts, small, ("a", "b", "c"))
    assert small.allocator.free_block_count == 2


def test_eight_bits_change_little(cuda):
    """Codes are within 2^-4 of the values, independently: the mean score of 400 tokens moves by far less than 2^-4."""
    model, cfg = llama(cuda)
    prompts = prompts_for(cfg, cuda, (400,))
    a = paged_score(model, prompts, cache_for(cfg, cuda, torch.bfloat16), ("a",))[0].logprobs.mean()
    b = paged_score(model, prompts, cache_for(cfg, cuda, F8), ("a",))[0].logprobs.mean()
    assert abs(float(a - b)) < 2.0**-4
