"""What the 8-bit cache's calls and token_logprobs refuse, and the plain forms themselves; no GPU."""

import pytest
import torch

import kv8_plain as plain
from nano_infer_engine_b200 import _native, ops

BF16 = torch.bfloat16


def cache(L=1, nb=4, bs=16, h=2, d=64):
    kc, vc = (torch.zeros(L, nb, bs, h, d, dtype=torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.ones(L, nb, h) for _ in range(2))
    return kc, vc, ks, vs


def append_args(T=3, hq=4, h=2, d=64, dtype=BF16):
    kc, vc, ks, vs = cache(h=h, d=d)
    return dict(q=torch.zeros(T, hq * d, dtype=dtype), k=torch.zeros(T, h * d, dtype=dtype), v=torch.zeros(T, h * d, dtype=dtype),
                sin=torch.zeros(T, d // 2, dtype=dtype), cos=torch.zeros(T, d // 2, dtype=dtype), key_cache=kc, value_cache=vc,
                key_scales=ks, value_scales=vs, layer=0, slot_mapping=torch.zeros(T, dtype=torch.int64), q_heads=hq)


@pytest.mark.parametrize("change, message", [
    (dict(q=torch.zeros(3, 128, dtype=BF16)), "q/k/v must be"),
    (dict(k=torch.zeros(2, 128, dtype=BF16)), "q/k/v must be"),
    (dict(v=torch.zeros(3, 128)), "q/k/v must be"),
    (dict(v=torch.zeros(128, 3, dtype=BF16).T), "q/k/v must be"),
    (dict(sin=torch.zeros(3, 32)), "sin/cos"),
    (dict(cos=torch.zeros(3, 64, dtype=BF16)), "sin/cos"),
    (dict(slot_mapping=torch.zeros(2, dtype=torch.int64)), "slot_mapping"),
    (dict(slot_mapping=torch.zeros(3, dtype=torch.int32)), "slot_mapping"),
    (dict(slot_mapping=torch.zeros(6, dtype=torch.int64)[::2]), "slot_mapping"),
    (dict(key_cache=torch.zeros(1, 4, 16, 2, 64, dtype=BF16)), "float8_e4m3fn"),
    (dict(value_cache=torch.zeros(1, 4, 16, 2, 32, dtype=torch.float8_e4m3fn)), "share a shape"),
    (dict(key_scales=torch.ones(1, 4, 3)), "scales must be"),
    (dict(value_scales=torch.ones(1, 4, 2, dtype=torch.float64)), "scales must be"),
    (dict(value_scales=torch.ones(1, 2, 4).transpose(1, 2)), "scales must be"),
])
def test_append_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        ops.rope_write_kv8(**{**append_args(), **change})


def test_append_refuses_layers_types_and_cpu_tensors():
    with pytest.raises(IndexError):
        ops.rope_write_kv8(**{**append_args(), "layer": 1})
    with pytest.raises(TypeError, match="unsupported dtype"):
        ops.rope_write_kv8(**append_args(dtype=torch.float64))
    with pytest.raises(RuntimeError, match="require CUDA"):
        ops.rope_write_kv8(**append_args())
    kc, vc, ks, vs = cache()
    x = torch.zeros(3, 2, 64, dtype=BF16)
    slots = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="require CUDA"):
        ops.write_kv8(x, x, kc, vc, ks, vs, 0, slots)
    with pytest.raises(ValueError, match="keys/values"):
        ops.write_kv8(x, x.float(), kc, vc, ks, vs, 0, slots)
    with pytest.raises(ValueError, match="keys/values"):
        ops.write_kv8(x[:, :1], x[:, :1], kc, vc, ks, vs, 0, slots)
    table = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="num_tokens"):
        ops.gather_kv8(kc, vc, ks, vs, 0, table, 33)
    with pytest.raises(ValueError, match="block_table"):
        ops.gather_kv8(kc, vc, ks, vs, 0, table.long(), 3)
    with pytest.raises(TypeError):
        ops.gather_kv8(kc, vc, ks, vs, 0, table, 3, dtype=torch.int8)


def attention_args(T=2, hq=4):
    kc, vc, ks, vs = cache()
    return dict(query=torch.zeros(T, hq, 64, dtype=BF16), key_cache=kc, value_cache=vc, key_scales=ks, value_scales=vs, layer=0,
                block_tables=torch.zeros(2, 3, dtype=torch.int32), seq_lens=torch.ones(2, dtype=torch.int32))


BAD_ATTENTION = [
    (dict(query=torch.zeros(2, 4, 32, dtype=BF16)), "query must be"),
    (dict(query=torch.zeros(2, 64, 4, dtype=BF16).transpose(1, 2)), "query must be"),
    (dict(query=torch.zeros(2, 3, 64, dtype=BF16)), "multiple of kv_heads"),
    (dict(block_tables=torch.zeros(2, 3, dtype=torch.int64)), "block_tables"),
    (dict(block_tables=torch.zeros(1, 3, dtype=torch.int32)), "a row per request"),
    (dict(block_tables=torch.zeros(1, 3, dtype=torch.int32).expand(2, 3)), "do not overlap"),
    (dict(seq_lens=torch.ones(2, dtype=torch.int64)), "seq_lens"),
    (dict(out=torch.zeros(2, 4, 64)), "out must"),
    (dict(out=torch.zeros(3, 4, 64, dtype=BF16)), "out must"),
    (dict(table_rows=torch.zeros(1, dtype=torch.int32)), "table_rows"),
    (dict(table_rows=torch.zeros(2, dtype=torch.int64)), "table_rows"),
    (dict(req_list=torch.zeros(2, dtype=torch.int64)), "req_list"),
    (dict(num_requests=3), "num_requests"),
    (dict(req_list=torch.zeros(1, dtype=torch.int32), num_requests=2), "num_requests"),
    (dict(key_scales=torch.ones(2, 4, 2)), "scales must be"),
]


@pytest.mark.parametrize("change, message", BAD_ATTENTION)
def test_attention_refuses(change, message):
    args = {**attention_args(), **change}
    with pytest.raises(ValueError, match=message):
        ops.paged_decode_kv8(**args)
    with pytest.raises(ValueError, match=message):
        ops.varlen_attention_kv8(**args, query_start_loc=torch.tensor([0, 1, 2]), max_query_len=1)


def test_attention_refuses_rows_and_boundaries():
    args = attention_args()
    with pytest.raises(ValueError, match="q_rows"):
        ops.paged_decode_kv8(**args, q_rows=torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="query_start_loc"):
        ops.varlen_attention_kv8(**args, query_start_loc=torch.tensor([0, 2]), max_query_len=1)
    with pytest.raises(ValueError, match="max_query_len"):
        ops.varlen_attention_kv8(**args, query_start_loc=torch.tensor([0, 1, 2]), max_query_len=0)
    with pytest.raises(RuntimeError, match="require CUDA"):
        ops.paged_decode_kv8(**args)


@pytest.mark.parametrize("change, message", [
    (dict(logits=torch.zeros(4)), "logits must be"),
    (dict(logits=torch.zeros(9, 4).T), "logits must be"),
    (dict(logits=torch.zeros(4, 0)), "logits must be"),
    (dict(tokens=torch.zeros(3, dtype=torch.int64)), "tokens must be"),
    (dict(tokens=torch.zeros(4, dtype=torch.int32)), "tokens must be"),
    (dict(top=-1), "top must be"),
    (dict(top=10), "top must be"),
    (dict(top=True), "top must be"),
    (dict(top=2.0), "top must be"),
    (dict(logits=torch.zeros(4, 100), top=33), "top must be"),
])
def test_logprobs_refuse(change, message):
    args = {**dict(logits=torch.zeros(4, 9), tokens=torch.zeros(4, dtype=torch.int64), top=0), **change}
    with pytest.raises(ValueError, match=message):
        ops.token_logprobs(args["logits"], args["tokens"], top=args["top"])


def test_logprobs_refuse_types_and_cpu_tensors():
    tokens = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(TypeError, match="unsupported dtype"):
        ops.token_logprobs(torch.zeros(4, 9, dtype=torch.float64), tokens)
    with pytest.raises(RuntimeError, match="require CUDA"):
        ops.token_logprobs(torch.zeros(4, 9), tokens)


def test_c_entries_refuse_before_any_launch():
    lib, bad = _native.lib, _native.NIE_ERR_INVALID
    fake = 4096
    assert lib.nie_token_logprobs(fake, 1, 9, 9, 1, fake, 33, fake, fake, fake, fake, None, None) == bad
    assert lib.nie_token_logprobs(fake, 1, 9, 8, 1, fake, 1, fake, fake, fake, fake, None, None) == bad
    assert lib.nie_token_logprobs(None, 1, 9, 9, 1, fake, 1, fake, fake, fake, fake, None, None) == bad
    assert lib.nie_token_logprobs(fake, 1, 9, 9, 7, fake, 1, fake, fake, fake, fake, None, None) == bad
    assert lib.nie_token_logprobs(fake, 0, 9, 9, 1, fake, 1, fake, fake, fake, fake, None, None) == _native.NIE_OK
    rope = [fake, 1, fake, 1, fake, 1, fake, fake, 3, 4, 2, 64, fake, fake, fake, fake, fake, 1, 0, 1, 4, 16, fake, None, None]
    for at, value in ((0, None), (8, -1), (9, 0), (11, 63), (11, 0), (17, 5), (18, 1), (18, -1), (20, 0), (21, 0), (22, None)):
        assert lib.nie_rope_write_kv8(*rope[:at], value, *rope[at + 1 :]) == bad, (at, value)
    assert lib.nie_rope_write_kv8(*rope[:8], 0, *rope[9:]) == _native.NIE_OK


# ------------------------------------------------------------------ the plain forms
def test_least_scale_holds_the_largest_value_and_no_smaller_one_does():
    for x in (1e-20, 1e-10, 1.75, 1.7500001, 447.9, 448.0, 448.0001, 3e4, 1e17, 1e30):
        s = plain.least_scale(x)
        assert plain.SCALE_MIN <= s <= plain.SCALE_MAX
        if plain.SCALE_MIN < s < plain.SCALE_MAX:
            assert x <= 448 * s and x > 448 * s / 2
    assert plain.least_scale(0.0) == plain.SCALE_MIN


def test_runs():
    assert plain.runs_of([3, 4, 5, 8, 9, -1, 10, 16, 2, 40], 4, 32) == [(0, 1), (1, 2), (3, 2), (6, 1), (7, 1), (8, 1)]


# ------------------------------------------------------------------ the cache's bookkeeping
def test_an_8_bit_cache_has_scales_and_others_have_none():
    from nano_infer_engine_b200.paged_cache import PagedKVCache

    c = PagedKVCache(8, 16, 2, 4, 64, torch.float8_e4m3fn, "cpu")
    assert c.quantized and c.key_scales.shape == c.value_scales.shape == (2, 8, 4) and c.keys.element_size() == 1
    d = PagedKVCache(8, 16, 2, 4, 64, BF16, "cpu")
    assert not d.quantized and d.key_scales is None and d.value_scales is None
    with pytest.raises(ValueError, match="even head_dim"):
        PagedKVCache(8, 16, 2, 4, 63, torch.float8_e4m3fn, "cpu")
    d.ensure_capacity("s", 3)
    with pytest.raises(ValueError, match="only an 8-bit cache"):
        d.gather(0, "s", 2, dtype=torch.float32)


def test_processes_do_not_hand_8_bit_pools_over():
    from nano_infer_engine_b200.generation.pd_disagg import export_pool
    from nano_infer_engine_b200.paged_cache import PagedKVCache

    with pytest.raises(ValueError, match="8-bit caches"):
        export_pool(PagedKVCache(8, 16, 2, 4, 64, torch.float8_e4m3fn, "cpu"))


def test_score_refuses_before_it_touches_the_cache():
    from nano_infer_engine_b200.generation.score import paged_score
    from nano_infer_engine_b200.paged_cache import PagedKVCache

    c = PagedKVCache(8, 16, 1, 1, 8, BF16, "cpu")
    prompt = torch.zeros(1, 5, dtype=torch.int64)
    for change, message in ((dict(chunk_size=0), "chunk_size"), (dict(chunk_size=True), "chunk_size"), (dict(top=33), "top"),
                            (dict(top=1.0), "top")):
        with pytest.raises(ValueError, match=message):
            paged_score(None, (prompt,), c, ("a",), **change)
    with pytest.raises(ValueError, match="two tokens"):
        paged_score(None, (prompt[:, :1],), c, ("a",))

    class Broken:
        def __call__(self, x, kv_cache, sequence_id):
            kv_cache.ensure_capacity(sequence_id, 5)
            raise RuntimeError("no")

    with pytest.raises(RuntimeError, match="no"):
        paged_score(Broken(), (prompt, prompt), c, ("a", "b"))
    assert c.allocator.free_block_count == 8
