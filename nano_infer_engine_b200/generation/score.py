"""Log probabilities of prompts through the paged model (no reference counterpart).

Perplexity, the ``logprobs`` of an echoed prompt, or what an 8-bit cache does to a
model's answers next to the same prompts through a bf16 cache.
"""

from __future__ import annotations

import torch

from .. import ops
from ..paged_cache import PagedKVCache
from .paged_prefill import _validate_paged_prefill_inputs


@torch.inference_mode()
def paged_score(
    model,
    prompts: tuple[torch.Tensor, ...],
    paged_cache: PagedKVCache,
    sequence_ids: tuple[str, ...],
    *,
    top: int = 0,
    chunk_size: int = 2048,
) -> tuple[ops.TokenLogprobs, ...]:
    """Score each prompt ``[1, n]`` (n >= 2): row ``i`` of its result is token ``i + 1`` given the tokens up to ``i``.

    Prompts are prefilled in chunks of ``chunk_size`` tokens, so that the logits of one chunk are
    alive at a time.  The sequences stay in the cache, as after ``paged_prefill``; if one fails, all
    are released and the error is raised.
    """
    _validate_paged_prefill_inputs(prompts, paged_cache, sequence_ids)
    if isinstance(chunk_size, bool) or not isinstance(chunk_size, int) or chunk_size <= 0:
        raise ValueError("chunk_size must be a positive integer")
    if isinstance(top, bool) or not isinstance(top, int) or not 0 <= top <= ops.LOGPROBS_MAX_TOP:
        raise ValueError(f"top must be an integer in [0, {ops.LOGPROBS_MAX_TOP}]")
    if any(p.shape[1] < 2 for p in prompts):
        raise ValueError("each prompt must contain at least two tokens to score")
    bs = paged_cache.block_size
    if sum(-(-p.shape[1] // bs) for p in prompts) > paged_cache.allocator.free_block_count:
        raise ValueError("not enough free blocks")
    scores = []
    try:
        for prompt, sequence_id in zip(prompts, sequence_ids):
            n = prompt.shape[1]
            parts = []
            for at in range(0, n, chunk_size):
                logits = model(prompt[:, at : at + chunk_size], kv_cache=paged_cache, sequence_id=sequence_id)[0]
                following = prompt[0, at + 1 : at + 1 + logits.shape[0]]
                if following.numel():
                    parts.append(ops.token_logprobs(logits[: following.numel()], following, top=top))
            scores.append(parts[0] if len(parts) == 1 else ops.TokenLogprobs(
                torch.cat([p.logprobs for p in parts]),
                torch.cat([p.entropy for p in parts]),
                torch.cat([p.top_logprobs for p in parts]),
                torch.cat([p.top_ids for p in parts]),
            ))
    except Exception:
        for sequence_id in sequence_ids:
            try:
                paged_cache.release(sequence_id)
            except KeyError:
                pass
        raise
    return tuple(scores)
