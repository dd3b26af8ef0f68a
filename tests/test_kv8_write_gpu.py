"""PagedKVCache.write of an 8-bit cache at any position: the rows around the new ones keep their values."""

import pytest
import torch

from nano_infer_engine_b200 import ops
from nano_infer_engine_b200.paged_cache import PagedKVCache, transfer_sequence

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
BS, H, D = 16, 2, 64


def new_cache(cuda, blocks=12):
    return PagedKVCache(blocks, BS, 2, H, D, F8, cuda)


class Mirror:
    """A cache's sequence and the values that it should hold."""

    def __init__(self, cache, name, capacity, dtype=torch.bfloat16, seed=0):
        self.cache, self.name, self.dtype = cache, name, dtype
        self.g = torch.Generator(device=cache.device).manual_seed(seed)
        cache.ensure_capacity(name, capacity)
        self.held = [{}, {}]  # per layer: position -> key and value
        self.top = [{}, {}]  # and the largest scales of its block [2, H] since they were written

    def write(self, start, count, size, layers=(0, 1)):
        for layer in layers:
            k, v = (size * torch.randn(count, H, D, device=self.cache.device, generator=self.g) for _ in range(2))
            k, v = k.to(self.dtype), v.to(self.dtype)
            self.cache.write(layer, self.name, start, k, v)
            for j in range(count):
                self.held[layer][start + j] = (k[j].double(), v[j].double())
                self.top[layer].pop(start + j, None)
            self.note(layer)

    def note(self, layer):
        for pos in self.held[layer]:
            block = self.cache.get_block_table(self.name)[pos // BS]
            now = torch.stack([self.cache.key_scales[layer, block], self.cache.value_scales[layer, block]]).double()
            self.top[layer][pos] = torch.maximum(self.top[layer].get(pos, now), now)

    def check(self):
        """A value is rounded to 3 bits (2^-4 of it) or to a multiple of the least step, off by 2^-10 s at a scale s;
        again where its block's scale grows: 2^-10 s_1 + 2^-10 s_2 + ... < 2^-9 s for scales that at least double up
        to s.  Where the scale falls the stored value keeps its place, and so it does where the scale grows again up to
        where it was: it is a multiple of that scale's least step by then, or has 3 bits.  So s is the largest
        scale that the block has had since (not its present one, by which the first form of this test went: a
        fall does not bring back what the rounding took)."""
        for layer, held in enumerate(self.held):
            if not held:
                continue
            got = self.cache.gather(layer, self.name, max(held) + 1, dtype=torch.float32)
            for kv in range(2):
                for pos, want in held.items():
                    d = (got[kv][pos].double() - want[kv]).abs()
                    s = self.top[layer][pos][kv][:, None]
                    assert (d <= 2.0**-4 * want[kv].abs() + 2.0**-9 * s).all(), (layer, kv, pos)
        ops.check_device_errors(self.cache.device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_the_second_half_of_a_block_before_the_first(cuda, dtype):
    for sizes in ((1.0, 4.0), (4.0, 1.0), (1.0, 1000.0), (1000.0, 1.0)):
        m = Mirror(new_cache(cuda), "s", 16, dtype)
        m.write(8, 8, sizes[0])
        m.write(0, 8, sizes[1])
        m.check()


@pytest.mark.parametrize("at, count", [(3, 1), (0, 1), (15, 1), (0, 16), (4, 9)])
def test_tokens_of_a_full_block_written_again(cuda, at, count):
    for size in (16.0, 1.0, 1 / 16):
        m = Mirror(new_cache(cuda), "s", 40, seed=at)
        m.write(0, 40, 1.0)
        for c in (False, True):
            if c:
                m.cache.advance("s", 40)
            m.write(16 + at, count, size)
            m.check()


def test_a_scale_falls_with_the_loud_token_that_needed_it(cuda):
    """Written from its first slot, a block's scale is what its tokens need: quiet ones are no zeros."""
    m = Mirror(new_cache(cuda), "s", 16)
    m.write(0, 12, 1.0)
    m.write(2, 1, 1e6)
    m.check()
    m.write(0, 12, 1.0)
    m.check()
    assert (m.cache.key_scales[:, m.cache.get_block_table("s")[0]] < 2.0**-4).all()


def test_a_run_over_several_blocks_that_ends_inside_one(cuda):
    m = Mirror(new_cache(cuda), "s", 60)
    m.write(0, 50, 1.0)
    m.write(5, 20, 30.0)  # 5 .. 24: 25 .. 31 stay
    m.check()
    m.write(48, 12, 8.0)  # past what was stored
    m.check()


def test_a_block_that_another_sequence_had(cuda):
    """A first write inside a block is not bound to the scale of the block's owner before."""
    cache = new_cache(cuda, blocks=1)
    loud = Mirror(cache, "loud", 16)
    loud.write(0, 16, 1e9)
    cache.release("loud")
    m = Mirror(cache, "quiet", 16, seed=1)
    m.write(5, 4, 1e-3)
    m.check()
    assert (cache.key_scales < 2.0**-12).all()
    m.write(0, 5, 1e-3)
    m.write(9, 2, 1.0)
    m.check()


def test_layers_have_their_own_state(cuda):
    m = Mirror(new_cache(cuda), "s", 32)
    m.write(8, 8, 1.0, layers=(0,))
    m.write(0, 8, 50.0, layers=(0,))
    m.write(0, 20, 1.0, layers=(1,))
    m.write(3, 2, 50.0, layers=(1,))
    m.check()


def test_after_a_hand_over(cuda):
    a, b, c = new_cache(cuda), new_cache(cuda), new_cache(cuda)
    m = Mirror(a, "s", 37)
    m.write(0, 37, 1.0)
    a.advance("s", 37)
    b.import_sequence("s", a.export_sequence("s"))
    transfer_sequence(a, c, "s")
    for cache in (b, c):
        other = Mirror(cache, "s", 37, seed=2)
        other.held, other.top = [dict(h) for h in m.held], [dict(t) for t in m.top]
        other.write(32, 2, 40.0)
        other.write(17, 3, 40.0)
        other.check()


@pytest.mark.parametrize("seed", range(4))
def test_writes_in_any_order(cuda, seed):
    g = torch.Generator().manual_seed(seed)
    m = Mirror(new_cache(cuda), "s", 90, seed=seed)
    for _ in range(14):
        at = int(torch.randint(0, 90, (1,), generator=g))
        count = min(90 - at, int(torch.randint(1, 24, (1,), generator=g)))
        m.write(at, count, float(2.0 ** torch.randint(-6, 7, (1,), generator=g)))
        m.check()
