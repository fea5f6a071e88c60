"""The append into the 8-bit cache where a block's rows are not neighbours in the call: the scale and
the codes of a block are a matter of the call's rows, whatever their order."""

from __future__ import annotations

import math

import pytest
import torch

from vflorence_b200 import _native as N
from vflorence_b200 import paged_ops as ops

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def append_call(x, cache, scale, slots):
    """The append's definition for the blocks of a call, in float32 on the host (in place)."""
    bs = cache.shape[2]
    slots = torch.as_tensor(slots)
    real = slots >= 0
    x, slots = x.float()[real], slots[real]
    for b in torch.unique(slots // bs).tolist():
        at = slots // bs == b
        part, offs = x[at], slots[at] % bs
        a = torch.where(part.isfinite(), part.abs(), 0.0).amax(-1).amax(0)
        want = a * torch.tensor(1.0 / 127.0, dtype=F32)
        want = torch.where(want < 2.0 ** -100, 0.0, want)
        fresh = bool((offs == 0).any())
        old = torch.zeros_like(scale[b]) if fresh else torch.where(scale[b] > 0, scale[b], 0.0)
        new = torch.maximum(old, want)
        inv = torch.where(new > 0, 1.0 / new, 0.0)
        if not fresh:
            ratio = torch.where(new > old, old * inv, 1.0)
            cache[b] = (cache[b].float() * ratio[:, None, None]).round().to(torch.int8)
        codes = (part * inv[None, :, None]).nan_to_num(0.0, math.inf, -math.inf).round().clamp(-127, 127)
        cache[b][:, offs] = codes.to(torch.int8).transpose(0, 1)
        scale[b] = new


def stale_cache(n, h, bs, d, seed):
    """What earlier owners left: codes everywhere, scales from far below to far above the new tokens'."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-127, 128, (2, n, h, bs, d), generator=g, dtype=torch.int8)
    scale = 0.02 * 10.0 ** (torch.rand((2, n, h), generator=g) * 4 - 2)
    return [codes[0].clone(), codes[1].clone(), scale[0].clone(), scale[1].clone()]


def check(slots, h, d, bs, dtype, seed=0, touch=None):
    slots = torch.as_tensor(slots)
    n = int(slots.max()) // bs + 2
    g = torch.Generator().manual_seed(seed)
    size = 10.0 ** (torch.rand((slots.numel(), 1, 1), generator=g) * 2 - 1)
    key, value = ((torch.randn((slots.numel(), h, d), generator=g) * size).to(dtype) for _ in range(2))
    if touch is not None:
        touch(key, value)
    cache = stale_cache(n, h, bs, d, seed + 1)
    dev = [t.cuda() for t in cache]
    ops.reshape_and_cache_int8(key.cuda(), value.cuda(), *dev, slots.cuda())
    append_call(key, cache[0], cache[2], slots)
    append_call(value, cache[1], cache[3], slots)
    for got, want, what in zip(dev, cache, ("K codes", "V codes", "K scales", "V scales")):
        assert torch.equal(got.cpu(), want), what


def time_major(requests, first, tokens, bs, seed=0):
    """Slots of `tokens` tokens of each request from position first[i] on, all requests' token 0
    first, then all requests' token 1, in blocks of their own in random order."""
    per = max(-(-(f + tokens) // bs) for f in first)
    perm = torch.randperm(requests * per, generator=torch.Generator().manual_seed(seed)).tolist()
    return [perm[i * per + (first[i] + t) // bs] * bs + (first[i] + t) % bs
            for t in range(tokens) for i in range(requests)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("slots", [
    [0, -1, 1],                                   # a padding row in a new block
    [17, -1, 16, -1, 18],                         # its first slot in the middle
    [33, 0, 34, 1, 32, 2],                        # two new blocks in turn, one's first slot last
    [5, 20, 6, 21, 7, 22],                        # two blocks that go on
    [5, 20, 6, 16, 7, 22],                        # one goes on, one starts anew
    list(range(15, 0, -1)) + [16, 0],             # backwards, the first slot after another block
    list(range(16)) + [16] + list(range(32, 48)) + [17],  # whole blocks between
])
def test_rows_of_a_block_apart(slots, dtype):
    for seed in range(4):
        check(slots, 8, 64, 16, dtype, seed)


@pytest.mark.parametrize("h,d", [(1, 16), (3, 80), (5, 128), (12, 64)])
@pytest.mark.parametrize("requests,tokens", [(3, 40), (64, 20), (130, 33)])
def test_time_major_prompts(h, d, requests, tokens):
    """Every run is one row. Up to 4290 rows: more than one look of a CTA, windows of several rows."""
    check(time_major(requests, [0] * requests, tokens, 16), h, d, 16, BF16, requests)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bs", [16, 48, 64, 80, 256])
def test_time_major_continuations(dtype, bs):
    """Requests that start inside a block, in blocks of up to more slots than a word has bits."""
    check(time_major(37, [(5 * i) % bs for i in range(37)], 90, bs), 4, 64, bs, dtype, bs)


@pytest.mark.parametrize("gap", [1023, 1024, 1025, 5000])
def test_rows_of_a_block_far_apart(gap):
    """A block's first rows and its last ones with `gap` rows of other blocks between, both ways."""
    between = list(range(32, 32 + gap))
    check([3, 4] + between + [5, 0, 17], 2, 32, 16, BF16, gap)
    check([0, 17] + between + [16, 4, 5], 2, 32, 16, F32, gap)


def test_non_finite_values_among_rows_apart():
    def touch(key, value):
        key[4, 1, 3], key[1, 0, 0], value[3, 2, 7] = math.inf, -math.inf, math.nan
        value[0] = math.nan

    ops.read_device_errors()
    for slots in ([16, 0, 17, 1, 18, 2], [19, 0, 20, 1, 21, 2]):
        check(slots, 4, 48, 16, BF16, 7, touch)
        assert ops.read_device_errors() == N.DEVERR_NONFINITE


def test_the_same_codes_whatever_the_order_of_the_rows():
    h, d, bs, t = 4, 64, 16, 200
    g = torch.Generator().manual_seed(3)
    slots = torch.randperm(20 * bs, generator=g)[:t]
    key, value = (torch.randn((t, h, d), generator=g) for _ in range(2))
    cache = stale_cache(20, h, bs, d, 9)
    results = []
    for order in (torch.arange(t), torch.randperm(t, generator=g), slots.argsort()):
        dev = [x.cuda() for x in cache]
        ops.reshape_and_cache_int8(key[order].cuda(), value[order].cuda(), *dev, slots[order].cuda())
        results.append([x.cpu() for x in dev])
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


@pytest.mark.parametrize("share", [False, True])
def test_many_runs_of_few_rows(share):
    """Two rows a block, thousands of rows apart, replayed from a CUDA graph. `share`: the blocks' numbers
    all meet in one table of those by which the runs are told apart, more than it holds."""
    h, d, bs, blocks = 8, 16, 16, 4000
    pool = torch.arange(1, 50000 if share else blocks + 1)
    if share:
        pool = pool[(pool * 2654435761 >> 12) % 8 == 5][:blocks]
    assert pool.numel() == blocks
    n = int(pool.max()) + 1
    g = torch.Generator().manual_seed(1)
    blk = torch.cat([pool[torch.randperm(blocks, generator=g)] for _ in range(2)])
    off = torch.cat([torch.randint(1, 8, (blocks,), generator=g), torch.randint(8, 16, (blocks,), generator=g)])
    key, value = (torch.randn((2 * blocks, h, d), generator=g).to(BF16).cuda() for _ in range(2))
    blk, off = blk.cuda(), off.cuda()
    codes = [torch.zeros((n, h, bs, d), dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros((n, h), device="cuda") for _ in range(2)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.reshape_and_cache_int8(key, value, *codes, *scales, blk * bs + off)
    graph.replay()
    for x, c, s in ((key, codes[0], scales[0]), (value, codes[1], scales[1])):
        x = x.float()
        a = torch.zeros((n, h), device="cuda").index_reduce_(0, blk, x.abs().amax(-1), "amax")
        want_s = a * torch.tensor(1.0 / 127.0, device="cuda")
        inv = torch.where(want_s > 0, 1.0 / want_s, 0.0)
        want = torch.zeros_like(c)
        want[blk, :, off] = (x * inv[blk][..., None]).round().clamp(-127, 127).to(torch.int8)
        assert torch.equal(s, want_s) and torch.equal(c, want)
