"""The paged cache held in 8 bits on the GPU: append and read-back against a restatement of the
quantiser, attention against the 64-bit definition on the same codes."""

from __future__ import annotations

import math

import pytest
import torch

from vflorence_b200 import _native as N
from vflorence_b200 import paged_ops as ops

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


# ------------------------------------------------------------------------------ the quantiser

def runs_of(slots, bs):
    """(first row, last row + 1) of each run of neighbouring rows in one block."""
    out, i = [], 0
    while i < len(slots):
        if slots[i] < 0:
            i += 1
            continue
        j = i + 1
        while j < len(slots) and slots[j] >= 0 and slots[j] // bs == slots[i] // bs:
            j += 1
        out.append((i, j))
        i = j
    return out


def append_plain(x, cache, scale, slots):
    """The append's definition, run by run, in float32 on the host (in place)."""
    bs = cache.shape[2]
    slots = slots.tolist()
    x = x.float()
    for i, j in runs_of(slots, bs):
        b, offs = slots[i] // bs, [s % bs for s in slots[i:j]]
        part = x[i:j]
        a = torch.where(part.isfinite(), part.abs(), 0.0).amax(-1).amax(0)
        want = a * torch.tensor(1.0 / 127.0, dtype=F32)
        want = torch.where(want < 2.0 ** -100, 0.0, want)
        fresh = 0 in offs
        old = torch.zeros_like(scale[b]) if fresh else torch.where(scale[b] > 0, scale[b], 0.0)
        new = torch.maximum(old, want)
        inv = torch.where(new > 0, 1.0 / new, 0.0)
        if not fresh:
            grown = new > old
            ratio = torch.where(grown, old * inv, 1.0)
            cache[b] = (cache[b].float() * ratio[:, None, None]).round().to(torch.int8)
        codes = (part * inv[None, :, None]).nan_to_num(0.0, math.inf, -math.inf).round().clamp(-127, 127)
        for t, o in enumerate(offs):
            cache[b, :, o] = codes[t].to(torch.int8)
        scale[b] = new


def new_cache(n, h, bs, d, gen=None):
    gen = gen or torch.Generator().manual_seed(1)
    codes = torch.randint(-127, 128, (2, n, h, bs, d), generator=gen, dtype=torch.int8)
    scale = (0.5 + torch.rand((2, n, h), generator=gen)) * 0.02
    return codes[0].clone(), codes[1].clone(), scale[0].clone(), scale[1].clone()


def check_append(key, value, slots, cache):
    """Append on the GPU and by the definition: codes and scales equal bit for bit."""
    dev = [t.cuda() for t in cache]
    ops.reshape_and_cache_int8(key.cuda(), value.cuda(), *dev, slots.cuda())
    append_plain(key, cache[0], cache[2], slots)
    append_plain(value, cache[1], cache[3], slots)
    for got, want, what in zip(dev, cache, ("K codes", "V codes", "K scales", "V scales")):
        assert torch.equal(got.cpu(), want), what
    return dev


def rows(t, h, d, dtype, seed=0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((t, h, d), generator=g) * size).to(dtype), torch.randn((t, h, d), generator=g).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [16, 32, 48, 64, 80, 128, 512])
@pytest.mark.parametrize("bs", [16, 48])
def test_append_matches_the_definition_bit_for_bit(dtype, d, bs):
    """New blocks, partly filled blocks that grow or keep their scale, padding rows, odd lengths."""
    h, n = 3, 40
    gen = torch.Generator().manual_seed(d + bs)
    perm = torch.randperm(n, generator=gen).tolist()
    slots = []
    slots += [perm[0] * bs + o for o in range(bs)]              # a whole block
    slots += [perm[1] * bs + o for o in range(5)]               # a block's first tokens
    slots += [-1, -1]
    slots += [perm[2] * bs + o for o in range(7, bs)]           # the rest of a block
    slots += [perm[3 + i] * bs + (3 * i + 1) % bs for i in range(20)]  # one token each
    slots += [perm[30] * bs + bs - 1, perm[31] * bs]            # a block's last slot, another's first
    slots = torch.tensor(slots)
    key, value = rows(len(slots), h, d, dtype, seed=d)
    key[30:40] *= 0.01   # some tokens below the stored step, some above
    check_append(key, value, slots, new_cache(n, h, bs, d, gen))


@pytest.mark.parametrize("tokens", [1, 2, 255, 2311])
def test_append_lengths_and_windows(tokens):
    """Few rows (one row a window) and many (runs that cross the windows' ends), bf16."""
    h, d, bs = 12, 64, 16
    n = tokens // bs + 3
    perm = torch.randperm(n, generator=torch.Generator().manual_seed(5))
    pos = torch.arange(tokens) + 5  # the first block is partly filled
    slots = perm[pos // bs] * bs + pos % bs
    key, value = rows(tokens, h, d, BF16, seed=tokens)
    check_append(key, value, slots, new_cache(n, h, bs, d))


def test_append_one_token_at_a_time_keeps_within_its_steps():
    """A block filled token by token: each growth rounds the older codes once more, so a value is
    at most half a final step for its own rounding and half a step for each later growth off."""
    h, d, bs, n = 4, 64, 16, 3
    key, value = rows(bs, h, d, F32, seed=9)
    key *= torch.linspace(0.2, 2.0, bs)[:, None, None]
    cache = [t.cuda() for t in new_cache(n, h, bs, d)]
    plain = [t.cpu().clone() for t in cache]
    grown = torch.zeros(h)
    for t in range(bs):
        before = plain[2][1].clone()
        slot = torch.tensor([bs + t])
        ops.reshape_and_cache_int8(key[t:t + 1].cuda(), value[t:t + 1].cuda(), *cache, slot.cuda())
        append_plain(key[t:t + 1], plain[0], plain[2], slot)
        append_plain(value[t:t + 1], plain[1], plain[3], slot)
        if t > 0:
            grown += (plain[2][1] > before).float()
    assert all(torch.equal(a.cpu(), b) for a, b in zip(cache, plain))
    k, _ = ops.gather_kv_int8(*cache, torch.arange(bs, 2 * bs).cuda(), F32)
    step = plain[2][1]
    off = (k.cpu() - key).abs().amax(-1) / step[None]
    assert (off <= 0.5 * (1 + grown)[None] + 1e-4).all()
    assert grown.max() >= 3  # the case grows


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_zero_tiny_huge_and_non_finite_values(dtype):
    h, d, bs, n = 2, 64, 16, 8
    key, value = rows(6, h, d, dtype, seed=3)
    key[0] = 0.0                       # a zero scale and zero codes
    key[1] *= 2.0 ** -110              # below the smallest scale: zeros
    key[2] *= 2.0 ** 120
    key[3, 0, 5], key[3, 1, 6] = math.inf, -math.inf
    value[4, 0, 7] = math.nan
    key[5] = math.inf                  # nothing finite: a zero scale
    slots = torch.arange(6) * bs       # each starts a block
    ops.read_device_errors()
    dev = check_append(key, value, slots, new_cache(n, h, bs, d))
    assert ops.read_device_errors() == N.DEVERR_NONFINITE
    k, v = ops.gather_kv_int8(*dev, slots.cuda(), F32)
    assert (k[0] == 0).all() and (k[1] == 0).all() and (k[5] == 0).all() and v[4, 0, 7] == 0
    assert k[3, 0, 5] > 0 and k[3, 1, 6] < 0 and torch.isfinite(k).all()


def test_append_reads_strided_rows():
    """key and value as slices of one fused projection."""
    h, d, bs, n, t = 12, 64, 16, 8, 37
    fused = torch.randn((t, 3 * h * d), generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    key, value = (x.reshape(t, h, d) for x in fused.chunk(3, -1)[1:])
    assert key.stride(0) == 3 * h * d
    pos = torch.arange(t)
    slots = torch.tensor([5, 2, 7])[pos // bs] * bs + pos % bs
    cache = new_cache(n, h, bs, d)
    dev = [x.cuda() for x in cache]
    ops.reshape_and_cache_int8(key, value, *dev, slots.cuda())
    append_plain(key.cpu(), cache[0], cache[2], slots)
    append_plain(value.cpu(), cache[1], cache[3], slots)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, cache))


def test_append_rows_of_a_block_that_are_not_neighbours():
    """Such runs are stored one after the other, in no set order: every value is within half a
    step for its rounding and half a step for each of the other runs' growths."""
    h, d, bs, n = 8, 64, 16, 4
    blocks, t = 3, 48
    slots = torch.tensor([(i % blocks) * bs + i // blocks for i in range(t)])  # blocks interleaved
    key, value = rows(t, h, d, F32, seed=11)
    dev = [x.cuda() for x in new_cache(n, h, bs, d)]
    dev[2].zero_(), dev[3].zero_()
    live = slots.clone()
    order = torch.arange(t)
    first = slots % bs == 0  # starting a block anew among other runs would drop theirs: keep them out
    ops.reshape_and_cache_int8(key[order[first]].cuda(), value[order[first]].cuda(), *dev, slots[first].cuda())
    ops.reshape_and_cache_int8(key[order[~first]].cuda(), value[order[~first]].cuda(), *dev, slots[~first].cuda())
    k, v = ops.gather_kv_int8(*dev, live.cuda(), F32)
    for got, want, scale in ((k, key, dev[2]), (v, value, dev[3])):
        step = scale.cpu()[live // bs]
        amax = want.abs().amax(-1).view(t // blocks, blocks, h).amax(0)
        assert torch.allclose(scale.cpu()[:blocks] * 127.0, amax, rtol=1e-6)
        assert ((got.cpu() - want).abs().amax(-1) <= step * (0.5 * bs)).all()
        assert ((got.cpu() - want).abs().mean(-1) <= step * 1.0).all()


def test_append_flags_slots_past_the_pool_and_takes_no_rows():
    h, d, bs, n = 2, 64, 16, 4
    cache = new_cache(n, h, bs, d)
    dev = [x.cuda() for x in cache]
    key, value = rows(3, h, d, BF16)
    ops.read_device_errors()
    slots = torch.tensor([n * bs, 17, 2 ** 40])
    ops.reshape_and_cache_int8(key.cuda(), value.cuda(), *dev, slots.cuda())
    assert ops.read_device_errors() == N.DEVERR_SLOT
    append_plain(key[1:2], cache[0], cache[2], slots[1:2])
    append_plain(value[1:2], cache[1], cache[3], slots[1:2])
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, cache))
    k, v = ops.gather_kv_int8(*dev, torch.tensor([-1, n * bs, 17]).cuda(), BF16)
    assert ops.read_device_errors() == N.DEVERR_SLOT
    assert (k[:2] == 0).all() and (v[:2] == 0).all() and (k[2] != 0).any()
    ops.reshape_and_cache_int8(key[:0].cuda(), value[:0].cuda(), *dev, slots[:0].cuda())
    k, v = ops.gather_kv_int8(*dev, slots[:0].cuda(), BF16)
    assert k.shape == (0, h, d) and ops.read_device_errors() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gather_is_code_times_scale_rounded_once(dtype):
    n, h, bs, d = 6, 5, 32, 48
    cache = new_cache(n, h, bs, d)
    dev = [x.cuda() for x in cache]
    slots = torch.randperm(n * bs, generator=torch.Generator().manual_seed(3))[:57]
    k, v = ops.gather_kv_int8(*dev, slots.cuda(), dtype)
    for got, codes, scale in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
        want = (codes[slots // bs, :, slots % bs].float() * scale[slots // bs][:, :, None]).to(dtype)
        assert torch.equal(got.cpu(), want)


def test_copy_blocks_carries_codes_and_scales():
    """A beam fork copies an 8-bit block with the copy the other pools use."""
    n, h, bs, d = 6, 4, 16, 64
    cache = new_cache(n, h, bs, d)
    dev = [x.cuda() for x in cache]
    ops.copy_blocks([dev[0]], [dev[1]], [(1, 4)])
    ops.copy_blocks([dev[2]], [dev[3]], [(1, 4)])
    for got, want in zip(dev, cache):
        assert torch.equal(got[4].cpu(), want[1]) and torch.equal(got[5].cpu(), want[5])


# ------------------------------------------------------------------------------- the attention

def attention_exact(q, cache, qsl, lens, table, scale, causal):
    """The definition in 64 bits, request by request, and each row's largest |v| (0: no token)."""
    kc, vc, ks, vs = cache
    hkv, bs = kc.shape[1], kc.shape[2]
    group = q.shape[1] // hkv
    out = torch.zeros(q.shape, dtype=torch.float64)
    top = torch.zeros(q.shape[:2], dtype=torch.float64)
    for r, n in enumerate(lens.tolist()):
        q0, q1 = int(qsl[r]), int(qsl[r + 1])
        if n == 0:
            continue
        blocks = table[r, : -(-n // bs)].long()
        k, v = ((c[blocks].double() * s[blocks].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :n]
                for c, s in ((kc, ks), (vc, vs)))
        for i in range(q0, q1):
            seen = n - (q1 - 1 - i) if causal else n
            if seen <= 0:
                continue
            for h in range(q.shape[1]):
                s = (k[h // group, :seen] @ q[i, h].double()) * scale
                out[i, h] = torch.softmax(s, 0) @ v[h // group, :seen]
                top[i, h] = v[h // group, :seen].abs().max()
    return out, top


@pytest.fixture(params=[0, 1, 2, 4])
def warps(request):
    """Warps a CTA: as planned, and each count."""
    return request.param


def attend(warps, q, cache, qsl, lens, table, scale, causal, planned=None, out=None):
    dev = [t.cuda() for t in cache]
    meta = ops.get_scheduler_metadata_int8(len(lens), q.shape[1], cache[0].shape[1], q.shape[2],
                                           lens if planned is None else planned, q.dtype, qsl, causal,
                                           cache[0].shape[2])
    if warps:
        ops.set_shape_int8(meta, warps)
    qd = q.cuda()
    out = torch.full_like(qd, 7.0) if out is None else out
    ops.attention_with_kv_cache_int8(qd, *dev, out, qsl.cuda(), lens.cuda(), scale, causal, table.cuda(), meta)
    return out.cpu(), ops.plan_of_int8(meta)


def assert_close(got, want, top, dtype):
    """Weights are rounded to half precision for the product (2^-11 of each), the output to
    bfloat16 (2^-9 of itself); in float32 the weights are pairs of halves, and the score's own
    rounding (a few 2^-22 of scores of about 10) sets the error."""
    tol = 2.0 ** -10 * top[..., None] + 2.0 ** -8 * want.abs() if dtype == BF16 else 1e-5 * top[..., None]
    bad = ~((got.double() - want).abs() <= tol + 1e-30)
    assert not bad.any(), (int(bad.sum()), (got.double() - want).abs().max().item())


def batch(lens, rows_per, hkv, group, d, bs, dtype, seed=0, spare=3):
    g = torch.Generator().manual_seed(seed)
    lens = torch.tensor(lens, dtype=torch.int32)
    rows_per = torch.tensor(rows_per)
    qsl = torch.cat([torch.zeros(1, dtype=torch.long), rows_per.cumsum(0)]).to(torch.int32)
    counts = [-(-int(n) // bs) for n in lens]
    n = sum(counts) + spare
    perm = torch.randperm(n, generator=g).tolist()
    table = torch.zeros((len(lens), max(max(counts), 1)), dtype=torch.int32)
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = torch.tensor(perm[at:at + c], dtype=torch.int32)
        at += c
    cache = new_cache(n, hkv, bs, d, g)
    for unused in perm[at:]:  # nothing of a block outside the tables may be read into a sum
        cache[2][unused] = math.nan
        cache[3][unused] = math.nan
    q = torch.randn((int(qsl[-1]), hkv * group, d), generator=g).to(dtype)
    return q, cache, qsl, lens, table


@pytest.mark.parametrize("d", sorted(ops.HEAD_DIMS))
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_head_dims(warps, d, dtype):
    q, cache, qsl, lens, table = batch([1, 16, 17, 100, 0], [1, 1, 3, 2, 1], 2, 1, d, 16, dtype, seed=d)
    want, top = attention_exact(q, cache, qsl, lens, table, d ** -0.5, False)
    got, _ = attend(warps, q, cache, qsl, lens, table, d ** -0.5, False)
    assert_close(got, want, top, dtype)
    assert (got[int(qsl[4]):] == 0).all()  # a request without tokens


@pytest.mark.parametrize("hkv,group,rows_per,causal", [
    (4, 1, [1, 1, 1, 1], False), (2, 4, [1, 1, 1, 1], False), (3, 7, [1, 2, 0, 5], False),
    (1, 1, [9, 17, 1, 3], True), (2, 8, [3, 0, 4, 30], True), (1, 16, [2, 2, 2, 2], True),
])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_grouped_heads_and_causal_rows(warps, hkv, group, rows_per, causal, dtype):
    """Requests with more causal rows than tokens hold rows that see nothing."""
    q, cache, qsl, lens, table = batch([3, 33, 64, 21], rows_per, hkv, group, 64, 32, dtype, seed=group)
    want, top = attention_exact(q, cache, qsl, lens, table, 0.2, causal)
    got, _ = attend(warps, q, cache, qsl, lens, table, 0.2, causal)
    assert_close(got, want, top, dtype)
    assert (got[top == 0] == 0).all()


@pytest.mark.parametrize("bs", [16, 48, 64, 1024])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_block_sizes_and_splits(warps, bs, dtype):
    """One long request next to short ones: its context is split and the pieces merged."""
    q, cache, qsl, lens, table = batch([1500, 1, 400, 17], [2, 1, 1, 3], 2, 1, 64, bs, dtype, seed=bs)
    want, top = attention_exact(q, cache, qsl, lens, table, 0.125, False)
    got, plan = attend(warps, q, cache, qsl, lens, table, 0.125, False)
    assert plan.num_splits > 1
    assert_close(got, want, top, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_scales_of_very_different_size(warps, dtype):
    """K and V scales that differ by many powers of ten from block to block, and zero scales."""
    q, cache, qsl, lens, table = batch([300, 150], [1, 2], 2, 2, 64, 16, dtype, seed=4)
    g = torch.Generator().manual_seed(8)
    for s, span in ((cache[2], 1.0), (cache[3], 25.0)):
        s *= 10.0 ** ((torch.rand(s.shape, generator=g) * 2 - 1) * span)
    zero = torch.rand(cache[3].shape, generator=g) < 0.2  # blocks of zeros, as the append leaves them
    cache[3][zero] = 0.0
    cache[1][zero] = 0
    want, top = attention_exact(q, cache, qsl, lens, table, 0.125, False)
    got, _ = attend(warps, q, cache, qsl, lens, table, 0.125, False)
    assert_close(got, want, top, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_query_sizes_and_non_finite_rows(warps, dtype):
    """Rows of very large, very small and zero queries, and a NaN or an infinity in one row, which
    stays in that row and head."""
    q, cache, qsl, lens, table = batch([50], [6], 2, 1, 64, 16, dtype, seed=6)
    q[0] *= 2.0 ** 60
    q[1] *= 2.0 ** -90
    q[2] = 0.0
    q[3, 0, 5] = math.nan
    q[4, 1] = math.inf
    want, top = attention_exact(q[:3], cache, torch.tensor([0, 3]), lens, table, 0.125, False)
    got, _ = attend(warps, q, cache, qsl, lens, table, 0.125, False)
    assert_close(got[1:3], want[1:3], top[1:3], dtype)
    # the huge row attends to one token alone: its score leads by far
    assert_close(got[:1], want[:1], top[:1], dtype)
    assert got[3, 0].isnan().all() and got[4, 1].isnan().all()
    assert got[3, 1].isfinite().all() and got[4, 0].isfinite().all() and got[5].isfinite().all()


def test_attention_splits_of_every_kind():
    """One to eight CTAs of a cluster, and several clusters with the launch that adds their pieces."""
    q, cache, qsl, lens, table = batch([1234, 3, 0, 160], [1, 2, 1, 1], 2, 2, 64, 16, BF16, seed=31)
    want, top = attention_exact(q, cache, qsl, lens, table, 0.125, False)
    dev = [t.cuda() for t in cache]
    for splits in (1, 2, 3, 4, 8, 16, 40, 100):
        meta = ops.get_scheduler_metadata_int8(4, 4, 2, 64, lens, BF16, qsl, False, 16)
        plan = ops.plan_of_int8(ops.set_shape_int8(meta, 2, splits))
        assert plan.num_splits <= splits < plan.num_splits * 2
        out = torch.full_like(q.cuda(), 7.0)
        ops.attention_with_kv_cache_int8(q.cuda(), *dev, out, qsl.cuda(), lens.cuda(), 0.125, False, table.cuda(), meta)
        assert_close(out.cpu(), want, top, BF16)


def test_attention_strides_stream_and_graph(warps):
    """Queries and outputs as slices of wider buffers, on a side stream, and replayed from a CUDA
    graph with other lengths than were captured (split plan)."""
    q, cache, qsl, lens, table = batch([700, 333], [1, 1], 4, 1, 64, 16, BF16, seed=12)
    want, top = attention_exact(q, cache, qsl, lens, table, 0.125, False)
    dev = [t.cuda() for t in cache]
    wide_q = torch.zeros((2, 4 * 64 + 64), dtype=BF16, device="cuda")
    wide_q[:, :256] = q.cuda().reshape(2, 256)
    wide_o = torch.full((2, 512), 3.0, dtype=BF16, device="cuda")
    qv, ov = wide_q[:, :256].reshape(2, 4, 64), wide_o[:, 256:].view(2, 4, 64)
    qv = wide_q[:, :256].unflatten(1, (4, 64))
    meta = ops.get_scheduler_metadata_int8(2, 4, 4, 64, lens, BF16, None, False, 16)
    assert ops.plan_of_int8(meta).num_splits > 1
    if warps:
        ops.set_shape_int8(meta, warps, 40)
    lens_d, qsl_d, table_d = lens.cuda(), qsl.cuda(), table.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.attention_with_kv_cache_int8(qv, *dev, ov, qsl_d, lens_d, 0.125, False, table_d, meta)
    torch.cuda.current_stream().wait_stream(side)
    assert_close(ov.cpu(), want, top, BF16)
    assert (wide_o[:, :256] == 3.0).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_with_kv_cache_int8(qv, *dev, ov, qsl_d, lens_d, 0.125, False, table_d, meta)
    shorter = torch.tensor([20, 0], dtype=torch.int32)
    lens_d.copy_(shorter)
    ov.fill_(9.0)
    graph.replay()
    want, top = attention_exact(q, cache, qsl, shorter, table, 0.125, False)
    assert_close(ov.cpu(), want, top, BF16)
    assert (ov[1] == 0).all()


@pytest.mark.parametrize("group,causal", [(1, False), (3, False), (3, True)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_many_requests_of_every_length(warps, group, causal, dtype):
    """Hundreds of items with empty requests among them."""
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 90, (150,), generator=g).tolist()
    lens[7], lens[8], lens[100] = 0, 1, 2000
    rows = torch.randint(0, 4, (150,), generator=g).tolist()
    q, cache, qsl, lens, table = batch(lens, rows, 2, group, 64, 16, dtype, seed=5)
    want, top = attention_exact(q, cache, qsl, lens, table, 0.125, causal)
    got, _ = attend(warps, q, cache, qsl, lens, table, 0.125, causal)
    assert_close(got, want, top, dtype)
    assert (got[top == 0] == 0).all()


def test_attention_flags_bad_lengths_blocks_and_rows(warps):
    q, cache, qsl, lens, table = batch([40, 20], [1, 1], 2, 1, 64, 16, BF16, seed=13)
    ops.read_device_errors()
    longer = torch.tensor([49, 20], dtype=torch.int32)  # more than its table holds
    attend(warps, q, cache, qsl, longer, table, 0.125, False, planned=longer)
    assert ops.read_device_errors() == N.DEVERR_CONTEXT
    broken = table.clone()
    broken[1, 0] = 10 ** 6
    want, top = attention_exact(q[:1], cache, qsl[:2], lens[:1], table, 0.125, False)
    got, _ = attend(warps, q, cache, qsl, lens, broken, 0.125, False)
    assert ops.read_device_errors() == N.DEVERR_BLOCK_ID
    assert_close(got[:1], want, top, BF16)
    dev = [t.cuda() for t in cache]
    meta = ops.get_scheduler_metadata_int8(2, 2, 2, 64, lens, BF16, None, False, 16)
    out = torch.full_like(q.cuda(), 5.0)
    ops.attention_with_kv_cache_int8(q.cuda(), *dev, out, torch.tensor([0, 1, 9], dtype=torch.int32).cuda(),
                                     lens.cuda(), 0.125, False, table.cuda(), meta)
    assert ops.read_device_errors() == N.DEVERR_QUERY
    assert (out[1] == 5.0).all() and (out[0] != 5.0).any()


def test_offsets_past_32_bits():
    """Blocks at the end of pools of more than 2^31 codes: append, read-back and attention."""
    h, bs, d = 16, 32, 64
    n = 2 ** 31 // (h * bs * d) + 40
    kc, vc = (torch.zeros((n, h, bs, d), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((n, h), device="cuda") for _ in range(2))
    key, value = rows(50, h, d, BF16, seed=21)
    pos = torch.arange(50)
    table = torch.tensor([[n - 1, n - 7]], dtype=torch.int32)
    slots = table[0].long()[pos // bs] * bs + pos % bs
    ops.reshape_and_cache_int8(key.cuda(), value.cuda(), kc, vc, ks, vs, slots.cuda())
    small = [torch.zeros((2, h, bs, d), dtype=torch.int8) for _ in range(2)] + [torch.zeros((2, h)) for _ in range(2)]
    append_plain(key, small[0], small[2], pos)
    append_plain(value, small[1], small[3], pos)
    at = table[0].long().cuda()
    for got, want in zip((kc, vc, ks, vs), small):
        assert torch.equal(got[at].cpu(), want)
    assert int((kc != 0).sum(dtype=torch.int64)) == int((small[0] != 0).sum())
    k, _ = ops.gather_kv_int8(kc, vc, ks, vs, slots.cuda(), F32)
    assert torch.equal(k.cpu(), small[0][pos // bs, :, pos % bs].float() * small[2][pos // bs][:, :, None])
    q = torch.randn((1, h, d), generator=torch.Generator().manual_seed(1)).to(BF16)
    lens, qsl = torch.tensor([50], dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    want, top = attention_exact(q, small, qsl, lens, torch.tensor([[0, 1]]), 0.125, False)
    meta = ops.get_scheduler_metadata_int8(1, h, h, d, lens, BF16, None, False, bs)
    out = torch.empty_like(q.cuda())
    ops.attention_with_kv_cache_int8(q.cuda(), kc, vc, ks, vs, out, qsl.cuda(), lens.cuda(), 0.125, False,
                                     table.cuda(), meta)
    assert_close(out.cpu(), want, top, BF16)
