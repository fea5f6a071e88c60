"""The 8-bit attention's error where scales, weights or query elements of one row differ by much:
against the 64-bit definition, with the head's own values as the measure."""

from __future__ import annotations

import math

import pytest
import torch

from vflorence_b200 import paged_ops as ops

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def exact(q, cache, lens, table, scale):
    """One row a request: (output, largest visible |v| of each head) in 64 bits."""
    kc, vc, ks, vs = (t.double() for t in cache)
    group, bs = q.shape[1] // kc.shape[1], kc.shape[2]
    out, top = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64)
    for r, n in enumerate(lens.tolist()):
        blocks = table[r, : -(-n // bs)].long()
        k, v = ((c[blocks] * s[blocks][..., None, None]).transpose(0, 1).flatten(1, 2)[:, :n] for c, s in ((kc, ks), (vc, vs)))
        for h in range(q.shape[1]):
            out[r, h] = torch.softmax((k[h // group] @ q[r, h].double()) * scale, 0) @ v[h // group]
            top[r, h] = v[h // group].abs().max()
    return out, top


def attend(q, cache, lens, table, scale, warps=0, splits=0):
    starts = torch.arange(len(lens) + 1, dtype=torch.int32)
    meta = ops.get_scheduler_metadata_int8(len(lens), q.shape[1], cache[0].shape[1], q.shape[2], lens, q.dtype, starts,
                                           False, cache[0].shape[2])
    if warps or splits:
        ops.set_shape_int8(meta, warps, splits)
    out = torch.full_like(q, 7.0).cuda()
    ops.attention_with_kv_cache_int8(q.cuda(), *[t.cuda() for t in cache], out, starts.cuda(), lens.cuda(), scale, False,
                                     table.cuda(), meta)
    return out.cpu()


def pool(lens, heads, d, bs, seed, v_scale):
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // bs) for n in lens]
    n = sum(counts)
    perm = torch.randperm(n, generator=g).to(torch.int32)
    table = torch.zeros((len(lens), max(counts)), dtype=torch.int32)
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = perm[at:at + c]
        at += c
    kc, vc = (torch.randint(-127, 128, (n, heads, bs, d), generator=g, dtype=torch.int8) for _ in range(2))
    ks = (0.5 + torch.rand((n, heads), generator=g)) * 0.02
    vs = (0.5 + torch.rand((n, heads), generator=g)) * v_scale
    return g, [kc, vc, ks, vs], torch.tensor(lens, dtype=torch.int32), table


def assert_within(got, want, top, dtype):
    """bfloat16: the output's rounding (2^-9 of itself) and the weights' (2^-11 each). float32: the
    exponent of a score of about 10 is off by a few 2^-24 of it."""
    tol = 2.0 ** -10 * top[..., None] + 2.0 ** -8 * want.abs() if dtype == BF16 else 1e-5 * top[..., None]
    over = (got.double() - want).abs() / tol
    assert bool((over <= 1).all()), over.max().item()


@pytest.mark.parametrize("warps,splits", [(0, 0), (1, 1), (2, 1), (4, 1), (2, 4), (1, 24)])
@pytest.mark.parametrize("v_scale", [1e-3, 1e-5, 1e-8, 2.0 ** -98])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_zero_v_blocks_among_small_scales(dtype, v_scale, warps, splits):
    """Blocks of zeros (scale 0, as the append leaves them) weigh in the sum of the weights alone."""
    g, cache, lens, table = pool([592, 100, 2000], 2, 64, 16, 3, v_scale)
    q = torch.randn((3, 2, 64), generator=g).to(dtype)
    for r, n in enumerate(lens.tolist()):
        for col in (0, 3, (n - 1) // 16):
            cache[3][table[r, col]] = 0.0
            cache[1][table[r, col]] = 0
    want, top = exact(q, cache, lens, table, 0.125)
    assert_within(attend(q, cache, lens, table, 0.125, warps, splits), want, top, dtype)


@pytest.mark.parametrize("lead", [4.0, 12.0, 60.0])
@pytest.mark.parametrize("v_scale", [0.02, 1e-3, 1e-8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_zero_v_block_with_most_of_the_weight(dtype, v_scale, lead):
    """A block of zeros whose scores lead by `lead`: the output is what is left for the others. Its
    error is a share of itself, and no longer of the largest value."""
    g, cache, lens, table = pool([700], 1, 64, 16, 5, v_scale)
    q = torch.randn((1, 1, 64), generator=g).to(dtype)
    b = int(table[0, 20])
    cache[0][b, 0] = (q[0, 0].float() / q.float().abs().max() * 100).round().to(torch.int8)
    cache[1][b], cache[3][b] = 0, 0.0
    others = torch.ones(700, dtype=torch.bool)
    others[20 * 16:21 * 16] = False
    kc, ks = cache[0].double(), cache[2].double()
    k = (kc[table[0].long()] * ks[table[0].long()][..., None, None]).transpose(0, 1).flatten(1, 2)[0, :700]
    s = k @ q[0, 0].double() * 0.125
    cache[2][b] = (float(s[others].max()) + lead) / float(kc[b, 0, 0] @ q[0, 0].double() * 0.125)
    want, top = exact(q, cache, lens, table, 0.125)
    got = attend(q, cache, lens, table, 0.125, 1, 1).double()
    # the others' weights against one another, then the division: relative to the largest output,
    # and the lead's own rounding, a few 2^-24 of a score of up to 80, times their sum
    tol = (2.0 ** -7 if dtype == BF16 else 1e-4) * want.abs().max()
    assert bool(((got - want).abs() <= tol).all()), ((got - want).abs().max() / want.abs().max()).item()


def test_a_nan_scale_shows():
    """A V or K block whose scale is a NaN makes the rows that see it NaN, and no others."""
    for which in (2, 3):
        g, cache, lens, table = pool([100, 90], 2, 64, 16, 7, 0.02)
        q = torch.randn((2, 2, 64), generator=g).to(BF16)
        cache[which][table[0, 2], 1] = math.nan
        got = attend(q, cache, lens, table, 0.125)
        assert got[0, 1].isnan().all()
        assert got[0, 0].isfinite().all() and got[1].isfinite().all()


@pytest.mark.parametrize("warps,splits", [(0, 0), (1, 1), (4, 1)])
@pytest.mark.parametrize("n", [1024, 4096, 20000])
def test_many_small_weights_beside_one_token(n, warps, splits):
    """One token leads by 17.6; what thousands of tokens of one sign add is theirs alone (its own
    values are 0). A weight is held to 2^-32 of the largest or better: n of them to n 2^-32."""
    g, cache, lens, table = pool([n], 1, 64, 16, 9, 0.02)
    cache[0].zero_()
    cache[1].fill_(127)
    cache[3].fill_(0.02)
    q = torch.ones((1, 1, 64))
    b, t = int(table[0, n // 40]), 5
    cache[0][b, 0, t] = 100
    cache[1][b, 0, t] = 0
    cache[2][b] = 17.6 / (100 * 64 * 0.125)
    want, top = exact(q, cache, lens, table, 0.125)
    got = attend(q, cache, lens, table, 0.125, warps, splits).double()
    tol = n * 2.0 ** -32 * top[..., None] + 1e-5 * want
    assert bool(((got - want).abs() <= tol).all()), ((got - want).abs() / top[..., None]).max().item()


@pytest.mark.parametrize("d", [32, 64, 80, 128, 256])
@pytest.mark.parametrize("ratio", [64.0, 1000.0])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_large_channel_in_the_query(dtype, ratio, d):
    """A query channel `ratio` times the others whose cached keys are small (0 or one step): the
    others' products decide the scores."""
    g, cache, lens, table = pool([300, 40, 150], 2, d, 16, 11, 0.02)
    q = torch.randn((3, 4, d), generator=g)
    q[..., 1] = ratio
    q = q.to(dtype)
    cache[0][..., 1] = torch.randint(-1, 2, cache[0].shape[:-1], generator=g).to(torch.int8)
    scale = 4.0 / (0.02 * 73.0 * math.sqrt(d))  # scores of the others of about 4
    want, top = exact(q, cache, lens, table, scale)
    assert_within(attend(q, cache, lens, table, scale), want, top, dtype)
