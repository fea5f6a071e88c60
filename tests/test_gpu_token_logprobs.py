"""Log probabilities of given tokens, entropy and alternatives on the GPU against 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from vflorence_b200 import _native as N
from vflorence_b200 import paged_ops as ops

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def check(x, targets, k, got):
    """Sums of exponentials are off by a few 2^-22 of themselves, a log probability by that and by
    2^-23 of its own size. Alternatives: exact order, ties by lower index."""
    lp, ent, values, indices = (t.cpu() for t in got)
    x64 = x.double().cpu()
    ref = torch.log_softmax(x64, -1)
    want = ref.gather(1, targets.long().clamp(min=0)[:, None])[:, 0]
    want = torch.where(targets < 0, 0.0, want)
    entropy = torch.special.entr(ref.exp()).sum(-1)

    def close(a, b):
        same = torch.where(b.isinf(), a.double() == b, (a.double() - b).abs() <= 5e-6 + 1e-6 * b.abs())
        assert same.all(), (a, b)

    close(lp, want)
    close(ent, entropy)
    order = torch.sort(x64, dim=-1, descending=True, stable=True)
    assert torch.equal(indices.long(), order.indices[:, :k])
    close(values, ref.gather(1, order.indices[:, :k]))


def run(x, targets, k):
    return ops.token_logprobs(x, targets.cuda(), k)


def targets_of(rows, vocab, seed=0):
    return torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 7), (5, 33), (4, 255), (3, 1000), (2, 8193), (1, 50265),
                                        (37, 51289), (200, 4099)])
@pytest.mark.parametrize("k", [0, 1, 20, 64])
def test_rows_vocabularies_and_k(dtype, rows, vocab, k):
    k = min(k, vocab)
    x = (torch.randn((rows, vocab), generator=torch.Generator().manual_seed(vocab)) * 3).to(dtype).cuda()
    t = targets_of(rows, vocab)
    check(x, t, k, run(x, t, k))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("offset", [0, 1, 3, 5])
def test_row_alignment_and_stride(dtype, offset):
    wide = (torch.randn((9, 700), generator=torch.Generator().manual_seed(offset)) * 2).to(dtype).cuda()
    x = wide[:, offset:offset + 613]
    t = targets_of(9, 613)
    check(x, t, 7, run(x, t, 7))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_forbidden_entries_and_targets(dtype):
    """Rows with many entries of -inf, down to one that is left; targets that are forbidden, or
    not given."""
    x = torch.randn((6, 5000), generator=torch.Generator().manual_seed(4)).to(dtype)
    for i, keep in enumerate((4000, 300, 70, 20, 2, 1)):
        drop = torch.randperm(5000, generator=torch.Generator().manual_seed(i))[keep:]
        x[i, drop] = -math.inf
    t = x.float().argmax(-1).to(torch.int32)
    t[0] = int(torch.nonzero(x[0] == -math.inf)[0])
    t[2] = -1
    check(x, t, 64, run(x.cuda(), t, 64))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [5000, 70001, 600003])
def test_ties(dtype, vocab):
    """Equal rows, rows of few values, large entries next to one another, sorted rows: the lowest
    indices win, however many entries tie."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.stack([
        torch.zeros(vocab),
        torch.randint(0, 3, (vocab,), generator=g).float(),
        torch.arange(vocab).float().neg() / vocab,
        torch.arange(vocab).float() / vocab,
        torch.where(torch.arange(vocab) % 2048 < 8, 5.0, 0.0) + torch.rand(vocab, generator=g),
        torch.where(torch.arange(vocab) >= vocab - 5, 1.0, -math.inf),
    ]).to(dtype)
    t = targets_of(6, vocab)
    t[5] = vocab - 1
    check(x, t, 64, run(x.cuda(), t, 64))
    check(x, t, 1, run(x.cuda(), t, 1))


def test_entries_of_a_few_threads_alone():
    """The largest entries all lie where a handful of threads read (every 2048th group of 8): more
    of them reach the bound than the candidate list holds."""
    vocab = 51200
    at = torch.arange(vocab)
    x = torch.where(at % 2048 < 64, 100.0 + (at * 7919 % 100003) / 1e4, (at * 7919 % 1009) / 1e4)[None].repeat(2, 1)
    t = targets_of(2, vocab)
    check(x, t, 64, run(x.cuda(), t, 64))
    # one row on one CTA (many rows), the same entries
    big = x[:1].repeat(160, 1)
    t = targets_of(160, vocab)
    check(big, t, 64, run(big.cuda(), t, 64))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_extreme_values(dtype):
    x = torch.randn((5, 900), generator=torch.Generator().manual_seed(8)).to(dtype)
    x[0] *= 1e30
    x[1] += 300.0
    x[2, 17] = 1e38
    x[3] = -1e38
    x[4] *= 1e-30
    t = targets_of(5, 900)
    check(x, t, 5, run(x.cuda(), t, 5))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masks_of_the_lowest_value(dtype):
    """Entries held at the type's lowest value instead of -inf: all, all but one, and half."""
    low = torch.finfo(dtype).min
    x = torch.randn((3, 9000), generator=torch.Generator().manual_seed(9)).to(dtype)
    x[0] = low
    x[1, :4321], x[1, 4322:] = low, low
    x[2, ::2] = low
    t = torch.tensor([17, 4321, 4], dtype=torch.int32)
    check(x, t, 20, run(x.cuda(), t, 20))


def test_empty_nan_and_infinite_rows():
    x = torch.zeros((4, 300))
    x[0] = -math.inf
    x[1, 40] = math.nan
    x[2, 40] = math.inf
    x[3, :298] = math.nan
    t = torch.tensor([5, 5, 5, 299], dtype=torch.int32)
    lp, ent, values, indices = (a.cpu() for a in run(x.cuda(), t, 4))
    assert lp[0] == -math.inf and ent[0] == 0 and (values[0] == -math.inf).all() and indices[0].tolist() == [0, 1, 2, 3]
    assert lp[1:].isnan().all() and ent[1:].isnan().all() and values[1:].isnan().all()
    assert indices[1].tolist() == [0, 1, 2, 3] and indices[2].tolist() == [40, 0, 1, 2]
    assert indices[3].tolist() == [298, 299, -1, -1]


def test_targets_past_the_vocabulary_and_none():
    x = torch.randn((2, 100), generator=torch.Generator().manual_seed(1)).cuda()
    ops.read_device_errors()
    lp, ent, _, _ = ops.token_logprobs(x, torch.tensor([100, 3], dtype=torch.int32).cuda())
    assert ops.read_device_errors() == N.DEVERR_SLOT
    assert lp[0].isnan() and lp[1].isfinite() and ent.isfinite().all()
    lp, _, values, _ = ops.token_logprobs(x, None, 3)
    assert (lp == 0).all() and values.shape == (2, 3) and ops.read_device_errors() == 0
    assert ops.token_logprobs(x[:0], None, 3)[2].shape == (0, 3)


def test_rows_past_32_bit_offsets():
    """The last row of a matrix of more than 2^31 elements."""
    vocab = 50265
    rows = 2 ** 31 // vocab + 3
    x = torch.zeros((rows, vocab), dtype=BF16, device="cuda")
    x[-1] = torch.randn(vocab, generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    t = torch.full((rows,), 77, dtype=torch.int32)
    lp, ent, values, indices = run(x, t, 3)
    check(x[-1:], t[-1:], 3, (lp[-1:], ent[-1:], values[-1:], indices[-1:]))
    assert torch.allclose(ent[:-1], torch.full_like(ent[:-1], math.log(vocab)), rtol=1e-6)
