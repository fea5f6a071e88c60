"""The linear layer with 4-bit weights on the GPU against the 64-bit definition."""

from __future__ import annotations

import math

import pytest
import torch

from vflorence_b200 import paged_ops as ops

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def make(rows, n, k, group, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    scales = ((0.5 + torch.rand((n, k // group), generator=g)) * 0.02).to(dtype)
    x = torch.randn((rows, k), generator=g).to(dtype)
    bias = torch.randn(n, generator=g).to(dtype)
    return x, codes, scales, bias


def weight(codes, scales):
    w = torch.stack([codes & 15, codes >> 4], -1).double().flatten(1) - 8
    return w * scales.double().repeat_interleave(w.shape[1] // scales.shape[1], 1)


def check(got, x, codes, scales, bias, gelu):
    """Products are exact in the tensor instructions; float32 sums of k / 16 steps may lose a last
    place (2^-23) of the sum of magnitudes each, and the result is rounded to its type. GELU has
    a slope below 1.13."""
    w = weight(codes, scales)
    want = x.double() @ w.T
    size = x.double().abs() @ w.abs().T
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    tol = (x.shape[1] / 16 + 16) * 2.0 ** -23 * size
    if gelu:
        want, tol = torch.nn.functional.gelu(want), 1.13 * tol + 1e-6
    if x.dtype == BF16:
        tol = tol + 2.0 ** -8 * want.abs()
    bad = ~((got.cpu().double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), (got.cpu().double() - want).abs().max().item())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("rows,n,k", [(1, 16, 256), (3, 50, 512), (8, 1, 768), (9, 129, 256), (16, 33, 1280),
                                      (20, 17, 512), (33, 64, 256), (70, 24, 512)])
def test_linear_shapes(dtype, group, rows, n, k):
    x, codes, scales, bias = make(rows, n, k, group, dtype, seed=rows * n)
    dev = [t.cuda() for t in (x, codes, scales, bias)]
    check(ops.linear_int4(*dev), x, codes, scales, bias, False)
    check(ops.linear_int4(*dev[:3], None, "gelu"), x, codes, scales, None, True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("group,k", [(32, 32), (32, 96), (64, 64), (64, 192), (32, 8224), (128, 128), (128, 16512)])
def test_linear_k_ends_inside_a_chunk_and_long_k(dtype, group, k):
    x, codes, scales, bias = make(5, 40, k, group, dtype, seed=k)
    check(ops.linear_int4(x.cuda(), codes.cuda(), scales.cuda()), x, codes, scales, None, False)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("group,k", [(32, 4224), (64, 4224), (32, 4192), (128, 4224), (256, 4352), (32, 10368)])
def test_linear_reads_nothing_past_its_operands(dtype, group, k):
    """A long k is cut over several CTAs, whose last one has less: what lies behind the scales, the
    codes and x is not read (a NaN would meet zeros there and stay)."""
    x, codes, scales, bias = make(3, 40, k, group, dtype, seed=k)

    def walled(t, wall):
        room = torch.full((t.numel() + 4096,), wall, dtype=t.dtype, device="cuda")
        room[: t.numel()] = t.flatten().cuda()
        return room[: t.numel()].view(t.shape)

    got = ops.linear_int4(walled(x, math.nan), walled(codes, 255), walled(scales, math.nan), walled(bias, math.nan))
    check(got, x, codes, scales, bias, False)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_strides_and_out(dtype):
    x, codes, scales, bias = make(4, 48, 256, 64, dtype)
    wide = torch.zeros((4, 320), dtype=dtype, device="cuda")
    wide[:, :256] = x.cuda()
    out = torch.full((4, 100), 3.0, dtype=dtype, device="cuda")
    got = ops.linear_int4(wide[:, :256], codes.cuda(), scales.cuda(), bias.cuda(), out=out[:, :48])
    check(got, x, codes, scales, bias, False)
    assert (out[:, 48:] == 3.0).all()
    assert ops.linear_int4(x[:0].cuda(), codes.cuda(), scales.cuda()).shape == (0, 48)


def test_linear_float32_keeps_24_bits_and_large_values():
    """x with long mantissas and very different sizes, weights of one: the sum is that of x."""
    k = 256
    codes = torch.full((16, k // 2), 0x99, dtype=torch.uint8)  # 9 - 8 = 1
    scales = torch.ones((16, k // 64))
    x = torch.zeros((3, k))
    x[0, 37] = 1.0 + 2.0 ** -23
    x[1, 200] = 3.3e38
    x[2, 5] = 2.0 ** -80 * (2.0 - 2.0 ** -23)
    got = ops.linear_int4(x.cuda(), codes.cuda(), scales.cuda()).cpu()
    assert torch.equal(got, x.sum(1, keepdim=True).expand(3, 16))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_infinities_and_nans_stay_in_their_rows(dtype):
    x, codes, scales, _ = make(3, 16, 128, 32, dtype)
    x[1, 7] = math.nan
    codes[:] = 0x9a  # weights of 2 and 1 steps: no zero to meet an infinity
    x[2] = x[2].abs()
    x[2, 9] = math.inf
    got = ops.linear_int4(x.cuda(), codes.cuda(), scales.cuda()).cpu()
    assert got[0].isfinite().all() and got[1].isnan().all() and (got[2] == math.inf).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("group", [32, 128])
def test_quantize_int4_round_trip(dtype, group):
    """Half a step off at most (the scale's own rounding in bfloat16: 7 steps of 2^-9 more, and a
    value past the largest code by as much)."""
    w = torch.randn((24, 512), generator=torch.Generator().manual_seed(1)).to(dtype)
    w[3] = 0.0
    codes, scales = ops.quantize_int4(w, group)
    step = scales.double().repeat_interleave(group, 1)
    off = (weight(codes, scales) - w.double()).abs()
    assert (off <= step * (0.5 + (7 * 2.0 ** -8 if dtype == BF16 else 1e-5))).all()
    x = torch.randn((2, 512), generator=torch.Generator().manual_seed(2)).to(dtype)
    check(ops.linear_int4(x.cuda(), codes.cuda(), scales.cuda()), x, codes, scales, None, False)
