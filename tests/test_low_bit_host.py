"""Refusals of the 8-bit cache, 4-bit linear and token-score entry points before any launch, and
the attention's plan: no GPU needed."""

from __future__ import annotations

import ctypes

import pytest
import torch

PTR = 1 << 20  # never dereferenced: every call is refused on the host


def test_append_and_gather_refuse_bad_arguments(native):
    def append(key=PTR, value=PTR, kc=PTR, vc=PTR, ks=PTR, vs=PTR, slots=PTR, tokens=4, heads=2, dim=64, bs=16,
               blocks=8, stride=128, vstride=128, dtype=1):
        return native.vfl_reshape_and_cache_int8(key, value, kc, vc, ks, vs, slots, tokens, heads, dim, bs, blocks,
                                                 stride, vstride, dtype, None)

    assert append(dtype=2) == 2 and append(dim=40, stride=80, vstride=80) == 2
    for bad in (dict(key=None), dict(ks=None), dict(slots=None), dict(tokens=-1), dict(heads=0), dict(bs=0),
                dict(blocks=0), dict(stride=64), dict(vstride=132), dict(kc=PTR + 8), dict(value=PTR + 2)):
        assert append(**bad) == 1, bad
    assert append(tokens=0) == 0

    def gather(kc=PTR, out=PTR, tokens=4, dim=64, blocks=8, dtype=0):
        return native.vfl_gather_kv_int8(kc, PTR, PTR, PTR, PTR, out, PTR, tokens, 2, dim, 16, blocks, dtype, None)

    assert gather(dtype=3) == 2 and gather(dim=24) == 2
    for bad in (dict(kc=None), dict(out=PTR + 4), dict(tokens=-2), dict(blocks=-1)):
        assert gather(**bad) == 1, bad
    assert gather(tokens=0) == 0


def _plan(lens, heads=8, kv=8, d=64, dtype=torch.bfloat16, qsl=None, causal=False, bs=16):
    from vflorence_b200 import paged_ops as ops

    lens = torch.tensor(lens, dtype=torch.int32)
    qsl = None if qsl is None else torch.tensor(qsl, dtype=torch.int32)
    return ops.get_scheduler_metadata_int8(len(lens), heads, kv, d, lens, dtype, qsl, causal, bs)


def test_plan_splits_few_long_requests_and_covers_them(native):
    from vflorence_b200 import paged_ops as ops

    for lens, kv in (([4096], 16), ([100000], 1), ([1, 2000, 64], 4), ([0, 0], 2), ([15], 3), ([2048] * 512, 16)):
        p = ops.plan_of_int8(_plan(lens, heads=kv, kv=kv))
        assert p.cluster in (1, 2, 4, 8) and p.num_splits % p.cluster == 0
        assert (p.workspace_bytes == 0) == (p.num_splits == p.cluster)
    assert ops.plan_of_int8(_plan([100000], heads=1, kv=1)).num_splits > 64
    assert ops.plan_of_int8(_plan([2048] * 512, heads=16, kv=16)).num_splits == 1
    p = ops.plan_of_int8(_plan([], heads=4, kv=4))
    assert p.num_reqs == 0 and p.workspace_bytes == 0


def test_plan_refuses_bad_input(native):
    from vflorence_b200 import paged_ops as ops

    for kwargs in (dict(heads=6, kv=4), dict(d=40), dict(bs=24), dict(heads=0, kv=1), dict(qsl=[0, 3, 2])):
        with pytest.raises(RuntimeError):
            _plan([5, 6], **kwargs)
    with pytest.raises(RuntimeError):
        _plan([-1])
    with pytest.raises(ValueError):
        _plan([5], dtype=torch.float16)
    with pytest.raises(ValueError):
        ops.plan_of_int8(torch.zeros(32, dtype=torch.int64))
    meta = _plan([5])
    with pytest.raises(ValueError):  # the other attention's metadata is another struct
        ops.plan_of(torch.cat([meta, meta, meta]))


def _attend(native, plan, **kw):
    a = dict(query=PTR, q_stride=512, kc=PTR, vc=PTR, ks=PTR, vs=PTR, blocks=64, out=PTR, o_stride=512, qsl=PTR,
             lens=PTR, table=PTR, t_stride=8, cols=8, scale=0.125, ws=None, ws_bytes=0)
    a.update(kw)
    return native.vfl_attention_with_kv_cache_int8(
        ctypes.byref(plan) if plan is not None else None, a["query"], a["q_stride"], a["kc"], a["vc"], a["ks"], a["vs"],
        a["blocks"], a["out"], a["o_stride"], a["qsl"], a["lens"], a["table"], a["t_stride"], a["cols"], a["scale"],
        a["ws"], a["ws_bytes"], None)


def test_attention_refuses_bad_arguments(native):
    from vflorence_b200 import paged_ops as ops

    meta = _plan([100, 7])
    plan = ops.plan_of_int8(meta)
    assert plan.workspace_bytes == 0
    assert _attend(native, None) == 1
    for bad in (dict(query=None), dict(ks=None), dict(out=None), dict(table=None), dict(blocks=0), dict(q_stride=500),
                dict(o_stride=256), dict(t_stride=4), dict(kc=PTR + 1), dict(query=PTR + 8),
                dict(scale=float("nan")), dict(scale=float("inf"))):
        assert _attend(native, plan, **bad) == 1, bad
    split_meta = _plan([20000], heads=8, kv=8, d=64)
    split = ops.plan_of_int8(split_meta)
    assert split.workspace_bytes > 0
    assert _attend(native, split, cols=1300, t_stride=1300) == 3
    assert _attend(native, split, cols=1300, t_stride=1300, ws=PTR, ws_bytes=16) == 3
    empty = _plan([], heads=4, kv=4)
    assert _attend(native, ops.plan_of_int8(empty)) == 0


@pytest.mark.parametrize("field,value", [("num_heads", 7), ("num_kv_heads", 0), ("head_dim", 40), ("block_size", 17),
                                         ("dtype", 5), ("causal", 2), ("num_splits", 0), ("cluster", 3), ("cluster", 0),
                                         ("num_splits", 12), ("rows_per_cta", 4), ("rows_per_cta", 16),
                                         ("total_q", -1), ("max_q_len", 70000), ("workspace_bytes", 8),
                                         ("num_splits", 70000), ("warps", 3), ("warps", 0)])
def test_attention_refuses_a_corrupted_plan(native, field, value):
    from vflorence_b200 import paged_ops as ops

    meta = _plan([9000, 300], d=160, heads=1, kv=1)
    plan = ops.plan_of_int8(meta)
    assert plan.num_splits > plan.cluster == 8
    setattr(plan, field, value)
    assert _attend(native, plan, cols=600, t_stride=600, ws=PTR, ws_bytes=1 << 40) == 1


def test_linear_int4_refuses_bad_arguments(native):
    def linear(x=PTR, xs=256, codes=PTR, scales=PTR, bias=None, y=PTR, ys=64, rows=2, n=64, k=256, group=64, dtype=1,
               act=0):
        return native.vfl_linear_int4(x, xs, codes, scales, bias, y, ys, rows, n, k, group, dtype, act, None)

    assert linear(dtype=4) == 2 and linear(group=48) == 2 and linear(group=0) == 2 and linear(k=288, xs=288) == 2
    for bad in (dict(x=None), dict(codes=None), dict(scales=None), dict(y=None), dict(act=3), dict(rows=-1), dict(n=0),
                dict(k=0), dict(xs=128), dict(ys=32), dict(x=PTR + 2), dict(codes=PTR + 4), dict(xs=260),
                dict(bias=PTR + 1), dict(y=PTR + 1)):
        assert linear(**bad) == 1, bad
    assert linear(rows=0) == 0


def test_token_logprobs_refuses_bad_arguments(native):
    def score(x=PTR, dtype=0, rows=2, vocab=100, stride=100, targets=PTR, k=4, lp=PTR, ent=PTR, values=PTR, idx=PTR):
        return native.vfl_token_logprobs(x, dtype, rows, vocab, stride, targets, k, lp, ent, values, idx, None)

    assert score(dtype=7) == 2
    for bad in (dict(x=None), dict(lp=None), dict(ent=None), dict(values=None), dict(idx=None), dict(rows=-1),
                dict(vocab=0), dict(stride=99), dict(k=-1), dict(k=65), dict(vocab=3, stride=3), dict(x=PTR + 2)):
        assert score(**bad) == 1, bad
    assert score(rows=0) == 0


def test_wrappers_refuse_cpu_tensors_and_wrong_types(native):
    from vflorence_b200 import paged_ops as ops

    kc = torch.zeros((4, 2, 16, 64), dtype=torch.int8)
    ks = torch.zeros((4, 2))
    x = torch.zeros((3, 2, 64))
    slots = torch.zeros(3, dtype=torch.int64)
    for call in (lambda: ops.reshape_and_cache_int8(x, x, kc, kc, ks, ks, slots),
                 lambda: ops.gather_kv_int8(kc, kc, ks, ks, slots, torch.float32),
                 lambda: ops.token_logprobs(torch.zeros((2, 5)), None),
                 lambda: ops.linear_int4(torch.zeros((1, 64)), torch.zeros((8, 32), dtype=torch.uint8),
                                         torch.zeros((8, 1))),
                 lambda: ops.attention_with_kv_cache_int8(x, kc, kc, ks, ks, x, slots, slots, 1.0, False, slots,
                                                          _plan([3], heads=2, kv=2))):
        with pytest.raises(ValueError):
            call()
    for weight, group in ((torch.zeros(64), 32), (torch.zeros((4, 64), dtype=torch.float16), 32),
                          (torch.zeros((4, 64)), 48), (torch.zeros((4, 96)), 64)):
        with pytest.raises(ValueError):
            ops.quantize_int4(weight, group)


def test_quantize_int4_packs_the_lower_half_first(native):
    from vflorence_b200 import paged_ops as ops

    w = torch.zeros((1, 32))
    w[0, 0], w[0, 1], w[0, 2] = 7.0, -7.0, 3.0
    codes, scales = ops.quantize_int4(w, 32)
    assert scales.item() == 1.0 and codes[0, 0].item() == 15 | (1 << 4) and codes[0, 1].item() == 11 | (8 << 4)
