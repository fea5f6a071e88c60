"""Edges of the 8-bit cache and 4-bit linear entry points on the host: no GPU needed."""

from __future__ import annotations

import ctypes

import torch

PTR = 1 << 20  # never dereferenced


def test_attention_of_requests_without_rows_launches_nothing(native):
    """Requests of no query row behind rows that belong to none: nothing to do, and no empty grid."""
    from vflorence_b200 import paged_ops as ops

    lens, qsl = torch.tensor([5, 6], dtype=torch.int32), torch.tensor([3, 3, 3], dtype=torch.int32)
    meta = ops.get_scheduler_metadata_int8(2, 8, 8, 64, lens, torch.bfloat16, qsl, False, 16)
    plan = ops.plan_of_int8(meta)
    assert plan.total_q == 3 and plan.max_q_len == 0
    assert native.vfl_attention_with_kv_cache_int8(ctypes.byref(plan), PTR, 512, PTR, PTR, PTR, PTR, 64, PTR, 512, PTR,
                                                   PTR, PTR, 8, 8, 0.125, None, 0, None) == 0
