"""CPU-only: rotary_cache_write refuses to drop a gradient."""
from __future__ import annotations

import pytest
import torch


def _call(q, cos_sin, k=None):
    from cta_b200 import ops

    ints = torch.zeros(8, dtype=torch.int64)
    k = torch.empty(8, 2, 64, dtype=q.dtype) if k is None else k
    cache = torch.empty(4, 16, 2, 64, dtype=q.dtype)
    return ops.rotary_cache_write(q, k, k, cache, cache, ints, ints, cos_sin)


def test_gradients_are_not_dropped():
    q, table = torch.empty(8, 4, 64, dtype=torch.bfloat16), torch.empty(10, 64)
    for bad in ((q.clone().requires_grad_(), table), (q, table.clone().requires_grad_()),
                (torch.empty_like(q).requires_grad_() * 2, table)):
        with pytest.raises(ValueError, match="gradient"):
            _call(*bad)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # the next check
            _call(*bad)
        with torch.inference_mode(), pytest.raises(ValueError, match="CUDA"):
            _call(*bad)
        with pytest.raises(ValueError, match="CUDA"):
            _call(*(x.detach() for x in bad))
    # the cache takes none
    with pytest.raises(ValueError, match="CUDA"):
        _call(q, table, torch.empty(8, 2, 64, dtype=torch.bfloat16, requires_grad=True))


def test_tangents_are_not_dropped():
    from torch.autograd import forward_ad

    q, table = torch.empty(8, 4, 64), torch.empty(10, 64)
    with forward_ad.dual_level():
        for bad in ((forward_ad.make_dual(q, torch.ones_like(q)), table), (q, forward_ad.make_dual(table, torch.ones_like(table)))):
            with pytest.raises(ValueError, match="gradient"):
                _call(*bad)
        with pytest.raises(ValueError, match="CUDA"):
            _call(q, table)
