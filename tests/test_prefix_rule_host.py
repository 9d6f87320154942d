"""CPU-only checks of how a shared prefix is cut into parts: by the prefix and the batch, whatever the block table's width."""
from __future__ import annotations

import pytest

from test_more_attention_host import _paged


def _bytes(prefix, **kw):
    from cta_b200 import _lib

    return _lib.load().cta_prefix_paged_attention_workspace_bytes(_paged(**kw), prefix)


def _plain(**kw):
    from cta_b200 import _lib

    return _lib.load().cta_paged_attention_workspace_bytes(_paged(**kw))


@pytest.mark.parametrize("quantized", [0, 1])
@pytest.mark.parametrize("dtype", [1, 2])
@pytest.mark.parametrize("heads,kv", [(32, 8), (8, 2), (32, 32)])
@pytest.mark.parametrize("batch,prefix", [(4, 16384), (16, 2048), (16, 8192), (16, 16384), (64, 1024), (64, 8192), (128, 16384)])
def test_parts_do_not_depend_on_the_tables_width(batch, prefix, heads, kv, dtype, quantized):
    """The workspace holds the parts' sums."""
    kw = dict(rows=batch, batch=batch, heads=heads, kv=kv, dim=128, dtype=dtype, quantized=quantized, pages=1 << 16)
    sizes = {_bytes(prefix, width=(prefix + own) // 16, **kw) for own in (16, 512, 1024, 8192, 131072 - prefix, 131072)}
    assert len(sizes) == 1


def test_a_part_has_no_more_than_16_key_tiles():
    """... as long as the parts fit 112 SMs."""
    row = 32 * (128 + 4) * 4  # of sums
    for batch, prefix in ((16, 8192), (16, 16384), (64, 8192), (64, 16384), (32, 4096)):
        kw = dict(rows=batch, batch=batch, heads=32, kv=8, dim=128, pages=1 << 16, width=1 << 13)
        parts = (_bytes(prefix, **kw) - _plain(**kw)) // (batch * row) - 1
        ctas = -(-batch // 64) * 8
        assert 64 <= parts * ctas <= 112
        assert parts * 16 >= prefix // 128
