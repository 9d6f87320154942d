"""CPU-only: the workspace of chunks over an e4m3 cache under a window follows from the rows and the window."""
from __future__ import annotations

import pytest

from test_more_attention_host import _paged


def _chunk(width, batch=4, rows=512, page=16, **kw):
    return _paged(rows=batch * rows, batch=batch, heads=32, kv=8, dim=128, page=page, width=width, pages=1 << 16, quantized=1, cu=16,
                  **kw)


def _bytes(args, window, sinks):
    from cta_b200 import _lib

    return _lib.load().cta_window_paged_attention_workspace_bytes(args, window, sinks)


def _rows(args, rows):
    # max_rows is the fourth 64-bit size from the end of the sizes: repack through the struct
    from cta_b200 import _lib

    x = list(_lib.PAGED_ATTENTION_ARGS.unpack(args))
    x[-5] = rows
    return _lib.PAGED_ATTENTION_ARGS.pack(*x)


@pytest.mark.parametrize("batch,rows", [(4, 512), (16, 512), (1, 2000), (64, 128)])
@pytest.mark.parametrize("window,sinks", [(1024, 4), (512, 0), (4000, 200)])
def test_width_does_not_count(batch, rows, window, sinks):
    sizes = {_bytes(_rows(_chunk(width, batch, rows), rows), window, sinks) for width in (2048, 8192, 16384)}
    assert len(sizes) == 1
    (size,) = sizes
    # codes as 16-bit rows and two fractions beside them, for the window, the first keys and the rows, in tiles of 128
    keys = batch * (window + sinks + 4 * 128) + batch * rows + 128
    assert 0 < size <= keys * 8 * (4 * 128 + 8) + 64


def test_no_more_than_the_table():
    wide, narrow = (_bytes(_rows(_chunk(width, 2, 300, page=64), 300), 900, 4) for width in (4096, 16))
    assert narrow < wide
    # a window as long as the table costs what the table does
    assert narrow <= 2 * 1024 * 8 * (4 * 128 + 8) + 64
