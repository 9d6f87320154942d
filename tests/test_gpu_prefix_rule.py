"""A shared prefix costs no call more than leaving it out, however many keys of their own the sequences have and however
wide their block table is."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _time(call, n=10):
    """Median device time of a call in a captured graph of n of them."""
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(n):
            call()
    graph.replay()
    torch.cuda.synchronize()
    times = []
    for _ in range(7):
        a, b = torch.cuda.Event(True), torch.cuda.Event(True)
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) / n)
    return sorted(times)[3]


def _both(batch, prefix, low, high, width=None):
    """(with, without): 32/8 heads of 128 over 16 bits."""
    from cta_b200 import ops

    page = 16
    gen = torch.Generator().manual_seed(batch)
    own = torch.randint(low, high + 1, (batch,), generator=gen)
    counts = (own + page - 1) // page
    pages = prefix // page + int(counts.sum())
    table = torch.zeros(batch, width or (prefix + high) // page + 1, dtype=torch.int32)
    table[:, : prefix // page] = torch.arange(prefix // page)
    at = prefix // page
    for b, n in enumerate(counts.tolist()):
        table[b, prefix // page : prefix // page + n] = torch.arange(at, at + n)
        at += n
    table, lens = table.cuda(), (own + prefix).int().cuda()
    q = torch.randn(batch, 32, 128, device="cuda").bfloat16()
    kc, vc = (torch.randn(pages, page, 8, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2))

    def call(shared):
        return ops.paged_attention(q, kc, vc, table, lens, shared_prefix=shared)

    return _time(lambda: call(prefix)), _time(lambda: call(0))


def test_long_own_keys():
    """The split kernel runs beside the parts without losing its L1 to their shared memory."""
    shared, plain = _both(64, 2048, 2048, 4096)
    # 0.9 of it; 1.5 where it lost its L1.  A clock that changes between the two moves this by a few percent.
    assert shared < 1.2 * plain, (shared, plain)


@pytest.mark.parametrize("batch,prefix,low,high", [(16, 8192, 16, 64), (4, 16384, 16, 1024), (16, 8192, 2048, 4096), (64, 8192, 16, 1024),
                                                  (16, 2048, 2048, 4096)])
def test_wide_block_tables(batch, prefix, low, high):
    """Tables of an engine whose sequences may be 131072 keys long."""
    shared, plain = _both(batch, prefix, low, high, width=131072 // 16)
    # 0.3 to 1.02 of it; 2 to 6 times as much where the table's width was taken for the sequences'
    assert shared < 1.2 * plain, (shared, plain)
