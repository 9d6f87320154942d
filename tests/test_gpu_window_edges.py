"""Sliding windows at the edges of what a call may hold: lengths past the block table, gradients of very different
sizes, few keys a row at every size of a call, padding longer than the window; against the definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

from test_gpu_attention import _check_sequence, _inputs, _run
from test_gpu_paged import Setup
from test_gpu_window import _reach

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error():
    from cta_b200 import _lib

    yield
    assert _lib.device_error() == 0


def _poisoned(s, **kw):
    """paged_attention of the setup in a workspace of NaN, as an earlier call may have left it."""
    from cta_b200 import _lib, ops

    q, out, fn, args, nbytes, held = ops._paged_plan(
        s.q, s.kc, s.vc, s.table, s.seq_lens, s.cu, max(s.rows), None, s.ks, s.vs, None, kw["window"], kw["sinks"])
    ws = torch.full((nbytes,), 0xFF, dtype=torch.uint8, device="cuda")
    _lib.enqueue(fn, q, *args, ws.data_ptr(), nbytes)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("rows", [[1, 1], [40, 200]])
@pytest.mark.parametrize("past", [1, 17, 100, 1000, 2**31 - 1 - 640])
def test_lengths_past_the_table(past, rows, quantized, dtype):
    """Reported, and computed as if the sequence ended with the table: no row holds what nobody wrote."""
    from cta_b200 import _lib

    s = Setup([640, 640], rows, 32, 8, 64, 16, dtype, quantized, seed=past % 1000)
    for window, sinks in ((100, 8), (30, 0), (257, 33)):
        want = _poisoned(s, window=window, sinks=sinks)
        assert _lib.device_error() == 0 and torch.isfinite(want.float()).all()
        for b in (0, 1):
            s.seq_lens[b] = 640 + past
            got = _poisoned(s, window=window, sinks=sinks)
            assert _lib.device_error() == 2
            assert torch.equal(got, want)
            s.seq_lens[b] = 640


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 1, 64), (4, 1, 128)])
@pytest.mark.parametrize("scale,size", [(2e-6, 1.5e4), (2e-7, 1.5e4), (0.1, 1.0)])
def test_gradients_far_behind_rows_without(scale, size, heads, kv_heads, dim, dtype):
    """Only late rows have a gradient, as where a prompt's tokens carry no loss: what reaches the first keys comes from the
    rows behind their tile alone, and is right for any scale."""
    n, window, sinks = 3000, 128, 4
    q, k, v, g = _inputs((1, n), heads, kv_heads, dim, dtype, seed=12)
    q, g = ((x.float() * size).clamp(-6e4, 6e4).to(dtype) for x in (q, g))  # fp16's largest number is 65504
    g[:, :500] = 0
    got = _run(q, k, v, g, causal=True, window=window, sinks=sinks, scale=scale)
    _check_sequence([x[0] for x in got], q[0], k[0], v[0], g[0], _reach(n, n, window, sinks), scale, dtype)


def _graph_time(call, n=10):
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(n):
            call()
    times = []
    for _ in range(7):
        a, b = torch.cuda.Event(True), torch.cuda.Event(True)
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) / n)
    return sorted(times)[3]


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,window,sinks", [(256, 32, 8, 128, 4, 4), (256, 32, 8, 128, 4, 0), (1024, 8, 2, 128, 4, 4),
                                                                   (2048, 8, 8, 64, 4, 4), (1024, 8, 8, 64, 16, 4)])
def test_windows_of_few_keys_cost_what_others_do(tokens, heads, kv_heads, dim, window, sinks):
    """Where the FP32 pipe would take longer than a training call takes to make, or is no more exact, the tensor cores
    compute the gradients, as under wider windows."""
    from cta_b200 import ops

    q, k, v, g = _inputs((1, tokens), heads, kv_heads, dim, torch.bfloat16, seed=3)
    times = []
    for w in (window, 40):
        kw = dict(causal=True, window=w, sinks=sinks)
        low = torch.empty_like(q)
        out, lse = ops.attention_forward(q, k, v, out_low=low, **kw)
        times.append(_graph_time(lambda: ops.attention_backward(g, q, k, v, out, lse, out_low=low, **kw)))
    # the same steps of work, within the few percent of a clock that moves; 2.7 to 14 times on the FP32 pipe
    assert times[0] < 1.5 * times[1], times


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim", [(300, 4, 4, 64), (300, 4, 1, 128), (9, 6, 2, 96)])
@pytest.mark.parametrize("window,sinks", [(2, 0), (3, 0), (1, 1), (4, 4), (8, 0), (9, 0), (5, 4)])
def test_few_keys_on_either_side_of_the_rule(window, sinks, tokens, heads, kv_heads, dim, dtype):
    q, k, v, g = _inputs((2, tokens), heads, kv_heads, dim, dtype, seed=window)
    got = _run(q, k, v, g, causal=True, window=window, sinks=sinks)
    for b in range(2):
        _check_sequence([x[b] for x in got], q[b], k[b], v[b], g[b], _reach(tokens, tokens, window, sinks), dim**-0.5, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 4), (100, 0), (128, 130), (257, 33), (700, 300), (1000, 1)])
@pytest.mark.parametrize("rows,more", [([40, 200, 1, 0, 64], (0, 77, 900, 3, 1000)), ([130, 1, 127, 129], (1000, 640, 5, 333)),
                                       ([1, 300, 2, 2, 2, 2, 90, 1], (5, 0, 700, 701, 702, 100, 64, 1500))])
def test_chunks_with_wide_tables(rows, more, window, sinks, dtype):
    """An e4m3 cache's copy holds what the rows can reach, however wide the block table: nothing else is read, the results
    are those of a narrow table bit for bit, and right."""
    from test_gpu_window import _check_paged

    lens = [r + x for r, x in zip(rows, more)]
    for heads, kv_heads, dim, page in ((32, 8, 64, 16), (12, 6, 80, 48), (32, 8, 128, 64)):
        s = Setup(lens, rows, heads, kv_heads, dim, page, dtype, True, seed=window, tail=3)
        narrow = s.table
        want = _poisoned(s, window=window, sinks=sinks)
        wide = torch.full((len(lens), 131072 // page), 2**31 - 1, dtype=torch.int32, device="cuda")
        wide[:, : narrow.shape[1]] = narrow
        s.table = wide
        got = _poisoned(s, window=window, sinks=sinks)
        total = sum(rows)
        assert torch.equal(got[:total], want[:total])
        _check_paged(s, got, window, sinks)
