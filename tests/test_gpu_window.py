"""Sliding windows whose first tokens stay visible, of prompts (with gradients) and over the paged cache, against
the definition in 64 bits (oracle/attention_oracle.py) with the bounds derived there."""
from __future__ import annotations

import pytest
import torch

from oracle import attention_oracle as A
from test_gpu_attention import DTYPES, _check_sequence, _inputs, _run, _within
from test_gpu_paged import Setup

pytestmark = pytest.mark.gpu

REACHES = [(1, 0), (1, 3), (7, 0), (64, 4), (100, 130), (128, 0), (129, 1), (200, 64)]


@pytest.fixture(autouse=True)
def no_device_error():
    from cta_b200 import _lib

    yield
    assert _lib.device_error() == 0


def _reach(rows, keys, window, sinks, valid=None, first=None):
    """[rows, keys]: the rows are the last ones of `keys` tokens, or begin at place `first`."""
    i = torch.arange(rows, device="cuda")[:, None] + (keys - rows if first is None else first)
    j = torch.arange(keys, device="cuda")[None, :]
    start = 0
    if valid is not None and bool(valid.any()):
        start = int(valid.nonzero()[0])
    see = (j <= i) & ((j > i - window) | (j < start + sinks))
    return see if valid is None else see & valid.to("cuda")[None, :]


# ---------------------------------------------------------------------------
# prompts
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", REACHES)
@pytest.mark.parametrize("length", [1, 2, 64, 65, 127, 129, 257, 400, 700])
def test_padded_lengths(length, window, sinks, dtype):
    q, k, v, g = _inputs((2, length), 4, 2, 64, dtype, seed=length)
    got = _run(q, k, v, g, causal=True, window=window, sinks=sinks)
    for b in range(2):
        _check_sequence([x[b] for x in got], q[b], k[b], v[b], g[b], _reach(length, length, window, sinks), 64**-0.5, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 20, 32, 72, 96, 128, 136, 256])
def test_head_dims(dim, dtype):
    q, k, v, g = _inputs((1, 333), 2, 1, dim, dtype, seed=dim)
    got = _run(q, k, v, g, causal=True, window=50, sinks=5)
    _check_sequence([x[0] for x in got], q[0], k[0], v[0], g[0], _reach(333, 333, 50, 5), dim**-0.5, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(33, 0), (150, 4)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(3, 3, 64), (6, 2, 128), (8, 1, 64), (12, 2, 128), (32, 4, 32)])
def test_head_groups(heads, kv_heads, dim, window, sinks, dtype):
    q, k, v, g = _inputs((1, 520), heads, kv_heads, dim, dtype, seed=heads)
    got = _run(q, k, v, g, causal=True, window=window, sinks=sinks)
    _check_sequence([x[0] for x in got], q[0], k[0], v[0], g[0], _reach(520, 520, window, sinks), dim**-0.5, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (60, 4), (300, 0), (128, 200)])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 4), (128, 8, 2)])
def test_packed(dim, heads, kv_heads, window, sinks, dtype):
    lens = [1, 700, 0, 130, 257, 64, 3]
    total = sum(lens) + 9  # rows behind the last sequence
    q, k, v, g = _inputs((total,), heads, kv_heads, dim, dtype, seed=dim)
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32).cuda()
    for x in (q, k, v, g):
        x[sum(lens):] = float("nan")
    got = _run(q, k, v, g, causal=True, cu_seqlens=cu, window=window, sinks=sinks)
    at = 0
    for n in lens:
        part = slice(at, at + n)
        at += n
        if n:
            _check_sequence([x[part] for x in got], q[part], k[part], v[part], g[part], _reach(n, n, window, sinks),
                            dim**-0.5, dtype, f"{n}: ")
    for x in got:
        assert (x[at:] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(70, 4), (70, 0), (5, 0), (200, 150)])
@pytest.mark.parametrize("kind", ["right", "left", "holes", "gap", "none", "one"])
def test_key_masks(kind, window, sinks, dtype):
    """Rows whose windows hold no valid key are zero and take no part, whatever they hold; first tokens count from the
    first valid one."""
    L = 450
    q, k, v, g = _inputs((3, L), 4, 2, 64, dtype, seed=7)
    mask = torch.ones(3, L, dtype=torch.bool)
    if kind == "right":
        mask[0, 333:], mask[1, 1:], mask[2, 128:] = False, False, False
    elif kind == "left":
        mask[0, :200], mask[1, :1], mask[2, :449] = False, False, False
    elif kind == "holes":
        mask = torch.rand(3, L, generator=torch.Generator().manual_seed(1)) < 0.4
    elif kind == "gap":  # longer than the shorter windows
        mask[0, 100:300], mask[1, 2:440], mask[2, 128:256] = False, False, False
    elif kind == "none":
        mask[0] = False
    else:
        mask[:] = False
        mask[0, 0], mask[1, 77], mask[2, L - 1] = True, True, True
    sees = [_reach(L, L, window, sinks, m) for m in mask]
    for b in range(3):
        blind = ~sees[b].any(1)
        for x in (k, v):
            x[b][~mask[b].cuda()] = float("nan")
        q[b][blind], g[b][blind] = float("inf"), float("nan")
    got = _run(q, k, v, g, causal=True, key_mask=mask.cuda(), window=window, sinks=sinks)
    for b in range(3):
        blind = ~sees[b].any(1)
        clean = [x[b].clone() for x in (q, g)]
        for x in clean:
            x[blind] = 0
        kc, vc = (torch.where(mask[b].cuda()[:, None, None], x[b], torch.zeros_like(x[b])) for x in (k, v))
        _check_sequence([x[b] for x in got], clean[0], kc, vc, clean[1], sees[b], 0.125, dtype, f"{kind} {b}: ")
        assert (got[0][b][blind] == 0).all() and (got[1][b][blind] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(513, 0), (400, 113), (10**9, 0), (2**40, 2**50), (1, 512)])
def test_window_over_everything_is_none(window, sinks, dtype):
    q, k, v, g = _inputs((1, 513), 4, 2, 64, dtype)
    for x, y in zip(_run(q, k, v, g, causal=True, window=window, sinks=sinks), _run(q, k, v, g, causal=True)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,window,sinks", [([3, 0, 1, 20, 8], 2**40, 0), ([32], 40, 3), ([33], 20, 12), ([700, 31, 2], 1, 31),
                                               ([300, 9], 2, 0)])
def test_few_keys(lens, window, sinks, dtype):
    """Gradients of rows that see few keys, up to the sizes from which the tensor cores compute them and beyond."""
    for heads, kv_heads, dim in ((2, 1, 40), (16, 4, 128)):
        total = sum(lens) + 3
        q, k, v, g = _inputs((total,), heads, kv_heads, dim, dtype, seed=total)
        cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32).cuda()
        for x in (q, k, v, g):
            x[sum(lens):] = float("nan")
        got = _run(q, k, v, g, causal=True, cu_seqlens=cu, window=window, sinks=sinks)
        at = 0
        for n in lens:
            part = slice(at, at + n)
            at += n
            if n > 0:
                _check_sequence([x[part] for x in got], q[part], k[part], v[part], g[part], _reach(n, n, window, sinks),
                                dim**-0.5, dtype)
        assert all((x[at:] == 0).all() for x in got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,heads,kv_heads,window,sinks", [(64, 8, 8, 1024, 4), (128, 8, 2, 500, 16), (128, 4, 1, 2000, 300),
                                                            (64, 2, 2, 31, 129)])
def test_long(dim, heads, kv_heads, window, sinks, dtype):
    """Long enough for the first keys' gradients to be summed in parts."""
    n = 5000
    q, k, v, g = _inputs((1, n), heads, kv_heads, dim, dtype, seed=5)
    got = _run(q, k, v, g, causal=True, window=window, sinks=sinks)
    group = heads // kv_heads
    see = _reach(n, n, window, sinks)
    for h in range(kv_heads):
        part = slice(h * group, (h + 1) * group)
        one = [got[0][0][:, part], got[1][0][:, part], got[2][0][:, h : h + 1], got[3][0][:, h : h + 1]]
        _check_sequence(one, q[0][:, part], k[0][:, h : h + 1], v[0][:, h : h + 1], g[0][:, part], see, dim**-0.5, dtype)


@pytest.mark.parametrize("dim,heads,kv_heads,window,sinks,dtype", [(64, 2, 2, 200, 4, torch.float32), (128, 2, 1, 60, 70, torch.float32),
                                                                  (192, 2, 1, 31, 40, torch.bfloat16), (20, 4, 4, 5, 3, torch.float16)])
def test_long_without_tensor_cores(dim, heads, kv_heads, window, sinks, dtype):
    n = 2500
    q, k, v, g = _inputs((2, n), heads, kv_heads, dim, dtype, seed=9)
    got = _run(q, k, v, g, causal=True, window=window, sinks=sinks)
    see = _reach(n, n, window, sinks)
    for b in range(2):
        _check_sequence([x[b] for x in got], q[b], k[b], v[b], g[b], see, dim**-0.5, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,window,sinks", [([3000, 40, 4100, 1500], 300, 20), ([5] * 40 + [70] * 50 + [600, 0, 411] + [3] * 30, 30, 4),
                                               ([9, 333, 1200], 12, 4)])
def test_long_packed(lens, window, sinks, dtype):
    q, k, v, g = _inputs((sum(lens),), 4, 1, 64, dtype, seed=6)
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32).cuda()
    got = _run(q, k, v, g, causal=True, cu_seqlens=cu, window=window, sinks=sinks)
    at = 0
    for n in lens:
        part = slice(at, at + n)
        at += n
        if n == 0:
            continue
        _check_sequence([x[part] for x in got], q[part], k[part], v[part], g[part], _reach(n, n, window, sinks), 0.125, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_masked(dtype):
    """First tokens in the middle of a key tile, and over the edge of one; their rows far behind."""
    L, window = 3300, 200
    q, k, v, g = _inputs((3, L), 2, 1, 128, dtype, seed=8)
    mask = torch.ones(3, L, dtype=torch.bool)
    mask[0, :700] = False
    mask[1, :1000], mask[1, 3000:] = False, False
    mask[2, 1:] = False
    for sinks in (4, 40):
        got = _run(q, k, v, g, causal=True, key_mask=mask.cuda(), window=window, sinks=sinks)
        for b in range(3):
            _check_sequence([x[b] for x in got], q[b], k[b], v[b], g[b], _reach(L, L, window, sinks, mask[b]), 128**-0.5,
                            dtype)


def test_gradient_against_differences():
    gen = torch.Generator().manual_seed(3)
    q, k, v, g = _inputs((1, 90), 2, 1, 16, torch.float32, seed=3)
    from cta_b200.attention import prompt_attention

    kw = dict(causal=True, window=20, sinks=3)
    grads = _run(q, k, v, g, **kw)[1:]
    for i, x in enumerate((q, k, v)):
        for _ in range(4):
            e = torch.randn(x.shape, generator=gen).cuda()
            step = 1e-2
            moved = []
            for s in (step, -step):
                args = [q, k, v]
                args[i] = x + s * e
                moved.append((prompt_attention(*args, **kw).double() * g.double()).sum())
            # fp32 outputs carry 2^-22 or so of their size, a third of which sums up by chance over 2880 terms; the
            # difference's own error is of the order of step^2
            want = (moved[0] - moved[1]) / (2 * step)
            have = (grads[i].double() * e.double()).sum()
            assert abs(want - have) < 2e-3 * (1 + abs(have)), (i, want, have)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_twice_the_same(dtype):
    q, k, v, g = _inputs((2, 300), 4, 4, 64, dtype, seed=11)
    both = torch.stack([q, k, v], dim=2)  # a projection's output
    kw = dict(causal=True, window=40, sinks=2)
    want = _run(q, k, v, g, **kw)
    for got in (_run(*both.unbind(2), g.transpose(1, 2).contiguous().transpose(1, 2), **kw), _run(q, k, v, g, **kw)):
        for x, y in zip(got, want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_and_on_two_streams(dtype):
    from cta_b200 import ops

    n, kw = 2600, dict(causal=True, window=300, sinks=8)
    cases = [_inputs((1, n), 4, 2, 64, dtype, seed=s) for s in (1, 2)]

    def step(q, k, v, g):
        low = None if dtype == torch.float32 else torch.empty_like(q)
        out, lse = ops.attention_forward(q, k, v, out_low=low, **kw)
        return (out, *ops.attention_backward(g, q, k, v, out, lse, out_low=low, **kw))

    want = [step(*c) for c in cases]
    graphs, outs = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*c))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for x in outs:
            for y in x:
                y.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(x, y))


def test_empty():
    from cta_b200.attention import prompt_attention

    for shape in ((0, 5), (2, 0)):
        x = torch.empty(*shape, 2, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        out = prompt_attention(x, x, x, causal=True, window=2, sinks=1)
        assert out.shape == x.shape
        out.sum().backward()


def test_only_wanted_gradients():
    q, k, v, g = _inputs((1, 2500), 2, 2, 64, torch.bfloat16)
    want = _run(q, k, v, g, causal=True, window=100, sinks=4)
    from cta_b200.attention import prompt_attention

    for i in range(3):
        x = [t.detach().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        out = prompt_attention(*x, causal=True, window=100, sinks=4)
        (got,) = torch.autograd.grad(out, (x[i],), g)
        assert torch.equal(got, want[1 + i])


# ---------------------------------------------------------------------------
# over the cache
# ---------------------------------------------------------------------------
def _check_paged(s, out, window, sinks):
    at = 0
    scale = s.dim**-0.5
    for b, (n, r) in enumerate(zip(s.lens, s.rows)):
        q, got = s.q[at : at + r], out[at : at + r]
        at += r
        if r == 0:
            continue
        if n == 0:
            assert (got == 0).all()
            continue
        see = _reach(r, n, window, sinks)
        want, _ = A.attention(q, s.k[b], s.v[b], see, scale)
        tol = A.bounds(q, s.k[b], s.v[b], see, scale, s.dtype, kv_error=2.0**-20 if s.quantized else 0.0)
        _within(got, want, tol, f"sequence {b} of {n}, {r} rows: ")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("window,sinks", [*REACHES, (1000, 4), (16, 16), (17, 33)])
def test_decode(window, sinks, quantized, dtype):
    s = Setup([1, 15, 16, 17, 79, 80, 200, 1333, 0], [1] * 9, 8, 2, 64, 16, dtype, quantized, seed=window)
    _check_paged(s, s.run(window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(3, 1, 128, 16), (16, 1, 32, 48), (8, 8, 128, 64), (40, 2, 80, 256), (71, 1, 64, 32)])
def test_decode_groups_and_pages(heads, kv_heads, dim, page, quantized):
    s = Setup([40, 700, 1, 259], [1] * 4, heads, kv_heads, dim, page, torch.bfloat16, quantized, seed=heads)
    for window, sinks in ((100, 5), (30, 0), (5, 70)):
        _check_paged(s, s.run(window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 4), (128, 0), (150, 140), (300, 20)])
@pytest.mark.parametrize("rows", [[2, 2, 2], [1, 0, 5], [17, 1, 130], [128, 129, 127], [300, 64, 0], [1, 400, 33]])
def test_chunks(rows, window, sinks, quantized, dtype):
    lens = [r + x for r, x in zip(rows, (0, 77, 800))]
    for heads, kv_heads, dim, page in ((4, 4, 64, 16), (32, 8, 128, 64), (6, 2, 80, 48)):
        s = Setup(lens, rows, heads, kv_heads, dim, page, dtype, quantized, seed=sum(rows))
        _check_paged(s, s.run(window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("rows,heads,kv_heads", [([1, 1, 1], 8, 2), ([3, 1, 20], 8, 2), ([200, 130, 300], 32, 8)])
@pytest.mark.parametrize("window,sinks", [(49, 4), (60, 0), (100, 17)])
@pytest.mark.parametrize("page", [16, 64])
def test_freed_pages_are_not_read(page, window, sinks, rows, heads, kv_heads, quantized):
    """Pages between the first tokens and the windows: their entries lie outside the cache or in pages of NaN."""
    lens = [r + x for r, x in zip(rows, (400, 1023, 640))]
    s = Setup(lens, rows, heads, kv_heads, 64, page, torch.bfloat16, quantized, seed=window)
    want = s.run(window=window, sinks=sinks)
    spare = (set(range(s.kc.shape[0])) - set(s.table.flatten().tolist())).pop()
    for x in (s.kc, s.vc):
        x.view(torch.uint8)[spare] = 0xFF  # NaN in e4m3 and in bf16
    for x in (s.ks, s.vs):
        if x is not None:
            x[spare] = float("nan")
    freed = 0
    for b, (n, r) in enumerate(zip(lens, rows)):
        for p in range(-(-n // page)):
            begin, end = p * page, (p + 1) * page
            if begin >= sinks and end <= n - r - window + 1:
                s.table[b, p] = (spare, 2**31 - 1, -1)[p % 3]
                freed += 1
    assert freed > 5
    assert torch.equal(s.run(window=window, sinks=sinks), want)
    _check_paged(s, want, window, sinks)


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("rows", [[1, 1], [40, 200]])
def test_paged_window_over_everything_is_none(rows, quantized):
    s = Setup([300, 513], rows, 8, 2, 64, 16, torch.bfloat16, quantized)
    want = s.run()
    for window, sinks in ((33 * 16, 0), (400, 128), (2**40, 3), (1, 2**45)):
        assert torch.equal(s.run(window=window, sinks=sinks), want)


@pytest.mark.parametrize("rows", [[1, 1], [40, 200]])
@pytest.mark.parametrize("quantized", [False, True])
def test_bad_pages_in_the_window(rows, quantized):
    """A page outside the cache among those that count is left out and reported."""
    from cta_b200 import _lib

    s = Setup([300, 513], rows, 8, 2, 64, 16, torch.bfloat16, quantized)
    s.table[1, 0] = 10**6
    out = s.run(window=100, sinks=8)
    torch.cuda.synchronize()
    assert _lib.device_error() == 2
    at = rows[0]
    valid = torch.ones(513, dtype=torch.bool)
    valid[:16] = False
    see = _reach(rows[1], 513, 100, 8) & valid.cuda()[None, :]
    want, _ = A.attention(s.q[at : at + rows[1]], s.k[1], s.v[1], see, 0.125)
    tol = A.bounds(s.q[at : at + rows[1]], s.k[1], s.v[1], see, 0.125, s.dtype, kv_error=2.0**-20 if quantized else 0.0)
    _within(out[at : at + rows[1]], want, tol, "")


@pytest.mark.parametrize("quantized", [False, True])
def test_large_window_batch(quantized):
    lens = [int(x) for x in torch.randint(1, 4000, (70,), generator=torch.Generator().manual_seed(2))]
    s = Setup(lens, [1] * 70, 8, 2, 128, 16, torch.bfloat16, quantized, seed=9)
    _check_paged(s, s.run(window=512, sinks=4), 512, 4)


@pytest.mark.parametrize("rows", [[1, 1, 1], [40, 200, 7]])
@pytest.mark.parametrize("quantized", [False, True])
def test_paged_captured_and_replayed_together(rows, quantized):
    setups = [Setup([300, 513, 77], rows, 8, 2, 64, 16, torch.bfloat16, quantized, seed=x) for x in (1, 2)]
    want = [s.run(window=64, sinks=4) for s in setups]
    graphs, outs = [], []
    for s in setups:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(s.run(window=64, sinks=4))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for x in outs:
            x.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("rows", [[1, 1], [40, 200]])
@pytest.mark.parametrize("quantized", [False, True])
def test_rows_behind_the_last_sequence(rows, quantized):
    s = Setup([300, 513], rows, 8, 2, 64, 16, torch.bfloat16, quantized, tail=5)
    out = torch.full_like(s.q, 7.0)
    s.run(out=out, window=50, sinks=2, cu_seqlens=s.cu)
    assert (out[sum(rows):] == 7).all()
    _check_paged(s, out, 50, 2)


# ---------------------------------------------------------------------------
# the language model
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("window,sinks", [(16, 0), (40, 4)])
@pytest.mark.parametrize("length", [1, 37, 200])
def test_language_model(length, window, sinks):
    """Logits and gradients are those of the stock layers under the same mask."""
    from cta_b200 import transformers as T

    torch.manual_seed(0)
    kw = dict(vocab_size=50, embed_dim=64, num_heads=4, hidden_dim=96, num_layers=2, pde_steps=2, max_length=256, dropout=0.0)
    model = T.PDETransformerLM(attention="fused", attention_window=window, attention_sinks=sinks, **kw).cuda()
    stock = T.PDETransformerLM(**kw).cuda()
    stock.load_state_dict(model.state_dict())
    ids = torch.randint(0, 50, (3, length), device="cuda")
    mask = torch.ones(3, length, dtype=torch.long, device="cuda")
    mask[1, max(1, length - 9):] = 0
    see = _reach(length, length, window, sinks)
    hidden = torch.zeros(length, length, device="cuda").masked_fill(~see, float("-inf"))
    patched = T.generate_causal_mask
    try:
        T.generate_causal_mask = lambda n, device: hidden
        want = stock(ids, mask)
    finally:
        T.generate_causal_mask = patched
    got = model(ids, mask)
    live = mask.bool()
    # the padding's rows see nothing once their windows have left the valid tokens: NaN in the stock softmax, so the
    # comparison is of valid rows, which no later row reaches (refinement is causal)
    scale = want[live].abs().max()
    assert ((got - want)[live].abs() <= 1e-5 * scale + 1e-6).all()
    weight = torch.randn_like(got[live])
    (got[live] * weight).sum().backward()
    if length > 1 and window < 40:
        return  # NaN of the stock padding rows reach its gradients
    (want[live] * weight).sum().backward()
    for (name, a), b in zip(model.named_parameters(), stock.parameters()):
        if b.grad is None or not torch.isfinite(b.grad).all():
            continue
        assert torch.isfinite(a.grad).all()
        # sums of fp32 products over up to 3 x 200 tokens and two layers: 1e-4 of the largest entry
        assert ((a.grad - b.grad).abs() <= 1e-4 * b.grad.abs().max() + 1e-6).all(), name


def test_language_model_saved_and_refused(tmp_path):
    from cta_b200 import transformers as T

    kw = dict(vocab_size=5, embed_dim=8, num_heads=2, hidden_dim=8, num_layers=1)
    with pytest.raises(ValueError, match="fused"):
        T.PDETransformerLM(attention_window=4, **kw)
    with pytest.raises(ValueError, match="window"):
        T.PDETransformerLM(attention="fused", attention_sinks=4, **kw)
    with pytest.raises(ValueError, match="window"):
        T.PDETransformerLM(attention="fused", attention_window=0, **kw)
    model = T.PDETransformerLM(attention="fused", attention_window=3, attention_sinks=1, **kw).cuda().eval()
    torch.save(model, tmp_path / "m.pt")
    again = torch.load(tmp_path / "m.pt", weights_only=False)
    ids, mask = torch.randint(0, 5, (2, 20), device="cuda"), torch.ones(2, 20, device="cuda")
    assert torch.equal(model(ids, mask), again(ids, mask))
    plain = T.PDETransformerLM(attention="fused", **kw).cuda().eval()
    plain.load_state_dict(model.state_dict())
    assert not torch.equal(model(ids, mask)[:, 4:], plain(ids, mask)[:, 4:])
    assert torch.equal(model(ids, mask)[:, :3], plain(ids, mask)[:, :3])
