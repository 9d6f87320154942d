"""Attention of prompts against its definition in 64 bits (oracle/attention_oracle.py),
with the bounds derived there."""
from __future__ import annotations

import pytest
import torch

from oracle import attention_oracle as A

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _rand(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen, dtype=torch.float32).to(dtype).cuda()


def _inputs(shape, heads, kv_heads, dim, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    q = _rand(gen, *shape, heads, dim, dtype=dtype)
    k = _rand(gen, *shape, kv_heads, dim, dtype=dtype)
    v = _rand(gen, *shape, kv_heads, dim, dtype=dtype)
    g = _rand(gen, *shape, heads, dim, dtype=dtype)
    return q, k, v, g


def _see(n, causal, valid=None, device="cuda"):
    see = torch.ones(n, n, dtype=torch.bool, device=device)
    if causal:
        see = see.tril()
    if valid is not None:
        see = see & valid.to(device)[None, :]
    return see


def _within(got, want, tol, what):
    got = got.detach().double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: {got[i].item()} for "
                             f"{want[i].item()}, bound {tol[i].item()}")


def _check_sequence(got, q, k, v, g, see, scale, dtype, what=""):
    out, dq, dk, dv = got
    want, _ = A.attention(q, k, v, see, scale)
    if dq is None:
        _within(out, want, A.bounds(q, k, v, see, scale, dtype), what + "out")
        return
    tol = A.bounds(q, k, v, see, scale, dtype, g)
    _within(out, want, tol[0], what + "out")
    for x, y, t, name in zip((dq, dk, dv), A.gradients(q, k, v, g, see, scale), tol[1:], ("dq", "dk", "dv")):
        _within(x, y, t, what + name)


def _run(q, k, v, g, **kw):
    from cta_b200.attention import prompt_attention

    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    out = prompt_attention(q, k, v, **kw)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), g)
    return out.detach(), dq, dk, dv


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("length", [1, 2, 31, 64, 65, 127, 128, 129, 255, 300, 513])
def test_padded_lengths(length, causal, dtype):
    q, k, v, g = _inputs((2, length), 4, 2, 64, dtype, seed=length)
    got = _run(q, k, v, g, causal=causal)
    for b in range(2):
        _check_sequence([x[b] for x in got], q[b], k[b], v[b], g[b], _see(length, causal), 64**-0.5, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 7, 8, 16, 24, 32, 40, 64, 72, 80, 96, 104, 128, 136, 192, 256])
def test_head_dims(dim, dtype):
    q, k, v, g = _inputs((1, 150), 2, 1, dim, dtype, seed=dim)
    got = _run(q, k, v, g, causal=True)
    _check_sequence([x[0] for x in got], q[0], k[0], v[0], g[0], _see(150, True), dim**-0.5, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (3, 1), (6, 2), (8, 1), (12, 2), (40, 8), (64, 1)])
def test_head_groups(heads, kv_heads, dtype):
    q, k, v, g = _inputs((1, 140), heads, kv_heads, 64, dtype, seed=heads)
    got = _run(q, k, v, g, causal=True)
    _check_sequence([x[0] for x in got], q[0], k[0], v[0], g[0], _see(140, True), 64**-0.5, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_packed(dim, causal, dtype):
    """Ragged sequences, empty ones among them, with rows behind the last sequence."""
    lengths = [0, 1, 130, 0, 0, 257, 64, 3, 128, 0]
    total = sum(lengths)
    q, k, v, g = _inputs((total + 5,), 4, 2, dim, dtype, seed=dim)
    for x in (q, k, v, g):
        x[total:] = float("nan")  # nothing there may be read into a sequence
    cu = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    got = _run(q, k, v, g, causal=causal, cu_seqlens=cu)
    at = 0
    for n in lengths:
        part = slice(at, at + n)
        if n:
            _check_sequence([x[part] for x in got], q[part], k[part], v[part], g[part], _see(n, causal), dim**-0.5,
                            dtype, f"at {at}: ")
        at += n
    for x in got:
        assert (x[total:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_packed_many_sequences(dtype):
    """More sequences than lanes of a warp."""
    gen = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 90, (150,), generator=gen).tolist()
    q, k, v, g = _inputs((sum(lengths),), 2, 2, 64, dtype, seed=9)
    cu = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    got = _run(q, k, v, g, causal=True, cu_seqlens=cu)
    at = 0
    for n in lengths:
        part = slice(at, at + n)
        if n:
            _check_sequence([x[part] for x in got], q[part], k[part], v[part], g[part], _see(n, True), 0.125, dtype)
        at += n


def test_packed_neighbours_do_not_mix():
    """A sequence's result does not depend on its neighbours' values, NaN among them."""
    from cta_b200.attention import prompt_attention

    for dtype in DTYPES:
        q, k, v, g = _inputs((300,), 2, 2, 64, dtype)
        cu = torch.tensor([0, 100, 170, 300], dtype=torch.int32, device="cuda")
        clean = _run(q, k, v, g, causal=False, cu_seqlens=cu)
        for x in (q, k, v, g):
            x[:100] = float("nan")
            x[170:] = float("inf")
        dirty = _run(q, k, v, g, causal=False, cu_seqlens=cu)
        for x, y in zip(clean, dirty):
            assert torch.equal(x[100:170], y[100:170])
        assert prompt_attention(q, k, v, cu_seqlens=cu)[:100].isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", ["right", "left", "holes", "none", "one", "all"])
def test_key_masks(kind, causal, dtype):
    n = 300
    q, k, v, g = _inputs((2, n), 2, 1, 64, dtype, seed=3)
    valid = torch.zeros(2, n, dtype=torch.bool)
    if kind == "right":
        valid[0, :131] = True
        valid[1, :7] = True
    elif kind == "left":
        valid[0, 140:] = True
        valid[1, 299:] = True
    elif kind == "holes":
        valid = torch.rand(2, n, generator=torch.Generator().manual_seed(1)) < 0.4
        valid[1, 128:256] = False
    elif kind == "one":
        valid[0, 130] = True
        valid[1, 0] = True
    elif kind == "all":
        valid[:] = True
    hidden = ~valid.cuda()
    k[hidden] = float("nan")  # masked places may hold anything
    v[hidden] = float("inf")
    got = _run(q, k, v, g, causal=causal, key_mask=valid.cuda())
    for b in range(2):
        see = _see(n, causal, valid[b])
        _check_sequence([x[b] for x in got], q[b], k[b], v[b], g[b], see, 0.125, dtype, f"{b}: ")
        assert (got[2][b][hidden[b]] == 0).all() and (got[3][b][hidden[b]] == 0).all()
        blind = ~see.any(1)
        assert (got[0][b][blind] == 0).all() and (got[1][b][blind] == 0).all()


@pytest.mark.parametrize("mask_dtype", [torch.bool, torch.uint8, torch.int32, torch.int64, torch.float32, torch.bfloat16])
def test_mask_types_and_strides(mask_dtype):
    q, k, v, g = _inputs((2, 70), 2, 2, 32, torch.bfloat16)
    valid = torch.rand(70, 2, generator=torch.Generator().manual_seed(2)) < 0.5
    a = _run(q, k, v, g, key_mask=valid.t().contiguous().cuda())
    b = _run(q, k, v, g, key_mask=valid.to(mask_dtype).cuda().t())
    for x, y in zip(a, b):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", ["projection", "head_major", "odd_offset", "wide_rows", "last_strided"])
def test_strides(form, dtype):
    """Views as models make them give what contiguous copies give, bit for bit."""
    gen = torch.Generator().manual_seed(4)
    B, L, H, d = 2, 150, 4, 64
    if form == "projection":
        x = _rand(gen, B, L, 3, H, d, dtype=dtype)
        q, k, v = x.unbind(2)
    elif form == "head_major":
        q, k, v = (_rand(gen, B, H, L, d, dtype=dtype).transpose(1, 2) for _ in range(3))
    elif form == "odd_offset":  # rows that TMA cannot address
        q, k, v = (_rand(gen, B, L, H, d + 3, dtype=dtype)[..., 1 : d + 1] for _ in range(3))
    elif form == "wide_rows":
        q, k, v = (_rand(gen, B, L, H, 2 * d, dtype=dtype)[..., d:] for _ in range(3))
    else:
        q, k, v = (_rand(gen, B, L, H, d, 2, dtype=dtype)[..., 0] for _ in range(3))
    g = _rand(gen, B, H, L, d, dtype=dtype).transpose(1, 2)
    got = _run(q, k, v, g, causal=True)
    for b in range(B):
        _check_sequence([x[b] for x in got], q[b], k[b], v[b], g[b], _see(L, True), d**-0.5, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_broadcast_keys(dtype):
    """Keys and values expanded over the batch (stride 0)."""
    q, k, v, g = _inputs((3, 80), 2, 2, 64, dtype)
    k1, v1 = k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1)
    got = _run(q, k1, v1, g)
    for b in range(3):
        _check_sequence([x[b] for x in got], q[b], k[0], v[0], g[b], _see(80, False), 0.125, dtype)
    # through autograd the gradient of the one row is the sum
    from cta_b200.attention import prompt_attention

    leaf = k[:1].detach().requires_grad_(True)
    prompt_attention(q, leaf.expand(3, -1, -1, -1), v1).backward(g)
    assert torch.allclose(leaf.grad[0].float(), got[2].float().sum(0), rtol=0.02, atol=0.02)


def test_offsets_past_31_bits():
    """Element offsets above 2^31 within one tensor."""
    n, d = 200, 64
    stride = (1 << 24) + 64  # 200 rows of it pass 2^31 elements
    for dtype in (torch.bfloat16, torch.float32):
        base = torch.zeros(n * stride, dtype=dtype, device="cuda")
        q, k, v, g = _inputs((1, n), 1, 1, d, dtype)
        wide = base.as_strided((1, n, 1, d), (0, stride, d, 1))
        wide.copy_(k)
        got = _run(q, wide, v, g, causal=True)
        want = _run(q, k, v, g, causal=True)
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        del base, wide


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(dtype):
    """Scores far outside the exponential's range: the maximum is taken off first."""
    q, k, v, g = _inputs((1, 200), 2, 2, 64, dtype)
    for scale in (0.0, 3.0, -2.0):
        got = _run(q, k, v, g, scale=scale)
        _check_sequence([x[0] for x in got], q[0], k[0], v[0], g[0], _see(200, False), scale, dtype, f"scale {scale}: ")


def test_lse():
    from cta_b200 import ops

    for dtype in DTYPES:
        q, k, v, _ = _inputs((2, 150), 4, 2, 64, dtype)
        valid = torch.ones(2, 150, dtype=torch.bool)
        valid[1, :5] = False
        out, lse = ops.attention_forward(q, k, v, causal=True, mask_words=ops.attention_mask(valid.cuda()))
        for b in range(2):
            _, want = A.attention(q[b], k[b], v[b], _see(150, True, valid[b]), 0.125)
            assert torch.equal(torch.isinf(lse[b]), torch.isinf(want))
            fin = torch.isfinite(want)
            # scores: (d + 4) u |q|.|k| / 8 with |q|.|k| below 64 * 3 * 3; sum and logarithm: 2^-20
            assert ((lse[b].double() - want)[fin].abs() <= 68 * 2.0**-24 * 72 + 2.0**-20 * (1 + want[fin].abs())).all()


def test_only_wanted_gradients():
    from cta_b200.attention import prompt_attention

    q, k, v, g = _inputs((1, 130), 2, 2, 64, torch.bfloat16)
    full = _run(q, k, v, g, causal=True)
    for want in ((0,), (1,), (2,), (0, 2)):
        t = [x.detach().requires_grad_(i in want) for i, x in enumerate((q, k, v))]
        got = torch.autograd.grad(prompt_attention(*t, causal=True), [t[i] for i in want], g)
        for i, x in zip(want, got):
            assert torch.equal(x, full[1 + i])


def test_gradient_against_differences():
    """fp32: the directional derivative against a central difference of the 64-bit definition."""
    q, k, v, g = _inputs((1, 90), 2, 1, 32, torch.float32)
    got = _run(q, k, v, g, causal=True)
    see = _see(90, True)
    gen = torch.Generator().manual_seed(8)
    for i, name in enumerate("qkv"):
        t = [q[0].double(), k[0].double(), v[0].double()]
        step = torch.randn(t[i].shape, generator=gen, dtype=torch.float64).cuda()
        f = []
        for e in (1e-5, -1e-5):
            u = list(t)
            u[i] = t[i] + e * step
            f.append((A.attention(*u, see, 32**-0.5)[0] * g[0].double()).sum())
        slope = (f[0] - f[1]) / 2e-5
        mine = (got[1 + i][0].double() * step).sum()
        # the difference is off by O(e^2) and 2^-53 / e; the gradient's bound is summed up
        tol = (A.bounds(q[0], k[0], v[0], see, 32**-0.5, torch.float32, g[0])[1 + i] * step.abs()).sum() + 1e-6
        assert (mine - slope).abs() <= tol, name


def test_twice_the_same():
    for dtype in DTYPES:
        q, k, v, g = _inputs((2, 400), 4, 2, 64, dtype)
        a, b = _run(q, k, v, g, causal=True), _run(q, k, v, g, causal=True)
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_empty():
    from cta_b200.attention import prompt_attention

    for shape in ((0, 5), (2, 0)):
        q, k, v, g = _inputs(shape, 2, 2, 64, torch.bfloat16)
        got = _run(q, k, v, g)
        assert got[0].shape == (*shape, 2, 64)
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    q, k, v, _ = _inputs((0,), 2, 2, 64, torch.bfloat16)
    assert prompt_attention(q, k, v, cu_seqlens=cu).shape == (0, 2, 64)
    # rows, but all sequences empty
    q, k, v, _ = _inputs((3,), 2, 2, 64, torch.bfloat16)
    assert (prompt_attention(q, k, v, cu_seqlens=cu) == 0).all()
    assert (prompt_attention(q, k, v, cu_seqlens=cu[:1]) == 0).all()


def test_out_buffer_keeps_tail():
    from cta_b200 import ops

    for dtype in DTYPES:
        q, k, v, _ = _inputs((140,), 2, 2, 64, dtype)
        cu = torch.tensor([0, 60, 133], dtype=torch.int32, device="cuda")
        out = torch.full_like(q, 7.0)
        y, _ = ops.attention_forward(q, k, v, cu_seqlens=cu, out=out)
        assert y is out and (out[133:] == 7).all()
        z, _ = ops.attention_forward(q, k, v, cu_seqlens=cu)
        assert torch.equal(out[:133], z[:133]) and (z[133:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_and_replayed(dtype):
    """Forward and backward in one CUDA graph, replayed on new inputs."""
    from cta_b200.attention import prompt_attention

    q, k, v, g = _inputs((2, 200), 4, 2, 64, dtype)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            torch.autograd.grad(prompt_attention(*leaves, causal=True), leaves, g)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = prompt_attention(*leaves, causal=True)
        grads = torch.autograd.grad(out, leaves, g)
    q2, k2, v2, g2 = _inputs((2, 200), 4, 2, 64, dtype, seed=77)
    with torch.no_grad():
        for x, y in zip(leaves, (q2, k2, v2)):
            x.copy_(y)
        g.copy_(g2)
    graph.replay()
    want = _run(q2, k2, v2, g2, causal=True)
    for x, y in zip((out, *grads), want):
        assert torch.equal(x, y)


def test_other_stream():
    q, k, v, g = _inputs((1, 300), 4, 4, 64, torch.bfloat16)
    want = _run(q, k, v, g, causal=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _run(q, k, v, g, causal=True)
    torch.cuda.current_stream().wait_stream(s)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
def test_longer(dim, dtype):
    """Many tiles on both sides, grouped heads."""
    q, k, v, g = _inputs((1, 2100), 4, 2, dim, dtype)
    for causal in (True, False):
        got = _run(q, k, v, g, causal=causal)
        _check_sequence([x[0] for x in got], q[0], k[0], v[0], g[0], _see(2100, causal), dim**-0.5, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,dim", [(8, 64), (4, 128), (2, 200), (3, 20)])
def test_output_that_rounds_far(heads, dim, dtype):
    # Two keys of equal score with values a and a + step, a step of the type apart: the output a + step / 2 rounds
    # by half a step, which is all of dP - delta.  dS = -+ step / 4 per unit of the gradient.
    step = 2.0
    a = 2.0 / torch.finfo(dtype).eps
    q = torch.zeros(3, 2, heads, dim, dtype=dtype, device="cuda")
    k = torch.randn(3, 2, heads, dim, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    v = torch.zeros_like(q)
    v[:, 0, :, 0], v[:, 1, :, 0] = a, a + step
    g = torch.zeros_like(q)
    g[..., 0] = 1.0
    dq = _run(q, k, v, g)[1].double()
    want = dim**-0.5 * step / 4 * (k[:, 1:] - k[:, :1].double()).expand(-1, 2, -1, -1)
    # Relative to |dS| = step / 4, as large as a * eps / 8: P and delta, both of a few fp32 roundings (lse, the
    # exponential, the sum over dim: 2^-21 in all), err by 2^-21 a = 2^-18 / eps of it.  dS and dq are rounded
    # once more (eps / 2 each).  The terms of the two keys add up.
    eps = torch.finfo(dtype).eps
    tol = dim**-0.5 * step / 4 * (2.0**-18 / eps + eps / 2) * (k.double().abs().sum(1, keepdim=True)) + eps / 2 * want.abs()
    tol = tol + torch.finfo(dtype).smallest_normal * eps
    _within(dq, want, tol.expand_as(want), "dq")


def test_low_part_refusals():
    from cta_b200 import ops

    q, k, v, _ = (x.cuda() for x in _inputs((2, 5), 2, 2, 32, torch.bfloat16, seed=0))
    for low in (q.float(), q[:, :4], torch.empty(2, 5, 2, 64, dtype=q.dtype, device="cuda")[..., :32], q.cpu()):
        with pytest.raises(ValueError, match="out_low"):
            ops.attention_forward(q, k, v, out_low=low)
    with pytest.raises(ValueError, match="out_low"):
        ops.attention_forward(q.float(), k.float(), v.float(), out_low=q.float())
    low = torch.full_like(q, float("nan"))
    out, lse = ops.attention_forward(q, k, v, out_low=low)
    with pytest.raises(ValueError, match="out_low"):
        ops.attention_backward(q, q, k, v, out, lse, out_low=low[:1])
    # out + low is the output with 16 bits more or less: within the weights' error of the formula's, below one rounding
    see = _see(5, False)
    want, _ = A.attention(q[0], k[0], v[0], see, 32**-0.5)
    tol = A.bounds(q[0], k[0], v[0], see, 32**-0.5, q.dtype) - 2.0**-9 * (1 - 2.0**-7) * want.abs()
    _within(out[0].double() + low[0].double(), want, tol, "out + low")


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 20)])
def test_rows_without_sequences(dtype, dim):
    """Packed rows of no sequence are zero and have no gradient, whatever the memory held before."""
    cu = torch.zeros(1, dtype=torch.int32, device="cuda")
    q, k, v, g = (x.cuda() for x in _inputs((70,), 4, 2, dim, dtype))
    for _ in range(3):
        held = [torch.full_like(x, float("nan")) for x in (q, q, q, k, k, k)]
        del held
        for x in _run(q, k, v, g, cu_seqlens=cu):
            assert (x == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_two_streams_at_once(dtype):
    """Calls that run side by side give what they give alone, bit for bit: the gradients' kernels of one call also run
    beside each other, and those of the next call of a stream start only when both are done."""
    from cta_b200 import ops

    sets = [[x.cuda() for x in _inputs((2, n), 8, 2, 64, dtype, seed=n)] for n in (700, 333)]

    def call(q, k, v, g):
        o, lse = ops.attention_forward(q, k, v, causal=True)
        return (o, lse, *ops.attention_backward(g, q, k, v, o, lse, causal=True))

    alone = [call(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(6):
        for i, (s, stream) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(stream):
                x = call(*s)
                got[i].append(tuple(y.clone() for y in x))  # reads the gradients right behind their kernels
    torch.cuda.synchronize()
    for want, all_of in zip(alone, got):
        for x in all_of:
            for a, b in zip(want, x):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_forward_mode_raises(dtype):
    """A tangent is refused, as by the framework's other operators, and not dropped."""
    import torch.autograd.forward_ad as fw

    from cta_b200.attention import prompt_attention

    q, k, v, g = _inputs((1, 40), 2, 2, 64, dtype)
    for i in range(3):
        for grad in (True, False):
            with fw.dual_level(), torch.set_grad_enabled(grad):
                t = [q, k, v]
                t[i] = fw.make_dual(t[i], g)
                with pytest.raises(RuntimeError, match="forward mode AD"):
                    prompt_attention(*t)
    with fw.dual_level():  # inside a level, without a tangent
        assert torch.equal(prompt_attention(q, k, v), prompt_attention(q, k, v))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 2, 1), (128, 4, 4), (72, 8, 1), (20, 2, 2), (160, 2, 1)])
def test_rows_that_see_nothing_take_no_part(dim, heads, kv_heads, dtype):
    """Left padding, causal: q and the output's gradient of rows that see no key may hold anything, NaN included,
    and reach no gradient."""
    n = 300
    q, k, v, g = _inputs((3, n), heads, kv_heads, dim, dtype, seed=dim)
    valid = torch.ones(3, n, dtype=torch.bool)
    valid[0, :140] = False
    valid[1, :5] = False
    valid[1, 9] = False
    valid[2] = False
    hidden = ~valid.cuda()
    blind = hidden.cumprod(1).bool()
    k[hidden], v[hidden] = float("nan"), float("inf")
    q[blind], g[blind] = float("nan"), float("inf")
    got = _run(q, k, v, g, causal=True, key_mask=valid.cuda())
    clean_q, clean_g = q.masked_fill(blind[..., None, None], 0), g.masked_fill(blind[..., None, None], 0)
    for b in range(3):
        _check_sequence([x[b] for x in got], clean_q[b], k[b], v[b], clean_g[b], _see(n, True, valid[b]), dim**-0.5, dtype,
                        f"{b}: ")
        assert (got[0][b][blind[b]] == 0).all() and (got[1][b][blind[b]] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_equal_weights_of_little_size(dim, dtype):
    """41891 keys of equal weight: 1 / 41891 is 400.497 steps of fp16's smallest, 1.2e-3 off when rounded to one.  dV
    is then the same everywhere, the sum of g over 41891."""
    n, m = 41891, 64
    q = torch.zeros(1, n, 1, dim, dtype=dtype, device="cuda")
    k, v = (torch.randn(1, n, 1, dim, generator=torch.Generator().manual_seed(i)).to(dtype).cuda() for i in (1, 2))
    g = torch.zeros_like(q)
    g[0, 1000 : 1000 + m] = (torch.rand(m, 1, dim, generator=torch.Generator().manual_seed(3)) * 64 + 32).to(dtype).cuda()
    dv = _run(q, k, v, g)[3].double()
    want = (g.double().sum(1, keepdim=True) / n).expand_as(dv)
    # P and dv are rounded once each; m terms are summed in fp32; lse = 10.6 and the sum of n weights, each 1 exactly,
    # (its logarithm 15.4) are rounded a few times, by 3e-6 in all; the exponential is off by 2^-21
    eps = torch.finfo(dtype).eps
    tol = want * (eps + (m + 8) * 2.0**-24 + 2.0**-18) + torch.finfo(dtype).smallest_normal * eps
    _within(dv, want, tol, "dv")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
def test_small_weights_beside_a_large_one(dim, dtype):
    """One key of weight 1 and value 0, 4000 of weight exp(-11.4453125) = 179.507 steps of fp16's smallest."""
    from cta_b200.attention import prompt_attention

    n, dot = 4001, -11.4453125
    q = torch.zeros(1, n, 2, dim, dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    k = torch.zeros_like(q)
    k[:, 1:, :, 0] = dot
    v = torch.ones_like(q)
    v[:, 0] = 0.0
    out = prompt_attention(q, k, v, scale=1.0).double()
    w = torch.exp(torch.tensor(k[0, 1, 0, 0].item(), dtype=torch.float64)).item()
    want = torch.full_like(out, 4000 * w / (1 + 4000 * w))
    # weights and output are rounded once each; the exponential 2^-21, the scores 2^-24 * 11.4 * 4, the sums below
    # (n / 64 + 80) 2^-24 of themselves: every 64 weights are added by themselves first
    eps = torch.finfo(dtype).eps
    _within(out, want, want * (eps + 2.0**-20 + 50 * 2.0**-24 + (n / 64 + 80) * 2.0**-24), "out")



@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", [1.0, 2.0**-13, 2.0**-17, 2.0**8])
def test_fp16_gradients_of_any_size(size, causal, dim):
    """P (dP - delta) over thousands of keys lies far below fp16's smallest step when the output's gradient is small;
    the sums over it do not.  Only what the gradients' own type cannot hold may be lost: the bounds here allow
    no step of fp16 per key, but 2^-39 of the largest weight for P and of 2 |g| |v| for dS."""
    n = 4200
    q, k, v, g = _inputs((1, n), 2, 1, dim, torch.float16, seed=dim)
    q, g = (q * 0.5).half(), (g * size).half()
    got = _run(q, k, v, g, causal=causal)
    see = _see(n, causal)
    q, k, v, g = (x[0] for x in (q, k, v, g))
    most = 2 * g.double().norm(dim=-1).max() * v.double().norm(dim=-1).max()
    tol = A.bounds(q, k, v, see, dim**-0.5, torch.float16, g, weight_step=2.0**-31, grad_steps=(2.0**-39, 2.0**-39 * most))
    for x, y, t, name in zip(got[1:], A.gradients(q, k, v, g, see, dim**-0.5), tol[1:], ("dq", "dk", "dv")):
        _within(x[0], y, t, name)


@pytest.mark.parametrize("dim", [64, 128])
def test_fp16_gradients_of_other_sequences_and_rows(dim):
    """Sizes that differ by 2^20 between sequences, padded and packed, and between the heads of a batch: each keeps its
    own precision.  Values of masked keys and of rows behind the last sequence count for nothing."""
    n = 700
    sizes = [2.0**-14, 1.0, 2.0**6]
    q, k, v, g = _inputs((3, n), 4, 2, dim, torch.float16, seed=dim)
    g = (g * torch.tensor(sizes, device="cuda")[:, None, None, None]).half()
    v[1, :, 1] *= 2.0**8
    valid = torch.ones(3, n, dtype=torch.bool, device="cuda")
    valid[:, 600:] = False
    v[:, 600:], k[:, 600:] = 60000.0, float("nan")

    def check(got, what, part):
        for b in range(3):
            m = 600 if part else n
            x = [t[b][:m] for t in (q, k, v, g)]
            see = _see(m, True)
            most = 2 * x[3].double().norm(dim=-1).max() * x[2].double().norm(dim=-1).amax(0)
            per_head = most.repeat_interleave(2)[:, None, None]
            tol = A.bounds(*x[:3], see, dim**-0.5, torch.float16, x[3], weight_step=2.0**-31,
                           grad_steps=(2.0**-39, 2.0**-39 * per_head))
            for y, w, t, name in zip(got[1:], A.gradients(*x, see, dim**-0.5), tol[1:], ("dq", "dk", "dv")):
                _within(y[b][:m], w, t, f"{what}, {b}: {name}")

    g[:, 600:] = 0
    check(_run(q, k, v, g, causal=True, key_mask=valid), "padded", True)
    packed = [torch.cat([x[:, :600].flatten(0, 1), torch.full_like(x[0, :9], 60000.0)]) for x in (q, k, v, g)]
    cu = torch.tensor([0, 600, 1200, 1800], dtype=torch.int32, device="cuda")
    got = _run(*packed, causal=True, cu_seqlens=cu)
    check([x[:1800].unflatten(0, (3, 600)) for x in got], "packed", True)
    assert all((x[1800:] == 0).all() for x in got)


def test_fp16_backward_with_one_plane_of_scratch():
    """Through the C interface with room for delta alone: the plain kernels, within the same bounds."""
    from cta_b200 import _lib, ops

    n, d = 300, 64
    q, k, v, g = _inputs((1, n), 4, 2, d, torch.float16)
    out, lse = ops.attention_forward(q, k, v, causal=True)
    grads = [torch.empty_like(x) for x in (q, k, v)]
    delta = torch.full((2, *lse.shape), 7.0, device="cuda")

    def strides(t):
        return t.stride()[:3]

    for planes in (0, 1, 2):
        args = _lib.ATTENTION_ARGS.pack(
            *(t.data_ptr() for t in (q, k, v, out)), 0, lse.data_ptr(), g.data_ptr(), delta.data_ptr(),
            *(t.data_ptr() for t in grads), 0, 0, *strides(q), *strides(k), *strides(v), *strides(out), *strides(g),
            *(x for t in grads for x in strides(t)), 1, n, 4, 2, d, 2, 1, 0, planes, d**-0.5, 0.0)
        _lib.enqueue(_lib.load().cta_attention_backward, q, args)
        assert (delta[1] == 7).all()
        see = _see(n, True)
        tol = A.bounds(q[0], k[0], v[0], see, d**-0.5, q.dtype, g[0])
        for x, y, t, name in zip(grads, A.gradients(q[0], k[0], v[0], g[0], see, d**-0.5), tol[1:], ("dq", "dk", "dv")):
            _within(x[0], y, t, name)
    bad = bytearray(args)
    bad[-12:-8] = (-1).to_bytes(4, "little", signed=True)
    assert _lib.load().cta_attention_backward(bytes(bad), None) == _lib.CTA_EINVAL


@pytest.mark.parametrize("dim", [64, 128])
def test_fp16_captured_and_on_two_streams(dim):
    """fp16's backward, whose scratch holds the norms too: captured and replayed on new inputs, and beside another call
    of other sizes, bit for bit."""
    from cta_b200.attention import prompt_attention

    first, second = _inputs((2, 300), 4, 2, dim, torch.float16), _inputs((2, 300), 4, 2, dim, torch.float16, seed=5)
    second[3].mul_(2.0**-12)
    want = [_run(*x, causal=True) for x in (first, second)]
    held = [x.clone() for x in first]
    leaves = [x.requires_grad_(True) for x in held[:3]]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(prompt_attention(*leaves, causal=True), leaves, held[3])
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = prompt_attention(*leaves, causal=True)
        grads = torch.autograd.grad(out, leaves, held[3])
    for inputs, expected in zip((second, first), reversed(want)):
        with torch.no_grad():
            for x, y in zip((*leaves, held[3]), inputs):
                x.copy_(y)
        graph.replay()
        for x, y in zip((out, *grads), expected):
            assert torch.equal(x, y)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i, (inputs, st) in enumerate(zip((first, second), streams)):
            with torch.cuda.stream(st):
                got[i].append(_run(*inputs, causal=True))
    torch.cuda.synchronize()
    for expected, all_of in zip(want, got):
        for x in all_of:
            for a, b in zip(x, expected):
                assert torch.equal(a, b)
