"""Queries and keys rotated by their positions on the way into the paged cache, against the formula in 64 bits."""
from __future__ import annotations

import pytest
import torch

from oracle import attention_oracle as A
from test_gpu_paged import _cache, _codes

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def no_device_error():
    from cta_b200 import _lib

    yield
    assert _lib.device_error() == 0


def _turned(x, table, positions, interleaved):
    """(value, size) in 64 bits: the rotated rows, and |a cos| + |b sin| of each element."""
    x, t = x.double(), table.double()[positions][:, None]
    pairs = table.shape[1] // 2
    a, b = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    y, size = x.clone(), x.abs()
    c, s = t[..., :pairs], t[..., pairs:]
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    size[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, size


def _tol(want, size, dtype):
    # two products and their sum in fp32 (one of the products exact in the fused operation), then one rounding
    r = torch.finfo(dtype).eps / 2
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return (1 + r) * 2.0**-23 * size + r * want.abs() + least


class Setup:
    def __init__(self, tokens, heads, kv_heads, dim, rotary, dtype, quantized, page=16, positions=5000, table_dtype=None, seed=0,
                 head_major=False):
        from cta_b200 import ops

        gen = torch.Generator().manual_seed(seed)
        pages = -(-tokens // page) + 2
        self.q = torch.randn(tokens, heads, dim, generator=gen).to(dtype).cuda()
        self.k, self.v = ((torch.randn(tokens, kv_heads, dim, generator=gen)
                           * torch.exp(torch.randn(tokens, kv_heads, 1, generator=gen))).to(dtype).cuda() for _ in range(2))
        self.kc, self.vc, self.ks, self.vs = _cache(pages, page, kv_heads, dim, dtype, quantized, head_major=head_major)
        self.slots = torch.randperm(pages * page, generator=gen)[:tokens].cuda()
        self.positions = torch.randint(0, positions, (tokens,), generator=gen).cuda()
        self.table = ops.rotary_table(positions, rotary, dtype=table_dtype or torch.float32)
        self.dtype, self.quantized, self.page = dtype, quantized, page

    def run(self, **kw):
        from cta_b200 import ops

        return ops.rotary_cache_write(self.q, self.k, self.v, self.kc, self.vc, self.slots, self.positions, self.table,
                                      k_scale=self.ks, v_scale=self.vs, **kw)

    def check(self, out, q=None, live=None, interleaved=False):
        live = torch.ones_like(self.slots, dtype=torch.bool) if live is None else live
        want, size = _turned(self.q if q is None else q, self.table, self.positions, interleaved)
        assert ((out.double() - want).abs() <= _tol(want, size, self.dtype)).all()
        slots = self.slots[live]
        at = (slots // self.page, slots % self.page)
        k, size = (x[live] for x in _turned(self.k, self.table, self.positions, interleaved))
        v = self.v[live]
        if not self.quantized:
            assert ((self.kc[at].double() - k).abs() <= _tol(k, size, self.dtype)).all()
            assert torch.equal(self.vc[at], v)
            return
        # the scale: the largest element's own error and one rounding; the code: half a step of the quotient, whose
        # error is that of the element, of the scale and of four operations in fp32
        ks, vs = (x[slots // self.page, :, slots % self.page].double() for x in (self.ks, self.vs))
        most = k.abs().amax(-1).clamp_min(2.0**-100)
        off = 2.0**-23 * size.amax(-1)
        assert ((ks - most / 448).abs() <= off / 448 + 2.0**-23 * most / 448).all()
        y = k * 448 / most[..., None]
        e = torch.frexp(y.abs().clamp_min(2.0**-6)).exponent - 1
        step = torch.ldexp(torch.ones_like(y), e - 3)
        moved = 448 / most[..., None] * (2.0**-23 * size + k.abs() / most[..., None] * off[..., None]) + 2.0**-21 * y.abs()
        got = _codes(self.kc, slots)
        # past a power of two the step doubles: what has moved there may round by a step of the next binade
        assert ((got - y).abs() <= step / 2 * (1 + 2.0**-10) + moved + (y.abs() + moved >= 16 * step) * step / 2).all()
        codes, scale = A.quantise(v)
        assert torch.equal(_codes(self.vc, slots), codes)
        assert torch.equal(vs.float(), scale.float())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(16, 16), (32, 16), (64, 64), (64, 32), (80, 80), (96, 48), (128, 128), (128, 64), (144, 144),
                                        (256, 256), (256, 96)])
def test_dims(dim, rotary, interleaved, quantized, dtype):
    s = Setup(77, 6, 2, dim, rotary, dtype, quantized, seed=dim + rotary)
    s.check(s.run(interleaved=interleaved), interleaved=interleaved)


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (1, 32, 8), (3, 5, 5), (64, 32, 8), (1000, 9, 3), (257, 4, 1)])
@pytest.mark.parametrize("table", [torch.float32, torch.bfloat16])
def test_sizes(tokens, heads, kv_heads, table, quantized):
    s = Setup(tokens, heads, kv_heads, 128, 128, torch.bfloat16, quantized, table_dtype=table, seed=tokens)
    s.check(s.run())


def test_far_positions_and_table():
    """Angles of positions up to 2^17 come from 64 bits."""
    s = Setup(64, 4, 2, 64, 64, torch.float16, False, positions=1 << 17, seed=3)
    s.positions[:3] = torch.tensor([0, (1 << 17) - 1, 99999])
    out = s.run()
    s.check(out)
    turn = 10000.0 ** (-torch.arange(32, dtype=torch.float64, device="cuda") / 32)
    angle = s.positions.double()[:, None] * turn
    assert ((s.table[s.positions].double() - torch.cat([angle.cos(), angle.sin()], 1)).abs() <= 2.0**-24).all()


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_and_strides(interleaved, quantized):
    s = Setup(50, 8, 2, 64, 48, torch.bfloat16, quantized, seed=4, head_major=True)
    both = torch.cat([s.q.flatten(1), s.k.flatten(1), s.v.flatten(1)], 1)  # one projection's output
    q = both[:, : 8 * 64].view(50, 8, 64)
    s.k, s.v = both[:, 512:640].view(50, 2, 64), both[:, 640:].view(50, 2, 64)
    before, s.q = q.clone(), q
    out = s.run(out=q, interleaved=interleaved)
    assert out.data_ptr() == q.data_ptr()
    s.check(out, q=before, interleaved=interleaved)
    # rows off 16 bytes are copied
    odd = torch.empty(50 * 8 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(50, 8, 64)
    odd.copy_(before)
    s.q = odd
    assert torch.equal(s.run(interleaved=interleaved), out)


@pytest.mark.parametrize("quantized", [False, True])
def test_padding_bad_slots_and_positions(quantized):
    from cta_b200 import _lib

    s = Setup(40, 4, 2, 64, 64, torch.bfloat16, quantized, seed=5)
    live = torch.ones(40, dtype=torch.bool, device="cuda")
    kept = [x.clone() for x in (s.kc.view(torch.uint8), s.vc.view(torch.uint8))]
    s.slots[7], s.slots[39] = -1, -5
    s.q[39], s.k[39], s.v[39] = float("nan"), float("inf"), float("nan")
    s.positions[39] = -3  # padding may hold anything
    live[7], live[39] = False, False
    out = s.run()
    assert _lib.device_error() == 0
    assert (out[39] == 0).all()
    s.q[39], s.positions[39] = 0.0, 0
    s.check(torch.where(live[:, None, None] | (s.slots == -1)[:, None, None], out, torch.zeros_like(out)), live=live)
    untouched = torch.ones(s.kc.shape[0] * s.page, dtype=torch.bool, device="cuda")
    untouched[s.slots[live]] = False
    for x, y in zip((s.kc, s.vc), kept):
        assert torch.equal(x.view(torch.uint8).flatten(0, 1)[untouched], y.flatten(0, 1)[untouched])
    # past the cache, and positions outside the table
    s.slots[7] = s.kc.shape[0] * s.page
    assert torch.equal(s.run()[7], out[7])
    torch.cuda.synchronize()
    assert _lib.device_error() == 2
    s.slots[7] = -1
    for bad in (-1, 5000, 2**40):
        s.positions[3] = bad
        at = (s.slots[3] // s.page, s.slots[3] % s.page)
        before = [x.view(torch.uint8)[at].clone() for x in (s.kc, s.vc)]
        s.k[3] += 1
        s.v[3] += 1
        got = s.run()
        torch.cuda.synchronize()
        assert _lib.device_error() == 2
        assert (got[3] == 0).all() and torch.equal(got[4:39], out[4:39])
        for x, y in zip((s.kc, s.vc), before):
            assert torch.equal(x.view(torch.uint8)[at], y)


def test_plain_rows_are_those_of_the_plain_write():
    """Angles of zero: the caches hold what kv_cache_write leaves, code by code."""
    from cta_b200 import ops

    for quantized in (False, True):
        for dtype in DTYPES:
            s = Setup(300, 4, 2, 128, 64, dtype, quantized, seed=6)
            s.table[:, :32], s.table[:, 32:] = 1.0, 0.0
            assert torch.equal(s.run(), s.q)
            held = [x.view(torch.uint8) for x in (s.kc, s.vc, s.ks, s.vs) if x is not None]  # bits: the rest is NaN
            got = [x.clone() for x in held]
            ops.kv_cache_write(s.k, s.v, s.kc, s.vc, s.slots, k_scale=s.ks, v_scale=s.vs)
            for x, y in zip(got, held):
                assert torch.equal(x, y)


def test_empty_and_captured():
    s = Setup(30, 4, 2, 64, 64, torch.bfloat16, True, seed=7)
    empty = Setup(30, 4, 2, 64, 64, torch.bfloat16, True, seed=7)
    for n in ("q", "k", "v", "slots", "positions"):
        setattr(empty, n, getattr(empty, n)[:0])
    assert empty.run().shape == (0, 4, 64)
    want = s.run().clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = s.run()
    stream = torch.cuda.Stream()
    for _ in range(2):
        out.zero_()
        s.kc.view(torch.uint8).zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        s.check(out)


def test_large_cache():
    """Offsets in the cache past 2^31 elements."""
    from cta_b200 import ops

    pages = 1100
    kc = torch.zeros(pages, 128, 64, 256, dtype=torch.bfloat16, device="cuda")  # 4.6 GB
    vc = torch.zeros_like(kc)
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, 64, 256, generator=gen).to(torch.bfloat16).cuda() for _ in range(3))
    slots = torch.tensor([pages * 128 - 1, 0]).cuda()
    positions = torch.tensor([3, 9]).cuda()
    table = ops.rotary_table(16, 256)
    ops.rotary_cache_write(q, k, v, kc, vc, slots, positions, table)
    want, size = _turned(k, table, positions, False)
    got = torch.stack([kc[-1, -1], kc[0, 0]])
    assert ((got.double() - want).abs() <= _tol(want, size, torch.bfloat16)).all()
    assert torch.equal(torch.stack([vc[-1, -1], vc[0, 0]]), v)
