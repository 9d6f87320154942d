"""The paged key/value cache and the attention that reads it, against their definitions in
64 bits (oracle/attention_oracle.py)."""
from __future__ import annotations

import pytest
import torch

from oracle import attention_oracle as A

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
E4M3 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def no_device_error():
    from cta_b200 import _lib

    _lib.device_error()
    yield
    assert _lib.device_error() == 0


def _cache(pages, page, heads, dim, dtype, quantized, fill=None, head_major=False):
    """(k_cache, v_cache, k_scale, v_scale), filled with NaN as memory never written may be."""
    def one():
        shape = (pages, heads, page, dim) if head_major else (pages, page, heads, dim)
        if quantized:
            t = torch.full(shape, 0x7F, dtype=torch.uint8, device="cuda").view(E4M3)
        else:
            t = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
        return t.transpose(1, 2) if head_major else t

    scales = [torch.full((pages, heads, page), float("nan"), device="cuda") if quantized else None for _ in range(2)]
    return one(), one(), *scales


def _rows(n, heads, dim, dtype, seed, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    size = torch.exp(spread * torch.randn(n, heads, 1, generator=gen))
    return (torch.randn(n, heads, dim, generator=gen) * size).to(dtype).cuda()


def _codes(cache, slots):
    """The cache's entries at slots, as 64-bit values."""
    page = cache.shape[1]
    if cache.dtype == E4M3:
        return cache.view(torch.uint8)[slots // page, slots % page].view(E4M3).double()
    return cache[slots // page, slots % page].double()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("head_major", [False, True])
@pytest.mark.parametrize("dim", [16, 64, 80, 128, 144, 256])
@pytest.mark.parametrize("tokens", [1, 3, 64, 1000])
def test_write_and_read(tokens, dim, head_major, dtype):
    from cta_b200 import ops

    heads, page, pages = 3, 16, 70
    k, v = _rows(tokens, heads, dim, dtype, 1, 2.0), _rows(tokens, heads, dim, dtype, 2, 2.0)
    if tokens >= 64:
        k[5] = 0  # a row of zeros
        v[6] *= 2.0**-10
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(3))[:tokens].cuda()
    others = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    others[slots] = False
    others = others.nonzero()[:, 0]
    for quantized in (False, True):
        kc, vc, ks, vs = _cache(pages, page, heads, dim, dtype, quantized, head_major=head_major)
        ops.kv_cache_write(k, v, kc, vc, slots, k_scale=ks, v_scale=vs)
        back = ops.kv_cache_read(kc, vc, slots, k_scale=ks, v_scale=vs, dtype=dtype)
        for x, c, s, y in ((k, kc, ks, back[0]), (v, vc, vs, back[1])):
            assert y.dtype == dtype and y.shape == x.shape
            assert _codes(c, others).isnan().all()  # nothing else was written
            if not quantized:
                assert torch.equal(_codes(c, slots), x.double()) and torch.equal(y, x)
                continue
            codes, scale = A.quantise(x)
            got = s[slots // page, :, slots % page].double()
            assert ((got - scale).abs() <= 2.0**-24 * scale).all()
            mine = _codes(c, slots)
            # x * (448 / m) carries two roundings of 2^-24: a value that close to the middle
            # between two codes may go to the other
            m = x.double().abs().amax(-1, keepdim=True).clamp_min(2.0**-100)
            y64 = x.double() * (448.0 / m)
            assert ((mine - y64).abs() <= (codes - y64).abs() + 2.0**-22 * y64.abs()).all()
            want = mine * got[..., None]
            assert ((y.double() - want).abs() <= want.abs() * (torch.finfo(dtype).eps / 2 + 2.0**-23)
                    + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all()


def test_extreme_rows():
    """Zeros, the smallest and the largest values, infinities and NaN."""
    from cta_b200 import ops

    k = torch.zeros(6, 1, 16, dtype=torch.bfloat16, device="cuda")
    k[1] = torch.finfo(torch.bfloat16).tiny
    k[2] = torch.finfo(torch.bfloat16).max
    k[2, 0, 0] *= -1
    k[3] = float("inf")
    k[4, 0, 3] = float("nan")
    k[5] = 2.0**-100
    slots = torch.arange(6, device="cuda")
    kc, vc, ks, vs = _cache(1, 16, 1, 16, torch.bfloat16, True)
    ops.kv_cache_write(k, k, kc, vc, slots, k_scale=ks, v_scale=vs)
    y = ops.kv_cache_read(kc, vc, slots, k_scale=ks, v_scale=vs)[0]
    assert (y[0] == 0).all()
    assert (y[1].abs() <= 2.0**-100).all()  # below the floor: rounded in steps of the floor's scale
    assert ((y[2].double() - k[2].double()).abs() <= 2.0**-8 * k[2].double().abs()).all()
    assert y[3].isnan().all()
    assert y[4, 0, 3].isnan()
    assert ((y[5].double() - 2.0**-100).abs() <= 2.0**-107).all()


@pytest.mark.parametrize("quantized", [False, True])
def test_padding_and_bad_slots(quantized):
    from cta_b200 import _lib, ops

    k = _rows(5, 2, 32, torch.bfloat16, 1)
    kc, vc, ks, vs = _cache(2, 16, 2, 32, torch.bfloat16, quantized)
    slots = torch.tensor([3, -1, 31, -7, 0], device="cuda")
    ops.kv_cache_write(k, k, kc, vc, slots, k_scale=ks, v_scale=vs)
    assert _lib.device_error() == 0
    assert int(kc.float().isnan().sum()) == (32 - 3) * 2 * 32
    y, _ = ops.kv_cache_read(kc, vc, slots, k_scale=ks, v_scale=vs)
    assert (y[1] == 0).all() and (y[3] == 0).all() and (y[0] != 0).any()
    before = [c.clone().view(torch.uint8) for c in (kc, vc)]
    slots[1] = 32  # past the cache: skipped and reported
    ops.kv_cache_write(k[1:2], k[1:2], kc, vc, slots[1:2], k_scale=ks, v_scale=vs)
    assert _lib.device_error() == 2 and _lib.device_error() == 0
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(before, (kc, vc)))
    y, _ = ops.kv_cache_read(kc, vc, slots, k_scale=ks, v_scale=vs)
    assert _lib.device_error() == 2
    assert (y[1] == 0).all()
    # int32 slots
    a = ops.kv_cache_read(kc, vc, torch.tensor([3], dtype=torch.int32, device="cuda"), k_scale=ks, v_scale=vs)[0]
    assert torch.equal(a[0], y[0])


def test_strided_rows():
    """Rows as views of a fused projection, 16-byte aligned or not."""
    from cta_b200 import ops

    for off in (0, 3):
        x = torch.randn(20, 3 * 2 * 64 + 8, device="cuda").to(torch.bfloat16)
        k = x[:, off : off + 128].view(20, 2, 64)
        v = x[:, off + 128 : off + 256].view(20, 2, 64)
        kc, vc, _, _ = _cache(2, 16, 2, 64, torch.bfloat16, False)
        slots = torch.arange(20, device="cuda")
        ops.kv_cache_write(k, v, kc, vc, slots)
        y = ops.kv_cache_read(kc, vc, slots)
        assert torch.equal(y[0], k) and torch.equal(y[1], v)


# ---------------------------------------------------------------------------
# attention over the cache
# ---------------------------------------------------------------------------
class Setup:
    """Sequences of `lens` keys, the newest `rows` of them queried, in shuffled pages."""

    def __init__(self, lens, rows, heads, kv_heads, dim, page, dtype, quantized, seed=0, head_major=False, spread=0.5,
                 width=None, tail=0):
        from cta_b200 import ops

        gen = torch.Generator().manual_seed(seed)
        self.lens, self.rows = lens, rows
        counts = [-(-n // page) for n in lens]
        pages = sum(counts) + 3
        order = torch.randperm(pages, generator=gen).tolist()
        width = max([1, *counts]) if width is None else width
        table = torch.full((len(lens), width), 2**31 - 1, dtype=torch.int32)  # entries past the length are not read
        self.kc, self.vc, self.ks, self.vs = _cache(pages, page, kv_heads, dim, dtype, quantized, head_major=head_major)
        self.k, self.v = [], []
        for b, n in enumerate(lens):
            mine = [order.pop() for _ in range(counts[b])]
            table[b, : len(mine)] = torch.tensor(mine, dtype=torch.int32)
            k, v = _rows(n, kv_heads, dim, dtype, 10 * b + 1 + seed, spread), _rows(n, kv_heads, dim, dtype, 10 * b + 2 + seed, spread)
            slots = torch.tensor([mine[j // page] * page + j % page for j in range(n)], dtype=torch.int64).cuda()
            ops.kv_cache_write(k, v, self.kc, self.vc, slots, k_scale=self.ks, v_scale=self.vs)
            if quantized:  # what the cache holds, exactly
                at = (slots // page, slice(None), slots % page)
                k = _codes(self.kc, slots) * self.ks[at].double()[..., None]
                v = _codes(self.vc, slots) * self.vs[at].double()[..., None]
            self.k.append(k)
            self.v.append(v)
        self.table = table.cuda()
        self.seq_lens = torch.tensor(lens, dtype=torch.int32).cuda()
        total = sum(rows)
        self.q = torch.randn(total + tail, heads, dim, generator=gen).to(dtype).cuda()
        self.cu = torch.tensor([0] + torch.tensor(rows).cumsum(0).tolist(), dtype=torch.int32).cuda()
        self.dtype, self.quantized, self.dim = dtype, quantized, dim

    def run(self, **kw):
        from cta_b200 import ops

        if not all(r == 1 for r in self.rows):
            kw.setdefault("cu_seqlens", self.cu)
        kw.setdefault("max_rows", max([1, *self.rows]))
        return ops.paged_attention(self.q, self.kc, self.vc, self.table, self.seq_lens, k_scale=self.ks,
                                   v_scale=self.vs, **kw)

    def check(self, out, scale=None):
        scale = self.dim**-0.5 if scale is None else scale
        at = 0
        for b, (n, r) in enumerate(zip(self.lens, self.rows)):
            q, got = self.q[at : at + r], out[at : at + r].double()
            at += r
            if r == 0:
                continue
            if n == 0:
                assert (got == 0).all()
                continue
            i = torch.arange(n - r, n, device="cuda")
            see = torch.arange(n, device="cuda")[None, :] <= i[:, None]
            want, _ = A.attention(q, self.k[b], self.v[b], see, scale)
            # e4m3, few rows: q is rounded to fp16 after an exact scaling, elements below 2^-14 of the largest to
            # 2^-25 of it: with d elements that is d 2^-25 of |q||k|, inside the (d + 4) 2^-24 of the scores'
            # bound.  More rows than one operand holds: codes and scales stay exact, each product is fp32.
            kv_error = 2.0**-20 if self.quantized else 0.0
            tol = A.bounds(q, self.k[b], self.v[b], see, scale, self.dtype, kv_error=kv_error)
            bad = ~((got - want).abs() <= tol)
            assert not bad.any(), (b, n, r, int(bad.sum()), (got - want).abs().max().item(), tol.min().item())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 128])
def test_decode_dims(dim, quantized, dtype):
    s = Setup([1, 15, 16, 17, 200, 333], [1] * 6, 8, 2, dim, 16, dtype, quantized, seed=dim)
    s.check(s.run())


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (2, 2), (3, 1), (5, 1), (8, 8), (16, 2), (9, 1), (16, 1), (17, 1), (40, 2), (71, 1)])
def test_decode_groups(heads, kv_heads, quantized):
    s = Setup([40, 300, 1], [1] * 3, heads, kv_heads, 64, 32, torch.bfloat16, quantized, seed=heads)
    s.check(s.run())


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("page", [16, 32, 48, 64, 128, 256])
def test_pages(page, quantized):
    s = Setup([page - 1, page, page + 1, 3 * page + 5, 700], [1, 1, 1, 1, 1], 4, 2, 128, page, torch.bfloat16,
              quantized, seed=page)
    s.check(s.run())
    s = Setup([page - 1, page, page + 1, 3 * page + 5, 700], [3, 16, 1, 40, 200], 4, 2, 128, page, torch.bfloat16,
              quantized, seed=page)
    s.check(s.run())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("rows", [[2, 2, 2], [1, 0, 5], [17, 1, 130], [128, 129, 127], [300, 64, 0], [1, 400, 33]])
def test_chunks(rows, quantized, dtype):
    lens = [r + x for r, x in zip(rows, (0, 77, 500))]
    for heads, kv_heads, dim in ((4, 4, 64), (8, 2, 128), (6, 2, 80)):
        s = Setup(lens, rows, heads, kv_heads, dim, 16, dtype, quantized, seed=sum(rows))
        s.check(s.run())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("rows", [[64, 64, 64], [1, 0, 300], [17, 1, 130], [128, 129, 127], [300, 64, 0], [1, 400, 33]])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(32, 8, 128, 16), (24, 8, 64, 48), (32, 32, 80, 128), (64, 4, 32, 64)])
def test_chunks_of_many_heads(heads, kv_heads, dim, page, rows, quantized, dtype):
    """Enough rows and heads for the tensor-core kernel."""
    lens = [r + x for r, x in zip(rows, (0, 77, 500))]
    s = Setup(lens, rows, heads, kv_heads, dim, page, dtype, quantized, seed=sum(rows), tail=2)
    out = torch.full_like(s.q, 7.0)
    s.run(out=out)
    s.check(out)
    assert (out[sum(rows):] == 7).all()
    if dim == 128 and not quantized:
        # any scale, the signs of it too
        s.check(s.run(scale=0.02), 0.02)
        s.check(s.run(scale=-0.02), -0.02)


@pytest.mark.parametrize("quantized", [False, True])
def test_lengths_zero_and_short(quantized):
    """No keys at all; more rows than keys (the first rows see nothing)."""
    s = Setup([0, 5, 0, 200], [1, 1, 1, 1], 4, 2, 64, 16, torch.bfloat16, quantized)
    s.check(s.run())
    for more in (0, 150):  # split and tensor-core kernels
        s = Setup([0, 3, 50 + more], [2, 3, 7 + more], 32, 8, 64, 16, torch.bfloat16, quantized)
        s.check(s.run())
        s.seq_lens[2] = 4 + more
        out = s.run()
        rows = out[5:12 + more]
        assert (rows[:3] == 0).all() and (rows[3:] != 0).any() and torch.isfinite(rows.float()).all()


@pytest.mark.parametrize("quantized", [False, True])
def test_one_long_sequence(quantized):
    """A single sequence over many workers; another with one very long sequence among short ones."""
    s = Setup([9000], [1], 4, 1, 128, 16, torch.bfloat16, quantized)
    s.check(s.run())
    s = Setup([3, 6000, 17, 1], [1, 1, 1, 1], 8, 2, 64, 64, torch.float16, quantized, width=200)
    s.check(s.run())


@pytest.mark.parametrize("quantized", [False, True])
def test_many_short_sequences(quantized):
    gen = torch.Generator().manual_seed(1)
    lens = torch.randint(1, 60, (150,), generator=gen).tolist()
    s = Setup(lens, [1] * 150, 4, 4, 64, 16, torch.bfloat16, quantized)
    s.check(s.run())


@pytest.mark.parametrize("quantized", [False, True])
def test_head_major_cache_and_strided_q(quantized):
    s = Setup([100, 260], [1, 1], 4, 2, 64, 16, torch.bfloat16, quantized, head_major=True)
    s.check(s.run())
    wide = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16, device="cuda")
    wide[:, 1] = s.q
    want = s.run()
    s.q = wide[:, 1]
    assert torch.equal(s.run(), want)
    odd = torch.zeros(2, 4, 67, dtype=torch.bfloat16, device="cuda")
    odd[..., 3:] = s.q
    s.q = odd[..., 3:]
    assert torch.equal(s.run(), want)


@pytest.mark.parametrize("spread", [6.0])
def test_e4m3_scales_far_apart(spread):
    """Scales over many orders of magnitude: neither overflow nor vanish in 16 bits."""
    for dtype in DTYPES:
        s = Setup([300, 40], [1, 1], 4, 2, 64, 16, torch.bfloat16, True, spread=0.3)
        for c in (s.vs,):
            c *= 2.0**-12
        s.v = [x * 2.0**-12 for x in s.v]
        s.check(s.run())
        s = Setup([300, 40], [1, 1], 4, 2, 64, 16, torch.bfloat16, True, spread=0.3)
        s.vs *= 2.0**14
        s.v = [x * 2.0**14 for x in s.v]
        s.check(s.run())
        s = Setup([300, 40], [1, 1], 4, 2, 64, 16, torch.bfloat16, True, spread=0.3)
        s.ks *= 2.0**-9
        s.k = [x * 2.0**-9 for x in s.k]
        s.q = s.q * 2.0**12
        s.check(s.run())


@pytest.mark.parametrize("rows", [[1, 1], [40, 200]])
@pytest.mark.parametrize("quantized", [False, True])
def test_rows_behind_the_last_sequence(rows, quantized):
    s = Setup([100, 300], rows, 32, 8, 64, 16, torch.bfloat16, quantized, tail=3)
    out = torch.full_like(s.q, 7.0)
    y = s.run(out=out, cu_seqlens=s.cu)
    assert y is out and (out[sum(rows):] == 7).all()
    s.check(out)


@pytest.mark.parametrize("rows", [[1, 1], [40, 200]])
@pytest.mark.parametrize("quantized", [False, True])
def test_bad_pages_and_lengths(rows, quantized):
    """Skipped and reported; the other sequence keeps its result."""
    from cta_b200 import _lib

    s = Setup([100, 300], rows, 32, 8, 64, 16, torch.bfloat16, quantized)
    want = s.run()
    good = s.table.clone()
    for bad in (-1, s.kc.shape[0], 2**31 - 1, -(2**31)):
        s.table[0, 2] = bad
        got = s.run()
        assert _lib.device_error() == 2
        assert torch.equal(got[rows[0]:], want[rows[0]:])
        assert torch.isfinite(got.float()).all()
        s.table.copy_(good)
    for n in (s.table.shape[1] * 16 + 1, 2**31 - 1, -5):
        s.seq_lens[0] = n
        s.table[0] = 0
        s.run()
        assert _lib.device_error() == 2
    s.table.copy_(good)
    s.seq_lens[0] = 100
    assert torch.equal(s.run(), want)


@pytest.mark.parametrize("rows", [[1, 1], [40, 200]])
def test_max_rows_is_a_hint(rows):
    s = Setup([100, 300], rows, 32, 8, 64, 16, torch.bfloat16, False)
    for hint in (1, 3, 100, 1000):
        s.check(s.run(max_rows=hint, cu_seqlens=s.cu))


@pytest.mark.parametrize("quantized", [False, True])
def test_large_cache(quantized):
    """Byte and element offsets past 2^31 and 2^32 in the pool."""
    from cta_b200 import ops

    page, heads, dim = 128, 8, 128
    pages = 36000  # 4.7e9 elements
    dtype = torch.bfloat16
    t = E4M3 if quantized else dtype
    kc, vc = (torch.empty(pages, page, heads, dim, dtype=t, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(pages, heads, page, device="cuda") if quantized else None for _ in range(2))
    mine = [35999, 17000, 3, 33000]
    n = 4 * page - 5
    k, v = _rows(n, heads, dim, dtype, 1), _rows(n, heads, dim, dtype, 2)
    slots = torch.tensor([mine[j // page] * page + j % page for j in range(n)], dtype=torch.int64).cuda()
    ops.kv_cache_write(k, v, kc, vc, slots, k_scale=ks, v_scale=vs)
    kr, vr = ops.kv_cache_read(kc, vc, slots, k_scale=ks, v_scale=vs, dtype=dtype)
    if not quantized:
        assert torch.equal(kr, k) and torch.equal(vr, v)
    small = [0, 1, 2, 3]
    kc2, vc2, ks2, vs2 = _cache(4, page, heads, dim, dtype, quantized)
    slots2 = torch.arange(n, device="cuda")
    ops.kv_cache_write(k, v, kc2, vc2, slots2, k_scale=ks2, v_scale=vs2)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    for rows in (1, 400):
        q = torch.randn(rows, 16, dim, device="cuda").to(dtype)
        cu = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
        a = ops.paged_attention(q, kc, vc, torch.tensor([mine], dtype=torch.int32, device="cuda"), lens, cu_seqlens=cu,
                                max_rows=rows, k_scale=ks, v_scale=vs)
        b = ops.paged_attention(q, kc2, vc2, torch.tensor([small], dtype=torch.int32, device="cuda"), lens,
                                cu_seqlens=cu, max_rows=rows, k_scale=ks2, v_scale=vs2)
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [[1, 1, 1], [40, 200, 7]])
@pytest.mark.parametrize("quantized", [False, True])
def test_captured_twice_and_replayed_together(rows, quantized):
    """Two graphs captured on one stream, replayed at the same time on two: each has its own workspace."""
    s = Setup([1500, 300, 2200], rows, 32, 8, 128, 16, torch.bfloat16, quantized)
    other = Setup([900, 2000, 800], rows, 32, 8, 128, 16, torch.bfloat16, quantized, seed=5)
    want, want2 = s.run(), other.run()
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for x in (s, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(x.run())
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want2)


def test_twice_the_same():
    for quantized in (False, True):
        for rows in ([1, 1, 1], [50, 3, 170]):
            s = Setup([1500, 300, 2200], rows, 32, 8, 128, 16, torch.bfloat16, quantized)
            assert torch.equal(s.run(), s.run())


def test_no_rows_or_sequences():
    from cta_b200 import ops

    s = Setup([10], [1], 2, 2, 64, 16, torch.bfloat16, False)
    assert ops.paged_attention(s.q[:0], s.kc, s.vc, s.table[:0], s.seq_lens[:0]).shape == (0, 2, 64)
    cu = torch.zeros(2, dtype=torch.int32, device="cuda")
    out = torch.full_like(s.q, 3.0)
    ops.paged_attention(s.q, s.kc, s.vc, s.table, s.seq_lens, cu_seqlens=cu, out=out)
    assert (out == 3).all()


@pytest.mark.parametrize("quantized", [False, True])
def test_two_streams_at_once(quantized):
    """Decode and a chunk side by side give what they give alone, bit for bit."""
    from cta_b200 import ops

    sets = [Setup([900, 33, 2100], [1, 1, 1], 8, 2, 128, 16, torch.bfloat16, quantized),
            Setup([1500, 700], [300, 260], 8, 2, 128, 32, torch.bfloat16, quantized)]
    alone = [s.run() for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(6):
        for i, (s, stream) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(stream):
                got[i].append(s.run().clone())
    torch.cuda.synchronize()
    for want, all_of in zip(alone, got):
        for x in all_of:
            assert torch.equal(want, x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("heads,kv_heads,rows,hint", [(32, 8, 8, 8), (8, 8, 24, 1), (16, 2, 40, 1), (4, 4, 40, 40)])
@pytest.mark.parametrize("keys", [1, 3, 4, 7, 17])
def test_tiles_whose_rows_all_see_nothing(keys, heads, kv_heads, rows, hint, quantized, dtype):
    """So many more rows than keys that whole tiles of 8 or 16 (row, head) pairs see none of the keys there are."""
    s = Setup([keys, 200], [rows, 1], heads, kv_heads, 64, 16, dtype, quantized, seed=keys)
    out = s.run(max_rows=hint)
    blind = max(0, rows - keys)
    assert (out[:blind] == 0).all()
    s.check(out)


@pytest.mark.parametrize("quantized", [False, True])
def test_empty_pool(quantized):
    """A cache without pages, or a view of none: every sequence is without keys, by whatever kernel the rows choose."""
    from cta_b200 import _lib, ops

    for rows in ([1, 1], [40, 200]):
        s = Setup([rows[0], rows[1]], rows, 32, 8, 64, 16, torch.bfloat16, quantized)
        for empty in (lambda t: t[:0], torch.empty_like):
            kc, vc, ks, vs = (None if t is None else empty(t[:0]) for t in (s.kc, s.vc, s.ks, s.vs))
            s.kc, s.vc, s.ks, s.vs = kc, vc, ks, vs
            s.seq_lens.zero_()
            assert (s.run(cu_seqlens=s.cu, out=torch.full_like(s.q, 7.0)) == 0).all()
            s.seq_lens.fill_(5)  # pages that are not there: skipped and reported
            assert (s.run(cu_seqlens=s.cu, out=torch.full_like(s.q, 7.0)) == 0).all()
            assert _lib.device_error() == 2
            slots = torch.full((3,), -1, device="cuda")
            new = torch.ones(3, 8, 64, dtype=torch.bfloat16, device="cuda")
            ops.kv_cache_write(new, new, kc, vc, slots, k_scale=ks, v_scale=vs)
            assert all((x == 0).all() for x in ops.kv_cache_read(kc, vc, slots, k_scale=ks, v_scale=vs))
            slots[1] = 0
            ops.kv_cache_write(new, new, kc, vc, slots, k_scale=ks, v_scale=vs)
            assert _lib.device_error() == 2
    s = Setup([0, 0], [40, 200], 32, 8, 64, 16, torch.bfloat16, quantized, width=0)  # a table without entries
    assert s.table.numel() == 0 and (s.run() == 0).all()


def _rescaled(s, ks=1.0, vs=1.0, q=1.0):
    """Other scales over the same codes: powers of two, so that the cache's values stay known exactly."""
    s.ks *= ks
    s.vs *= vs
    s.k, s.v = [x * ks for x in s.k], [x * vs for x in s.v]
    s.q = s.q * q


def _check_scaled(s, out):
    """Against the definition, with no allowance for what 16 bits cannot hold of a weight but this: weight times
    value's scale is held relative to the largest of them so far, with a smallest step of 2^-31 of it (fp16:
    2^-24, shifted by 2^7), so each key is off by at most 2^-32 of the row's largest weight * scale, times its
    code, 448 at most and 448 in the largest element of each row.  A scale that joins a weight through its
    logarithm (up to 64 here, 2^-24 of it) moves it by 2^-18."""
    at = 0
    for b, (n, r) in enumerate(zip(s.lens, s.rows)):
        q, got = s.q[at : at + r], out[at : at + r].double()
        at += r
        see = torch.arange(n, device="cuda")[None, :] <= torch.arange(n - r, n, device="cuda")[:, None]
        scale = s.dim**-0.5
        want, _ = A.attention(q, s.k[b], s.v[b], see, scale)
        assert want.abs().max() < torch.finfo(s.dtype).max
        tol = A.bounds(q, s.k[b], s.v[b], see, scale, s.dtype, kv_error=2.0**-20, weight_step=0.0)
        p, _ = A.weights(q, s.k[b], see, scale)
        v = s.v[b].abs().transpose(0, 1).repeat_interleave(q.shape[1] // s.v[b].shape[1], 0)  # [H, n, dim]
        most = (p * v.amax(-1)[:, None]).amax(-1, keepdim=True)
        tol = tol + (n * 2.0**-32 * most + 2.0**-18 * torch.matmul(p, v)).transpose(0, 1)
        bad = ~((got - want).abs() <= tol)
        assert not bad.any(), (b, n, r, int(bad.sum()), (got - want).abs().max().item(), want.abs().max().item())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [[1, 1], [40, 200]])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("written", DTYPES)
def test_e4m3_scales_outside_the_type(written, dim, rows, dtype):
    """Scales that fp32 holds and fp16 does not, codes times them included: decode and chunks alike, whatever type
    the cache was written from."""
    def setup(**kw):
        s = Setup([300, 250], rows, 32, 8, dim, 16, written, True, **kw)
        s.q, s.dtype = s.q.to(dtype), dtype
        return s

    for kw in (dict(ks=2.0**19, q=2.0**-19), dict(ks=2.0**17, q=2.0**-14), dict(ks=2.0**-13, q=2.0**12),
               dict(ks=2.0**-40, q=2.0**13), dict(vs=2.0**-10), dict(vs=2.0**-17), dict(vs=2.0**11),
               dict(ks=2.0**-13, q=2.0**11, vs=2.0**9)):
        s = setup()
        _rescaled(s, **kw)
        _check_scaled(s, s.run())
    # rows of different size in one sequence, as a whole far down and up
    for vs in (1.0, 2.0**-10, 2.0**4):
        s = setup(spread=1.5, seed=3)
        _rescaled(s, vs=vs)
        _check_scaled(s, s.run())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [[1, 1], [40, 200]])
def test_e4m3_large_values_of_little_weight(rows, dtype):
    """Every fourth key has values 2^17 times the others', past fp16, and a weight that makes up for it."""
    from cta_b200 import ops

    s = Setup([300, 250], rows, 32, 8, 64, 16, dtype, True, seed=4)
    s.q = s.q.abs() + 1
    page = s.kc.shape[1]
    # their scores are about -115 * 0.85 / 8 = -12, a weight of 2^-17.6
    for b, n in enumerate(s.lens):
        j = torch.arange(0, n, 4, device="cuda")
        slots = s.table[b].long()[j // page] * page + j % page
        far = -(0.7 + 0.3 * torch.rand(len(j), 8, 64, generator=torch.Generator().manual_seed(b))).cuda().to(dtype)
        ops.kv_cache_write(far, s.v[b][j].to(dtype), s.kc, s.vc, slots, k_scale=s.ks, v_scale=s.vs)
        at = (slots // page, slice(None), slots % page)
        s.vs[at] *= 2.0**17
        s.k[b][j] = _codes(s.kc, slots) * s.ks[at].double()[..., None]
        s.v[b][j] = _codes(s.vc, slots) * s.vs[at].double()[..., None]
    assert s.v[0].abs().max() > torch.finfo(torch.float16).max
    _check_scaled(s, s.run())


@pytest.mark.parametrize("dtype", DTYPES)
def test_codes_are_the_nearest(dtype):
    """Every element's code is the e4m3 number nearest to x * 448 / m, ties to the even one.  In 64 bits x * 448 is exact
    and the quotient exact to 2^-53, while a quotient that is no tie lies 2^-17 or further from one: x * 448 and
    the tie times m are whole numbers of at most 17 bits."""
    from cta_b200 import ops

    bits = 7 if dtype == torch.bfloat16 else 10
    # all fractions of x against the fractions of m: those with ties (m = 7 i) and others
    fractions = torch.arange(2**bits, 2 ** (bits + 1), dtype=torch.float64)
    mine = fractions if bits == 7 else torch.cat([fractions[fractions % 7 == 0][::4], fractions[::31]])
    binades = 17 if bits == 7 else 14
    x = (fractions[None, :] * 2.0 ** -torch.arange(binades, dtype=torch.float64)[:, None]).flatten()
    per = 255
    x = torch.cat([x, x[: -len(x) % per]]).view(-1, per)
    x[:, ::2] *= -1
    for scale in ((2.0**-106, 2.0**-7, 1.0, 2.0**120) if bits == 7 else (2.0**-10, 2.0**5)):
        rows = []
        for m in mine:
            keep = torch.where(x.abs() > m, x / 2, x)
            rows.append(torch.cat([torch.full((len(x), 1), m.item(), dtype=torch.float64), keep], 1))
        wide = torch.cat(rows) * scale
        k = wide.to(dtype)
        wide = k.double()  # fp16's subnormal numbers are rounded here
        n = len(k)
        k = k.cuda()[:, None]
        kc, vc, ks, vs = _cache(-(-n // 16), 16, 1, 256, dtype, True)
        slots = torch.arange(n, device="cuda")
        ops.kv_cache_write(k, -k, kc, vc, slots, k_scale=ks, v_scale=vs)
        codes, scales = A.quantise(k)
        assert torch.equal(_codes(kc, slots), codes)
        assert torch.equal(_codes(vc, slots), -codes)
        assert torch.equal(ks[slots // 16, :, slots % 16], scales.float())


def test_fp16_chunks_over_e4m3_captured_together():
    """Chunks whose expansion lies in a workspace of their own: two graphs replayed at the same time, bit for bit."""
    sets = [Setup(lens, [40, 200, 7], 32, 8, 128, 16, torch.float16, True, seed=i)
            for i, lens in enumerate(([1500, 300, 2200], [900, 2000, 800]))]
    _rescaled(sets[1], vs=2.0**6)
    want = [s.run() for s in sets]
    assert all(torch.equal(s.run(), x) for s, x in zip(sets, want))
    side, graphs, outs = torch.cuda.Stream(), [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(s.run())
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(outs, want):
        assert torch.equal(x, y)
