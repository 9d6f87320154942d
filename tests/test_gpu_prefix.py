"""Paged attention of a batch whose sequences begin with the same keys, against the definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

from oracle import attention_oracle as A
from test_gpu_attention import _within
from test_gpu_paged import Setup as Plain

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def no_device_error():
    """The prefix is read once at these sizes too, where that need not pay."""
    from cta_b200 import _lib

    before = _lib.set_tuning(6, 1)
    yield
    _lib.set_tuning(6, before)
    assert _lib.device_error() == 0


class Setup(Plain):
    """Sequences of `lens` keys, of which the first `prefix` (whole pages) are sequence 0's; as many sequences as lens."""

    def __init__(self, prefix, lens, rows, heads, kv_heads, dim, page, dtype, quantized, **kw):
        assert prefix % page == 0 and lens[0] >= prefix
        super().__init__(lens, rows, heads, kv_heads, dim, page, dtype, quantized, **kw)
        self.prefix, shared = prefix, prefix // page
        for b in range(1, len(lens)):
            mine = min(shared, -(-lens[b] // page))
            self.table[b, :mine] = self.table[0, :mine]
            n = min(prefix, lens[b])
            self.k[b] = torch.cat([self.k[0][:n], self.k[b][n:]])
            self.v[b] = torch.cat([self.v[0][:n], self.v[b][n:]])

    def run(self, **kw):
        kw.setdefault("shared_prefix", self.prefix)
        return super().run(**kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("prefix", [16, 128, 144, 400, 1024, 2000])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 4, 64)])
def test_prefixes(heads, kv_heads, dim, prefix, quantized, dtype):
    lens = [prefix + x for x in (1, 17, 100, 1, 300, 33)]
    s = Setup(prefix, lens, [1] * 6, heads, kv_heads, dim, 16, dtype, quantized, seed=prefix)
    s.check(s.run())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(1, 1, 16, 16), (3, 1, 48, 32), (32, 8, 128, 64), (12, 2, 80, 48), (71, 1, 64, 128),
                                                     (16, 1, 96, 256), (24, 8, 32, 16)])
def test_heads_dims_pages(heads, kv_heads, dim, page, quantized, dtype):
    prefix = page * (1000 // page)
    s = Setup(prefix, [prefix + x for x in (5, 1, 260)], [1] * 3, heads, kv_heads, dim, page, dtype, quantized, seed=heads)
    s.check(s.run())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("batch", [2, 33, 64, 65, 200])
def test_batches(batch, quantized, dtype):
    lens = [512 + 1 + int(x) for x in torch.randint(0, 90, (batch,), generator=torch.Generator().manual_seed(batch))]
    s = Setup(512, lens, [1] * batch, 8, 2, 64, 32, dtype, quantized, seed=batch)
    s.check(s.run())


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("rows", [[2, 3, 1, 4], [1, 0, 2, 1], [40, 1, 200, 0], [16, 16, 16, 16]])
def test_more_rows(rows, quantized):
    """Speculated tokens, sequences without rows, chunks."""
    for heads, kv_heads, dim in ((8, 2, 128), (32, 8, 64)):
        lens = [640 + r + x for r, x in zip(rows, (0, 77, 300, 1))]
        s = Setup(640, lens, rows, heads, kv_heads, dim, 64, torch.bfloat16, quantized, seed=sum(rows))
        s.check(s.run())


@pytest.mark.parametrize("quantized", [False, True])
def test_sequences_that_end_within_the_prefix(quantized):
    """Also empty ones, as the padding of a captured batch has them."""
    s = Setup(1024, [1100, 1024, 1000, 17, 1, 0, 0, 1030], [1] * 8, 8, 2, 64, 16, torch.bfloat16, quantized, seed=2)
    s.check(s.run())
    s = Setup(1024, [1100, 1024, 1000, 17, 3, 0, 0, 1030], [3, 3, 3, 3, 3, 3, 0, 2], 8, 2, 64, 16, torch.bfloat16, quantized, seed=2)
    at = 0
    out = s.run()
    for b, (n, r) in enumerate(zip(s.lens, s.rows)):
        q, got = s.q[at : at + r], out[at : at + r]
        at += r
        if n == 0 or r == 0:
            assert (got == 0).all()
            continue
        i = torch.arange(n - r, n, device="cuda")
        see = torch.arange(n, device="cuda")[None, :] <= i[:, None]
        want, _ = A.attention(q, s.k[b], s.v[b], see, 0.125)
        _within(got, want, A.bounds(q, s.k[b], s.v[b], see, 0.125, s.dtype, kv_error=2.0**-20 if quantized else 0.0), f"{b}: ")


@pytest.mark.parametrize("quantized", [False, True])
def test_a_page_in_part_does_not_count(quantized):
    """shared_prefix within a page: the keys of that page are each sequence's own."""
    s = Setup(640, [700, 650, 641], [1] * 3, 8, 2, 64, 64, torch.bfloat16, quantized, seed=3)
    for extra in (1, 17, 63):
        s.check(s.run(shared_prefix=640 + extra))


@pytest.mark.parametrize("quantized", [False, True])
def test_far_scores(quantized):
    """Prefix or own keys that outweigh the others by far: the join is relative to both."""
    for which in (0, 1):
        s = Setup(512, [600, 530, 513], [1] * 3, 8, 2, 64, 16, torch.float16, quantized, seed=4)
        if quantized:
            pages = s.table[0, :32].long() if which == 0 else torch.cat([s.table[b, 32 : -(-n // 16)] for b, n in enumerate(s.lens)]).long()
            s.ks[pages] *= 64.0
            for b in range(3):
                part = slice(0, 512) if which == 0 else slice(512, None)
                s.k[b] = s.k[b].clone()
                s.k[b][part] *= 64.0
        else:
            s.q *= 30
        out = s.run()
        for b, n in enumerate(s.lens):
            see = torch.ones(1, n, dtype=torch.bool, device="cuda")
            want, _ = A.attention(s.q[b : b + 1], s.k[b], s.v[b], see, 0.125)
            _within(out[b : b + 1], want, A.bounds(s.q[b : b + 1], s.k[b], s.v[b], see, 0.125, s.dtype,
                                                   kv_error=2.0**-20 if quantized else 0.0), f"{which} {b}: ")


@pytest.mark.parametrize("quantized", [False, True])
def test_bad_page_in_the_prefix(quantized):
    from cta_b200 import _lib

    s = Setup(512, [600, 530, 513], [1] * 3, 8, 2, 64, 16, torch.bfloat16, quantized, seed=5)
    s.table[:, 3] = s.kc.shape[0]
    out = s.run()
    torch.cuda.synchronize()
    assert _lib.device_error() == 2
    for b, n in enumerate(s.lens):
        see = torch.ones(1, n, dtype=torch.bool, device="cuda")
        see[:, 48:64] = False
        want, _ = A.attention(s.q[b : b + 1], s.k[b], s.v[b], see, 0.125)
        _within(out[b : b + 1], want, A.bounds(s.q[b : b + 1], s.k[b], s.v[b], see, 0.125, s.dtype,
                                               kv_error=2.0**-20 if quantized else 0.0), f"{b}: ")


def test_strided_q_and_out():
    s = Setup(512, [600, 530, 513], [1] * 3, 8, 2, 64, 16, torch.bfloat16, False, seed=6)
    want = s.run()
    wide = torch.zeros(3, 8, 128, dtype=torch.bfloat16, device="cuda")
    wide[..., :64] = s.q
    s.q = wide[..., :64]
    out = torch.zeros(3, 16, 64, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(s.run(), want)
    assert torch.equal(s.run(out=out[:, ::2]), want) and (out[:, 1::2] == 0).all()


@pytest.mark.parametrize("quantized", [False, True])
def test_tail_and_twice_the_same(quantized):
    s = Setup(1024, [1100, 1030, 1025], [1, 2, 1], 8, 2, 64, 16, torch.bfloat16, quantized, seed=7, tail=4)
    out = torch.full_like(s.q, 7.0)
    s.run(out=out)
    assert (out[4:] == 7).all()
    s.check(out)
    assert torch.equal(s.run(out=torch.full_like(s.q, 7.0)), out)


@pytest.mark.parametrize("quantized", [False, True])
def test_captured_and_replayed_together(quantized):
    setups = [Setup(1024, [1100, 1030, 1025], [1] * 3, 8, 2, 64, 16, torch.bfloat16, quantized, seed=x) for x in (1, 2)]
    want = [s.run() for s in setups]
    graphs, outs = [], []
    for s in setups:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(s.run())
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


@pytest.mark.parametrize("quantized", [False, True])
def test_where_it_pays(quantized):
    """Small batches go without it, to the bit; large ones use it."""
    from cta_b200 import _lib

    _lib.set_tuning(6, 0)
    s = Setup(512, [600, 530, 513], [1] * 3, 8, 2, 64, 16, torch.bfloat16, quantized, seed=8)
    assert torch.equal(s.run(), s.run(shared_prefix=0))
    n = 80
    s = Setup(3200, [3200 + 1 + b % 7 for b in range(n)], [1] * n, 8, 2, 64, 64, torch.bfloat16, quantized, seed=9)
    out = s.run()
    s.check(out)
    assert not torch.equal(out, s.run(shared_prefix=0))


def test_empty():
    s = Setup(64, [70, 65], [1, 1], 8, 2, 64, 16, torch.bfloat16, False)
    s.q, s.rows, s.lens = s.q[:0], [], []
    s.table, s.seq_lens = s.table[:0], s.seq_lens[:0]
    assert s.run().shape == (0, 8, 64)


def test_prefix_longer_than_the_table():
    """As far as the table goes; more cannot be shared."""
    s = Setup(512, [520, 513], [1, 1], 8, 2, 64, 16, torch.bfloat16, False)
    s.table[1] = s.table[0]
    s.k[1], s.v[1] = s.k[0][:513], s.v[0][:513]
    s.check(s.run(shared_prefix=10**12))


def test_refusals():
    s = Setup(64, [70, 65], [1, 1], 8, 2, 64, 16, torch.bfloat16, False)
    with pytest.raises(ValueError, match="shared_prefix"):
        s.run(shared_prefix=-1)
    with pytest.raises(TypeError):
        s.run(shared_prefix=1.5)
