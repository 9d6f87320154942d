"""The operators where the framework calls them: the PDE Transformers with fused attention,
and the serving mixer over a paged cache."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from oracle import attention_oracle as A

pytestmark = pytest.mark.gpu


def _models(kind, **kw):
    from cta_b200 import transformers as T

    cls = T.PDETransformerClassifier if kind == "classifier" else T.PDETransformerLM
    if kind == "classifier":
        kw["num_classes"] = 3
    torch.manual_seed(0)
    stock = cls(**kw).cuda()
    fused = cls(attention="fused", **kw).cuda()
    fused.load_state_dict(stock.state_dict())  # same parameters under the same names
    return stock, fused


@pytest.mark.parametrize("kind", ["classifier", "lm"])
@pytest.mark.parametrize("length", [1, 37, 200])
def test_models_match_stock_attention(kind, length):
    """fp32, dropout 0: fused and stock attention differ by fp32 rounding.  A layer's attention is off by
    about 64 * 2^-24 relative to its largest value (dot products of 16 elements, sums of up to 200); two
    layers with norms and projections pass that on with factors of a few: 1e-4 of the largest value is 25
    times that."""
    kw = dict(vocab_size=101, embed_dim=64, num_heads=4, hidden_dim=128, num_layers=2, pde_steps=2, pde_layout="bld",
              max_length=256, dropout=0.0)
    stock, fused = _models(kind, **kw)
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 101, (3, length), generator=gen).cuda()
    mask = torch.ones(3, length, dtype=torch.long)
    mask[1, (length + 1) // 2:] = 0
    mask = mask.cuda()
    outs = []
    for net in (stock, fused):
        net.train()
        y = net(ids, mask)
        (y * torch.linspace(-1, 1, y.shape[-1], device="cuda")).square().sum().backward()
        outs.append((y.detach(), {n: p.grad for n, p in net.named_parameters()}))
    (y0, g0), (y1, g1) = outs
    assert (y0 - y1).abs().max() <= 1e-4 * y0.abs().max()
    assert g0.keys() == g1.keys()
    for n in g0:
        if g0[n] is None:
            assert g1[n] is None
            continue
        assert (g0[n] - g1[n]).abs().max() <= 1e-3 * g0[n].abs().max() + 1e-6, n


def test_model_left_padding_is_finite():
    """Rows that see nothing get zeros from their attention; no NaN reaches the loss or a gradient."""
    _, fused = _models("lm", vocab_size=50, embed_dim=64, num_heads=4, hidden_dim=64, num_layers=2, pde_steps=1,
                       max_length=64, dropout=0.0)
    for dtype in (torch.float32, torch.bfloat16):
        net = fused.to(dtype)
        net.zero_grad()
        mask = torch.ones(2, 40, dtype=torch.long, device="cuda")
        mask[0, :13] = 0
        mask[1] = 0
        y = net(torch.randint(0, 50, (2, 40), device="cuda"), mask)
        assert torch.isfinite(y).all()
        y.float().square().mean().backward()
        assert all(torch.isfinite(p.grad).all() for p in net.parameters() if p.grad is not None)


def test_model_in_eval_and_unknown_attention():
    from cta_b200 import transformers as T

    stock, fused = _models("lm", vocab_size=50, embed_dim=64, num_heads=2, hidden_dim=64, num_layers=1, pde_steps=1,
                           max_length=64, dropout=0.3)
    ids = torch.randint(0, 50, (2, 30), device="cuda")
    mask = torch.ones(2, 30, dtype=torch.long, device="cuda")
    with torch.no_grad():
        a, b = stock.eval()(ids, mask), fused.eval()(ids, mask)
    assert (a - b).abs().max() <= 1e-4 * a.abs().max()
    with pytest.raises(ValueError, match="attention"):
        T.PDETransformerLM(vocab_size=5, embed_dim=8, num_heads=2, hidden_dim=8, num_layers=1, attention="flash")


# ---------------------------------------------------------------------------
# serving
# ---------------------------------------------------------------------------
class Server:
    """One layer's cache and the sequences in it."""

    def __init__(self, heads, kv_heads, dim, page, pages, dtype, quantized):
        self.heads, self.kv_heads, self.dim, self.page, self.dtype = heads, kv_heads, dim, page, dtype
        t = torch.float8_e4m3fn if quantized else dtype
        self.kc, self.vc = (torch.full((pages, page, kv_heads, dim), 0x7F, dtype=torch.uint8, device="cuda").view(t)
                            if quantized else torch.full((pages, page, kv_heads, dim), float("nan"), dtype=t, device="cuda")
                            for _ in range(2))
        self.ks, self.vs = (torch.full((pages, kv_heads, page), float("nan"), device="cuda") if quantized else None
                            for _ in range(2))
        self.free = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).tolist()
        self.pages, self.k, self.v = {}, {}, {}

    def batch(self, new, seed, padding=0):
        """Metadata and rows for {sequence: new tokens}."""
        gen = torch.Generator().manual_seed(seed)
        slots, lens, starts = [], [], [0]
        k_rows, v_rows = [], []
        for s, n in new.items():
            old = self.k[s].shape[0] if s in self.k else 0
            mine = self.pages.setdefault(s, [])
            while len(mine) * self.page < old + n:
                mine.append(self.free.pop())
            k, v = (torch.randn(n, self.kv_heads, self.dim, generator=gen).to(self.dtype).cuda() for _ in range(2))
            k_rows.append(k)
            v_rows.append(v)
            self.k[s] = torch.cat([self.k[s], k]) if old else k
            self.v[s] = torch.cat([self.v[s], v]) if old else v
            slots += [mine[j // self.page] * self.page + j % self.page for j in range(old, old + n)]
            lens.append(old + n)
            starts.append(starts[-1] + n)
        total = starts[-1]
        width = max(len(self.pages[s]) for s in new) + 2
        table = torch.zeros(len(new), width, dtype=torch.int32)
        for b, s in enumerate(new):
            table[b, : len(self.pages[s])] = torch.tensor(self.pages[s], dtype=torch.int32)
        pad = torch.full((padding, self.kv_heads, self.dim), float("nan"), dtype=self.dtype, device="cuda")
        md = SimpleNamespace(slot_mapping=torch.tensor(slots + [-1] * padding, dtype=torch.int64).cuda(),
                             block_table=table.cuda(), seq_lens=torch.tensor(lens, dtype=torch.int32).cuda(),
                             query_start_loc=torch.tensor(starts, dtype=torch.int32).cuda(),
                             max_query_len=max(new.values()))
        q = torch.randn(total + padding, self.heads, self.dim, generator=gen).to(self.dtype).cuda()
        return md, q, torch.cat([*k_rows, pad]), torch.cat([*v_rows, pad])

    def check(self, out, q, new):
        at = 0
        for s, n in new.items():
            k, v = self.k[s], self.v[s]
            if self.ks is not None:
                # what the cache holds, exactly (what the write makes of a row has its own tests: a value near
                # the middle of two codes may go to either, which moves a score by more than this bound)
                j = torch.arange(k.shape[0], device="cuda")
                pages, slot = torch.tensor(self.pages[s], device="cuda")[j // self.page], j % self.page
                k, v = (c.view(torch.uint8)[pages, slot].view(torch.float8_e4m3fn).double() * x[pages, :, slot].double()[..., None]
                        for c, x in ((self.kc, self.ks), (self.vc, self.vs)))
            total = k.shape[0]
            i = torch.arange(total - n, total, device="cuda")
            see = torch.arange(total, device="cuda")[None, :] <= i[:, None]
            want, _ = A.attention(q[at : at + n], k, v, see, self.dim**-0.5)
            tol = A.bounds(q[at : at + n], k, v, see, self.dim**-0.5, self.dtype,
                           kv_error=2.0**-20 if self.ks is not None else 0.0)
            bad = (out[at : at + n].double() - want).abs() > tol
            assert not bad.any(), (s, n, total, int(bad.sum()))
            at += n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 4, 64)])
def test_prompts_chunks_and_decode(heads, kv_heads, dim, quantized, dtype):
    """Prompts, chunks of prompts, single tokens and mixed batches of them, one after another in one cache."""
    from cta_b200.serving_vllm import CtaConfig, CtaPostAttnMixer

    mixer = CtaPostAttnMixer(CtaConfig(enabled=False))  # the attention alone
    server = Server(heads, kv_heads, dim, 16, 200, dtype, quantized)
    steps = [{0: 130, 1: 17}, {2: 300}, {0: 1, 1: 1, 2: 1}, {0: 1, 3: 64, 2: 1}, {1: 200, 3: 5}, {0: 1, 1: 1, 2: 1, 3: 1}]
    for i, new in enumerate(steps):
        md, q, k, v = server.batch(new, i, padding=3)
        out = mixer.attend(q, k, v, server.kc, server.vc, attn_metadata=md, k_scale=server.ks, v_scale=server.vs)
        assert out.shape == (q.shape[0], heads * dim)
        server.check(out.view(-1, heads, dim), q, new)


def test_attention_with_mixer_and_residual():
    """attend() is write, attention and mixer in turn, the residual included."""
    from cta_b200 import ops
    from cta_b200.serving_vllm import CtaConfig, CtaPostAttnMixer

    mixer = CtaPostAttnMixer(CtaConfig(steps=4, alpha=0.1))
    server = Server(8, 2, 64, 16, 60, torch.bfloat16, True)
    md, q, k, v = server.batch({0: 100, 1: 33, 2: 1}, 1)
    residual = torch.randn(q.shape[0], 512, device="cuda").to(torch.bfloat16)
    out = mixer.attend(q, k, v, server.kc, server.vc, attn_metadata=md, k_scale=server.ks, v_scale=server.vs,
                       residual=residual)
    a = ops.paged_attention(q, server.kc, server.vc, md.block_table, md.seq_lens, cu_seqlens=md.query_start_loc,
                            max_rows=100, k_scale=server.ks, v_scale=server.vs).view(q.shape[0], -1)
    assert torch.equal(out, mixer(a, attn_metadata=md, residual=residual))
    for name in ("slot_mapping", "block_table", "seq_lens", "query_start_loc", "max_query_len"):
        bad = SimpleNamespace(**vars(md))
        delattr(bad, name)
        with pytest.raises(ValueError, match=name):
            mixer.attend(q, k, v, server.kc, server.vc, attn_metadata=bad, k_scale=server.ks, v_scale=server.vs)


def test_decode_step_captured():
    """A decode step (write, attention) in a CUDA graph, replayed as the sequences grow."""
    from cta_b200.serving_vllm import CtaConfig, CtaPostAttnMixer

    mixer = CtaPostAttnMixer(CtaConfig(enabled=False))
    server = Server(8, 2, 64, 16, 60, torch.bfloat16, False)
    md, q, k, v = server.batch({0: 60, 1: 15}, 0)
    mixer.attend(q, k, v, server.kc, server.vc, attn_metadata=md)
    new = {0: 1, 1: 1}
    md, q, k, v = server.batch(new, 1)
    md.block_table = torch.nn.functional.pad(md.block_table, (0, 4))
    graph = torch.cuda.CUDAGraph()
    mixer.attend(q, k, v, server.kc, server.vc, attn_metadata=md)  # warm-up: writes the same rows
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = mixer.attend(q, k, v, server.kc, server.vc, attn_metadata=md)
    for i in range(4):
        if i:
            nmd, nq, nk, nv = server.batch(new, 10 + i)
            q.copy_(nq), k.copy_(nk), v.copy_(nv)
            md.slot_mapping.copy_(nmd.slot_mapping)
            md.seq_lens.copy_(nmd.seq_lens)
            md.block_table[:, : nmd.block_table.shape[1]].copy_(nmd.block_table)
        graph.replay()
        server.check(out.view(-1, 8, 64), q, new)


@pytest.mark.parametrize("quantized", [False, True])
def test_attend_without_rows(quantized):
    """A step without tokens (an idle rank): no row out, nothing written."""
    from cta_b200.serving_vllm import CtaConfig, CtaPostAttnMixer

    for enabled in (False, True):
        mixer = CtaPostAttnMixer(CtaConfig(enabled=enabled))
        server = Server(8, 2, 64, 16, 20, torch.bfloat16, quantized)
        md, q, k, v = server.batch({0: 40}, 0)
        before = server.kc.clone().view(torch.uint8)
        for starts, lens, longest in (([0], 0, 0), ([0, 0], 1, 0), ([0, 0], 1, 5)):
            md.query_start_loc = torch.tensor(starts, dtype=torch.int32, device="cuda")
            md.block_table, md.seq_lens = md.block_table[:lens], torch.full((lens,), 7, dtype=torch.int32, device="cuda")
            if lens == 1:
                md.block_table = torch.zeros(1, 3, dtype=torch.int32, device="cuda")
            md.max_query_len, md.slot_mapping = longest, torch.zeros(0, dtype=torch.int64, device="cuda")
            for residual in (None, torch.zeros(0, 512, dtype=torch.bfloat16, device="cuda")):
                out = mixer.attend(q[:0], k[:0], v[:0], server.kc, server.vc, attn_metadata=md, k_scale=server.ks,
                                   v_scale=server.vs, residual=residual)
                assert out.shape == (0, 512)
        assert torch.equal(before, server.kc.view(torch.uint8))


def test_attend_refuses_before_it_writes():
    """Whatever the attention refuses is refused before the cache is touched."""
    from cta_b200.serving_vllm import CtaConfig, CtaPostAttnMixer

    mixer = CtaPostAttnMixer(CtaConfig(enabled=False))

    def refused(server, md, q, k, v, match, **kw):
        before = [c.clone().view(torch.uint8) for c in (server.kc, server.vc)]
        with pytest.raises(ValueError, match=match):
            mixer.attend(q, k, v, server.kc, server.vc, attn_metadata=md, k_scale=server.ks, v_scale=server.vs, **kw)
        assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(before, (server.kc, server.vc)))

    for quantized in (False, True):
        for dim in (144, 256):  # the cache takes them, the attention does not
            server = Server(4, 2, dim, 16, 20, torch.bfloat16, quantized)
            refused(server, *server.batch({0: 40}, 0), "head dim")
        server = Server(4, 2, 64, 8, 20, torch.bfloat16, quantized)
        refused(server, *server.batch({0: 40}, 0), "page size")
        server = Server(4, 2, 64, 16, 20, torch.bfloat16, quantized)
        md, q, k, v = server.batch({0: 40, 1: 3}, 0)
        refused(server, md, q[:, :3], k, v, "does not go with")
        refused(server, md, torch.cat([q, q], -1), k, v, "does not go with")
        refused(server, md, q.float(), k, v, "must be|bf16 or fp16")
        for name, value, match in (("block_table", md.block_table[:1], "block_table"),
                                   ("seq_lens", md.seq_lens.float(), "seq_lens"),
                                   ("query_start_loc", md.query_start_loc[:2], "cu_seqlens")):
            bad = SimpleNamespace(**vars(md))
            setattr(bad, name, value)
            refused(server, bad, q, k, v, match)
