"""Serving steps with rotated keys, a window over the cache and a shared prefix, through CtaPostAttnMixer.attend, against
the definition in 64 bits."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from oracle import attention_oracle as A
from test_gpu_attention_models import Server as Plain
from test_gpu_rotary import _turned

pytestmark = pytest.mark.gpu


class Server(Plain):
    """Keeps the rotated keys and what each row may see."""

    def __init__(self, *args, window=None, sinks=0, rotary=0, interleaved=False):
        super().__init__(*args)
        from cta_b200 import ops

        self.window, self.sinks, self.interleaved = window, sinks, interleaved
        self.table = ops.rotary_table(4096, rotary) if rotary else None

    def positions(self, new, padding=0):
        out = []
        for s, n in new.items():
            total = self.k[s].shape[0]
            out += range(total - n, total)
        return torch.tensor(out + [0] * padding).cuda()

    def check(self, out, q, new):
        at = 0
        for s, n in new.items():
            k, v = self.k[s], self.v[s]
            total = k.shape[0]
            rows = q[at : at + n]
            j = torch.arange(total, device="cuda")
            pages, slot = torch.tensor(self.pages[s], device="cuda")[j // self.page], j % self.page
            if self.table is not None:
                # q as it is rounded after the rotation; k as the cache holds it (rounding it has its own tests)
                rows = _turned(rows, self.table, torch.arange(total - n, total, device="cuda"), self.interleaved)[0].to(self.dtype)
            if self.ks is not None:
                k, v = (c.view(torch.uint8)[pages, slot].view(torch.float8_e4m3fn).double() * x[pages, :, slot].double()[..., None]
                        for c, x in ((self.kc, self.ks), (self.vc, self.vs)))
            elif self.table is not None:
                k = self.kc[pages, slot]
            i = torch.arange(total - n, total, device="cuda")[:, None]
            see = j[None, :] <= i
            if self.window is not None:
                see &= (j[None, :] > i - self.window) | (j[None, :] < self.sinks)
            want, _ = A.attention(rows, k, v, see, self.dim**-0.5)
            # q may round the other way where its fp32 value lies next to the middle of two numbers: one step of q, which
            # enters the scores like an error of k
            kv_error = (2.0**-20 if self.ks is not None else 0.0)
            tol = A.bounds(rows, k, v, see, self.dim**-0.5, self.dtype, kv_error=kv_error)
            if self.table is not None:
                near = A.bounds(rows, k, v, see, self.dim**-0.5, self.dtype, kv_error=kv_error + torch.finfo(self.dtype).eps)
                # few elements are that close; all of them being so would be the bound `near`
                off = (out[at : at + n].double() - want).abs()
                assert (off <= near).all()
                assert (off > tol).float().mean() < 1e-3
            else:
                assert ((out[at : at + n].double() - want).abs() <= tol).all(), (s, n, total)
            at += n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,rotary,interleaved", [(8, 2, 128, 128, False), (4, 4, 64, 32, True)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 4)])
def test_prompts_chunks_and_decode(window, sinks, heads, kv_heads, dim, rotary, interleaved, quantized, dtype):
    from cta_b200.serving_vllm import CtaConfig, CtaPostAttnMixer

    mixer = CtaPostAttnMixer(CtaConfig(enabled=False))  # the attention alone
    server = Server(heads, kv_heads, dim, 16, 200, dtype, quantized, window=window, sinks=sinks, rotary=rotary,
                    interleaved=interleaved)
    steps = [{0: 130, 1: 17}, {2: 300}, {0: 1, 1: 1, 2: 1}, {0: 1, 3: 64, 2: 1}, {1: 200, 3: 5}, {0: 1, 1: 1, 2: 1, 3: 1}]
    for i, new in enumerate(steps):
        md, q, k, v = server.batch(new, i, padding=3)
        before = q.clone()
        out = mixer.attend(q, k, v, server.kc, server.vc, attn_metadata=md, k_scale=server.ks, v_scale=server.vs,
                           positions=server.positions(new, 3), cos_sin=server.table, interleaved=interleaved, window=window,
                           sinks=sinks)
        assert torch.equal(q, before)
        server.check(out.view(-1, heads, dim), q, new)


@pytest.mark.parametrize("quantized", [False, True])
def test_shared_prefix(quantized):
    """A prompt is prefilled once, other sequences go on from its pages."""
    from cta_b200 import _lib
    from cta_b200.serving_vllm import CtaConfig, CtaPostAttnMixer

    mixer = CtaPostAttnMixer(CtaConfig(enabled=False))
    server = Server(8, 2, 128, 16, 300, torch.bfloat16, quantized)
    kw = dict(k_scale=server.ks, v_scale=server.vs)
    md, q, k, v = server.batch({0: 640}, 0)
    server.check(mixer.attend(q, k, v, server.kc, server.vc, attn_metadata=md, **kw).view(-1, 8, 128), q, {0: 640})
    for s in range(1, 40):
        server.pages[s], server.k[s], server.v[s] = list(server.pages[0]), server.k[0], server.v[0]
    for step in range(4):
        new = {s: (1 if step else 1 + s % 5) for s in range(40)}
        md, q, k, v = server.batch(new, step + 1, padding=2)
        _lib.set_tuning(6, int(step < 3))
        out = mixer.attend(q, k, v, server.kc, server.vc, attn_metadata=md, shared_prefix=640, **kw)
        server.check(out.view(-1, 8, 128), q, new)


def test_steps_with_the_mixer_are_their_parts():
    from cta_b200 import ops
    from cta_b200.serving_vllm import CtaConfig, CtaPostAttnMixer

    mixer = CtaPostAttnMixer(CtaConfig(steps=4, alpha=0.1))
    server = Server(8, 2, 64, 16, 60, torch.bfloat16, True, rotary=64)
    md, q, k, v = server.batch({0: 100, 1: 33, 2: 1}, 1)
    positions = server.positions({0: 100, 1: 33, 2: 1})
    out = mixer.attend(q, k, v, server.kc, server.vc, attn_metadata=md, k_scale=server.ks, v_scale=server.vs,
                       positions=positions, cos_sin=server.table, window=30, sinks=2)
    turned = ops.rotary_cache_write(q, k, v, server.kc, server.vc, md.slot_mapping, positions, server.table, k_scale=server.ks,
                                    v_scale=server.vs)
    a = ops.paged_attention(turned, server.kc, server.vc, md.block_table, md.seq_lens, cu_seqlens=md.query_start_loc,
                            max_rows=100, k_scale=server.ks, v_scale=server.vs, window=30, sinks=2).view(q.shape[0], -1)
    assert torch.equal(out, mixer(a, attn_metadata=md))


def test_attend_refuses_before_it_writes():
    from cta_b200 import ops
    from cta_b200.serving_vllm import CtaConfig, CtaPostAttnMixer

    mixer = CtaPostAttnMixer(CtaConfig(enabled=False))
    server = Server(8, 2, 64, 16, 60, torch.bfloat16, False, rotary=64)
    md, q, k, v = server.batch({0: 20, 1: 3}, 1)
    p = server.positions({0: 20, 1: 3})
    kept = server.kc.clone()
    good = dict(positions=p, cos_sin=server.table)
    for bad, match in ((dict(positions=p), "cos_sin"), (dict(cos_sin=server.table), "positions"),
                       (dict(good, positions=p[:5]), "positions"), (dict(good, window=0), "window"),
                       (dict(good, sinks=3), "window"), (dict(good, shared_prefix=-2), "shared_prefix"),
                       (dict(good, cos_sin=server.table.double()), "cos_sin"),
                       (dict(good, cos_sin=ops.rotary_table(64, 24)), "rotary_dim"),
                       (dict(good, cos_sin=ops.rotary_table(64, 80)), "rotary_dim")):
        with pytest.raises(ValueError, match=match):
            mixer.attend(q, k, v, server.kc, server.vc, attn_metadata=md, **bad)
    torch.cuda.synchronize()
    assert torch.equal(kept.view(torch.int16), server.kc.view(torch.int16))


def test_decode_step_captured():
    """Rotation, write and windowed attention in one graph, replayed as the sequences grow."""
    from cta_b200.serving_vllm import CtaConfig, CtaPostAttnMixer

    mixer = CtaPostAttnMixer(CtaConfig(enabled=False))
    server = Server(8, 2, 64, 16, 60, torch.bfloat16, False, window=40, sinks=3, rotary=64)
    first = {0: 60, 1: 35, 2: 90}
    md, q, k, v = server.batch(first, 0)
    mixer.attend(q, k, v, server.kc, server.vc, attn_metadata=md, positions=server.positions(first), cos_sin=server.table,
                 window=40, sinks=3)
    new = {0: 1, 1: 1, 2: 1}
    held = None
    for step in range(1, 5):
        md, q, k, v = server.batch(new, step)
        fresh = dict(q=q, k=k, v=v, positions=server.positions(new), slots=md.slot_mapping, lens=md.seq_lens,
                     starts=md.query_start_loc)
        table = torch.zeros(3, 16, dtype=torch.int32, device="cuda")
        table[:, : md.block_table.shape[1]] = md.block_table
        fresh["table"] = table
        if held is None:
            held = {n: x.clone() for n, x in fresh.items()}
            meta = SimpleNamespace(slot_mapping=held["slots"], block_table=held["table"], seq_lens=held["lens"],
                                   query_start_loc=held["starts"], max_query_len=1)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = mixer.attend(held["q"], held["k"], held["v"], server.kc, server.vc, attn_metadata=meta,
                                   positions=held["positions"], cos_sin=server.table, window=40, sinks=3)
        for n, x in fresh.items():
            held[n].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        server.check(out.view(-1, 8, 64), q, new)
