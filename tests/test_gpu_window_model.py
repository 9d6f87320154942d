"""Gradients of the language model under an attention window against the same model with attention by its definition:
padding shorter and longer than the window, on either side."""
from __future__ import annotations

import pytest
import torch

from test_gpu_window import _reach

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error():
    from cta_b200 import _lib

    yield
    assert _lib.device_error() == 0


def _definition(mask):
    """prompt_attention from products, exponentials and sums in 64 bits; a row that sees nothing is zero."""

    def attend(q, k, v, *, causal, mask_words, window=None, sinks=0):
        assert causal
        length = q.shape[1]
        out = []
        for b in range(q.shape[0]):
            see = _reach(length, length, window, sinks, mask[b].bool())
            s = torch.einsum("ihd,jhd->hij", q[b].double(), k[b].double()) * q.shape[-1] ** -0.5
            s = s.masked_fill(~see, float("-inf"))
            some = see.any(-1)[None, :, None]
            # exp of a row without keys: of zeros, then times zero, so that no gradient is NaN
            s = torch.where(some, s, torch.zeros_like(s))
            p = torch.exp(s - s.amax(-1, keepdim=True).detach()) * some
            p = p / torch.where(some, p.sum(-1, keepdim=True), torch.ones_like(p[..., :1]))
            out.append(torch.einsum("hij,jhd->ihd", p, v[b].double()))
        return torch.stack(out).to(q.dtype)

    return attend


@pytest.mark.parametrize("window,sinks", [(16, 0), (16, 3), (5, 0), (40, 4)])
@pytest.mark.parametrize("length", [37, 200])
@pytest.mark.parametrize("padding", ["few", "right", "left", "none"])
def test_gradients(padding, length, window, sinks, monkeypatch):
    from cta_b200 import transformers as T

    torch.manual_seed(0)
    kw = dict(vocab_size=50, embed_dim=64, num_heads=4, hidden_dim=96, num_layers=2, pde_steps=2, max_length=256, dropout=0.0)
    model = T.PDETransformerLM(attention="fused", attention_window=window, attention_sinks=sinks, **kw).cuda()
    ids = torch.randint(0, 50, (3, length), device="cuda")
    mask = torch.ones(3, length, dtype=torch.long, device="cuda")
    long = length * 3 // 4 if length == 37 else 100  # longer than every window here at length 200
    if padding == "few":
        mask[1, length - 9:] = 0
    elif padding == "right":
        mask[1, length - long:] = 0
    elif padding == "left":
        mask[1, :long] = 0
        mask[2, :1] = 0
    if padding == "right" and sinks == 0:  # windows that have left the valid tokens
        see = _reach(length, length, window, sinks, mask[1].bool())
        assert bool((~see.any(1)).any()) == (long >= window)
    weight = torch.randn(3, length, 50, device="cuda")
    results = []
    for attend in (None, _definition(mask)):
        if attend is not None:
            monkeypatch.setattr(T, "prompt_attention", attend)
        model.zero_grad()
        logits = model(ids, mask)
        # the padding's rows count too: zeros from their attention are a value like others
        (logits * weight).sum().backward()
        results.append((logits.detach(), {n: p.grad.clone() for n, p in model.named_parameters()}))
    (got, grads), (want, wants) = results
    assert torch.isfinite(want).all() and all(torch.isfinite(x).all() for x in wants.values())
    assert ((got - want).abs() <= 1e-5 * want.abs().max() + 1e-6).all()
    for name, x in wants.items():
        # sums of fp32 products over up to 3 x 200 tokens and two layers: 1e-4 of the largest entry
        assert ((grads[name] - x).abs() <= 1e-4 * x.abs().max() + 1e-6).all(), name
    assert any(name.endswith("in_proj_weight") and bool((x != 0).any()) for name, x in wants.items())
