"""CPU-only checks of the attention and cache operators: refusals before any launch, and the
oracle against torch's own attention and casts."""
from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import attention_oracle as A


def test_oracle_matches_autograd():
    gen = torch.Generator().manual_seed(0)
    q, g = (torch.randn(37, 4, 16, generator=gen, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(37, 2, 16, generator=gen, dtype=torch.float64) for _ in range(2))
    see = torch.ones(37, 37, dtype=torch.bool).tril()
    see[:, 5] = False
    see[0] = False
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    kk, vv = (x.transpose(0, 1).repeat_interleave(2, 0) for x in leaves[1:])
    s = leaves[0].transpose(0, 1) @ kk.transpose(1, 2) * 0.25
    p = torch.softmax(s.masked_fill(~see, -1e300), -1) * see.any(-1, keepdim=True)
    out = (p @ vv).transpose(0, 1)
    want = torch.autograd.grad(out, leaves, g)
    got = A.gradients(q, k, v, g, see, 0.25)
    assert torch.allclose(A.attention(q, k, v, see, 0.25)[0], out, atol=1e-13)
    for x, y in zip(got, want):
        assert torch.allclose(x, y, atol=1e-12)


def test_oracle_quantises_as_torch_casts():
    x = torch.randn(500, 3, 64, generator=torch.Generator().manual_seed(1)) * 10
    codes, scale = A.quantise(x)
    m = x.abs().amax(-1)
    cast = (x.double() * (448.0 / m.double())[..., None]).to(torch.float32).to(torch.float8_e4m3fn)
    assert (codes == cast.double()).float().mean() > 0.9999  # the cast rounds twice
    assert torch.equal(scale, m.double() / 448)


def _qkv(shape=(2, 8), heads=4, kv=2, dim=16, dtype=torch.bfloat16, device="meta"):
    return (torch.empty(*shape, heads, dim, dtype=dtype, device=device),
            torch.empty(*shape, kv, dim, dtype=dtype, device=device),
            torch.empty(*shape, kv, dim, dtype=dtype, device=device))


def test_cpu_tensors_are_refused():
    from cta_b200 import ops
    from cta_b200.attention import prompt_attention

    q, k, v = _qkv(device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        prompt_attention(q, k, v)
    with pytest.raises(ValueError, match="CUDA"):
        ops.attention_mask(torch.ones(2, 8))
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_cache_write(q[0], q[0], k, v, torch.zeros(8))
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_cache_read(k, v, torch.zeros(8))
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(q[0], k, v, torch.zeros(1, 1), torch.zeros(1))


def _null():
    return ctypes.c_void_p(0)


def test_attention_arguments_fail_before_launch():
    from cta_b200 import _lib

    lib = _lib.load()

    def call(fn="cta_attention_forward", pointers=(16,) * 4 + (0,) * 9, batch=1, length=8, heads=4, kv=2, dim=64,
             dtype=1):
        args = _lib.ATTENTION_ARGS.pack(*pointers, *(64,) * 24, batch, length, heads, kv, dim, dtype, 0, 0, 0, 0.1, 0.0)
        return getattr(lib, fn)(args, None), lib.cta_last_error()

    for fn in ("cta_attention_forward", "cta_attention_backward"):
        assert lib.__getattr__(fn)(None, None) == _lib.CTA_EINVAL
        for kw, word in ((dict(dtype=7), b"dtype"), (dict(heads=5), b"heads"), (dict(kv=0), b"heads"),
                         (dict(dim=0), b"head dim"), (dict(dim=257), b"head dim"), (dict(batch=-1), b"shape"),
                         (dict(length=-1), b"shape"), (dict(pointers=(0,) * 13), b"null"),
                         (dict(pointers=(16,) * 13), b"key mask")):
            rc, msg = call(fn, **kw)
            assert rc == _lib.CTA_EINVAL and word in msg, (fn, kw, msg)
        assert call(fn, length=1 << 30)[0] == _lib.CTA_EUNSUPPORTED
        assert call(fn, batch=0)[0] == _lib.CTA_OK and call(fn, length=0)[0] == _lib.CTA_OK
    # the backward's own inputs; dk without dv
    assert call("cta_attention_backward")[0] == _lib.CTA_EINVAL
    rc, msg = call("cta_attention_backward", pointers=(16,) * 10 + (0,) * 3)
    assert rc == _lib.CTA_EINVAL and b"dk and dv" in msg
    assert lib.cta_attention_mask_words_per_row(1) == 8
    assert lib.cta_attention_mask_words_per_row(129) == 12
    assert lib.cta_attention_mask_words(None, 9, 0, 0, 1, 1, None, None) == _lib.CTA_EINVAL
    assert lib.cta_attention_mask_words(None, 0, 0, 0, 1, 1, None, None) == _lib.CTA_EINVAL


def test_cache_arguments_fail_before_launch():
    from cta_b200 import _lib

    lib = _lib.load()

    def call(fn, pointers=(16,) * 7, rows=(64, 64), cells=(1024, 64, 64), tokens=2, heads=2, dim=64, pages=4, page=16,
             dtype=1, quantized=0):
        args = _lib.KV_CACHE_ARGS.pack(*pointers, *rows, *rows, *cells, *cells, tokens, heads, dim, pages, page, dtype,
                                       quantized)
        return getattr(lib, fn)(args, None), lib.cta_last_error()

    for fn in ("cta_kv_cache_write", "cta_kv_cache_read"):
        assert getattr(lib, fn)(None, None) == _lib.CTA_EINVAL
        for kw, word in ((dict(dtype=0), b"bf16 or fp16"), (dict(dim=24), b"multiple of 16"), (dict(dim=272), b"head dim"),
                         (dict(heads=0), b"shape"), (dict(page=0), b"shape"), (dict(rows=(60, 64)), b"16 bytes"),
                         (dict(cells=(1024, 65, 64)), b"16 bytes"), (dict(cells=(1024, 72, 72), quantized=1), b"16 bytes"),
                         (dict(pointers=(8,) * 7), b"16 bytes"), (dict(pointers=(0,) * 7), b"null"),
                         (dict(pointers=(16, 16, 16, 16, 0, 16, 16), quantized=1), b"scales")):
            rc, msg = call(fn, **kw)
            assert rc == _lib.CTA_EINVAL and word in msg, (fn, kw, msg)
        assert call(fn, pages=1 << 28)[0] == _lib.CTA_EUNSUPPORTED
        assert call(fn, tokens=0)[0] == _lib.CTA_OK


def test_paged_arguments_fail_before_launch():
    from cta_b200 import _lib

    lib = _lib.load()

    def call(pointers=(16,) * 9, q=(256, 64), cells=(1024, 64, 64), rows=2, batch=2, heads=4, kv=2, dim=64, pages=4,
             page=16, width=3, max_rows=1, dtype=1, quantized=0, ws=16, ws_bytes=0):
        args = _lib.PAGED_ATTENTION_ARGS.pack(*pointers, *q, *q, *cells, *cells, width, rows, batch, heads, kv, dim,
                                              pages, page, width, max_rows, dtype, quantized, 0.1, 0.0)
        return lib.cta_paged_attention(args, ws, ws_bytes, None), lib.cta_last_error()

    assert lib.cta_paged_attention(None, None, 0, None) == _lib.CTA_EINVAL
    for kw, word in ((dict(dtype=0), b"bf16 or fp16"), (dict(heads=3), b"heads"), (dict(dim=40), b"head dim"),
                     (dict(dim=144), b"head dim"), (dict(page=8), b"page size"), (dict(page=40), b"page size"),
                     (dict(max_rows=0), b"max_rows"), (dict(pointers=(16,) * 8 + (0,), rows=3), b"one row"),
                     (dict(pointers=(16,) * 4 + (0,) * 5, quantized=1), b"scales"), (dict(pointers=(0,) * 9), b"null"),
                     (dict(q=(256, 60)), b"16 bytes"), (dict(cells=(1024, 60, 64)), b"16 bytes"),
                     (dict(pointers=(24,) * 9), b"16 bytes"), (dict(), b"workspace"), (dict(ws=None), b"workspace")):
        rc, msg = call(**kw)
        assert rc == _lib.CTA_EINVAL and word in msg, (kw, msg)
    assert call(width=1 << 28)[0] == _lib.CTA_EUNSUPPORTED
    assert call(rows=0)[0] == _lib.CTA_OK and call(batch=0)[0] == _lib.CTA_OK


def test_sizes_past_the_kernels_numbers_are_refused():
    """Index arithmetic of the kernels is 32-bit in places: sizes past it are refused before any launch."""
    from cta_b200 import _lib

    lib = _lib.load()

    def cache(tokens, heads, pages=4, page=16):
        args = _lib.KV_CACHE_ARGS.pack(*(16,) * 7, *(64,) * 4, *(64,) * 6, tokens, heads, 64, pages, page, 1, 1)
        return lib.cta_kv_cache_write(args, None)

    def paged(width=4, page=16, pages=4, rows=2, heads=4):
        args = _lib.PAGED_ATTENTION_ARGS.pack(*(16,) * 9, *(64,) * 4, *(64,) * 6, width, rows, rows, heads, 2, 64, pages,
                                              page, width, 1, 1, 0, 0.1, 0.0)
        return lib.cta_paged_attention(args, None, 0, None)

    # 2^27 groups of up to 32 lanes are 2^32 threads
    assert cache(1 << 27, 1) == _lib.CTA_EUNSUPPORTED
    assert cache(1 << 25, 13) == _lib.CTA_EUNSUPPORTED
    assert cache(2, 2, pages=1 << 40, page=1 << 40) == _lib.CTA_EUNSUPPORTED
    # a tile of 128 keys past the last one still has a number
    assert paged(width=(1 << 27) - 8) == _lib.CTA_EUNSUPPORTED
    assert paged(width=1 << 40, page=1 << 40) == _lib.CTA_EUNSUPPORTED
    assert paged(pages=1 << 40, page=1 << 40) == _lib.CTA_EUNSUPPORTED
    assert paged(rows=1 << 27, heads=16) == _lib.CTA_EUNSUPPORTED


def test_paged_workspace_size_of_refused_arguments():
    """Minus the status that the call itself returns, with its message."""
    from cta_b200 import _lib

    lib = _lib.load()

    def size(dim=64, page=16, width=3):
        args = _lib.PAGED_ATTENTION_ARGS.pack(*(16,) * 9, 256, 64, 256, 64, *(1024, 64, 64) * 2, width, 2, 2, 4, 2, dim, 4,
                                              page, width, 1, 1, 0, 0.1, 0.0)
        return lib.cta_paged_attention_workspace_bytes(args), lib.cta_last_error()

    assert size()[0] > 0
    for kw, status, word in ((dict(dim=144), _lib.CTA_EINVAL, b"head dim"), (dict(page=24), _lib.CTA_EINVAL, b"page size"),
                             (dict(width=1 << 28), _lib.CTA_EUNSUPPORTED, b"2^31")):
        rc, msg = size(**kw)
        assert rc == -status and word in msg, (kw, rc, msg)


def test_paged_kernel_goes_by_what_tma_addresses():
    """Chunks take the tensor-core kernel, which needs no workspace over a 16-bit cache; with strides that a tensor map
    cannot hold, or no pages, the split kernel, which does."""
    from cta_b200 import _lib

    lib = _lib.load()

    def size(q=(2048, 64), cells=(8192, 512, 64), pages=100, heads=32):
        args = _lib.PAGED_ATTENTION_ARGS.pack(*(16,) * 9, *q, *q, *cells, *cells, 64, 512, 1, heads, 8, 64, pages, 16, 64,
                                              512, 1, 0, 0.1, 0.0)
        return lib.cta_paged_attention_workspace_bytes(args)

    assert size() == 0
    assert size(pages=0) > 0
    assert size(pages=1, cells=(0, 512, 64)) == 0  # an axis of one entry has no stride
    for kw in (dict(q=(0, 64)), dict(q=(2048, -64)), dict(cells=(1 << 39, 512, 64)), dict(cells=(8192, 0, 64))):
        assert size(**kw) > 0, kw


def test_models_saved_whole_before_the_choice_of_attention():
    """A model object from before there was a choice has no such attribute and runs as it did."""
    from cta_b200 import transformers as T

    for cls, kw in ((T.PDETransformerLM, {}), (T.PDETransformerClassifier, dict(num_classes=3))):
        net = cls(vocab_size=11, embed_dim=16, num_heads=2, hidden_dim=16, num_layers=1, pde_steps=0, max_length=32, **kw)
        net.eval()
        ids, mask = torch.randint(0, 11, (2, 9)), torch.ones(2, 9, dtype=torch.long)
        want = net(ids, mask)
        net.__dict__.pop("attention", None)
        assert torch.equal(net(ids, mask), want)


def _plain_prompt_attention(q, k, v, *, causal=False, mask_words=None):
    """What the CPU has in place of the kernel; ``mask_words``: the mask itself."""
    s = torch.einsum("bihd,bjhd->bhij", q, k) * q.shape[-1] ** -0.5
    see = mask_words[:, None, None, :] != 0
    if causal:
        see = see & torch.ones(s.shape[-2:], dtype=torch.bool).tril()
    return torch.einsum("bhij,bjhd->bihd", torch.softmax(s.masked_fill(~see, -1e30), -1), v)


@pytest.fixture
def plain(monkeypatch):
    from cta_b200 import transformers as T

    monkeypatch.setattr(T, "prompt_attention", _plain_prompt_attention)
    monkeypatch.setattr(T.ops, "attention_mask", lambda mask: mask)
    return T


KW = dict(vocab_size=11, embed_dim=16, num_heads=2, hidden_dim=16, num_layers=2, pde_steps=0, max_length=32, dropout=0.0)


def test_fused_attention_runs_through_its_module(plain):
    """The attention of a layer is the call of its ``self_attn``: hooks there fire, and what they do counts."""
    torch.manual_seed(0)
    stock = plain.PDETransformerLM(**KW)
    torch.manual_seed(0)
    net = plain.PDETransformerLM(attention="fused", **KW)
    for (a, x), (b, y) in zip(stock.state_dict().items(), net.state_dict().items()):
        assert a == b and torch.equal(x, y)  # the same draws under the same names
    ids, mask = torch.randint(0, 11, (2, 9)), torch.ones(2, 9, dtype=torch.long)
    want = stock(ids, mask)
    assert (net(ids, mask) - want).abs().max() <= 1e-5 * want.abs().max()
    att = net.transformer_layers[0].self_attn
    assert isinstance(att, torch.nn.MultiheadAttention)
    seen = []
    handles = [att.register_forward_pre_hook(lambda m, args: seen.append("before")),
               att.register_forward_hook(lambda m, args, out: seen.append("after")),
               att.out_proj.register_forward_hook(lambda m, args, out: seen.append("out_proj"))]
    net(ids, mask)
    assert seen == ["before", "out_proj", "after"]
    for h in handles:
        h.remove()
    # a weight that a hook recomputes
    half = att.register_forward_pre_hook(lambda m, args: (m.in_proj_weight.data.mul_(0.5), None)[1])
    net(ids, mask)
    half.remove()
    with torch.no_grad():
        stock.transformer_layers[0].self_attn.in_proj_weight.mul_(0.5)
    want = stock(ids, mask)
    assert (net(ids, mask) - want).abs().max() <= 1e-5 * want.abs().max()


def test_gradients_reach_the_fused_attention(plain):
    torch.manual_seed(0)
    stock = plain.PDETransformerClassifier(num_classes=3, **KW)
    net = plain.PDETransformerClassifier(num_classes=3, attention="fused", **KW)
    net.load_state_dict(stock.state_dict())
    ids, mask = torch.randint(0, 11, (2, 9)), torch.ones(2, 9, dtype=torch.long)
    mask[1, 5:] = 0
    for x in (stock, net):
        x.train()
        x(ids, mask).square().sum().backward()
    for (n, a), b in zip(stock.named_parameters(), net.parameters()):
        assert (a.grad - b.grad).abs().max() <= 1e-4 * a.grad.abs().max() + 1e-7, n


def test_fused_models_are_saved_and_copied_whole(plain, tmp_path):
    """Copies and pickles keep the fused module; one that was saved with the stock module in its place gets it."""
    import copy

    torch.manual_seed(0)
    net = plain.PDETransformerLM(attention="fused", **KW)
    ids, mask = torch.randint(0, 11, (2, 9)), torch.ones(2, 9, dtype=torch.long)
    want = net(ids, mask)
    old = copy.deepcopy(net)
    for layer in old.transformer_layers:
        layer.self_attn.__class__ = torch.nn.MultiheadAttention
    for i, x in enumerate((net, old)):
        torch.save(x, tmp_path / f"{i}.pt")
        back = torch.load(tmp_path / f"{i}.pt", weights_only=False)
        assert torch.equal(back(ids, mask), want)
    assert torch.equal(copy.deepcopy(net)(ids, mask), want)


def test_fused_models_refuse_a_mask_of_another_length(plain):
    for cls, kw in ((plain.PDETransformerLM, {}), (plain.PDETransformerClassifier, dict(num_classes=3))):
        net = cls(attention="fused", **KW, **kw)
        ids = torch.randint(0, 11, (2, 9))
        for shape in ((2, 8), (2, 10), (1, 9), (2, 9, 1)):
            with pytest.raises(ValueError, match="attention_mask"):
                net(ids, torch.ones(*shape, dtype=torch.long))
