"""CPU-only checks of windows, shared prefixes and the rotated cache write: refusals before any launch, workspace sizes,
the table of angles, the models' arguments."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch


def _prompt(batch=2, length=64, heads=4, kv=2, dim=64, dtype=1, causal=1, pointers=(16,) * 11 + (0, 0)):
    from cta_b200 import _lib

    return _lib.ATTENTION_ARGS.pack(*pointers, *(64,) * 24, batch, length, heads, kv, dim, dtype, causal, 0, 1, 0.1, 0.0)


def _message():
    from cta_b200 import _lib

    return _lib.load().cta_last_error().decode()


@pytest.mark.parametrize("window,sinks,causal,match", [(-1, 0, 1, "negative"), (8, -1, 1, "negative"), (0, 3, 1, "window"),
                                                      (8, 0, 0, "causal")])
def test_windows_of_prompts_are_refused(window, sinks, causal, match):
    from cta_b200 import _lib

    lib = _lib.load()
    args = _prompt(causal=causal)
    assert lib.cta_window_attention_forward(args, window, sinks, None) == _lib.CTA_EINVAL and match in _message()
    assert lib.cta_window_attention_backward(args, window, sinks, None, 0, None) == _lib.CTA_EINVAL and match in _message()
    assert lib.cta_window_attention_workspace_bytes(args, window, sinks) == -_lib.CTA_EINVAL


def test_window_calls_refuse_what_the_plain_ones_do():
    from cta_b200 import _lib

    lib = _lib.load()
    for args, match in ((None, "null"), (_prompt(dim=300), "dim"), (_prompt(heads=3), "shape"), (_prompt(dtype=7), "dtype"),
                        (_prompt(pointers=(0,) * 13), "null")):
        assert lib.cta_window_attention_forward(args, 8, 2, None) == _lib.CTA_EINVAL and match in _message()
        assert lib.cta_window_attention_workspace_bytes(args, 8, 2) == -_lib.CTA_EINVAL
    # nothing to do is no error
    for args in (_prompt(batch=0), _prompt(length=0)):
        assert lib.cta_window_attention_forward(args, 8, 2, None) == _lib.CTA_OK
        assert lib.cta_window_attention_backward(args, 8, 2, None, 0, None) == _lib.CTA_OK
        assert lib.cta_window_attention_workspace_bytes(args, 8, 2) == 0


def test_backward_workspace():
    """For the far rows of first keys; nothing where there are none."""
    from cta_b200 import _lib

    lib = _lib.load()

    def size(window, sinks, **kw):
        return lib.cta_window_attention_workspace_bytes(_prompt(batch=1, **kw), window, sinks)

    assert size(100, 4, length=5000) > 0
    assert size(100, 0, length=5000) == 0 and size(0, 0, length=5000) == 0
    assert size(100, 4, length=200) == 0 and size(4996, 4, length=5000) == 0
    assert size(100, 4, length=5000, dtype=0) > 0 and size(100, 4, length=5000, dim=20) > 0
    no_dk = (16,) * 9 + (0, 0, 0, 0)
    assert size(100, 4, length=5000, pointers=no_dk) == 0
    # many first keys of long rows: bounded, beyond one part for each
    assert size(64, 10**6, length=1 << 21) < 2 * (10**6 + 128) * 2 * 2 * 64 * 4 + (1 << 29)
    args = _prompt(batch=1, length=5000)
    need = size(100, 4, length=5000)
    for ws, nbytes in ((None, need), (ctypes.c_void_p(16), need - 1)):
        assert lib.cta_window_attention_backward(args, 100, 4, ws, nbytes, None) == _lib.CTA_EINVAL and "workspace" in _message()
    assert lib.cta_window_attention_backward(args, 100, 4, ctypes.c_void_p(8), need, None) == _lib.CTA_EINVAL


def _paged(rows=4, heads=4, kv=2, dim=64, pages=64, page=16, width=8, batch=4, dtype=1, quantized=0, cu=0, pointers=(16,) * 8):
    from cta_b200 import _lib

    cells = (page * kv * dim, kv * dim, dim)
    return _lib.PAGED_ATTENTION_ARGS.pack(*pointers, cu, heads * dim, dim, heads * dim, dim, *cells, *cells, width, rows, batch,
                                          heads, kv, dim, pages, page, width, 1, dtype, quantized, 0.1, 0.0)


def test_paged_windows_and_prefixes_are_refused():
    from cta_b200 import _lib

    lib = _lib.load()
    good = _paged()
    for window, sinks in ((-1, 0), (4, -2), (0, 1)):
        assert lib.cta_window_paged_attention(good, window, sinks, None, 0, None) == _lib.CTA_EINVAL
        assert lib.cta_window_paged_attention_workspace_bytes(good, window, sinks) == -_lib.CTA_EINVAL
    assert lib.cta_prefix_paged_attention(good, -1, None, 0, None) == _lib.CTA_EINVAL and "shared_prefix" in _message()
    assert lib.cta_prefix_paged_attention_workspace_bytes(good, -1) == -_lib.CTA_EINVAL
    for args in (None, _paged(dim=24), _paged(page=8), _paged(heads=3), _paged(dtype=0), _paged(rows=3)):
        assert lib.cta_window_paged_attention(args, 8, 2, None, 0, None) == _lib.CTA_EINVAL
        assert lib.cta_prefix_paged_attention(args, 64, None, 0, None) == _lib.CTA_EINVAL
    # key numbers past a window's groups
    wide = _paged(width=1 << 26, pages=1 << 10)
    assert lib.cta_window_paged_attention_workspace_bytes(wide, 8, 2) == -_lib.CTA_EUNSUPPORTED
    assert lib.cta_window_paged_attention_workspace_bytes(wide, 0, 0) > 0
    # a prefix that cannot be used is none
    assert (lib.cta_prefix_paged_attention_workspace_bytes(wide, 1 << 20)
            == lib.cta_window_paged_attention_workspace_bytes(wide, 0, 0))
    # no workspace, no pointers
    need = lib.cta_window_paged_attention_workspace_bytes(good, 8, 2)
    assert need > 0
    assert lib.cta_window_paged_attention(good, 8, 2, None, need, None) == _lib.CTA_EINVAL and "workspace" in _message()
    assert lib.cta_window_paged_attention(good, 8, 2, ctypes.c_void_p(16), need - 1, None) == _lib.CTA_EINVAL
    none = _paged(pointers=(0,) * 8)
    assert lib.cta_window_paged_attention(none, 8, 2, ctypes.c_void_p(16), need, None) == _lib.CTA_EINVAL and "null" in _message()
    # no rows
    assert lib.cta_window_paged_attention(_paged(rows=0, batch=0), 8, 2, None, 0, None) == _lib.CTA_OK
    assert lib.cta_prefix_paged_attention(_paged(rows=0, batch=0), 64, None, 0, None) == _lib.CTA_OK


def test_prefix_workspace():
    from cta_b200 import _lib

    lib = _lib.load()
    big = dict(rows=64, batch=64, heads=32, kv=8, dim=128, width=600, pages=4096)
    plain = lib.cta_window_paged_attention_workspace_bytes(_paged(**big), 0, 0)

    def size(prefix, **kw):
        return lib.cta_prefix_paged_attention_workspace_bytes(_paged(**{**big, **kw}), prefix)

    assert size(0) == plain and size(15) == plain  # not one page
    assert size(8192) > plain  # the parts' sums
    assert size(10**15) > plain  # as far as the table goes
    assert size(8192, quantized=1) > size(8192)  # and the prefix's pages, expanded
    few = dict(rows=2, batch=2)
    assert size(256, **few) == lib.cta_window_paged_attention_workspace_bytes(_paged(**{**big, **few}), 0, 0)
    before = _lib.set_tuning(6, 1)
    try:
        assert before == 0 and size(256, **few) > 0
        assert size(256, **few) != lib.cta_window_paged_attention_workspace_bytes(_paged(**{**big, **few}), 0, 0)
    finally:
        assert _lib.set_tuning(6, before) == 1


def _rotary(tokens=4, heads=4, kv=2, dim=64, rotary=64, end=100, table_dtype=0, dtype=1, pointers=(16, 16, 16, 16), q=(256, 64), table=64,
            interleaved=0):
    from cta_b200 import _lib

    cells = (16 * kv * dim, kv * dim, dim)
    cache = _lib.KV_CACHE_ARGS.pack(*(16,) * 7, kv * dim, dim, kv * dim, dim, *cells, *cells, tokens, kv, dim, 8, 16, dtype, 0)
    return cache, _lib.ROTARY_ARGS.pack(*pointers, *q, *q, table, heads, rotary, end, table_dtype, interleaved)


@pytest.mark.parametrize("kw,match", [
    (dict(heads=0), "heads"), (dict(heads=1 << 20), "heads"), (dict(rotary=8), "rotary_dim"), (dict(rotary=0), "rotary_dim"),
    (dict(rotary=24), "rotary_dim"), (dict(rotary=80), "rotary_dim"), (dict(rotary=-16), "rotary_dim"),
    (dict(table_dtype=2), "table"), (dict(table_dtype=9), "table"), (dict(end=-1), "table"), (dict(q=(257, 64)), "16 bytes"),
    (dict(table=66), "16 bytes"), (dict(pointers=(0, 16, 16, 16)), "null"), (dict(pointers=(16, 0, 16, 16)), "null"),
    (dict(pointers=(16, 16, 0, 16)), "null"), (dict(pointers=(16, 16, 16, 0)), "null"), (dict(pointers=(8, 16, 16, 16)), "16 bytes"),
    (dict(pointers=(16, 8, 16, 16)), "16 bytes"), (dict(pointers=(16, 16, 16, 8)), "16 bytes"), (dict(dim=24, rotary=16), "dim"),
    (dict(dtype=0), "bf16")])
def test_rotary_arguments_fail_before_launch(kw, match):
    from cta_b200 import _lib

    assert _lib.load().cta_rotary_cache_write(*_rotary(**kw), None) == _lib.CTA_EINVAL
    assert match in _message()


def test_rotary_sizes_and_nothing_to_do():
    from cta_b200 import _lib

    lib = _lib.load()
    assert lib.cta_rotary_cache_write(*_rotary(tokens=0), None) == _lib.CTA_OK
    assert lib.cta_rotary_cache_write(_rotary()[0], None, None) == _lib.CTA_EINVAL
    assert lib.cta_rotary_cache_write(None, _rotary()[1], None) == _lib.CTA_EINVAL
    assert lib.cta_rotary_cache_write(*_rotary(tokens=1 << 25, heads=64), None) == _lib.CTA_EUNSUPPORTED


def test_cpu_tensors_and_wrong_shapes_are_refused():
    from cta_b200 import ops
    from cta_b200.attention import prompt_attention

    def t(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype)

    q, k = t(8, 4, 64), t(8, 2, 64)
    cache = t(4, 16, 2, 64)
    ints = torch.zeros(8, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rotary_cache_write(q, k, k, cache, cache, ints, ints, t(10, 64, dtype=torch.float32))
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(q, cache, cache, ints[:, None].int(), ints.int(), window=4)
    with pytest.raises(ValueError, match="CUDA"):
        prompt_attention(q[None], k[None], k[None], causal=True, window=4)
    for kw, match in ((dict(causal=False, window=4), "causal"), (dict(causal=True, window=0), "window"),
                      (dict(causal=True, window=-3), "window"), (dict(causal=True, sinks=2), "window"),
                      (dict(causal=True, window=4, sinks=-1), "sinks")):
        with pytest.raises(ValueError, match=match):
            prompt_attention(q[None], k[None], k[None], **kw)
        if kw["causal"]:
            with pytest.raises(ValueError, match=match):
                ops.paged_attention(q, cache, cache, ints[:, None].int(), ints.int(), **{n: x for n, x in kw.items() if n != "causal"})
    with pytest.raises(TypeError):
        prompt_attention(q[None], k[None], k[None], causal=True, window=2.5)


def test_table_of_angles():
    from cta_b200 import ops

    table = ops.rotary_table(200, 32, device="cpu")
    assert table.shape == (200, 32) and table.dtype == torch.float32
    for p in (0, 1, 77, 199):
        for i in range(16):
            a = p / 10000.0 ** (2 * i / 32)
            assert abs(table[p, i].item() - math.cos(a)) <= 2.0**-24
            assert abs(table[p, 16 + i].item() - math.sin(a)) <= 2.0**-24
    assert ops.rotary_table(3, 16, base=500.0, dtype=torch.bfloat16, device="cpu").dtype == torch.bfloat16
    assert ops.rotary_table(0, 16, device="cpu").shape == (0, 16)
    for bad in ((-1, 16), (4, 15), (4, 0)):
        with pytest.raises(ValueError):
            ops.rotary_table(*bad, device="cpu")


def test_models_take_a_window_with_the_fused_attention_only():
    from cta_b200 import transformers as T

    kw = dict(vocab_size=5, embed_dim=8, num_heads=2, hidden_dim=8, num_layers=2)
    model = T.PDETransformerLM(attention="fused", attention_window=7, attention_sinks=2, **kw)
    assert all(layer.self_attn.reach == {"window": 7, "sinks": 2} for layer in model.transformer_layers)
    assert all(layer.self_attn.reach == {} for layer in T.PDETransformerLM(attention="fused", **kw).transformer_layers)
    for bad, match in ((dict(attention_window=7), "fused"), (dict(attention="fused", attention_sinks=1), "window"),
                       (dict(attention="fused", attention_window=0), "window")):
        with pytest.raises(ValueError, match=match):
            T.PDETransformerLM(**bad, **kw)
    # the parameters are those of a model without it
    again = T.PDETransformerLM(**kw)
    again.load_state_dict(model.state_dict())


def test_window_reaches_the_fused_attention(monkeypatch):
    """Each layer's call carries the model's window; a model without one calls as before."""
    from cta_b200 import transformers as T

    calls = []

    def plain(q, k, v, **kw):
        calls.append({n: x for n, x in kw.items() if n in ("window", "sinks")})
        return v

    monkeypatch.setattr(T, "prompt_attention", plain)
    monkeypatch.setattr(T.ops, "attention_mask", lambda m: m)
    monkeypatch.setattr(T, "_refine", lambda x, *a: x)
    kw = dict(vocab_size=5, embed_dim=8, num_heads=2, hidden_dim=8, num_layers=2, dropout=0.0)
    ids, mask = torch.zeros(1, 4, dtype=torch.long), torch.ones(1, 4)
    T.PDETransformerLM(attention="fused", attention_window=3, attention_sinks=1, **kw)(ids, mask)
    assert calls == [{"window": 3, "sinks": 1}] * 2
    calls.clear()
    T.PDETransformerLM(attention="fused", **kw)(ids, mask)
    assert calls == [{}] * 2
