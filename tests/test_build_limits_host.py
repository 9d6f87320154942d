"""CPU-only: the build's limit on stack frames is that of the unit."""
from __future__ import annotations


def _log(nbytes):
    return "\n".join([
        "ptxas info    : Compiling entry function '_Z6kernelILi5EEvv' for 'sm_100a'",
        "ptxas info    : Function properties for _Z6kernelILi5EEvv",
        f"    {nbytes} bytes stack frame, 16 bytes spill stores, 16 bytes spill loads",
    ])


def test_march_units_keep_the_small_limit():
    from cta_b200 import build as B

    assert B.MAX_STACK_BYTES == 64
    assert B.stack_frames(_log(64)) == [] and B.stack_frames(_log(72)) == [("_Z6kernelILi5EEvv", 72)]
    assert set(B.UNIT_STACK_BYTES) <= set(B.SOURCES)
    assert all(name.startswith("attn_") and most <= 96 for name, most in B.UNIT_STACK_BYTES.items())


def test_a_unit_with_its_own_limit(monkeypatch, tmp_path):
    """The limit that compiling a unit applies."""
    from types import SimpleNamespace

    import pytest

    from cta_b200 import build as B

    monkeypatch.setattr(B, "BUILD_DIR", tmp_path)
    monkeypatch.setattr(B.subprocess, "run", lambda cmd, **kw: SimpleNamespace(returncode=0, stdout="", stderr=_log(88)))
    monkeypatch.setattr(B.os, "replace", lambda a, b: None)
    monkeypatch.setattr(B, "SOURCES", ["attn_simt.cu", "attn_tc_fwd_reach.cu"])
    B.build(force=True, out=tmp_path / "x.so")
    for name in ("bld_fwd_f32.cu", "stencil_bdl.cu", "attn_tc_fwd.cu", "kv_cache.cu"):
        monkeypatch.setattr(B, "SOURCES", [name])
        with pytest.raises(RuntimeError, match="above 64 bytes"):
            B.build(force=True, out=tmp_path / "x.so")
