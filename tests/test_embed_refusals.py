"""Argument checks of nm_embed_fwd / nm_embed_bwd. They are made on the host before any device call, so they run without a
GPU; the pointers below are never followed."""
import pytest

from test_capi_load import lib  # noqa: F401  (the built library)

A = 1 << 20      # an aligned address that is only compared and checked


def _refused(call, *args, text):
    import nmce
    with pytest.raises(nmce.NmError) as e:
        call(*args)
    assert e.value.status == 1 and text in str(e.value), str(e.value)


def test_forward_refusals(lib):  # noqa: F811
    good = dict(dtype=1, table=A, tokens=A, out=A, scale=1.0, T=4, D=16, V=10, stream=None)

    def refuse(text, **change):
        _refused(lib.nm_embed_fwd, *{**good, **change}.values(), text=text)

    refuse("storage 0 (f32) or 1 (bf16)", dtype=2)
    refuse("cannot be negative", T=-1)
    refuse("multiple of 8", D=12)
    refuse("multiple of 8", D=0)
    refuse("D <= 65536", D=65544)
    refuse("vocabulary size", V=0)
    refuse("required", table=None)
    refuse("required", tokens=None)
    refuse("required", out=None)
    refuse("16-byte aligned", table=A + 8)
    refuse("16-byte aligned", out=A + 2)
    refuse("4-byte aligned", tokens=A + 1)
    assert lib.nm_embed_fwd(1, None, None, None, 1.0, 0, 16, 10, None) == 0


def test_backward_refusals(lib):  # noqa: F811
    need = lib.nm_embed_bwd_workspace_bytes(4, 16, 10)
    assert need > 0 and need % 256 == 0
    good = dict(dtype=1, dy=A, tokens=A, dtable=A, scale=1.0, accumulate=0, T=4, D=16, V=10, ws=A, ws_bytes=need, stream=None)

    def refuse(text, **change):
        _refused(lib.nm_embed_bwd, *{**good, **change}.values(), text=text)

    refuse("storage 0 (f32) or 1 (bf16)", dtype=-1)
    refuse("cannot be negative", T=-4)
    refuse("multiple of 8", D=20)
    refuse("D <= 65536", D=131072)
    refuse("vocabulary size", V=-3)
    refuse("required", dy=None)
    refuse("required", tokens=None)
    refuse("dtable is required", dtable=None)
    refuse("dtable is required", dtable=A + 4)
    refuse("16-byte aligned", dy=A + 2)
    refuse("4-byte aligned", tokens=A + 2)
    refuse("256-byte aligned workspace", ws=None)
    refuse("256-byte aligned workspace", ws=A + 16)
    refuse("smaller than", ws_bytes=need - 1)
    assert lib.nm_embed_bwd(1, None, None, None, 1.0, 1, 0, 16, 10, None, 0, None) == 0


def test_workspace_size_is_bounded_by_a_section(lib):  # noqa: F811
    """A call longer than 131072 tokens runs in sections, so its scratch does not grow further."""
    one = lib.nm_embed_bwd_workspace_bytes(131072, 2048, 128256)
    assert lib.nm_embed_bwd_workspace_bytes(10 ** 7, 2048, 128256) == one
    assert lib.nm_embed_bwd_workspace_bytes(-1, 2048, 128256) == 0 and b"negative" in lib.nm_last_error()
