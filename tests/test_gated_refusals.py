"""Argument checks of the gated sandwich tail, made on the host before any device call (no GPU needed; the pointers are never
followed)."""
import pytest

from test_capi_load import lib  # noqa: F401  (the built library)

A = 1 << 20


def _refused(call, *args, text):
    import nmce
    with pytest.raises(nmce.NmError) as e:
        call(*args)
    assert e.value.status == 1 and text in str(e.value), str(e.value)


def test_forward_refusals(lib):  # noqa: F811
    good = dict(dtype=1, kind=2, branch=A, x_in=A, gate=A, res_scale=A, g_post=A, g_next=A, x_out=A, a_next=A, rstd_post=A,
                rstd_next=A, T=4, D=64, eps=1e-5, stream=None)

    def refuse(text, **change):
        _refused(lib.nm_gated_tail_fwd, *{**good, **change}.values(), text=text)

    refuse("storage 0 (f32) or 1 (bf16)", dtype=3)
    refuse("gate_kind 0 (none)", kind=3)
    refuse("gate_kind 0 (none)", kind=-1)
    refuse("goes with gate_kind", gate=None)
    refuse("goes with gate_kind", kind=0)
    refuse("cannot be negative", T=-1)
    refuse("multiple of 8", D=12)
    refuse("D <= 8192", D=8200)
    refuse("D <= 8192 (bf16 storage) or 4096 (f32)", dtype=0, D=4104)
    refuse("required", branch=None)
    refuse("required", x_in=None)
    refuse("required", x_out=None)
    refuse("a_next needs g_next", g_next=None)
    for name in ("branch", "x_in", "res_scale", "g_post", "g_next", "x_out", "a_next"):
        refuse("16-byte aligned", **{name: A + 8})
    refuse("gate per element must be 16-byte aligned", gate=A + 2)


def test_backward_refusals(lib):  # noqa: F811
    need = lib.nm_gated_tail_workspace_bytes(4, 64)
    assert need >= 3 * 4 * 64 * 4
    good = dict(dtype=1, kind=1, dx_out=A, da_next=A, x_in=A, branch=A, gate=A + 2, res_scale=A, g_post=A, g_next=A,
                rstd_post=A, rstd_next=A, dx_in=A, dbranch=A, dgate=A + 2, dg_next=A, dg_post=A, dres_scale=A, T=4, D=64, ws=A,
                ws_bytes=need, stream=None)

    def refuse(text, **change):
        _refused(lib.nm_gated_tail_bwd, *{**good, **change}.values(), text=text)

    refuse("storage 0 (f32) or 1 (bf16)", dtype=2)
    refuse("gate_kind 0 (none)", kind=7)
    refuse("goes with gate_kind", gate=None)
    refuse("dgate goes with a gate", dgate=None)
    refuse("dgate goes with a gate", kind=0, gate=None)
    refuse("multiple of 8", D=4)
    refuse("cannot be negative", T=-2)
    for name in ("da_next", "x_in", "branch", "g_next", "rstd_next"):
        refuse("are required", **{name: None})
    refuse("needs rstd_post", rstd_post=None)
    refuse("dx_in and dbranch", dx_in=None)
    refuse("dx_in and dbranch", dbranch=None)
    refuse("dg_post without g_post", g_post=None)
    refuse("dres_scale without res_scale", res_scale=None)
    for name in ("dx_out", "da_next", "x_in", "branch", "res_scale", "g_post", "g_next", "dx_in", "dbranch"):
        refuse("16-byte aligned", **{name: A + 4})
    refuse("per element must be 16-byte aligned", kind=2)
    refuse("16-byte aligned workspace", ws=None)
    refuse("smaller than", ws_bytes=need - 1)
    assert lib.nm_gated_tail_workspace_bytes(4, 12) == 0 and b"multiple of 8" in lib.nm_last_error()
