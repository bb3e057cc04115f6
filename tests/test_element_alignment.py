"""Pointers of single elements (gates per token, statistics, [D] gradients, row vectors) that are not aligned to their element
size are refused on the host: on the device such an address is a fault. No GPU needed; the pointers are never followed."""
import pytest

from test_capi_load import lib  # noqa: F401  (the built library)

A = 1 << 20


def _refused(call, args, text):
    import nmce
    with pytest.raises(nmce.NmError) as e:
        call(*args.values())
    assert e.value.status == 1 and text in str(e.value), str(e.value)


@pytest.mark.parametrize("dtype,off", [(1, 1), (0, 1), (0, 2)])
def test_gated_tail(lib, dtype, off):  # noqa: F811
    fwd = dict(dtype=dtype, kind=1, branch=A, x_in=A, gate=A, res_scale=A, g_post=A, g_next=A, x_out=A, a_next=A, rstd_post=A,
               rstd_next=A, T=4, D=64, eps=1e-5, stream=None)
    bwd = dict(dtype=dtype, kind=1, dx_out=A, da_next=A, x_in=A, branch=A, gate=A, res_scale=A, g_post=A, g_next=A, rstd_post=A,
               rstd_next=A, dx_in=A, dbranch=A, dgate=A, dg_next=A, dg_post=A, dres_scale=A, T=4, D=64, ws=A,
               ws_bytes=lib.nm_gated_tail_workspace_bytes(4, 64), stream=None)
    for call, good, gates, words in ((lib.nm_gated_tail_fwd, fwd, ("gate",), ("rstd_post", "rstd_next")),
                                     (lib.nm_gated_tail_bwd, bwd, ("gate", "dgate"),
                                      ("rstd_post", "rstd_next", "dg_next", "dg_post", "dres_scale"))):
        for name in gates:
            _refused(call, {**good, name: A + off}, "aligned to its element size")
        for name in words:
            _refused(call, {**good, name: A + 2}, "4-byte aligned")


def test_no_rows_but_gradients(lib):  # noqa: F811
    _refused(lib.nm_gated_tail_bwd, dict(dtype=1, kind=0, **{str(i): None for i in range(13)}, dg_next=A + 2, dg_post=None,
                                         dres_scale=None, T=0, D=64, ws=A, ws_bytes=1 << 20, stream=None), "4-byte aligned")


def test_distillation(lib):  # noqa: F811
    good = dict(teacher_dtype=0, x=A, w=A, ids=A, logits=A, tlse=A, targets=A, weight=A, gs=A, tau=1.0, soft=0.5, hard=0.5,
                loss=A, kl=A, lse=A, partial=A, dx=A + 4096, acc=0, dw=A, fwd=0, T=4, D=64, V=100, K=3, chunk=128, ignore=0,
                ws=A, ws_bytes=1 << 30, stream=None)
    for name in ("tlse", "targets", "weight", "gs", "loss", "kl", "lse", "partial"):
        for off in (1, 2, 3):
            _refused(lib.nm_ce_distill, {**good, name: A + off}, "4-byte aligned")
