"""Argument checks of the distillation head, made on the host before any device call (no GPU needed; the pointers are never
followed)."""
import pytest

from test_capi_load import lib  # noqa: F401  (the built library)

A = 1 << 20


def test_refusals(lib):  # noqa: F811
    import nmce
    need = lib.nm_ce_distill_workspace_bytes(4, 64, 100, 3, 128, 0)
    assert need > 0 and need % 256 == 0
    good = dict(teacher_dtype=0, x=A, w=A, ids=A, logits=A, tlse=None, targets=A, weight=A, gs=A, tau=1.0, soft=0.5, hard=0.5,
                loss=A, kl=None, lse=None, partial=None, dx=A + 4096, acc=0, dw=A, fwd=0, T=4, D=64, V=100, K=3, chunk=128,
                ignore=0, ws=A, ws_bytes=need, stream=None)

    def refuse(text, **change):
        with pytest.raises(nmce.NmError) as e:
            lib.nm_ce_distill(*{**good, **change}.values())
        assert e.value.status == 1 and text in str(e.value), str(e.value)

    refuse("teacher_dtype 0 (f32) or 1 (bf16)", teacher_dtype=2)
    for name in ("x", "w", "ids", "logits", "weight", "loss"):
        refuse("are required", **{name: None})
    for tau in (0.0, -1.0, float("inf"), float("nan")):
        refuse("temperature must be positive", tau=tau)
    refuse("cannot be negative", soft=-0.1)
    refuse("cannot be negative", hard=float("nan"))
    refuse("hard term needs targets", targets=None)
    refuse("forward-only call has no dx", fwd=1)
    refuse("needs the device scalar grad_scale", gs=None)
    refuse("may be x or accumulate, not both", dx=A, acc=1)
    for name in ("x", "w", "dx", "dw"):
        refuse("16-byte aligned", **{name: A + 8})
    refuse("aligned to their size", ids=A + 2)
    refuse("aligned to their size", logits=A + 2)
    refuse("256-byte aligned workspace", ws=None)
    refuse("256-byte aligned workspace", ws=A + 128)
    refuse("smaller than", ws_bytes=need - 1)
    refuse("cannot be negative", T=-1)
    refuse("multiple of 8", D=60)
    refuse("must be positive", V=0)
    refuse("1 to 512 teacher entries", K=0)
    refuse("1 to 512 teacher entries", K=513)
    refuse("chunk_rows must be positive", chunk=0)
    assert lib.nm_ce_distill_workspace_bytes(4, 60, 100, 3, 128, 0) == 0 and b"multiple of 8" in lib.nm_last_error()


def test_forward_only_needs_no_logits_store(lib):  # noqa: F811
    full = lib.nm_ce_distill_workspace_bytes(8192, 2048, 128256, 64, 8192, 0)
    assert full > 8192 * 128256 * 4 > 20 * lib.nm_ce_distill_workspace_bytes(8192, 2048, 128256, 64, 8192, 1)
    # chunk_rows beyond the call's rows costs nothing
    assert lib.nm_ce_distill_workspace_bytes(100, 64, 1000, 4, 10 ** 6, 0) == lib.nm_ce_distill_workspace_bytes(100, 64, 1000, 4, 100, 0)
