"""The largest extents that the distillation head takes, checked on the host (no GPU needed)."""
import pytest

from test_capi_load import lib  # noqa: F401  (the built library)

A, TOP = 1 << 20, 1 << 30


@pytest.mark.parametrize("fwd", [0, 1])
def test_vocabularies_beyond_the_coordinates_are_refused(lib, fwd):  # noqa: F811
    """The gradient of a row is 2 V bf16 columns wide, and a column is a 32-bit coordinate."""
    import nmce
    assert lib.nm_ce_distill_workspace_bytes(1, 8, TOP, 1, 128, fwd) > 0
    for V in (TOP + 1, TOP + 6400, 2 ** 31 - 65, 2 ** 31 - 1):
        assert lib.nm_ce_distill_workspace_bytes(1, 8, V, 1, 128, fwd) == 0 and b"at most 2^30" in lib.nm_last_error()
        grads = (None, None) if fwd else (A, A)
        with pytest.raises(nmce.NmError) as e:
            lib.nm_ce_distill(0, A, A, A, A, None, None, A, A, 1.0, 1.0, 0.0, A, None, None, None, grads[0], 0, grads[1], fwd, 1, 8,
                              V, 1, 128, 0, A, 2 ** 62, None)
        assert e.value.status == 1 and "at most 2^30" in str(e.value)


def test_chunks_beyond_the_coordinates_are_refused(lib):  # noqa: F811
    assert lib.nm_ce_distill_workspace_bytes(TOP, 8, 16, 1, 2 ** 31 - 1, 1) > 0
    assert lib.nm_ce_distill_workspace_bytes(TOP + 1, 8, 16, 1, TOP, 1) > 0
    assert lib.nm_ce_distill_workspace_bytes(100, 8, 16, 1, 2 ** 31 - 1, 1) > 0          # a chunk beyond the call's rows
    assert lib.nm_ce_distill_workspace_bytes(TOP + 1, 8, 16, 1, 2 ** 31 - 1, 1) == 0
    assert b"at most 2^30 rows" in lib.nm_last_error()
