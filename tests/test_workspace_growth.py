"""A workspace that a program planned for its longest call serves the shorter ones: the sizes never fall as the rows grow. No GPU
needed."""
import pytest

from test_capi_load import lib  # noqa: F401  (the built library)

LENGTHS = sorted({n + d for n in [16 << i for i in range(15)] + [2560, 5120, 10240, 49152, 98304, 131072, 150000]
                  for d in (-1, 0, 1, 17)})


@pytest.mark.parametrize("D", [8, 64, 320, 512, 768, 1024, 2048, 4104, 65536])
def test_embedding_gradient(lib, D):  # noqa: F811
    sizes = [lib.nm_embed_bwd_workspace_bytes(T, D, 64256) for T in LENGTHS]
    assert sizes[0] > 0 and sizes == sorted(sizes)


def test_the_other_operators(lib):  # noqa: F811
    for D in (8, 1024, 4096):
        sizes = [lib.nm_gated_tail_workspace_bytes(T, D) for T in LENGTHS]
        assert sizes[0] > 0 and sizes == sorted(sizes)
        for fwd in (0, 1):
            sizes = [lib.nm_ce_distill_workspace_bytes(T, D, 1000, 9, 4096, fwd) for T in LENGTHS]
            assert sizes[0] > 0 and sizes == sorted(sizes)
