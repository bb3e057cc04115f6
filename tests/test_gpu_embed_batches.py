"""nm_embed_fwd in the form of its large calls, where a row group takes eight batches of two rows: it begins at
groups * 2 * 8 * 8 rows per SM (groups: rows that 256 threads hold side by side). Ragged ends inside a batch, between batches
and beyond whole groups, ids outside the vocabulary, both storage types, rows of less and of more than one piece per thread.

The result is the f32 product rounded to the storage type, both of which torch forms too: equal bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {1: torch.bfloat16, 0: torch.float32}


def _threshold(D):
    G = 32
    while G < D // 8 and G < 256:
        G *= 2
    return 256 // G * 2 * 8 * 8 * torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("dtype", [1, 0])
@pytest.mark.parametrize("D,more", [(2056, 57), (2056, 0), (2056, -1), (1024, 123), (1032, 16), (520, 31), (264, 2), (64, 48), (8, 3)])
def test_batched_rows(dtype, D, more):
    from gpu_common import lib, nmce
    T, V = _threshold(D) + more, 5000
    g = torch.Generator(device="cuda").manual_seed(T + D)
    table = torch.randn(V, D, generator=g, device="cuda").to(TYPES[dtype])
    tokens = torch.randint(0, V, (T,), generator=g, device="cuda").int()
    drop = torch.rand(T, generator=g, device="cuda")
    tokens = torch.where(drop < 0.02, torch.full_like(tokens, -1), torch.where(drop > 0.98, torch.full_like(tokens, V), tokens))
    tokens[0], tokens[-1], tokens[-2] = V - 1, V - 2, -7
    guard = torch.full((T + 2, D), 7.0, dtype=TYPES[dtype], device="cuda")
    guard[1:-1] = float("nan")
    scale = float(torch.tensor(D ** 0.5))
    lib().nm_embed_fwd(dtype, nmce.ptr(table), nmce.ptr(tokens), nmce.ptr(guard[1]), scale, T, D, V, None)
    ok = (tokens >= 0) & (tokens < V)
    want = (table[tokens.long().clamp(0, V - 1)].float() * scale).to(TYPES[dtype])
    want[~ok] = 0
    assert torch.equal(guard[1:-1], want)
    assert bool((guard[0] == 7).all()) and bool((guard[-1] == 7).all())
