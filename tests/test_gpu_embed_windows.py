"""nm_embed_bwd at every window size and on both sides of the lengths where it changes, in one section and in several: runs that
begin, end and cross at every offset of a window, counted exactly and held to the float64 bound of test_gpu_embed.py, in a
workspace whose end is watched.

That bound has one rounding for the addition to the old value, of the final one. A call of s sections adds s times (an overwriting
one s - 1 times), and rounds a running value each time, which is at most |old| + |scale| sum|term|: so much u more per section
after the first."""
import numpy as np
import pytest
import torch

from test_gpu_embed import U32, _bwd, _check_bwd, _lib

pytestmark = pytest.mark.gpu


def _check(dy, tokens, V, scale, before, got):
    T = dy.shape[0]
    sections = -(-T // 131072)
    if sections == 1:
        return _check_bwd(dy, tokens, V, scale, before, got)
    keep = (tokens >= 0) & (tokens < V)
    ids, rows = tokens[keep].long(), dy[keep].double()
    total = torch.zeros(V, dy.shape[1], dtype=torch.float64, device="cuda").index_add_(0, ids, rows) * scale
    size = torch.zeros_like(total).index_add_(0, ids, rows.abs()) * abs(scale)
    count = torch.bincount(ids, minlength=V).double()[:, None]
    old = torch.zeros_like(total) if before is None else before.double()
    want = total + old
    tol = U32 * ((count + 1) * size + want.abs() + (sections - 1) * (old.abs() + size))
    assert bool(((got.double() - want).abs() <= 1.01 * tol).all())


def _tokens(rng, T):
    """Runs of lengths around 16, 32, 64 and a few long ones, T positions in all, in random order; and the lengths."""
    lengths = []
    while sum(lengths) < T:
        lengths.append(int(rng.choice([1, 1, 2, 3, 7, 8, 9, 15, 16, 17, 23, 24, 25, 31, 32, 33, 47, 48, 49, 63, 64, 65, 96, 100, 129, 400])))
    lengths[-1] -= sum(lengths) - T
    lengths = [n for n in lengths if n > 0]
    return torch.from_numpy(np.repeat(np.arange(len(lengths), dtype=np.int32), lengths)[rng.permutation(T)]).cuda(), lengths


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,D", [(4096, 72), (4097, 72), (9001, 72), (16384, 72), (16385, 72), (10240, 512), (10241, 512), (2560, 2048),
                                 (2561, 2048), (40000, 72), (98304, 72), (98305, 72), (131072, 72), (131072 + 3000, 72),
                                 (131072 + 16384, 72), (131072 + 50001, 72), (131072 + 98304, 8), (2 * 131072 + 1, 8)])
def test_runs_around_the_cuts(T, D, dtype):
    lib, _ = _lib()
    rng = np.random.default_rng(T + D)
    tok, lengths = _tokens(rng, T)
    V = len(lengths)
    g = torch.Generator(device="cuda").manual_seed(T)
    dy = torch.randn(T, D, generator=g, device="cuda").to(dtype)
    dy[:, 0] = 1.0                                       # whole numbers: exact in any order
    need = lib.nm_embed_bwd_workspace_bytes(T, D, V)
    ws = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    got = _bwd(dy, tok, V, 1.0, ws=ws[:need])
    assert torch.equal(got[:, 0].cpu(), torch.tensor(lengths, dtype=torch.float32))
    _check(dy, tok, V, 1.0, None, got)
    assert bool((ws[need:] == 0x5A).all())
    before = torch.randn(V, D, generator=g, device="cuda")
    _check(dy, tok, V, 0.5, before, _bwd(dy, tok, V, 0.5, before, ws=ws[:need]))


@pytest.mark.parametrize("T", [500, 2560, 16384, 98304, 131072])
def test_one_id(T):
    """Cut at every edge; ids outside the vocabulary at both ends of the sorted order's last run."""
    D, V = 136, 40
    tok = torch.full((T,), 7, dtype=torch.int32, device="cuda")
    tok[::17], tok[5::31] = -1, V
    g = torch.Generator(device="cuda").manual_seed(T)
    dy = torch.randn(T, D, generator=g, device="cuda").bfloat16()
    for before in (None, torch.ones(V, D, device="cuda")):
        got = _bwd(dy, tok, V, 1.5, before)
        _check_bwd(dy, tok, V, 1.5, before, got)
        assert torch.equal(got, _bwd(dy, tok, V, 1.5, before))


def test_a_workspace_of_a_longer_call():
    lib, _ = _lib()
    D, V = 72, 3000
    ws = torch.empty(lib.nm_embed_bwd_workspace_bytes(140000, D, V), dtype=torch.uint8, device="cuda")
    for T in (140000, 131072, 98304, 32768, 16384, 2560, 1):
        g = torch.Generator(device="cuda").manual_seed(T)
        dy = torch.randn(T, D, generator=g, device="cuda")
        tok = torch.randint(-1, V + 1, (T,), generator=g, device="cuda").int()
        want = _bwd(dy, tok, V, 1.0)
        assert torch.equal(_bwd(dy, tok, V, 1.0, ws=ws), want)
        _check(dy, tok, V, 1.0, None, want)
