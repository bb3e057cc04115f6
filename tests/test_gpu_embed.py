"""nm_embed_fwd / nm_embed_bwd against plain float64: types, odd sizes, ids outside the vocabulary, runs of every length
around the places where the backward cuts them, sections, repeatability, graphs, streams and untouched memory.

Tolerances. Forward: the product in f32 is off by at most 2^-24 relative, the store in bf16 by another 2^-8 (half a step).
Backward: a sum of n terms added one by one in f32, in any grouping, is off by at most (n - 1) 2^-24 sum|term| (first
order), the product with the scale and the addition to the old value by one rounding each."""
import ctypes

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
TYPES = {1: torch.bfloat16, 0: torch.float32}


def _lib():
    from gpu_common import lib, nmce
    return lib(), nmce.ptr


def _bwd(dy, tokens, V, scale, before=None, stream=None, ws=None):
    """before: the old gradient (accumulate) or None (overwrite). Returns f32 [V, D]."""
    lib, ptr = _lib()
    T, D = dy.shape
    out = torch.full((V, D), float("nan"), device="cuda") if before is None else before.clone()
    need = lib.nm_embed_bwd_workspace_bytes(T, D, V)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda") if ws is None else ws
    lib.nm_embed_bwd(int(dy.dtype == torch.bfloat16), ptr(dy), ptr(tokens), ptr(out), scale, int(before is not None), T, D,
                     V, ptr(ws), ws.numel(), stream)
    return out


def _check_bwd(dy, tokens, V, scale, before, got):
    keep = (tokens >= 0) & (tokens < V)
    ids, rows = tokens[keep].long(), dy[keep].double()
    scale = float(np.float32(scale))
    total = torch.zeros(V, dy.shape[1], dtype=torch.float64, device="cuda").index_add_(0, ids, rows)
    size = torch.zeros_like(total).index_add_(0, ids, rows.abs())
    count = torch.zeros(V, dtype=torch.float64, device="cuda").index_add_(0, ids, torch.ones_like(ids, dtype=torch.float64))
    want = total * scale
    tol = (count[:, None] + 1) * U32 * size * abs(scale)
    if before is not None:
        want = want + before.double()
        tol = tol + U32 * want.abs()
    # second-order terms: under a hundredth of the first-order bound for up to 10^5 terms
    assert bool(((got.double() - want).abs() <= 1.01 * tol).all())
    if before is None:
        assert bool((got[count == 0] == 0).all())
    else:
        assert torch.equal(got[count == 0].view(torch.int32), before[count == 0].view(torch.int32))


@pytest.mark.parametrize("dtype", [1, 0])
@pytest.mark.parametrize("T,D,V", [(1, 8, 1), (3, 64, 5), (17, 520, 100), (2125, 768, 8256), (64, 2048, 128256),
                                   (1000, 4104, 77)])
def test_forward(dtype, T, D, V):
    lib, ptr = _lib()
    g = torch.Generator(device="cuda").manual_seed(T + D)
    table = torch.randn(V, D, generator=g, device="cuda").to(TYPES[dtype])
    tokens = torch.randint(-1, V + 2, (T,), generator=g, device="cuda").int()
    tokens[0] = V - 1
    guard = torch.full((T + 2, D), 7.0, dtype=TYPES[dtype], device="cuda")
    scale = float(np.float32(D ** 0.5))
    lib.nm_embed_fwd(dtype, ptr(table), ptr(tokens), ptr(guard[1]), scale, T, D, V, None)
    ok = (tokens >= 0) & (tokens < V)
    want = torch.where(ok[:, None], table.double()[tokens.long().clamp(0, V - 1)] * scale, torch.zeros((), dtype=torch.float64, device="cuda"))
    tol = (U32 + (2.0 ** -8 if dtype else 0.0)) * want.abs() * (1 + 2.0 ** -20)
    assert bool(((guard[1:-1].double() - want).abs() <= tol).all())
    assert bool((guard[0] == 7).all()) and bool((guard[-1] == 7).all())


def test_forward_keeps_what_is_not_finite():
    lib, ptr = _lib()
    table = torch.ones(3, 16, device="cuda").bfloat16()
    table[1, 3], table[1, 4] = float("inf"), float("nan")
    tokens = torch.tensor([0, 1, -5, 2], dtype=torch.int32, device="cuda")
    out = torch.empty(4, 16, dtype=torch.bfloat16, device="cuda")
    lib.nm_embed_fwd(1, ptr(table), ptr(tokens), ptr(out), 2.0, 4, 16, 3, None)
    assert torch.isposinf(out[1, 3]) and torch.isnan(out[1, 4])
    assert bool(torch.isfinite(out[[0, 2, 3]]).all()) and bool((out[2] == 0).all())


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("dtype", [1, 0])
@pytest.mark.parametrize("T,D,V", [(1, 8, 1), (1, 512, 8256), (31, 64, 2), (2125, 768, 64256), (5000, 136, 40),
                                   (20000, 264, 511), (20000, 64, 512), (9000, 4104, 300)])
def test_backward(dtype, T, D, V, add):
    g = torch.Generator(device="cuda").manual_seed(T + V)
    dy = torch.randn(T, D, generator=g, device="cuda").to(TYPES[dtype])
    u = torch.rand(T, generator=g, device="cuda")
    tokens = ((V + 3.0) ** u).int() - 2          # -1 and some ids beyond V among them; frequencies fall as 1 / rank
    before = torch.randn(V, D, generator=g, device="cuda") if add else None
    got = _bwd(dy, tokens, V, 0.37, before)
    _check_bwd(dy, tokens, V, 0.37, before, got)
    assert torch.equal(got, _bwd(dy, tokens, V, 0.37, before)), "the same call gave other bits"


@pytest.mark.parametrize("seed", range(6))
def test_backward_runs_around_the_cuts(seed):
    """Run lengths at and around 16, 32, 48, 64 and long ones, so that runs begin, end and cross at every offset of a
    window; every position is checked through a column that counts."""
    rng = np.random.default_rng(seed)
    lengths = []
    while sum(lengths) < 6000:
        lengths.append(int(rng.choice([1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 100, 400])))
    T, V = sum(lengths), len(lengths)
    tokens = np.repeat(np.arange(V, dtype=np.int32), lengths)
    perm = rng.permutation(T)
    tok = torch.from_numpy(tokens[perm]).cuda()
    dy = torch.from_numpy(rng.standard_normal((T, 72)).astype(np.float32)).cuda()
    dy[:, 0] = 1.0                                 # whole numbers: exact in any order
    got = _bwd(dy, tok, V, 1.0)
    assert torch.equal(got[:, 0].cpu(), torch.tensor(lengths, dtype=torch.float32))
    _check_bwd(dy, tok, V, 1.0, None, got)


@pytest.mark.parametrize("n_ids", [1, 2, 7])
def test_backward_few_ids_many_rows(n_ids):
    T, D, V = 131072 + 1000, 64, 1000             # two sections; runs cross the section's end
    g = torch.Generator(device="cuda").manual_seed(n_ids)
    dy = torch.randn(T, D, generator=g, device="cuda").bfloat16()
    tokens = (torch.randint(0, n_ids, (T,), generator=g, device="cuda") * 137).int()
    for before in (None, torch.ones(V, D, device="cuda")):
        _check_bwd(dy, tokens, V, 1.5, before, _bwd(dy, tokens, V, 1.5, before))


def test_backward_full_step_shape():
    T, D, V = 131072, 512, 128256
    g = torch.Generator(device="cuda").manual_seed(9)
    dy = torch.randn(T, D, generator=g, device="cuda").bfloat16()
    tokens = (float(V) ** torch.rand(T, generator=g, device="cuda", dtype=torch.float64)).int() - 1
    _check_bwd(dy, tokens, V, 22.6, None, _bwd(dy, tokens, V, 22.6))


def test_backward_ids_beyond_eighteen_bits():
    """Three sorting passes (a vocabulary above 2^18)."""
    T, D, V = 3000, 8, 300000
    g = torch.Generator(device="cuda").manual_seed(4)
    dy = torch.randn(T, D, generator=g, device="cuda")
    tokens = (torch.randint(0, 500, (T,), generator=g, device="cuda") * 600 + 123).int()
    _check_bwd(dy, tokens, V, 1.0, None, _bwd(dy, tokens, V, 1.0))


def test_offsets_beyond_32_bits():
    """A table and a gradient of more than 2^31 elements: the last rows are found and nothing wraps."""
    lib, ptr = _lib()
    V, D, T = 1_050_000, 2056, 5
    table = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda")
    tokens = torch.tensor([V - 1, 0, V - 1, 1_045_000, -1], dtype=torch.int32, device="cuda")
    table[V - 1], table[1_045_000], table[0] = 3.0, 2.0, 1.0
    out = torch.empty(T, D, dtype=torch.bfloat16, device="cuda")
    lib.nm_embed_fwd(1, ptr(table), ptr(tokens), ptr(out), 1.0, T, D, V, None)
    assert out[:, 0].tolist() == [3, 1, 3, 2, 0] and bool((out == out[:, :1]).all())
    del table
    got = _bwd(out, tokens, V, 1.0)
    assert bool((got[V - 1] == 6).all()) and bool((got[1_045_000] == 2).all()) and bool((got[0] == 1).all())
    assert float(got[1:1_045_000].abs().amax()) == 0 and float(got[1_045_001:V - 1].abs().amax()) == 0


def test_no_rows():
    lib, ptr = _lib()
    out = torch.full((5, 16), 3.0, device="cuda")
    ws = torch.empty(lib.nm_embed_bwd_workspace_bytes(0, 16, 5), dtype=torch.uint8, device="cuda")
    assert lib.nm_embed_fwd(1, None, None, None, 1.0, 0, 16, 5, None) == 0
    lib.nm_embed_bwd(1, None, None, ptr(out), 1.0, 1, 0, 16, 5, ptr(ws), ws.numel(), None)
    assert bool((out == 3).all())
    lib.nm_embed_bwd(1, None, None, ptr(out), 1.0, 0, 0, 16, 5, ptr(ws), ws.numel(), None)
    assert bool((out == 0).all())


def test_gradient_against_differences():
    """<dE, delta> against the forward's central difference along delta, in f32 storage: the lookup is linear, so the
    difference is exact up to the rounding of its sums."""
    lib, ptr = _lib()
    T, D, V = 300, 64, 50
    g = torch.Generator(device="cuda").manual_seed(1)
    table, delta = (torch.randn(V, D, generator=g, device="cuda") for _ in range(2))
    tokens = torch.randint(-1, V, (T,), generator=g, device="cuda").int()
    dy = torch.randn(T, D, generator=g, device="cuda")

    def value(sign):
        out, moved = torch.empty(T, D, device="cuda"), table + sign * delta
        lib.nm_embed_fwd(0, ptr(moved), ptr(tokens), ptr(out), 3.0, T, D, V, None)
        return (out.double() * dy.double()).sum()

    difference = (value(1) - value(-1)) / 2
    dE = _bwd(dy, tokens, V, 3.0)
    slope = (dE.double() * delta.double()).sum()
    # each of the T D terms carries a few roundings of 2^-24 of values of size 3 (|table| + |delta|)
    bound = 8 * U32 * 3.0 * (dy.double().abs().sum() * float(table.abs().max() + delta.abs().max()))
    assert abs(float(difference - slope)) <= float(bound)


def test_captured_and_replayed_on_new_tokens():
    T, D, V = 4000, 128, 3000
    g = torch.Generator(device="cuda").manual_seed(6)
    lib, ptr = _lib()
    dy = torch.randn(T, D, generator=g, device="cuda").bfloat16()
    tokens = torch.randint(0, V, (T,), generator=g, device="cuda").int()
    out = torch.empty(V, D, device="cuda")
    y = torch.empty(T, D, dtype=torch.bfloat16, device="cuda")
    table = torch.randn(V, D, generator=g, device="cuda").bfloat16()
    ws = torch.empty(lib.nm_embed_bwd_workspace_bytes(T, D, V), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        lib.nm_embed_fwd(1, ptr(table), ptr(tokens), ptr(y), 2.0, T, D, V, st)
        lib.nm_embed_bwd(1, ptr(dy), ptr(tokens), ptr(out), 2.0, 0, T, D, V, ptr(ws), ws.numel(), st)
    for seed in (1, 2):
        g2 = torch.Generator(device="cuda").manual_seed(seed)
        tokens.copy_((torch.randint(0, V, (T,), generator=g2, device="cuda") // seed).int())
        graph.replay()
        torch.cuda.synchronize()
        _check_bwd(dy, tokens, V, 2.0, None, out)
        assert torch.equal(out, _bwd(dy, tokens, V, 2.0))
        assert torch.equal(y, (table.float()[tokens.long()] * 2.0).bfloat16())


def test_two_calls_at_once_with_a_workspace_each():
    T, D, V = 30000, 256, 900
    data = []
    for seed in (1, 2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        data.append((torch.randn(T, D, generator=g, device="cuda").bfloat16(),
                     torch.randint(0, V, (T,), generator=g, device="cuda").int()))
    want = [_bwd(dy, tok, V, 1.0) for dy, tok in data]
    streams = [torch.cuda.Stream() for _ in data]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, (dy, tok) in enumerate(data):
            with torch.cuda.stream(streams[i]):
                got[i] = _bwd(dy, tok, V, 1.0, stream=ctypes.c_void_p(streams[i].cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_nothing_outside_the_buffers_is_written():
    lib, ptr = _lib()
    T, D, V = 1500, 72, 40
    dy = torch.randn(T, D, device="cuda")
    tokens = torch.randint(0, V, (T,), device="cuda").int()
    need = lib.nm_embed_bwd_workspace_bytes(T, D, V)
    ws = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    out = torch.full((V + 2, D), 9.0, device="cuda")
    lib.nm_embed_bwd(0, ptr(dy), ptr(tokens), ptr(out[1]), 1.0, 0, T, D, V, ptr(ws), need, None)
    _check_bwd(dy, tokens, V, 1.0, None, out[1:-1])
    assert bool((ws[need:] == 0x5A).all()) and bool((out[0] == 9).all()) and bool((out[-1] == 9).all())


@pytest.mark.parametrize("T", [5, 5000])
def test_no_token_inside_the_vocabulary(T):
    V, D = 100, 64
    dy = torch.full((T, D), float("nan"), device="cuda")          # rows that do not count are not read
    tokens = torch.where(torch.arange(T, device="cuda") % 2 == 0, -1, V).int()
    assert bool((_bwd(dy, tokens, V, 1.0) == 0).all())
    before = torch.randn(V, D, device="cuda")
    assert torch.equal(_bwd(dy, tokens, V, 1.0, before), before)
    tokens[3] = 7
    dy[3] = 2.0
    got = _bwd(dy, tokens, V, 1.5)
    assert bool((got[7] == 3).all()) and float(got.abs().sum()) == 3 * D


@pytest.mark.parametrize("add", [False, True])
def test_a_gradient_that_is_only_16_byte_aligned(add):
    """Rows of the gradient that do not start on 32 bytes take the narrower stores: the same bits."""
    lib, p = _lib()
    T, D, V = 3000, 72, 500
    g = torch.Generator(device="cuda").manual_seed(8)
    dy = torch.randn(T, D, generator=g, device="cuda").bfloat16()
    tokens = torch.randint(-1, 40, (T,), generator=g, device="cuda").int()
    before = torch.randn(V, D, generator=g, device="cuda")
    want = _bwd(dy, tokens, V, 2.0, before if add else None)
    room = torch.full((V * D + 8,), 9.0, device="cuda")
    out = room[4:4 + V * D].view(V, D)
    out.copy_(before)
    assert out.data_ptr() % 32 == 16
    ws = torch.empty(lib.nm_embed_bwd_workspace_bytes(T, D, V), dtype=torch.uint8, device="cuda")
    lib.nm_embed_bwd(1, p(dy), p(tokens), p(out), 2.0, int(add), T, D, V, p(ws), ws.numel(), None)
    assert torch.equal(out, want) and bool((room[:4] == 9).all()) and bool((room[-4:] == 9).all())


def test_widest_rows():
    T, D, V = 40, 65536, 6
    g = torch.Generator(device="cuda").manual_seed(2)
    dy = torch.randn(T, D, generator=g, device="cuda")
    tokens = torch.randint(0, V, (T,), generator=g, device="cuda").int()
    _check_bwd(dy, tokens, V, 1.0, None, _bwd(dy, tokens, V, 1.0))
