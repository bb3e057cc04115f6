"""nm_gated_tail_fwd / nm_gated_tail_bwd against plain float64: storage types, gate kinds, optional parts, odd widths and row
counts, calls in place, extreme gates, repeatability, graphs, and the gradient against differences.

Tolerances. u = 2^-24 is half a step of f32. A row sum of D <= 8192 terms goes through at most 16 fma steps per lane of a
pair, one addition of the pair and 8 butterfly steps: 25 roundings, each at most u times the sum of the terms' magnitudes.
The products around it add at most 10 roundings; ex2.approx and rcp.approx are within 2 u and 1 u (2 ulp and 1 ulp are 4 u and
2 u at worst), and the argument of ex2 carries |gate| <= 10 roundings' worth. 25 + 10 + 6 + 10 < 64: a value built from
magnitudes M is off by at most 64 u M before it is stored; storing in bf16 adds half a step, 2^-8 of the value. The next norm
is held to the x_out that the kernel stored (its definition). Sums over T rows add T u times the sum of magnitudes."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
U, C = 2.0 ** -24, 64
TYPES = {1: torch.bfloat16, 0: torch.float32}
EPS = 1e-5


def _lib():
    from gpu_common import lib, nmce
    return lib(), nmce.ptr


def _inputs(dtype, T, D, kind, post, scaled, seed=0, carried=True):
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * T + D)
    dt = TYPES[dtype]
    r = lambda *s, std=1.0, mean=0.0: (torch.randn(*s, generator=g, device="cuda") * std + mean).to(dt)  # noqa: E731
    s = {"branch": r(T, D, std=2.0), "x_in": r(T, D, std=1.5), "g_next": r(D, std=0.2, mean=1.0),
         "dx_out": r(T, D) if carried else None, "da_next": r(T, D)}
    s["gate"] = None if kind == 0 else r(T, std=2.0).clamp(-10, 10) if kind == 1 else r(T, D, std=2.0).clamp(-10, 10)
    s["g_post"] = r(D, std=0.2, mean=1.0) if post else None
    s["scale"] = r(D, std=0.1, mean=0.8) if scaled else None
    return s


def _fwd(dtype, kind, s, stream=None, x_out=None, a_next=None, eps=EPS):
    lib, p = _lib()
    T, D = s["x_in"].shape
    x_out = torch.empty_like(s["x_in"]) if x_out is None else x_out
    a = torch.empty_like(s["x_in"]) if a_next is None else a_next
    rp, rn = torch.full((T,), -1.0, device="cuda"), torch.full((T,), -1.0, device="cuda")
    lib.nm_gated_tail_fwd(dtype, kind, p(s["branch"]), p(s["x_in"]), p(s["gate"]), p(s["scale"]), p(s["g_post"]),
                          p(s["g_next"]), p(x_out), p(a), p(rp), p(rn), T, D, eps, stream)
    return x_out, a, rp, rn


def _bwd(dtype, kind, s, rp, rn, stream=None, out=None, ws=None):
    lib, p = _lib()
    T, D = s["x_in"].shape
    o = {"dx_in": torch.empty_like(s["x_in"]), "dbranch": torch.empty_like(s["x_in"]),
         "dgate": None if kind == 0 else torch.empty_like(s["gate"]), "dg_next": torch.full((D,), -7.0, device="cuda"),
         "dg_post": None if s["g_post"] is None else torch.full((D,), -7.0, device="cuda"),
         "dscale": None if s["scale"] is None else torch.full((D,), -7.0, device="cuda")} if out is None else out
    ws = torch.empty(lib.nm_gated_tail_workspace_bytes(T, D), dtype=torch.uint8, device="cuda") if ws is None else ws
    lib.nm_gated_tail_bwd(dtype, kind, p(s["dx_out"]), p(s["da_next"]), p(s["x_in"]), p(s["branch"]), p(s["gate"]),
                          p(s["scale"]), p(s["g_post"]), p(s["g_next"]), p(rp), p(rn), p(o["dx_in"]), p(o["dbranch"]),
                          p(o["dgate"]), p(o["dg_next"]), p(o["dg_post"]), p(o["dscale"]), T, D, p(ws), ws.numel(), stream)
    return o


def _near(name, got, want, tol):
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (f"{name}: {int(bad.sum())} of {bad.numel()} outside, worst "
                                 f"{float(((got.double() - want).abs() / tol.clamp_min(1e-300)).max()):.2f} x the tolerance")


def _check(dtype, kind, s, fwd, bwd):
    half = 2.0 ** -8 if dtype else 0.0
    d = {k: None if v is None else v.double() for k, v in s.items()}
    T, D = d["x_in"].shape
    one = torch.ones((), dtype=torch.float64, device="cuda")
    x_out, a, rp, rn = fwd
    gate = None if kind == 0 else d["gate"][:, None] if kind == 1 else d["gate"]
    on = one if gate is None else torch.sigmoid(gate)
    slope = one if gate is None else torch.sigmoid(gate) * torch.sigmoid(-gate)
    sc = one if d["scale"] is None else d["scale"]
    gp = one if d["g_post"] is None else d["g_post"]
    if s["g_post"] is not None:
        want = (d["branch"].square().mean(1) + EPS).rsqrt()
        _near("rstd_post", rp, want, C * U * want)
        n = d["branch"] * rp.double()[:, None]
    else:
        assert bool((rp == -1).all())
        n = d["branch"]
    y = n * gp
    want = sc * d["x_in"] + on * y
    _near("x_out", x_out, want, half * want.abs() + C * U * ((sc * d["x_in"]).abs() + (on * y).abs()))
    xo = x_out.double()
    want = (xo.square().mean(1) + EPS).rsqrt()
    _near("rstd_next", rn, want, C * U * want)
    want = xo * want[:, None] * d["g_next"]
    _near("a_next", a, want, (half + C * U) * want.abs())
    if bwd is None:
        return
    r = rn.double()[:, None]
    av = d["g_next"] * d["da_next"]
    carried = torch.zeros_like(xo) if d["dx_out"] is None else d["dx_out"]
    m = carried + r * av - xo * r ** 3 * (xo * av).sum(1, keepdim=True) / D
    M = carried.abs() + r * av.abs() + xo.abs() * r ** 3 * (xo * av).abs().sum(1, keepdim=True) / D
    _near("dx_in", bwd["dx_in"], sc * m, half * (sc * m).abs() + C * U * sc.abs() * M)
    if kind == 1:
        want, mag = (m * y).sum(1) * slope[:, 0], (M * y.abs()).sum(1) * slope[:, 0]
        _near("dgate", bwd["dgate"], want, half * want.abs() + 2 * C * U * mag)
    elif kind == 2:
        want = m * y * slope
        _near("dgate", bwd["dgate"], want, half * want.abs() + C * U * M * y.abs() * slope)
    t, Tm = on * m, on * M
    if s["g_post"] is None:
        _near("dbranch", bwd["dbranch"], t, half * t.abs() + C * U * Tm)
    else:
        q = rp.double()[:, None]
        pv, P = gp * t, gp.abs() * Tm
        b = d["branch"]
        want = q * pv - b * q ** 3 * (b * pv).sum(1, keepdim=True) / D
        mag = q * P + b.abs() * q ** 3 * (b.abs() * P).sum(1, keepdim=True) / D
        _near("dbranch", bwd["dbranch"], want, half * want.abs() + 2 * C * U * mag)
        _near("dg_post", bwd["dg_post"], (t * n).sum(0), (T + C) * U * (Tm * n.abs()).sum(0))
    term = d["da_next"] * xo * r
    _near("dg_next", bwd["dg_next"], term.sum(0), (T + C) * U * term.abs().sum(0))
    if s["scale"] is not None:
        _near("dscale", bwd["dscale"], (m * d["x_in"]).sum(0), (T + C) * U * (M * d["x_in"].abs()).sum(0))


@pytest.mark.parametrize("dtype", [1, 0])
@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("post,scaled,carried", [(True, True, True), (False, True, True), (True, False, False),
                                                 (False, False, True)])
@pytest.mark.parametrize("T,D", [(1, 8), (17, 520), (301, 64), (40, 2048), (1201, 256)])
def test_against_float64(dtype, kind, post, scaled, carried, T, D):
    s = _inputs(dtype, T, D, kind, post, scaled, carried=carried)
    fwd = _fwd(dtype, kind, s)
    _check(dtype, kind, s, fwd, _bwd(dtype, kind, s, fwd[2], fwd[3]))


@pytest.mark.parametrize("dtype,T,D", [(1, 5, 8192), (1, 700, 4104), (0, 5, 4096), (0, 333, 2056), (1, 5000, 1024),
                                       (0, 2125, 1024), (1, 9, 8184)])
@pytest.mark.parametrize("kind", [1, 2])
def test_wide_rows_and_many_rows(dtype, T, D, kind):
    s = _inputs(dtype, T, D, kind, True, True)
    fwd = _fwd(dtype, kind, s)
    _check(dtype, kind, s, fwd, _bwd(dtype, kind, s, fwd[2], fwd[3]))


@pytest.mark.parametrize("dtype", [1, 0])
def test_extreme_gates_and_empty_rows(dtype):
    """Gates at both ends of the type (closed and open exactly), rows of zeros (rstd = 1 / sqrt(eps)): finite everywhere."""
    T, D = 12, 136
    s = _inputs(dtype, T, D, 2, True, True)
    big = float(torch.finfo(TYPES[dtype]).max)
    s["gate"][0], s["gate"][1], s["gate"][2], s["gate"][3] = big, -big, float("inf"), float("-inf")
    s["gate"][4], s["gate"][5] = 90.0, -90.0
    s["branch"][6] = 0
    s["branch"][7], s["x_in"][7] = 0, 0
    fwd = _fwd(dtype, 2, s)
    bwd = _bwd(dtype, 2, s, fwd[2], fwd[3])
    for v in list(fwd) + [v for v in bwd.values()]:
        assert bool(torch.isfinite(v).all())
    y = s["branch"].double() * fwd[2].double()[:, None] * s["g_post"].double()
    base = s["scale"].double() * s["x_in"].double()
    half = 2.0 ** -8 if dtype else 0.0
    for row, open_ in ((0, 1.0), (1, 0.0), (2, 1.0), (3, 0.0), (4, 1.0), (5, 0.0)):
        want = base[row] + open_ * y[row]
        # |gate| = 90 leaves 1e-39 of the branch, far below every tolerance
        _near("x_out", fwd[0][row], want, half * want.abs() + C * U * (base[row].abs() + y[row].abs()))
        assert float(bwd["dgate"][row].abs().max()) <= 1e-30
        if open_ == 0.0:
            assert float(bwd["dbranch"][row].abs().max()) <= 1e-30
    assert bool((fwd[1][7] == 0).all())
    assert abs(float(fwd[2][6]) - EPS ** -0.5) <= C * U * EPS ** -0.5


def test_what_is_not_finite_stays_in_its_row():
    s = _inputs(1, 9, 256, 2, True, True)
    s["branch"][2, 5], s["gate"][4, 9], s["x_in"][6, 1] = float("nan"), float("nan"), float("inf")
    fwd = _fwd(1, 2, s)
    bwd = _bwd(1, 2, s, fwd[2], fwd[3])
    clean = [0, 1, 3, 5, 7, 8]
    for v in (fwd[0], fwd[1], bwd["dx_in"], bwd["dbranch"], bwd["dgate"]):
        assert bool(torch.isfinite(v[clean]).all())
    assert bool(torch.isnan(fwd[0][4, 9])) and bool(torch.isnan(fwd[0][2]).all()) and bool(torch.isinf(fwd[0][6, 1]))


@pytest.mark.parametrize("dtype,kind", [(1, 2), (1, 1), (0, 2), (0, 1)])
def test_in_place_gives_the_same_bits(dtype, kind):
    s = _inputs(dtype, 700, 776, kind, True, True)
    fwd = _fwd(dtype, kind, s)
    bwd = _bwd(dtype, kind, s, fwd[2], fwd[3])
    c = {k: None if v is None else v.clone() for k, v in s.items()}
    over = _fwd(dtype, kind, c, x_out=c["x_in"], a_next=c["branch"])
    assert all(torch.equal(x, y) for x, y in zip(over, fwd))
    c = {k: None if v is None else v.clone() for k, v in s.items()}
    out = dict(bwd)
    out = {k: v.clone() for k, v in out.items()}
    out["dx_in"], out["dbranch"], out["dgate"] = c["dx_out"], c["branch"], c["gate"]
    over = _bwd(dtype, kind, c, fwd[2], fwd[3], out=out)
    assert all(torch.equal(over[k], bwd[k]) for k in bwd)


def test_repeats_give_the_same_bits_and_gradients_may_be_skipped():
    lib, p = _lib()
    s = _inputs(1, 3001, 512, 2, True, True)
    fwd = _fwd(1, 2, s)
    first = _bwd(1, 2, s, fwd[2], fwd[3])
    again = _bwd(1, 2, s, fwd[2], fwd[3])
    assert all(torch.equal(first[k], again[k]) for k in first)
    T, D = s["x_in"].shape
    o = {k: torch.empty_like(first[k]) for k in ("dx_in", "dbranch", "dgate")}
    lib.nm_gated_tail_bwd(1, 2, p(s["dx_out"]), p(s["da_next"]), p(s["x_in"]), p(s["branch"]), p(s["gate"]), p(s["scale"]),
                          p(s["g_post"]), p(s["g_next"]), p(fwd[2]), p(fwd[3]), p(o["dx_in"]), p(o["dbranch"]), p(o["dgate"]),
                          None, None, None, T, D, None, 0, None)
    assert all(torch.equal(o[k], first[k]) for k in o)


def test_without_the_next_norm():
    lib, p = _lib()
    s = _inputs(1, 33, 256, 2, True, True)
    want = _fwd(1, 2, s)
    x_out = torch.empty_like(s["x_in"])
    lib.nm_gated_tail_fwd(1, 2, p(s["branch"]), p(s["x_in"]), p(s["gate"]), p(s["scale"]), p(s["g_post"]), None, p(x_out), None,
                          None, None, 33, 256, EPS, None)
    assert torch.equal(x_out, want[0])


def test_ungated_unscaled_is_the_sandwich_tail():
    """Without gate and residual scale the accurate sandwich tail computes the same thing (its f32 steps are ordered
    otherwise, so a value next to a bf16 tie may land one step away: on under 1 % of the elements)."""
    lib, p = _lib()
    T, D = 500, 1024
    s = _inputs(1, T, D, 0, True, False)
    x_out, a, rp, rn = _fwd(1, 0, s)
    x2, a2 = torch.empty_like(x_out), torch.empty_like(a)
    rp2, rn2 = torch.empty_like(rp), torch.empty_like(rn)
    lib.nm_sandwich_tail_fwd(1, 1, p(s["branch"]), p(s["x_in"]), p(s["g_post"]), p(s["g_next"]), p(x2), p(a2), p(rp2), p(rn2), T,
                             D, EPS, None)
    for mine, other in ((x_out, x2), (a, a2)):
        assert float((mine != other).float().mean()) < 0.01
        assert float((mine.float() - other.float()).norm() / other.float().norm()) < 2.0 ** -9


def test_gradient_against_differences():
    """f32 storage. The directional derivative of <x_out, dx_out> + <a_next, da_next> along random directions of every input
    against a central difference taken in float64 on the same formula; the kernel's gradients carry f32 roundings (2^-24 of
    their magnitude, a few hundred of them), the difference its h^2 term."""
    s = _inputs(0, 29, 72, 2, True, True)
    fwd = _fwd(0, 2, s)
    bwd = _bwd(0, 2, s, fwd[2], fwd[3])
    names = {"x_in": "dx_in", "branch": "dbranch", "gate": "dgate", "g_next": "dg_next", "g_post": "dg_post", "scale": "dscale"}

    def value(moved):
        d = {k: v.double() for k, v in moved.items()}
        n = d["branch"] * (d["branch"].square().mean(1, keepdim=True) + EPS).rsqrt() * d["g_post"]
        xo = d["scale"] * d["x_in"] + torch.sigmoid(d["gate"]) * n
        a = xo * (xo.square().mean(1, keepdim=True) + EPS).rsqrt() * d["g_next"]
        return float((xo * d["dx_out"]).sum() + (a * d["da_next"]).sum())

    g = torch.Generator(device="cuda").manual_seed(3)
    h = 1e-4
    for k, out in names.items():
        dirn = torch.randn(s[k].shape, generator=g, device="cuda", dtype=torch.float64)
        up = value({**{j: v.double() for j, v in s.items()}, k: s[k].double() + h * dirn})
        down = value({**{j: v.double() for j, v in s.items()}, k: s[k].double() - h * dirn})
        slope = float((bwd[out].double() * dirn).sum())
        size = float((bwd[out].double() * dirn).abs().sum())
        # third derivatives of these forms are of the size of the gradient itself times a small constant: h^2 = 1e-8
        assert abs((up - down) / (2 * h) - slope) <= 1e-5 * size, k


def test_captured_and_replayed():
    s = _inputs(1, 800, 512, 2, True, True)
    lib, p = _lib()
    fwd = _fwd(1, 2, s)                                   # the first call on a device is made outside a capture
    want = _bwd(1, 2, s, fwd[2], fwd[3])
    ws = torch.empty(lib.nm_gated_tail_workspace_bytes(800, 512), dtype=torch.uint8, device="cuda")
    out = {k: torch.zeros_like(v) for k, v in want.items()}
    xo, a = torch.zeros_like(fwd[0]), torch.zeros_like(fwd[1])
    rp, rn = torch.zeros_like(fwd[2]), torch.zeros_like(fwd[3])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        lib.nm_gated_tail_fwd(1, 2, p(s["branch"]), p(s["x_in"]), p(s["gate"]), p(s["scale"]), p(s["g_post"]), p(s["g_next"]),
                              p(xo), p(a), p(rp), p(rn), 800, 512, EPS, st)
        _bwd(1, 2, s, rp, rn, stream=st, out=out, ws=ws)
    for seed in (0, 5):
        fresh = _inputs(1, 800, 512, 2, True, True, seed=seed)
        for k in s:
            s[k].copy_(fresh[k])
        graph.replay()
        torch.cuda.synchronize()
        fwd = _fwd(1, 2, fresh)
        want = _bwd(1, 2, fresh, fwd[2], fwd[3])
        assert torch.equal(xo, fwd[0]) and torch.equal(a, fwd[1])
        assert all(torch.equal(out[k], want[k]) for k in want)


def test_no_rows_and_nothing_outside_the_buffers():
    lib, p = _lib()
    dg = torch.full((64,), 5.0, device="cuda")
    ws = torch.empty(lib.nm_gated_tail_workspace_bytes(0, 64), dtype=torch.uint8, device="cuda")
    assert lib.nm_gated_tail_fwd(1, 0, None, None, None, None, None, None, None, None, None, None, 0, 64, EPS, None) == 0
    lib.nm_gated_tail_bwd(1, 0, None, None, None, None, None, None, None, None, None, None, None, None, None, p(dg), None, None,
                          0, 64, p(ws), ws.numel(), None)
    assert bool((dg == 0).all())
    T, D = 203, 264
    s = _inputs(1, T, D, 2, True, True)
    guard = torch.full((T + 2, D), 3.0, dtype=torch.bfloat16, device="cuda")
    guard2 = guard.clone()
    _fwd(1, 2, s, x_out=guard[1:-1], a_next=guard2[1:-1])
    need = lib.nm_gated_tail_workspace_bytes(T, D)
    big = torch.full((need + 1024,), 0x5A, dtype=torch.uint8, device="cuda")
    fwd = _fwd(1, 2, s)
    _bwd(1, 2, s, fwd[2], fwd[3], ws=big)
    assert torch.equal(guard[1:-1], fwd[0]) and torch.equal(guard2[1:-1], fwd[1])
    for v in (guard[0], guard[-1], guard2[0], guard2[-1]):
        assert bool((v == 3).all())
    assert bool((big[need:] == 0x5A).all())


def test_status_word_stays_clean():
    lib, _ = _lib()
    word = ctypes.c_uint32(9)
    lib.nm_norm_bwd_device_status(None, ctypes.byref(word))
    assert word.value == 0


@pytest.mark.parametrize("kind", [1, 2])
@pytest.mark.parametrize("T,D", [(333, 520), (40, 2048)])
def test_the_open_part_of_far_gates(kind, T, D):
    """f32 without the post norm, gates of magnitude up to 80. Counted in half steps u: the product branch g_post 1, exp 2 ulp
    (4 u), 1 + exp 1, the quotient 1 and a second-order rest, x_out's own rounding 1: under 9 u of |s x| + |open y|."""
    s = _inputs(0, T, D, kind, False, True)
    g = torch.Generator(device="cuda").manual_seed(T)
    s["gate"] = torch.rand(s["gate"].shape, generator=g, device="cuda") * 160 - 80
    x_out = _fwd(0, kind, s)[0]
    d = {k: v.double() for k, v in s.items() if v is not None}
    carried = d["scale"] * d["x_in"]
    through = torch.sigmoid(d["gate"][:, None] if kind == 1 else d["gate"]) * d["branch"]
    _near("x_out", x_out, carried + through, 9 * U * (carried.abs() + through.abs()))


@pytest.mark.parametrize("dtype", [1, 0])
@pytest.mark.parametrize("kind", [1, 2])
def test_an_infinite_branch_passes_the_gate(dtype, kind):
    s = _inputs(dtype, 6, 264, kind, False, True)
    s["branch"][1, 5], s["branch"][3, 260], s["branch"][4, 7] = float("inf"), float("-inf"), float("nan")
    x_out, a_next, _, _ = _fwd(dtype, kind, s)
    assert float(x_out[1, 5]) == float("inf") and float(x_out[3, 260]) == float("-inf") and bool(x_out[4, 7].isnan())
    assert int(x_out.isfinite().logical_not().sum()) == 3
    for row in (1, 3):      # the statistic of a row with an infinity is 0: its finite elements become 0
        assert int((a_next[row] == 0).sum()) == 263 and int(a_next[row].isnan().sum()) == 1
    assert bool(a_next[[0, 2, 5]].isfinite().all()) and bool(a_next[4].isnan().all())
