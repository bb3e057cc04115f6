"""The backward at rows of very large and very small size: its results are products of powers of rstd with sums over the row, of
which each is representable while r^3 alone is not. Tolerances as for rows of ordinary size: a value that is built from
magnitudes M in f32 is off by at most 64 half steps of M (row sums of 520 terms: 5 fma a lane, a pair, 8 butterfly steps; ten
products around them), and half a step of bf16 when stored in it."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U, EPS = 2.0 ** -24, 1e-5


@pytest.mark.parametrize("dtype", [1, 0])
@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("size", [1e-6, 1e10, 1e13, 1e15])
def test_projections_of_large_rows(dtype, kind, size):
    from gpu_common import lib, nmce
    T, D = 37, 520
    dt = (torch.float32, torch.bfloat16)[dtype]
    half = 2.0 ** -8 if dtype else 0.0
    g = torch.Generator(device="cuda").manual_seed(5)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    branch, x_in, da = (n(T, D) * size).to(dt), (n(T, D) * size).to(dt), n(T, D).to(dt)
    gate = (None, n(T).to(dt), n(T, D).to(dt))[kind]
    g_next, g_post = (1 + 0.2 * n(D)).to(dt), (1 + 0.2 * n(D)).to(dt)
    nan = lambda v: None if v is None else torch.full_like(v, float("nan"))  # noqa: E731
    x_out, a_next, dx_in, dbranch, dgate = nan(x_in), nan(x_in), nan(x_in), nan(x_in), nan(gate)
    rp, rn = torch.full((T,), float("nan"), device="cuda"), torch.full((T,), float("nan"), device="cuda")
    p = nmce.ptr
    lib().nm_gated_tail_fwd(dtype, kind, p(branch), p(x_in), p(gate), None, p(g_post), p(g_next), p(x_out), p(a_next), p(rp), p(rn),
                            T, D, EPS, None)
    lib().nm_gated_tail_bwd(dtype, kind, None, p(da), p(x_in), p(branch), p(gate), None, p(g_post), p(g_next), p(rp), p(rn), p(dx_in),
                            p(dbranch), p(dgate), None, None, None, T, D, None, 0, None)
    b, xo, r, q = branch.double(), x_out.double(), rn.double()[:, None], rp.double()[:, None]
    assert bool(((r - (xo.square().mean(1, keepdim=True) + EPS).rsqrt()).abs() <= 64 * U * r).all())
    av, gp = g_next.double() * da.double(), g_post.double()
    m = r * av - xo * r ** 3 * (xo * av).sum(1, keepdim=True) / D
    M = r * av.abs() + xo.abs() * r ** 3 * (xo * av).abs().sum(1, keepdim=True) / D

    def close(name, got, want, tol):
        bad = ~((got.double() - want).abs() <= tol)
        assert not bool(bad.any()), f"{name}: {int(bad.sum())} outside, {float(((got.double() - want).abs() / tol).max()):.2f} x"

    close("dx_in", dx_in, m, half * m.abs() + 64 * U * M)
    gd = None if gate is None else gate.double() if kind == 2 else gate.double()[:, None]
    on = torch.ones_like(m) if gd is None else torch.sigmoid(gd)
    pv, P = gp * on * m, gp.abs() * on * M
    want = q * pv - b * q ** 3 * (b * pv).sum(1, keepdim=True) / D
    mag = q * P + b.abs() * q ** 3 * (b.abs() * P).sum(1, keepdim=True) / D
    close("dbranch", dbranch, want, half * want.abs() + 128 * U * mag)
    if kind:
        slope = torch.sigmoid(gd) * torch.sigmoid(-gd)
        want, mag = m * b * q * gp * slope, M * (b * q * gp).abs() * slope
        if kind == 1:
            want, mag = want.sum(1), mag.sum(1)
        close("dgate", dgate, want, half * want.abs() + 128 * U * mag)
