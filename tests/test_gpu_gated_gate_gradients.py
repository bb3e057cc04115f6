"""f32 storage: what the gate passes back at gates up to 80 in magnitude, where sigmoid and its complement are far apart.

With da_next = 0 the gradient m of x_out is dx_out exactly, and without a post-norm
  dbranch = on m,   dgate = m branch on off  (summed over the row for a gate per token),   on = sigmoid(gate), off = 1 - on.
Counted in half steps u = 2^-24: exp 2 ulp (4 u), 1 + exp 1, the quotient 1 and a second-order rest: on within 7 u; off = exp on:
the same and a product, 8 u. dbranch: on and a product, 8 u of it. dgate of an element: on, off and four products, 19 u; of a
token: 19 u and the row's sum, under 25 u of the terms' magnitudes. A value below 2^-126 is held in steps of 2^-149, whatever its
size: a product that lands there is off by up to half of one, 2^-150 (dx_out = 6e-6 at gate -78.7 gives 4e-40, where half a step
is 28 u of the value). dbranch is one such product; dgate multiplies it by branch and by at most 1 and rounds twice more."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U, STEP = 2.0 ** -24, 2.0 ** -149


@pytest.mark.parametrize("kind", [1, 2])
@pytest.mark.parametrize("scaled", [False, True])
@pytest.mark.parametrize("T,D", [(64, 8), (333, 520), (40, 2048)])
def test_gradients_at_far_gates(kind, scaled, T, D):
    from gpu_common import lib, nmce
    g = torch.Generator(device="cuda").manual_seed(T + D + kind)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    branch, x_in, dx_out, g_next = n(T, D), n(T, D), n(T, D), 1 + 0.2 * n(D)
    scale = 0.8 + 0.1 * n(D) if scaled else None
    gate = torch.rand(*((T,) if kind == 1 else (T, D)), generator=g, device="cuda") * 160 - 80
    gate.view(-1)[:6] = torch.tensor([80.0, -80.0, 0.0, 1e-30, -17.25, 30.0], device="cuda")
    da, rn = torch.zeros(T, D, device="cuda"), torch.ones(T, device="cuda")
    dx_in, dbranch = (torch.full((T, D), float("nan"), device="cuda") for _ in range(2))
    dgate = torch.full_like(gate, float("nan"))
    p = nmce.ptr
    lib().nm_gated_tail_bwd(0, kind, p(dx_out), p(da), p(x_in), p(branch), p(gate), p(scale), None, p(g_next), None, p(rn), p(dx_in),
                            p(dbranch), p(dgate), None, None, None, T, D, None, 0, None)
    gd = gate.double() if kind == 2 else gate.double()[:, None]
    m, b = dx_out.double(), branch.double()
    on, off = torch.sigmoid(gd), torch.sigmoid(-gd)
    want = m * on
    tol = 8 * U * want.abs() + STEP / 2
    assert bool(((dbranch.double() - want).abs() <= tol).all()), float(((dbranch.double() - want).abs() / tol).max())
    want = m * b * on * off
    tol = 19 * U * want.abs() + STEP / 2 * (2 + b.abs())
    if kind == 1:
        want, tol = want.sum(1), (19 + 25) * U * want.abs().sum(1) + STEP / 2
    assert bool(((dgate.double() - want).abs() <= tol).all()), float(((dgate.double() - want).abs() / tol).max())
    want = m if scale is None else m * scale.double()
    assert bool(((dx_in.double() - want).abs() <= U * want.abs()).all())
