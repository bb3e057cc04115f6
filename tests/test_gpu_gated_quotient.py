"""The gate's quotient alone: with x_in = 0 and no post-norm x_out = branch / (1 + exp(-gate)) in f32 storage, rounded no further.

In half steps u = 2^-24: exp 2 ulp (4 u), 1 + exp 1, the quotient 1 and 2^-43 of what its one correction leaves: 6 u and 2^-19 u.
A value below 2^-126 is held in steps of 2^-149: half of one more. Both directions form it by the same operations."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("kind", [1, 2])
@pytest.mark.parametrize("T,D,spread", [(4000, 264, 80.0), (3000, 520, 4.0)])
def test_bound_of_the_quotient(kind, T, D, spread):
    from gpu_common import lib, nmce
    g = torch.Generator(device="cuda").manual_seed(T)
    branch = torch.randn(T, D, generator=g, device="cuda") * torch.exp(4 * torch.randn(T, D, generator=g, device="cuda"))
    gate = (torch.rand(*((T,) if kind == 1 else (T, D)), generator=g, device="cuda") * 2 - 1) * spread
    x_in, x_out = torch.zeros(T, D, device="cuda"), torch.full((T, D), float("nan"), device="cuda")
    p = nmce.ptr
    lib().nm_gated_tail_fwd(0, kind, p(branch), p(x_in), p(gate), None, None, None, p(x_out), None, None, None, T, D, 1e-5, None)
    gd = gate.double() if kind == 2 else gate.double()[:, None]
    want = branch.double() / (1 + torch.exp(-gd))
    tol = (6 + 2.0 ** -19) * U * want.abs() + 2.0 ** -150
    assert bool(((x_out.double() - want).abs() <= tol).all()), float(((x_out.double() - want).abs() / tol).max())
