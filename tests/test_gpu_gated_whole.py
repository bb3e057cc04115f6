"""The gated tail's float64 checks in a form that a NaN or an element left unwritten cannot pass: outputs begin as NaN, and a
value counts as right only when its error is known to be within the tolerance. Formulas, inputs and tolerances are those of
test_gpu_gated.py."""
import pytest
import torch

import test_gpu_gated as base

pytestmark = pytest.mark.gpu


def _near(name, got, want, tol):
    good = (got.double() - want).abs() <= tol
    assert good.shape == want.shape and bool(good.all()), (
        f"{name}: {int((~good).sum())} of {good.numel()} outside, {int(got.isnan().sum())} of them NaN")


def _nan(v):
    return None if v is None else torch.full_like(v, float("nan"))


def _both(dtype, kind, s):
    fwd = base._fwd(dtype, kind, s, x_out=_nan(s["x_in"]), a_next=_nan(s["x_in"]))
    f32 = lambda v: None if v is None else _nan(v.float())  # noqa: E731
    out = {"dx_in": _nan(s["x_in"]), "dbranch": _nan(s["x_in"]), "dgate": _nan(s["gate"]), "dg_next": f32(s["g_next"]),
           "dg_post": f32(s["g_post"]), "dscale": f32(s["scale"])}
    return fwd, base._bwd(dtype, kind, s, fwd[2], fwd[3], out=out)


def test_the_check_sees_a_nan():
    with pytest.raises(AssertionError):
        _near("x", torch.tensor([1.0, float("nan")]), torch.ones(2).double(), torch.ones(2).double())


@pytest.mark.parametrize("dtype", [1, 0])
@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("post,scaled,carried", [(True, True, True), (False, True, True), (True, False, False),
                                                 (False, False, True)])
@pytest.mark.parametrize("T,D", [(1, 8), (17, 520), (301, 64), (40, 2048), (1201, 256), (5, 4096), (700, 1032)])
def test_against_float64(monkeypatch, dtype, kind, post, scaled, carried, T, D):
    monkeypatch.setattr(base, "_near", _near)
    s = base._inputs(dtype, T, D, kind, post, scaled, carried=carried)
    base._check(dtype, kind, s, *_both(dtype, kind, s))


@pytest.mark.parametrize("dtype,T,D", [(1, 5, 8192), (1, 700, 4104), (0, 5, 4096), (0, 333, 2056), (1, 5000, 1024),
                                       (0, 2125, 1024), (1, 9, 8184)])
@pytest.mark.parametrize("kind", [0, 1, 2])
def test_wide_rows_and_many_rows(monkeypatch, dtype, T, D, kind):
    monkeypatch.setattr(base, "_near", _near)
    s = base._inputs(dtype, T, D, kind, True, True)
    base._check(dtype, kind, s, *_both(dtype, kind, s))
