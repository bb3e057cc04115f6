"""dX of the distillation head over the full vocabulary, where one accumulator adds up tens of thousands of products: two figures
of the whole matrix that single elements cannot show.

2-norm. The roundings of n to bf16 (its first term, calls of more than 128 rows) and of dX itself are at most 2^-8 of each value
and independent, so the error's norm is at most 2^-8 (|dX| + |n o W|), with |n o W|^2 the sum of n^2 W^2 over all products (root
mean squares stand a factor sqrt 3 below).
Slope of dX against float64. Those roundings average out: deviation s, s^2 = sum dX_i^2 (2^-16 / 3) (dX_i^2 + (n^2 W^2)_i) / |dX|^4;
five of them. What does not average is the cutting of the accumulator (one f32 step of 2 u, u = 2^-24, at most per product of 16 along
the vocabulary), and the error of n from that of the logits, 2 / tau times (D / 16 + 2) 2 u sum|x w| at most."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("T,D", [(16400, 256), (8192, 1024), (300, 512), (128, 512)])
def test_norm_and_slope(T, D):
    from gpu_common import lib, nmce
    V, K, tau = 128256, 16, 2.0
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, D, generator=g, device="cuda").bfloat16()
    w = (torch.randn(V, D, generator=g, device="cuda") * (2.0 / D ** 0.5)).bfloat16()
    ids = torch.randint(0, V, (T, K), generator=g, device="cuda").int()
    t = torch.randn(T, K, generator=g, device="cuda") * 2 + 3
    one, gs = torch.ones(T, device="cuda"), torch.ones(1, device="cuda")
    dx = torch.full((T, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(lib().nm_ce_distill_workspace_bytes(T, D, V, K, T, 0), dtype=torch.uint8, device="cuda")
    nmce.distill_call(lib(), x, w, ids, t, one, gs, tau=tau, dx=dx, chunk=T, ws=ws)
    del ws
    wd, w2 = w.double(), w.double().square()
    dot = norm2 = err2 = prod2 = var = 0.0
    logits = 0.0
    for r in range(0, T, 1024):
        at = slice(r, min(r + 1024, T))
        z = x[at].double() @ wd.T
        n = torch.softmax(z / tau, 1).mul_(tau)
        del z
        q = torch.softmax(t[at].double() / tau, 1)
        n.scatter_add_(1, ids[at].long(), -tau * q)
        want = n @ wd
        products = n.square_() @ w2
        got = dx[at].double()
        dot, norm2 = dot + float((got * want).sum()), norm2 + float(want.square().sum())
        err2, prod2 = err2 + float((got - want).square().sum()), prod2 + float(products.sum())
        var += float((want.square() * (want.square() + products)).sum()) * 2.0 ** -16 / 3
        logits = max(logits, float((x[at].double().norm(dim=1)).max() * wd.norm(dim=1).max()))    # >= sum|x w|
    assert err2 ** 0.5 <= 2.0 ** -8 * (norm2 ** 0.5 + prod2 ** 0.5)
    slope = dot / norm2
    bound = V / 16 * 2 * U + 5 * var ** 0.5 / norm2 + 2 / tau * (D / 16 + 2) * 2 * U * logits
    print(f"dX {T} x {D}: 2-norm {(err2 / norm2) ** 0.5:.2e}, slope - 1 = {slope - 1:.2e}, bound {bound:.2e}, "
          f"deviation {var ** 0.5 / norm2:.1e}")
    assert abs(slope - 1) <= bound
