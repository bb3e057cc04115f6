"""nm_ce_distill where the logits have a large common part: a softmax does not depend on it, so neither may its accuracy. The
logits are exact in f32 (few bits in x and W, D = 8), so that only the statistics are measured.

Tolerances, u = 2^-24, H the mean distance from the maximum in nats, X the distance of an element.
- The factor log2e / tau is off by 2 u, the exponent of an element by a rounding of itself: 3 u X; ex2 by 2 ulp, 4 u.
- A sum takes at most 10 additions in a chunk of 32 columns, and a step to another maximum (ex2 4 u, a product, an addition, and
  3 u of its size, whose sum over the steps of a term is at most its X) for 4 chunks, the other half of the tile, two tiles of a
  strip and the strips: 10 + 6 (4 + 1 + 2 + 1), a butterfly of 5: 63, with the element's own ex2 67. So S is off by
  sigma = (67 + 6 H) u.
- lse = max / tau + log S: a quotient, an addition, the log: u (|max / tau| + |lse| + 4 log S) + sigma.
- log p: sigma + 4 u (1 + |log p| + log S). log q: the difference from the largest entry and the quotient by tau, its sum (exp 2
  ulp, K / 32 + 5 additions), its log: u (4 |d| + 4 log K + 30).
- n: the dense part by sigma + (3 X + 12) u, the listed part by that of log q + 8 u, and what is below 2^-126 counts as 0.
- dW takes n as two bf16 terms, 2^-16, and adds T rows of them in the tensor core: under 24 u for 24 rows."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
T, V, D, K = 24, 1003, 8, 7


def _case(offset, tau, teacher_offset, given, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    unit = 1.0 / 64 if tau < 0.5 else 1.0 / 8
    x = torch.randint(-2, 3, (T, D), generator=g, device="cuda").float()
    x[:, 0] = torch.tensor([1.0, 0.5, -1.0] * (T // 3), device="cuda")
    w = torch.randint(-8, 9, (V, D), generator=g, device="cuda").float() * unit
    w[:, 0] = offset
    assert bool((x.bfloat16().float() == x).all()) and bool((w.bfloat16().float() == w).all())
    ids = torch.stack([torch.randperm(V, generator=g, device="cuda")[:K] for _ in range(T)]).int()
    t = teacher_offset + torch.randn(T, K, generator=g, device="cuda") * 3 * tau
    lse = (torch.logsumexp(t.double() / tau, 1) + 0.4).float() if given else None
    y = torch.randint(0, V, (T,), generator=g, device="cuda").int()
    return x.bfloat16(), w.bfloat16(), ids, t, lse, y


def _close(name, got, want, tol):
    ratio = (got.double() - want).abs() / tol
    assert bool((ratio <= 1).all()), f"{name}: worst {float(ratio.max()):.2f} x the tolerance"


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("hard", [0.0, 0.5])
@pytest.mark.parametrize("offset,tau,teacher_offset", [(0.0, 1.0, 0.0), (300.0, 1.0, 200.0), (50.0, 0.05, 40.0), (-300.0, 0.3, -100.0),
                                                       (20.0, 2.0, 20.0)])
def test_a_common_part_of_the_logits_costs_no_accuracy(offset, tau, teacher_offset, hard, given):
    from gpu_common import lib, nmce
    x, w, ids, t, tlse, y = _case(offset, tau, teacher_offset, given)
    weight, gs = torch.ones(T, device="cuda"), torch.full((1,), 1.0 / T, device="cuda")
    tau = float(torch.tensor(tau))                         # the value that the call gets
    z = x.double() @ w.double().T

    def softmax(s):
        m = s.amax(1, keepdim=True)
        total = torch.exp(s - m).sum(1, keepdim=True)
        logp = s - m - total.log()
        h = (torch.exp(logp) * (m - s)).sum(1, keepdim=True)
        return m, total, logp, (67 + 6 * h) * U

    top, total, logp, sigma = softmax(z / tau)
    top1, total1, logp1, sigma1 = softmax(z)
    lse = top + total.log()
    td = t.double() / tau
    norm = tlse.double()[:, None] if given else torch.logsumexp(td, 1, keepdim=True)
    lq, q = td - norm, torch.exp(td - norm)
    e_lq = U * (4 * (td - td.amax(1, keepdim=True)).abs() + 4 * math.log(K) + 30 + 2 * lq.abs())
    lp = logp.gather(1, ids.long())
    e_lp = sigma + 4 * U * (1 + lp.abs() + total.log())
    kl = (q * (lq - lp)).sum(1)
    e_kl = (q * ((lq - lp).abs() * (e_lq + (K / 32 + 10) * U) + e_lq + e_lp + 2 * U * (lq.abs() + lp.abs()))).sum(1)
    ce = -logp1.gather(1, y.long()[:, None])[:, 0]
    e_ce = sigma1[:, 0] + U * (4 + 4 * ce.abs() + 4 * total1.log()[:, 0])
    loss = 0.5 * tau * tau * kl + hard * ce
    e_loss = 0.5 * tau * tau * (e_kl + 4 * U * kl.abs()) + hard * e_ce + 2 * U * loss.abs()
    mass = q.sum(1, keepdim=True)
    n = 0.5 * tau * mass * torch.exp(logp) + hard * torch.exp(logp1)
    e_n = 0.5 * tau * mass * torch.exp(logp) * (sigma + e_lq.amax(1, keepdim=True) + U * (12 + 3 * (top - z / tau)))
    e_n = e_n + hard * torch.exp(logp1) * (sigma1 + U * (12 + 3 * (top1 - z)))
    listed = 0.5 * tau * q
    n = n.scatter_add(1, ids.long(), -listed).scatter_add(1, y.long()[:, None], torch.full((T, 1), -hard, device="cuda").double())
    e_n = e_n.scatter_add(1, ids.long(), listed * (e_lq + 8 * U)) + 4 * U * n.abs() + 2.0 ** -126
    dw = n.T @ x.double() / T
    e_dw = (e_n.T @ x.double().abs() + (2.0 ** -16 + 24 * U) * (n.abs().T @ x.double().abs())) / T

    for fwd in (False, True):
        dx_out = None if fwd else torch.full((T, D), float("nan"), dtype=torch.bfloat16, device="cuda")
        dw_out = None if fwd else torch.zeros(V, D, device="cuda")
        out = nmce.distill_call(lib(), x, w, ids, t, weight, gs, tau=tau, soft=0.5, hard=hard, teacher_lse=tlse,
                                targets=y if hard else None, dx=dx_out, dw=dw_out)
        _close("lse", out[2], lse[:, 0], U * (top.abs() + lse.abs() + 4 * total.log())[:, 0] + sigma[:, 0])
        _close("kl", out[1], kl, e_kl)
        _close("loss", out[0], loss, e_loss)
        if not fwd:
            _close("dw", dw_out, dw, e_dw)
            assert bool(torch.isfinite(dx_out).all())
