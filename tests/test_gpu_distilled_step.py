"""One step of a distilled student through the operators as a program uses them: embedding -> gated sandwich tail (whose branch
is a fixed elementwise block here) -> distillation head -> back through all three, in bf16, with the embedding tied to the head:
its gradient is added into the dW that the head has begun. The reference is the same step in float64 by automatic
differentiation, with the activations rounded where the operators store them (straight through).

Tolerances, relative in the 2-norm. Each gradient of the chain is stored in bf16 after every operator (half a step, 2^-8, at most,
of each element), so the distances of dX, the tail's gradients and dE's rows add up: two stored roundings behind dx_in and
dbranch (dX holds two itself: the gradient's and its own), three behind what reaches the embedding. The head's own dW holds none
of them (f32 through two bf16 terms). The activations' roundings are the same on both sides; where the two sides round to
neighbours (a value within 2^-20 of a tie: under one in 2^10 of them, by a step of 2^-7), a further 2^-7 * 2^-5 may appear."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8
FLIP = 2.0 ** -12
EPS = 1e-5


def _rounded(v):
    return v + (v.detach().bfloat16().double() - v.detach())


def _rel(a, b):
    return float((a.double() - b).norm() / b.norm())


@pytest.mark.parametrize("T,D,V,K", [(777, 512, 8256, 16), (130, 264, 1003, 5)])
def test_distilled_step(T, D, V, K):
    from gpu_common import lib, nmce
    L, p = lib(), nmce.ptr
    g = torch.Generator(device="cuda").manual_seed(T)
    W = (torch.randn(V, D, generator=g, device="cuda") * 0.05).bfloat16()          # tied: embedding and head
    tokens = torch.randint(-1, V, (T,), generator=g, device="cuda").int()
    targets = torch.randint(0, V, (T,), generator=g, device="cuda").int()
    ids = torch.randint(0, V, (T, K), generator=g, device="cuda").int()
    teacher = torch.randn(T, K, generator=g, device="cuda") * 2
    weight = (tokens >= 0).float()
    gs = 1.0 / weight.sum().reshape(1)
    gate = torch.randn(T, D, generator=g, device="cuda").bfloat16()
    g_post, g_next, scale = ((1 + 0.1 * torch.randn(D, generator=g, device="cuda")).bfloat16() for _ in range(3))
    branch_w = torch.randn(D, generator=g, device="cuda").bfloat16()               # the block: branch = round(x * branch_w)
    factor = float(D ** 0.5)

    # ---- the operators
    x = torch.empty(T, D, dtype=torch.bfloat16, device="cuda")
    L.nm_embed_fwd(1, p(W), p(tokens), p(x), factor, T, D, V, None)
    branch = (x.float() * branch_w.float()).bfloat16()
    x_out, a = torch.empty_like(x), torch.empty_like(x)
    rp, rn = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    L.nm_gated_tail_fwd(1, 2, p(branch), p(x), p(gate), p(scale), p(g_post), p(g_next), p(x_out), p(a), p(rp), p(rn), T, D, EPS,
                        None)
    da, dw = torch.empty_like(a), torch.zeros(V, D, device="cuda")
    loss, kl, lse = nmce.distill_call(L, a, W, ids, teacher, weight, gs, tau=2.0, soft=0.5, hard=0.5, targets=targets, dx=da, dw=dw,
                                      chunk=256)
    head = dw.clone()
    dx, db, dgate = torch.empty_like(x), torch.empty_like(x), torch.empty_like(gate)
    dgn, dgp, dsc = (torch.empty(D, device="cuda") for _ in range(3))
    ws = torch.empty(L.nm_gated_tail_workspace_bytes(T, D), dtype=torch.uint8, device="cuda")
    L.nm_gated_tail_bwd(1, 2, None, p(da), p(x), p(branch), p(gate), p(scale), p(g_post), p(g_next), p(rp), p(rn), p(dx), p(db),
                        p(dgate), p(dgn), p(dgp), p(dsc), T, D, p(ws), ws.numel(), None)
    dx_all = (dx.float() + db.float() * branch_w.float()).bfloat16()
    ws2 = torch.empty(L.nm_embed_bwd_workspace_bytes(T, D, V), dtype=torch.uint8, device="cuda")
    L.nm_embed_bwd(1, p(dx_all), p(tokens), p(dw), factor, 1, T, D, V, p(ws2), ws2.numel(), None)
    word = ctypes.c_uint32(1)
    L.nm_norm_bwd_device_status(None, ctypes.byref(word))
    assert word.value == 0

    # ---- float64
    leaf = {k: v.double().requires_grad_() for k, v in
            dict(E=W, H=W, gate=gate, g_post=g_post, g_next=g_next, scale=scale).items()}
    t = tokens.long()
    xe = _rounded(torch.where((t >= 0)[:, None], leaf["E"][t.clamp(min=0)] * factor, torch.zeros((), dtype=torch.float64, device="cuda")))
    xe.retain_grad()
    br = _rounded(xe * branch_w.double())
    br.retain_grad()
    n = br * (br.square().mean(1, keepdim=True) + EPS).rsqrt() * leaf["g_post"]
    xo = _rounded(leaf["scale"] * xe + torch.sigmoid(leaf["gate"]) * n)
    an = _rounded(xo * (xo.square().mean(1, keepdim=True) + EPS).rsqrt() * leaf["g_next"])
    an.retain_grad()
    z = an @ leaf["H"].T
    logq = torch.log_softmax(teacher.double() / 2.0, 1)
    klr = (logq.exp() * (logq - torch.log_softmax(z / 2.0, 1).gather(1, ids.long()))).sum(1)
    ce = -torch.log_softmax(z, 1).gather(1, targets.long()[:, None])[:, 0]
    lossr = 0.5 * 4.0 * klr + 0.5 * ce
    (lossr * weight.double()).sum().mul(gs.double()).backward()

    on = weight.double()
    assert _rel(loss, (lossr * on).detach()) < 2 * FLIP and _rel(kl, (klr * on).detach()) < 2 * FLIP
    assert _rel(da, an.grad) < 2 * HALF + FLIP
    assert _rel(head, leaf["H"].grad) < 2 * FLIP
    for name, got in (("gate", dgate), ("scale", dsc), ("g_next", dgn), ("g_post", dgp)):
        assert _rel(got, leaf[name].grad) < 3 * HALF + FLIP, name
    assert _rel(db, br.grad) < 3 * HALF + FLIP
    assert _rel(dx_all, xe.grad) < 5 * HALF + FLIP
    assert _rel(dw.double() - head.double(), leaf["E"].grad) < 5 * HALF + FLIP
    assert bool((da[tokens < 0] == 0).all())             # rows of padding have no weight
