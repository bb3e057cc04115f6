"""nm_ce_distill against the formulas of include/marincpp/kernels/distill_head.hpp in float64.

Tolerances, u = 2^-24. A logit is a sum of D products that the tensor core adds in D / 16 steps, each of which may cut the
running sum by one f32 step, 2 u of its size: |dz| <= Z = (D / 16 + 2) 2 u sum|x w|. The statistics move by as much, and by the
roundings of their exponents (a few u times the size of the numbers in them; 64 u (1 + |lse| + |t| / tau + |z| / tau) covers
exponentials of 2 ulp, the merges and the sums). So a probability is off by at most rho = 2 Z / tau + that, relative, a
divergence by (1 + mass) times rho, an element of n by rho times the sizes of its parts. dW takes n as two bf16 terms (each
half a step: 2^-8 * 2^-8 < 2^-15 would be the bound of the second term's rounding of a first remainder of 2^-8: 2^-16 of n) and adds
at most 1152 rows x 2 terms before it drains: 1152 / 8 steps of 2 u. dX takes the first term alone (2^-8 of n; both in short calls), adds up to V / 8 steps
of 2 u (all shares together), and is stored with half a step of bf16."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BIG_NEG = -(2 ** 31)


def _case(T, D, V, K, seed=0, teacher=torch.float32, pad=0.0, tau=1.0, given_lse=False):
    g = torch.Generator(device="cuda").manual_seed(1000 * seed + T + V)
    x = torch.randn(T, D, generator=g, device="cuda").bfloat16()
    w = (torch.randn(V, D, generator=g, device="cuda") * (2.0 / D ** 0.5)).bfloat16()
    ids = torch.randint(0, V, (T, K), generator=g, device="cuda").int()          # repeats within a row happen
    t = (torch.randn(T, K, generator=g, device="cuda") * 2 + 3).to(teacher)
    drop = torch.rand(T, K, generator=g, device="cuda") < pad
    ids = torch.where(drop, torch.where(torch.rand(T, K, generator=g, device="cuda") < 0.5, -1, V).int(), ids)
    t = torch.where(drop, torch.full_like(t, float("nan")), t)
    lse = None
    if given_lse:
        lse = torch.logsumexp(torch.nan_to_num(t.double(), nan=-1e9) / tau, 1).float() + 0.5
    targets = torch.randint(-1, V, (T,), generator=g, device="cuda").int()
    weight = (torch.rand(T, generator=g, device="cuda") < 0.9).float() * (0.5 + torch.rand(T, generator=g, device="cuda"))
    gs = torch.tensor([1.0 / max(T, 1)], device="cuda")
    return dict(x=x, w=w, ids=ids, t=t, lse=lse, targets=targets, weight=weight, gs=gs, tau=tau)


def _formula(c, soft, hard, ignore=BIG_NEG):
    """Everything in float64, with the sizes that the tolerances are made of."""
    x, w = c["x"].double(), c["w"].double()
    V, tau = w.shape[0], c["tau"]
    z = x @ w.T
    Z = (x.shape[1] / 16 + 2) * 2 * U * (x.abs() @ w.abs().T).amax(1, keepdim=True)
    logp = torch.log_softmax(z / tau, 1)
    lse = torch.logsumexp(z / tau, 1, keepdim=True)
    live = (c["weight"] != 0).double()[:, None]
    ok = (c["ids"] >= 0) & (c["ids"] < V)
    at = c["ids"].long().clamp(0, V - 1)
    t = torch.where(ok, c["t"].double(), torch.full_like(z[:, :1], 0.0)) / tau
    masked = t.masked_fill(~ok, float("-inf"))
    some = ok.any(1, keepdim=True)
    norm = c["lse"].double()[:, None] if c["lse"] is not None else torch.where(some, torch.logsumexp(masked, 1, keepdim=True), 0.0)
    q = torch.where(ok, torch.exp(t - norm), torch.zeros_like(t))
    kl = torch.where(q > 0, q * (t - norm - logp.gather(1, at)), torch.zeros_like(q)).sum(1, keepdim=True)   # 0 log 0 = 0
    t = torch.where(q > 0, t, torch.zeros_like(t))
    mass = q.sum(1, keepdim=True)
    y = c["targets"].long()[:, None]
    lab = ((y >= 0) & (y < V) & (y != ignore)).double() * (hard != 0)
    lse1 = torch.logsumexp(z, 1, keepdim=True)
    ce = lse1 - z.gather(1, y.clamp(0, V - 1))
    loss = soft * tau ** 2 * kl + hard * lab * ce
    wt = c["weight"].double()[:, None]
    p = torch.exp(logp)
    dense = soft * tau * mass * p + hard * lab * torch.softmax(z, 1)
    sparse = torch.zeros_like(z).scatter_add_(1, at, q * soft * tau).scatter_add_(1, y.clamp(0, V - 1), hard * lab)
    size = z.abs().amax(1, keepdim=True)
    rho = 2 * Z / min(tau, 1.0) + 64 * U * (1 + lse.abs() + lse1.abs() + t.abs().amax(1, keepdim=True) + size / min(tau, 1.0))
    n = wt * (dense - sparse)
    dn = wt * (dense + sparse) * rho
    return dict(z=z, lse=lse[:, 0], kl=(kl * live)[:, 0], loss=(loss * live)[:, 0], n=n, dn=dn, rho=rho[:, 0],
                mass=mass[:, 0], lab=lab[:, 0])


def _close(name, got, want, tol):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{name}: {int(bad.sum())} of {bad.numel()} outside, worst {float((err / tol).max()):.2f} x"


def _check(c, soft, hard, out, dx=None, dw=None, ignore=BIG_NEG, dx0=None, dw0=None):
    f = _formula(c, soft, hard, ignore)
    g = float(c["gs"].double())
    _close("lse", out[2], f["lse"], f["rho"])
    kl_tol = (1 + f["mass"]) * f["rho"]
    _close("kl", out[1], f["kl"], kl_tol)
    _close("loss", out[0], f["loss"], soft * c["tau"] ** 2 * kl_tol + hard * 2 * f["rho"] + 4 * U * f["loss"].abs())
    n, dn = f["n"].abs(), f["dn"]
    if dw is not None:
        want, size = g * (f["n"].T @ c["x"].double()), g * (n.T @ c["x"].double().abs())
        tol = g * (dn.T @ c["x"].double().abs()) + (2.0 ** -16 + (1152 / 8 + c["x"].shape[0] / 1024 + 4) * 2 * U) * size
        if dw0 is not None:
            want = want + dw0.double()
            tol = tol + (c["x"].shape[0] / 1024 + 2) * U * (dw0.double().abs() + size)
        _close("dw", dw, want, tol + 1e-30)
    if dx is not None:
        want, size = g * (f["n"] @ c["w"].double()), g * (n @ c["w"].double().abs())
        tol = g * (dn @ c["w"].double().abs()) + (2.0 ** -8 + (c["w"].shape[0] / 8 + 40) * 2 * U) * size
        if dx0 is not None:
            want = want + dx0.double()
        _close("dx", dx, want, tol + 2.0 ** -8 * (want.abs() + tol) + 1e-30)


def _run(c, soft=1.0, hard=0.0, fwd=False, **kw):
    from gpu_common import lib, nmce
    T, V, D = c["x"].shape[0], c["w"].shape[0], c["w"].shape[1]
    dx = dw = None
    if not fwd:
        dx = kw.pop("dx", torch.full((T, D), float("nan"), dtype=torch.bfloat16, device="cuda"))
        dw = kw.pop("dw", torch.zeros(V, D, device="cuda"))
    out = nmce.distill_call(lib(), c["x"], c["w"], c["ids"], c["t"], c["weight"], c["gs"], tau=c["tau"], soft=soft, hard=hard,
                            teacher_lse=c["lse"], targets=c["targets"] if hard else None, dx=dx, dw=dw, **kw)
    return out, dx, dw


@pytest.mark.parametrize("T,D,V,K,tau,hard,given,teacher,pad,chunk", [
    (1, 8, 1, 1, 1.0, 0.5, False, torch.float32, 0.0, 8192),
    (1, 64, 300, 1, 2.0, 0.0, False, torch.bfloat16, 0.0, 8192),
    (33, 136, 1003, 5, 0.7, 0.3, True, torch.float32, 0.3, 8192),
    (130, 512, 8256, 64, 2.0, 0.5, False, torch.bfloat16, 0.1, 8192),
    (700, 256, 5000, 16, 1.0, 0.0, False, torch.float32, 0.5, 256),
    (2100, 264, 600, 33, 4.0, 0.25, True, torch.bfloat16, 0.2, 8192),
    (257, 2048, 9, 512, 1.5, 0.5, False, torch.float32, 0.0, 100),
    (1025, 72, 255, 100, 1.0, 1.0, False, torch.float32, 0.9, 1025),
    (300, 1024, 20001, 8, 1.0, 0.5, False, torch.float32, 0.0, 8192),
])
def test_against_float64(T, D, V, K, tau, hard, given, teacher, pad, chunk):
    c = _case(T, D, V, K, teacher=teacher, pad=pad, tau=tau, given_lse=given)
    out, dx, dw = _run(c, soft=1.0 - 0.5 * hard, hard=hard, chunk=chunk)
    _check(c, 1.0 - 0.5 * hard, hard, out, dx, dw)
    again, dx2, dw2 = _run(c, soft=1.0 - 0.5 * hard, hard=hard, chunk=chunk)
    assert all(torch.equal(a, b) for a, b in zip(out, again)) and torch.equal(dx, dx2) and torch.equal(dw, dw2)
    ev, _, _ = _run(c, soft=1.0 - 0.5 * hard, hard=hard, chunk=chunk, fwd=True)
    _check(c, 1.0 - 0.5 * hard, hard, ev)
    assert torch.equal(ev[2], out[2])


def test_full_vocabulary_and_pairs_of_ctas():
    """Sizes at which the logits run on CTA pairs and dX in one share and in several."""
    for T, D, V in ((4100, 1024, 16384), (150, 512, 128256)):
        c = _case(T, D, V, 32, tau=2.0)
        out, dx, dw = _run(c, soft=0.5, hard=0.5)
        _check(c, 0.5, 0.5, out, dx, dw)


def test_rows_that_do_not_count():
    c = _case(200, 128, 777, 12, tau=1.0)
    c["weight"][3], c["weight"][150] = 0.0, 0.0
    c["ids"][7], c["t"][7] = -1, float("nan")                    # nothing listed
    c["t"][8] = float("-inf")                                    # listed, with no mass
    c["t"][9, :6] = float("-inf")
    c["ids"][10] = 5                                             # one id twelve times
    c["t"][3] = float("nan")                                     # a row without weight is not looked at
    c["targets"][11], c["targets"][12], c["targets"][13] = 42, -7, 777
    out, dx, dw = _run(c, soft=0.7, hard=0.3, ignore_index=42)
    c["t"][3] = 0.0
    c["t"][8] = 0.0
    c["ids"][8] = -1
    _check(c, 0.7, 0.3, out, dx, dw, ignore=42)
    for r in (3, 150):
        assert float(out[0][r]) == 0 and float(out[1][r]) == 0 and bool((dx[r] == 0).all())
    assert float(out[1][7]) == 0 and float(out[1][8]) == 0
    soft_only, dx_s, _ = _run(c, soft=1.0, hard=0.0)
    assert float(soft_only[0][7]) == 0 and bool((dx_s[7] == 0).all())


def test_a_student_equal_to_its_teacher_has_no_divergence():
    """Every id listed with the student's own logits: kl and gradient vanish up to the roundings."""
    T, D, V = 20, 64, 96
    c = _case(T, D, V, V, tau=1.0)
    c["ids"] = torch.arange(V, device="cuda").int().repeat(T, 1)
    c["t"] = (c["x"].double() @ c["w"].double().T).float()
    c["weight"] = torch.ones(T, device="cuda")
    out, dx, dw = _run(c)
    _check(c, 1.0, 0.0, out, dx, dw)
    f = _formula(c, 1.0, 0.0)
    assert bool((out[1].abs() <= 2 * f["rho"]).all())


def test_extreme_temperatures_and_logits():
    for tau in (0.05, 50.0):
        c = _case(60, 64, 500, 10, tau=tau)
        out, dx, dw = _run(c, soft=1.0, hard=0.5)
        _check(c, 1.0, 0.5, out, dx, dw)
        assert all(bool(torch.isfinite(v).all()) for v in (*out, dx, dw))
    c = _case(60, 64, 500, 10, tau=1.0)
    c["x"] = (c["x"].float() * 30).bfloat16()                    # logits of some hundreds: probabilities of 0 and 1
    out, dx, dw = _run(c, soft=1.0, hard=0.5)
    _check(c, 1.0, 0.5, out, dx, dw)
    assert all(bool(torch.isfinite(v).all()) for v in (*out, dx, dw))


def test_added_to_what_is_there_and_over_x():
    c = _case(500, 256, 2000, 20, tau=2.0)
    g = torch.Generator(device="cuda").manual_seed(5)
    dx0 = (torch.randn(500, 256, generator=g, device="cuda") * 1e-3).bfloat16()
    dw0 = torch.randn(2000, 256, generator=g, device="cuda") * 1e-3
    out, dx, dw = _run(c, dx=dx0.clone(), dw=dw0.clone(), acc_dx=True, chunk=200)
    _check(c, 1.0, 0.0, out, dx, dw, dx0=dx0, dw0=dw0)
    plain, want, _ = _run(c, chunk=200)
    over = dict(c, x=c["x"].clone())
    out2, dx2, _ = _run(over, dx=over["x"], chunk=200)
    assert torch.equal(dx2, want) and torch.equal(out2[0], plain[0])
    # either gradient alone
    from gpu_common import lib, nmce
    only = torch.empty_like(want)
    nmce.distill_call(lib(), c["x"], c["w"], c["ids"], c["t"], c["weight"], c["gs"], tau=2.0, dx=only, chunk=200)
    assert torch.equal(only, want)


def test_chunks_do_not_change_loss_and_sum_of_chunks():
    from gpu_common import nmce, lib
    c = _case(1000, 128, 3000, 9, tau=1.5)
    ref, _, _ = _run(c, soft=0.5, hard=0.5)
    for chunk in (1000, 333, 1):
        if chunk == 1:
            c1 = {k: v[:40] if torch.is_tensor(v) and v.dim() and v.shape[0] == 1000 else v for k, v in c.items()}
            out, _, _ = _run(c1, soft=0.5, hard=0.5, chunk=1)
            assert torch.equal(out[0], ref[0][:40])
            continue
        part = torch.empty(-(-1000 // chunk), device="cuda")
        out, _, _ = _run(c, soft=0.5, hard=0.5, chunk=chunk, loss_partial=part)
        assert all(torch.equal(a, b) for a, b in zip(out, ref))
        want = (out[0].double() * c["weight"].double()).sum()
        assert abs(float(part.double().sum() - want)) <= 1000 * U * float((out[0].double() * c["weight"].double()).abs().sum())
    assert lib() and nmce


def test_many_short_rows():
    """More rows in a chunk than one launch's grid has in its second extent."""
    c = _case(70001, 8, 16, 2, tau=1.0)
    out, dx, dw = _run(c, soft=1.0, hard=0.25, chunk=70001)
    _check(c, 1.0, 0.25, out, dx, dw)


def test_gradient_against_differences():
    """The directional derivative of sum weight loss along random directions of x and W, as a central difference of the
    float64 formula; the gradients carry the tolerances above (dX half a step of bf16 twice, 2^-7 of its size), the
    difference a term of h^2 = 1e-8."""
    c = _case(24, 64, 200, 6, tau=2.0)
    _, dx, dw = _run(c, soft=0.6, hard=0.4)
    g = torch.Generator(device="cuda").manual_seed(1)

    def value(x, w):
        f = _formula(dict(c, x=x, w=w), 0.6, 0.4)
        return float((f["loss"] * c["weight"].double()).sum() * c["gs"].double())

    h = 1e-4
    x, w = c["x"].double(), c["w"].double()
    for grad, move in ((dx, lambda s, d: (x + s * d, w)), (dw, lambda s, d: (x, w + s * d))):
        d = torch.randn(grad.shape, generator=g, device="cuda", dtype=torch.float64)
        slope = (value(*move(h, d)) - value(*move(-h, d))) / (2 * h)
        size = float((grad.double() * d).abs().sum())
        assert abs(slope - float((grad.double() * d).sum())) <= (2.0 ** -7 if grad is dx else 1e-4) * size


def test_captured_and_replayed():
    from gpu_common import lib, nmce
    c = _case(300, 128, 1500, 10, tau=2.0)
    want, dx_w, dw_w = _run(c, soft=0.5, hard=0.5)                # the first call on a device is made outside a capture
    T, D, V, K = 300, 128, 1500, 10
    ws = torch.empty(lib().nm_ce_distill_workspace_bytes(T, D, V, K, 128, 0), dtype=torch.uint8, device="cuda")
    dx, dw = torch.zeros_like(dx_w), torch.zeros_like(dw_w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dw.zero_()
        out = nmce.distill_call(lib(), c["x"], c["w"], c["ids"], c["t"], c["weight"], c["gs"], tau=2.0, soft=0.5, hard=0.5,
                                targets=c["targets"], dx=dx, dw=dw, chunk=128, ws=ws,
                                stream=torch.cuda.current_stream().cuda_stream, check=False)
    for seed in (0, 3):
        fresh = _case(300, 128, 1500, 10, seed=seed, tau=2.0)
        for k in ("x", "w", "ids", "t", "targets", "weight"):
            c[k].copy_(fresh[k])
        graph.replay()
        torch.cuda.synchronize()
        want, dx_w, dw_w = _run(fresh, soft=0.5, hard=0.5, chunk=128)
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(dx, dx_w) and torch.equal(dw, dw_w)


def test_two_calls_at_once_with_a_workspace_each():
    from gpu_common import lib, nmce
    cs = [_case(600, 256, 4000, 16, seed=s, tau=1.5) for s in (1, 2)]
    want = [_run(c) for c in cs]
    ws = [torch.empty(lib().nm_ce_distill_workspace_bytes(600, 256, 4000, 16, 8192, 0), dtype=torch.uint8, device="cuda")
          for _ in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    got = [[torch.empty_like(want[0][1]), torch.zeros_like(want[0][2])] for _ in cs]
    torch.cuda.synchronize()
    for i, c in enumerate(cs):
        with torch.cuda.stream(streams[i]):
            nmce.distill_call(lib(), c["x"], c["w"], c["ids"], c["t"], c["weight"], c["gs"], tau=1.5, dx=got[i][0],
                              dw=got[i][1], ws=ws[i], stream=streams[i].cuda_stream, check=False)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(got[i][0], want[i][1]) and torch.equal(got[i][1], want[i][2])


@pytest.mark.parametrize("fwd", [False, True])
def test_nothing_outside_the_buffers_is_written(fwd):
    from gpu_common import lib, nmce
    T, D, V, K = 190, 72, 1001, 7
    c = _case(T, D, V, K, tau=2.0)
    need = lib().nm_ce_distill_workspace_bytes(T, D, V, K, 64, int(fwd))
    ws = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    dx = torch.full((T + 2, D), 3.0, dtype=torch.bfloat16, device="cuda")
    dw = torch.zeros(V + 2, D, device="cuda")
    dw[0], dw[-1] = 9.0, 9.0
    kw = {} if fwd else dict(dx=dx[1:-1], dw=dw[1:-1])
    out = nmce.distill_call(lib(), c["x"], c["w"], c["ids"], c["t"], c["weight"], c["gs"], tau=2.0, soft=0.5, hard=0.5,
                            targets=c["targets"], chunk=64, ws=ws[:need], **kw)
    _check(c, 0.5, 0.5, out, None if fwd else dx[1:-1], None if fwd else dw[1:-1])
    assert bool((ws[need:] == 0x5A).all())
    assert bool((dx[0] == 3).all()) and bool((dx[-1] == 3).all()) and bool((dw[0] == 9).all()) and bool((dw[-1] == 9).all())
    status = ctypes.c_uint32(7)
    lib().nm_ce_device_status(nmce.ptr(ws), None, ctypes.byref(status))
    assert status.value == 0


def test_no_gradient_asked_of_a_full_call():
    """forward_only = 0 with neither dx nor dw: the losses of a forward-only call, in a workspace with a logits store."""
    from gpu_common import lib, nmce
    T, D, V, K = 300, 64, 5, 40                                  # more entries than vocabulary
    c = _case(T, D, V, K, tau=1.0)
    ev, _, _ = _run(c, soft=0.5, hard=0.5, fwd=True)
    ws = torch.empty(lib().nm_ce_distill_workspace_bytes(T, D, V, K, 128, 0), dtype=torch.uint8, device="cuda")
    out = torch.empty(3, T, device="cuda")
    p = nmce.ptr
    lib().nm_ce_distill(0, p(c["x"]), p(c["w"]), p(c["ids"]), p(c["t"]), None, p(c["targets"]), p(c["weight"]), None, 1.0, 0.5,
                        0.5, p(out[0]), p(out[1]), p(out[2]), None, None, 0, None, 0, T, D, V, K, 128, BIG_NEG, p(ws),
                        ws.numel(), None)
    assert all(torch.equal(a, b) for a, b in zip(out, ev))


def test_soft_and_hard_alone():
    c = _case(150, 128, 900, 9, tau=2.0)
    for soft, hard in ((0.0, 1.0), (2.5, 0.0), (0.0, 0.0)):
        out, dx, dw = _run(c, soft=soft, hard=hard)
        _check(c, soft, hard, out, dx, dw)
        if soft == hard == 0.0:
            assert bool((dx == 0).all()) and bool((dw == 0).all())


def test_no_rows():
    from gpu_common import lib, nmce
    assert lib().nm_ce_distill(0, *[None] * 8, 1.0, 1.0, 0.0, *[None] * 5, 0, None, 0, 0, 64, 100, 4, 128, 0, None, 0, None) == 0
    assert nmce
