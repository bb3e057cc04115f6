"""Workloads of the operators on either side of the fused head: embedding lookup and its gradient, the gated sandwich
tail (post-norm, gate, scaled residual, next pre-norm) forward and backward, and the distillation head over a teacher's
top logits. Sizes are those of this repository's benchmark and tests (vocabularies 8256, 64256 and 128256, hidden sizes
512 to 2048, 65536- and 131072-row steps) and odd ones between them.

With own = False, run() computes the operators with elementary torch operations in 32 bits; with own = True it calls
the library.
"""
import math
import os
import sys

import torch

own = False

_REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_LIB = []
_EPS = 1e-5
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _framework():
    """(nmce, lib), loaded once per process."""
    if not _LIB:
        sys.path.insert(0, os.path.join(_REPO, "marin.cpp_b200"))
        import nmce
        _LIB.extend((nmce, nmce.Lib()))
    return _LIB


# ---------------------------------------------------------------------------------------------------- cases
def _embed(name, back, T, D, V, dtype, accumulate=False, pad=0.0):
    return {"name": name, "op": "embed_bwd" if back else "embed_fwd", "T": T, "D": D, "V": V, "dtype": dtype,
            "accumulate": accumulate, "pad": pad, "scale": math.sqrt(D)}


def _tail(name, back, T, D, dtype, gating, post=True, scaled=True):
    return {"name": name, "op": "tail_bwd" if back else "tail_fwd", "T": T, "D": D, "dtype": dtype, "gating": gating,
            "post": post, "scaled": scaled}


def _distill(name, T, D, V, K, tau, hard, given_lse=False, teacher="f32", pad=0.0, back=True):
    return {"name": name, "op": "distill" if back else "distill_fwd", "T": T, "D": D, "V": V, "K": K, "tau": tau,
            "hard": hard, "given_lse": given_lse, "teacher": teacher, "pad": pad}


def listed():
    return [
        # the tokens of one short evaluation prompt
        _embed("embed_fwd_short", False, 64, 512, 8256, "bf16"),
        # one training step of the benchmark's flagship shape
        _embed("embed_fwd_step", False, 131072, 2048, 128256, "bf16"),
        # a ragged microbatch with padding ids, added into a gradient that a tied head has begun; f32 activations
        _embed("embed_bwd_ragged_add", True, 2125, 768, 64256, "f32", accumulate=True, pad=0.1),
        # the gradient of one training step of the flagship shape
        _embed("embed_bwd_step", True, 131072, 2048, 128256, "bf16", pad=0.01),
        # a few rows of an odd width, f32 storage: the call whose latency counts
        _tail("tail_fwd_short", False, 17, 520, "f32", "token"),
        # one layer of a training step
        _tail("tail_fwd_step", False, 65536, 2048, "bf16", "element"),
        # a ragged microbatch in f32 storage with one gate per token
        _tail("tail_bwd_ragged", True, 2125, 1024, "f32", "token"),
        # the backward of one layer of a training step
        _tail("tail_bwd_step", True, 65536, 2048, "bf16", "element"),
        # evaluating a narrow student against stored teacher logits: no gradients
        _distill("distill_eval", 2125, 512, 128256, 16, 1.0, 0.5, back=False),
        # a handful of rows on a small vocabulary: the call whose latency counts
        _distill("distill_short", 16, 512, 8256, 8, 1.0, 0.0),
        # stored teacher logits with their normaliser and padded lists, ragged microbatch
        _distill("distill_ragged", 2125, 1024, 64256, 64, 1.5, 0.0, given_lse=True, teacher="bf16", pad=0.15),
        # one microbatch of the flagship shape, soft and hard targets mixed
        _distill("distill_step", 8192, 2048, 128256, 64, 2.0, 0.5),
    ]


def _spread(rng, lo, hi):
    """A whole number whose logarithm is spread evenly over [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    return _spread(rng, lo // 8, hi // 8) * 8


def draw(rng):
    op = rng.choice(["embed_fwd", "embed_bwd", "tail_fwd", "tail_bwd", "distill", "distill", "distill_fwd"])
    if op.startswith("embed"):
        c = _embed("", op == "embed_bwd", _spread(rng, 1, 131072), _width(rng, 64, 2048), _spread(rng, 512, 128256),
                   rng.choice(["bf16", "f32"]), rng.random() < 0.5 and op == "embed_bwd",
                   rng.choice([0.0, 0.05, 0.5]))
        if c["dtype"] == "f32":
            c["T"] = min(c["T"], 65536)
    elif op.startswith("tail"):
        D = _width(rng, 64, 4096)
        dtype = rng.choice(["bf16", "bf16", "f32"])
        T = min(_spread(rng, 1, 65536), 65536 * 2048 // D // (2 if dtype == "f32" else 1))
        c = _tail("", op == "tail_bwd", T, D, dtype, rng.choice(["none", "token", "element"]), rng.random() < 0.7,
                  rng.random() < 0.7)
    else:
        c = _distill("", _spread(rng, 1, 8192), _width(rng, 64, 2048), _spread(rng, 512, 128256), _spread(rng, 1, 128),
                     rng.choice([1.0, 0.7, 2.0, 4.0]), rng.choice([0.0, 0.25, 0.5]), rng.random() < 0.5,
                     rng.choice(["f32", "bf16"]), rng.choice([0.0, 0.2]), op == "distill")
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------- inputs
def _tokens(g, T, V, pad):
    """Ids whose frequency falls as 1 / rank, and a share of padding ids (-1)."""
    u = torch.rand(T, generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(V + 1.0)) - 1.0).long().clamp_(0, V - 1).int()
    return torch.where(torch.rand(T, generator=g, device="cuda") < pad, torch.full_like(ids, -1), ids)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(std)

    s = dict(case)
    T, D = case["T"], case["D"]
    op = case["op"]
    if op.startswith("embed"):
        V, dt = case["V"], _TYPES[case["dtype"]]
        s["tokens"] = _tokens(g, T, V, case["pad"])
        if op == "embed_fwd":
            s["table"] = normal(V, D, dtype=dt, std=0.02)
            s["out"] = torch.empty(T, D, dtype=dt, device="cuda")
        else:
            s["dy"] = normal(T, D, dtype=dt, std=1e-3)
            s["dtable"] = normal(V, D, dtype=torch.float32, std=1e-2)   # what a tied head has left there
            s["ws"] = torch.empty(_scratch(case), dtype=torch.uint8, device="cuda")
    elif op.startswith("tail"):
        dt = _TYPES[case["dtype"]]
        s["branch"], s["x_in"] = normal(T, D, dtype=dt, std=2.0), normal(T, D, dtype=dt, std=1.5)
        shape = {"none": None, "token": (T,), "element": (T, D)}[case["gating"]]
        s["gate"] = None if shape is None else normal(*shape, dtype=dt, std=2.0)
        s["g_next"] = (1.0 + normal(D, dtype=torch.float32, std=0.1)).to(dt)
        s["g_post"] = (1.0 + normal(D, dtype=torch.float32, std=0.1)).to(dt) if case["post"] else None
        s["scale"] = (0.9 + normal(D, dtype=torch.float32, std=0.05)).to(dt) if case["scaled"] else None
        if op == "tail_fwd":
            s["x_out"], s["a_next"] = torch.empty_like(s["x_in"]), torch.empty_like(s["x_in"])
            s["rstd"] = torch.empty(2, T, device="cuda")
        else:
            s["dx_out"], s["da_next"] = normal(T, D, dtype=dt, std=1e-2), normal(T, D, dtype=dt, std=1e-2)
            s["rstd"] = torch.stack(_tail_forward(s)[2:])     # the statistics that the forward call has left
            s["dx_in"], s["dbranch"] = torch.empty_like(s["x_in"]), torch.empty_like(s["branch"])
            s["dgate"] = None if s["gate"] is None else torch.empty_like(s["gate"])
            s["dgains"] = torch.empty(3, D, device="cuda")
            s["ws"] = torch.empty(_scratch(case), dtype=torch.uint8, device="cuda")
    else:
        V, K = case["V"], case["K"]
        s["x"], s["w"] = normal(T, D), normal(V, D, std=0.02)
        start = torch.randint(0, V, (T, 1), generator=g, device="cuda")
        step = (torch.rand(T, 1, generator=g, device="cuda") * (V // K)).long() + 1
        s["ids"] = ((start + step * torch.arange(K, device="cuda")) % V).int()      # distinct within a row
        t = (8.0 + 2.0 * torch.randn(T, K, generator=g, device="cuda")).sort(dim=1, descending=True).values
        s["tlse"] = None
        if case["given_lse"]:
            s["tlse"] = torch.logsumexp(t.double() / case["tau"], dim=1).float() + 0.3   # a quarter of the mass is not listed
        drop = torch.rand(T, K, generator=g, device="cuda") < case["pad"]
        s["ids"] = torch.where(drop, torch.full_like(s["ids"], -1), s["ids"])
        s["teacher_logits"] = torch.where(drop, torch.full_like(t, float("nan")), t).to(_TYPES[case["teacher"]])
        s["targets"] = _tokens(g, T, V, 0.02)
        s["weight"] = (torch.rand(T, generator=g, device="cuda") < 0.95).float()
        s["gscale"] = 1.0 / s["weight"].sum().clamp_min(1.0).reshape(1)
        s["loss"] = torch.empty(3, T, device="cuda")
        if op == "distill":
            s["dx"] = torch.empty(T, D, dtype=torch.bfloat16, device="cuda")
            s["dw"] = torch.empty(V, D, device="cuda")
        s["ws"] = torch.empty(_scratch(case), dtype=torch.uint8, device="cuda")
    return s


def _chunk(case):
    return min(case["T"], 8192)


def _scratch(case):
    """Room for the scratch a program plans beside its tensors (an upper bound that both forms are given alike)."""
    T, D = case["T"], case["D"]
    if case["op"] == "embed_bwd":
        return 64 * T + 4 * D * (T // 16 + 64) + (1 << 20)
    if case["op"] == "tail_bwd":
        return 3 * 4 * D * (min(T, 1024) + 64) + (1 << 20)
    rows, V = _chunk(case), case["V"]
    return 4 * rows * (V + 128) + rows * (32 * (V // 256 + 2) + 32 * case["K"] + 1024) + 16 * 8192 * D + (4 << 20)


# ---------------------------------------------------------------------------------------------------- plain forms
def _tail_forward(s):
    """(x_out, a_next, rstd_post, rstd_next) in f32; x_out holds values of the storage type, which the next norm reads."""
    b, x = s["branch"].float(), s["x_in"].float()
    rp = torch.rsqrt((b * b).mean(1) + _EPS)
    y = b if s["g_post"] is None else b * rp[:, None] * s["g_post"].float()
    if s["gate"] is not None:
        gate = s["gate"].float()
        y = y / (1.0 + torch.exp(-(gate[:, None] if gate.dim() == 1 else gate)))
    xo = ((x if s["scale"] is None else x * s["scale"].float()) + y).to(s["x_in"].dtype).float()
    rn = torch.rsqrt((xo * xo).mean(1) + _EPS)
    return xo, xo * rn[:, None] * s["g_next"].float(), rp, rn


def _plain(s):
    op = s["op"]
    if op == "embed_fwd":
        t = s["tokens"].long()
        rows = s["table"][t.clamp_min(0)].float() * s["scale"]
        return (rows * (t >= 0)[:, None]).to(s["table"].dtype)
    if op == "embed_bwd":
        t = s["tokens"].long()
        keep = t >= 0
        d = s["dtable"]
        if not s["accumulate"]:
            d.zero_()
        return d.index_add_(0, t[keep], s["dy"][keep].float() * s["scale"])
    if op == "tail_fwd":
        xo, a, rp, rn = _tail_forward(s)
        dt = s["x_in"].dtype
        return [xo.to(dt), a.to(dt), rn] + ([] if s["g_post"] is None else [rp])
    if op == "tail_bwd":
        return _plain_tail_bwd(s)
    return _plain_distill(s)


def _plain_tail_bwd(s):
    dt, D = s["x_in"].dtype, s["D"]
    b, x, da, rp, rn = s["branch"].float(), s["x_in"].float(), s["da_next"].float(), s["rstd"][0], s["rstd"][1]
    xo = _tail_forward(s)[0]
    a = s["g_next"].float() * da
    xr = xo * rn[:, None]
    mid = s["dx_out"].float() + rn[:, None] * (a - xr * (a * xr).sum(1, keepdim=True) / D)
    dg_next = (da * xr).sum(0)
    dx_in = mid if s["scale"] is None else mid * s["scale"].float()
    dscale = None if s["scale"] is None else (mid * x).sum(0)
    yn = b * rp[:, None]
    y = b if s["g_post"] is None else yn * s["g_post"].float()
    dgate, dy = None, mid
    if s["gate"] is not None:
        gate = s["gate"].float()
        gate = gate[:, None] if gate.dim() == 1 else gate
        on, off = 1.0 / (1.0 + torch.exp(-gate)), 1.0 / (1.0 + torch.exp(gate))
        dy = mid * on
        dgate = mid * y
        dgate = (dgate.sum(1) * (on * off)[:, 0] if s["gate"].dim() == 1 else dgate * on * off).to(dt)
    dg_post, db = None, dy
    if s["g_post"] is not None:
        dg_post = (dy * yn).sum(0)
        ap = dy * s["g_post"].float()
        db = rp[:, None] * (ap - yn * (ap * yn).sum(1, keepdim=True) / D)
    return [v for v in (dx_in.to(dt), db.to(dt), dgate, dg_next, dg_post, dscale) if v is not None]


def _plain_distill(s):
    V, tau, hard, soft = s["V"], s["tau"], s["hard"], 1.0 - s["hard"]
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    zt = z / tau
    m = zt.amax(1, keepdim=True)
    lse = m + torch.exp(zt - m).sum(1, keepdim=True).log()
    listed_ids = s["ids"].long()
    ok = (listed_ids >= 0) & (listed_ids < V)
    at = listed_ids.clamp(0, V - 1)
    t = s["teacher_logits"].float() / tau
    t = torch.where(ok, t, torch.full_like(t, -math.inf))
    if s["tlse"] is None:
        top = t.amax(1, keepdim=True)
        top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
        norm = top + torch.exp(t - top).sum(1, keepdim=True).log()
    else:
        norm = s["tlse"][:, None]
    q = torch.where(ok, torch.exp(t - norm), torch.zeros_like(t))
    kl = torch.where(q > 0, q * ((t - norm) - (zt.gather(1, at) - lse)), torch.zeros_like(q)).sum(1)
    w_t = s["weight"]
    counted = w_t != 0
    loss = soft * tau * tau * kl
    y = s["targets"].long()
    labelled = (y >= 0) & (y < V)
    if hard != 0:
        m1 = z.amax(1, keepdim=True)
        lse1 = m1 + torch.exp(z - m1).sum(1, keepdim=True).log()
        loss = loss + hard * torch.where(labelled, lse1[:, 0] - z.gather(1, y.clamp(0, V - 1)[:, None])[:, 0],
                                         torch.zeros_like(kl))
    out = [torch.where(counted, loss, torch.zeros_like(loss)), torch.where(counted, kl, torch.zeros_like(kl)), lse[:, 0]]
    if s["op"] == "distill_fwd":
        return out
    n = torch.exp(zt - lse) * (q.sum(1, keepdim=True) * (soft * tau))
    n.scatter_add_(1, at, q * (-soft * tau))
    if hard != 0:
        on = labelled.float()[:, None] * hard
        n += torch.exp(z - lse1) * on
        n.scatter_add_(1, y.clamp(0, V - 1)[:, None], -on)
    n *= (w_t * s["gscale"])[:, None]
    return out + [(n @ w).to(torch.bfloat16), n.t() @ x]


# ---------------------------------------------------------------------------------------------------- the library
_GATE = {"none": 0, "token": 1, "element": 2}


def _own(s):
    nmce, lib = _framework()
    p = nmce.ptr
    op, T, D = s["op"], s["T"], s["D"]
    st = nmce.VP(torch.cuda.current_stream().cuda_stream)
    if op == "embed_fwd":
        lib.nm_embed_fwd(int(s["dtype"] == "bf16"), p(s["table"]), p(s["tokens"]), p(s["out"]), s["scale"], T, D, s["V"], st)
        return s["out"]
    if op == "embed_bwd":
        lib.nm_embed_bwd(int(s["dtype"] == "bf16"), p(s["dy"]), p(s["tokens"]), p(s["dtable"]), s["scale"],
                         int(s["accumulate"]), T, D, s["V"], p(s["ws"]), s["ws"].numel(), st)
        return s["dtable"]
    if op == "tail_fwd":
        rstd_post = None if s["g_post"] is None else s["rstd"][0]
        lib.nm_gated_tail_fwd(int(s["dtype"] == "bf16"), _GATE[s["gating"]],
                              p(s["branch"]), p(s["x_in"]), p(s["gate"]), p(s["scale"]), p(s["g_post"]), p(s["g_next"]),
                              p(s["x_out"]), p(s["a_next"]), p(rstd_post), p(s["rstd"][1]), T, D, _EPS, st)
        return [s["x_out"], s["a_next"], s["rstd"][1]] + ([] if rstd_post is None else [rstd_post])
    if op == "tail_bwd":
        dg = s["dgains"]
        dg_post = None if s["g_post"] is None else dg[1]
        dscale = None if s["scale"] is None else dg[2]
        lib.nm_gated_tail_bwd(int(s["dtype"] == "bf16"), _GATE[s["gating"]], p(s["dx_out"]), p(s["da_next"]), p(s["x_in"]),
                              p(s["branch"]), p(s["gate"]), p(s["scale"]), p(s["g_post"]), p(s["g_next"]),
                              p(s["rstd"][0]), p(s["rstd"][1]), p(s["dx_in"]), p(s["dbranch"]), p(s["dgate"]), p(dg[0]),
                              p(dg_post), p(dscale), T, D, p(s["ws"]), s["ws"].numel(), st)
        return [v for v in (s["dx_in"], s["dbranch"], s["dgate"], dg[0], dg_post, dscale) if v is not None]
    back = op == "distill"
    loss = s["loss"]
    if back:
        s["dw"].zero_()
    lib.nm_ce_distill(int(s["teacher"] == "bf16"), p(s["x"]), p(s["w"]), p(s["ids"]), p(s["teacher_logits"]), p(s["tlse"]),
                      p(s["targets"]) if s["hard"] != 0 else None, p(s["weight"]), p(s["gscale"]), s["tau"],
                      1.0 - s["hard"], s["hard"], p(loss[0]), p(loss[1]), p(loss[2]), None, p(s.get("dx")), 0,
                      p(s.get("dw")), int(not back), T, D, s["V"], s["K"], _chunk(s), -(2 ** 31), p(s["ws"]),
                      s["ws"].numel(), st)
    return [loss[0], loss[1], loss[2]] + ([s["dx"], s["dw"]] if back else [])


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---------------------------------------------------------------------------------------------------- work, exact values
def work(case):
    T, D = case["T"], case["D"]
    op = case["op"]
    if op.startswith("embed"):
        size, V = (2 if case["dtype"] == "bf16" else 4), case["V"]
        if op == "embed_fwd":
            return {"bytes": 4 * T + size * D * (T + min(T, V)), "flops": T * D}
        touched = 8 * D * min(T, V) if case["accumulate"] else 4 * D * V
        return {"bytes": 4 * T + size * D * T + touched, "flops": 2 * T * D}
    if op.startswith("tail"):
        size = 2 if case["dtype"] == "bf16" else 4
        gates = 1 if case["gating"] == "element" else 0
        if op == "tail_fwd":
            return {"bytes": size * T * D * (4 + gates) + 8 * T, "flops": 12 * T * D}
        return {"bytes": size * T * D * (6 + 2 * gates) + 8 * T, "flops": 30 * T * D}
    V, K = case["V"], case["K"]
    bytes_ = 2 * (T * D + V * D) + T * K * (8 if case["teacher"] == "f32" else 6) + 24 * T
    if op == "distill_fwd":
        return {"bytes": bytes_, "flops": 2 * T * D * V}
    return {"bytes": bytes_ + 2 * T * D + 4 * V * D, "flops": 6 * T * D * V}


def _rounded(v, dtype):
    """The value as the storage type holds it, with the gradient passing straight through."""
    return v + (v.detach().to(dtype).to(v.dtype) - v.detach())


def _exact_tail(s, back):
    dt = s["x_in"].dtype
    leaf = {k: s[k].double().requires_grad_(back) for k in ("branch", "x_in", "gate", "g_next", "g_post", "scale")
            if s[k] is not None}
    rms = lambda v: torch.sqrt(v.square().sum(-1, keepdim=True) / v.shape[-1] + _EPS)  # noqa: E731
    h = leaf["branch"]
    if "g_post" in leaf:
        h = h / rms(h) * leaf["g_post"]
    if "gate" in leaf:
        h = h * torch.sigmoid(leaf["gate"] if leaf["gate"].dim() == 2 else leaf["gate"].unsqueeze(1))
    x_out = _rounded(leaf["x_in"] * leaf["scale"] + h if "scale" in leaf else leaf["x_in"] + h, dt)
    a = x_out / rms(x_out) * leaf["g_next"]
    if not back:
        out = [x_out, a, 1.0 / rms(x_out)[:, 0]]
        return out + ([1.0 / rms(leaf["branch"])[:, 0]] if "g_post" in leaf else [])
    total = (x_out * s["dx_out"].double()).sum() + (a * s["da_next"].double()).sum()
    names = [k for k in ("x_in", "branch", "gate", "g_next", "g_post", "scale") if k in leaf]
    return list(torch.autograd.grad(total, [leaf[k] for k in names]))


def _exact_distill(s, back):
    V, tau, hard = s["V"], s["tau"], s["hard"]
    x, w = s["x"].double().requires_grad_(back), s["w"].double().requires_grad_(back)
    z = x @ w.T
    logp = torch.log_softmax(z / tau, dim=1)
    lse = (z[:, 0] / tau - logp[:, 0]).detach()
    inside = (s["ids"] >= 0) & (s["ids"] < V)
    t = (s["teacher_logits"].double() / tau).masked_fill(~inside, -1e30)
    logq = torch.log_softmax(t, dim=1) if s["tlse"] is None else t - s["tlse"].double().unsqueeze(1)
    q = torch.exp(logq) * inside
    kl = (q * (logq.masked_fill(~inside, 0.0) - logp.gather(1, s["ids"].long().clamp(0, V - 1)))).sum(1)
    loss = (1.0 - hard) * tau ** 2 * kl
    if hard != 0:
        y = s["targets"].long()
        good = ((y >= 0) & (y < V)).double()
        loss = loss - hard * good * torch.log_softmax(z, dim=1).gather(1, y.clamp(0, V - 1).unsqueeze(1)).squeeze(1)
    on = (s["weight"] != 0).double()
    out = [(loss * on).detach(), (kl * on).detach(), lse]
    if not back:
        return out
    total = (loss * s["weight"].double()).sum() * s["gscale"].double().sum()
    return out + list(torch.autograd.grad(total, [x, w]))


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "embed_fwd":
        t = s["tokens"].long()
        return torch.where((t < 0).unsqueeze(1), 0.0, s["table"].double()[t.clamp(min=0)] * case["scale"])
    if op == "embed_bwd":
        # rows in token order, then differences of running sums at the ends of each token's run
        t, order = torch.sort(s["tokens"].long(), stable=True)
        run_sum = torch.cat([torch.zeros(1, s["D"], dtype=torch.float64, device="cuda"),
                             torch.cumsum(s["dy"].double()[order], 0)])
        ids = torch.arange(s["V"], device="cuda")
        lo, hi = torch.searchsorted(t, ids), torch.searchsorted(t, ids, right=True)
        total = (run_sum[hi] - run_sum[lo]) * case["scale"]
        return total + s["dtable"].double() if case["accumulate"] else total
    if op.startswith("tail"):
        return _exact_tail(s, op == "tail_bwd")
    return _exact_distill(s, op == "distill")
