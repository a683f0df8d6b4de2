"""What is measured of the categorical-policy operators: their cases, inputs, plain forms and calls.

Three operators on rows of logits [N, V] (ppo_radiotherapy_amd.categorical):

* sample:  an action per row from given uniform numbers, under temperature, top-k, top-p and min-p
* ppo:     the clipped PPO loss of the actions with its gradient (fused, through autograd, or the loss alone)
* distill: KL from a teacher's top logits with its gradient (the same three forms)
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = float(1 << 40)  # sampling weights are whole numbers of 2^-40 of the row's largest
NARROW = 1024          # rows up to this long: the plain forms' sums over a row are in 64 bits throughout


def listed():
    return [
        # a rollout step of 4096 envs whose 6 action components are discretised to 11 bins each
        {"name": "sample actions", "op": "sample", "n": 24576, "v": 11, "dtype": "f32", "filter": "none", "pad": 0},
        # one sequence's next token: latency counts
        {"name": "sample one token", "op": "sample", "n": 1, "v": 131072, "dtype": "bf16", "filter": "k+p", "pad": 0},
        # a rollout batch of token policies, every row with parameters of its own
        {"name": "sample batch mixed", "op": "sample", "n": 256, "v": 131072, "dtype": "bf16", "filter": "mixed", "pad": 0},
        # a ragged batch: odd vocabulary, rows inside a wider buffer
        {"name": "sample odd f32 top-p", "op": "sample", "n": 63, "v": 50021, "dtype": "f32", "filter": "p", "pad": 11},
        # a PPO minibatch of 32768 samples with 6 discretised action components
        {"name": "ppo actions", "op": "ppo", "form": "fused", "n": 196608, "v": 11, "dtype": "f32", "ref": False, "pad": 0},
        # a large minibatch of tokens, loss and gradient in one call
        {"name": "ppo tokens", "op": "ppo", "form": "fused", "n": 4096, "v": 131072, "dtype": "bf16", "ref": True, "pad": 0},
        # a model trained through autograd in full precision, with a KL term to a reference policy
        {"name": "ppo autograd f32", "op": "ppo", "form": "autograd", "n": 1023, "v": 32003, "dtype": "f32", "ref": True, "pad": 0},
        # log-probabilities, entropies and the loss of stored tokens, no gradient
        {"name": "ppo score f16", "op": "ppo", "form": "loss", "n": 2048, "v": 50021, "dtype": "f16", "ref": False, "pad": 3},
        # a micro-batch of a few tokens over a wide vocabulary
        {"name": "ppo few tokens", "op": "ppo", "form": "fused", "n": 8, "v": 131072, "dtype": "bf16", "ref": False, "pad": 0},
        # a small policy distilled over its discretised actions
        {"name": "distill actions", "op": "distill", "form": "fused", "n": 32768, "v": 64, "k": 8, "dtype": "f32", "lse": False, "pad": 0},
        # a token policy distilled from a stored teacher's top logits
        {"name": "distill tokens", "op": "distill", "form": "fused", "n": 2048, "v": 131072, "k": 64, "dtype": "bf16", "lse": True, "pad": 0},
        # the same through autograd, ragged sizes, odd row strides
        {"name": "distill autograd f16", "op": "distill", "form": "autograd", "n": 777, "v": 50021, "k": 33, "dtype": "f16", "lse": False, "pad": 5},
    ]


def draw(rng):
    op = rng.choice(("sample", "ppo", "distill"))
    v = round(2 * 2 ** rng.uniform(0, 16.6))
    most = (1 << 25 if op == "sample" else 1 << 28) // v
    n = round(2 ** rng.uniform(0, math.log2(min(most, 200000))))
    c = {"op": op, "n": max(1, n), "v": v, "dtype": rng.choice(("f32", "bf16", "f16")), "pad": rng.choice((0, 0, 0, 1, 8, 13))}
    if op == "sample":
        return c | {"filter": rng.choice(("none", "k", "p", "k+p", "min_p", "mixed" if n >= 16 else "p"))}
    c["form"] = rng.choice(("fused", "fused", "autograd", "loss"))
    if op == "ppo":
        return c | {"ref": rng.random() < 0.5}
    return c | {"k": max(1, round(2 ** rng.uniform(0, min(7, math.log2(v))))), "lse": rng.random() < 0.5}


def _logits(c, g):
    """Rows as a policy's head gives them: a common slope over the vocabulary (few likely entries, many unlikely) and noise."""
    n, v = c["n"], c["v"]
    wide = torch.empty(n, v + c["pad"], dtype=DTYPES[c["dtype"]], device="cuda")
    bias = -torch.log1p(torch.randperm(v, generator=g, device="cuda").float()) if v > NARROW else torch.zeros(v, device="cuda")
    step = max(1, (1 << 27) // v)
    for i in range(0, n, step):
        k = min(step, n - i)
        wide[i:i + k, :v] = torch.randn(k, v, generator=g, device="cuda").mul_(1.5).add_(bias)
    wide[:, v:] = float("nan")  # what lies between the rows is nobody's
    return wide[:, :v]


def _logprob_of(x, a):
    """log softmax(x)[a], in chunks of rows."""
    out = torch.empty(a.shape, device=x.device)
    step = max(1, (1 << 27) // x.shape[1])
    for i in range(0, x.shape[0], step):
        f = x[i:i + step].float()
        out[i:i + step] = torch.gather(f, 1, a[i:i + step]) - torch.logsumexp(f, 1, keepdim=True)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, v = case["n"], case["v"]
    s = {"case": case, "x": _logits(case, g)}
    if case["op"] == "sample":
        s["u"] = torch.rand(n, generator=g, device="cuda")
        f = case["filter"]
        s["par"] = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
        if f in ("k", "k+p"):
            s["par"] |= {"top_k": 50, "temperature": 0.8}
        if f in ("p", "k+p"):
            s["par"] |= {"top_p": 0.9}
        if f == "min_p":
            s["par"] |= {"min_p": 0.05, "temperature": 1.2}
        if f == "mixed":  # what different users ask for, side by side in one batch
            pick = lambda *vals: torch.tensor(vals, device="cuda")[torch.randint(len(vals), (n,), generator=g, device="cuda")]  # noqa: E731
            s["par"] = {"temperature": pick(0.0, 0.6, 0.8, 1.0, 1.0, 1.3), "top_k": pick(0, 0, 1, 20, 50, 400).int(),
                        "top_p": pick(1.0, 1.0, 0.95, 0.9, 0.5), "min_p": pick(0.0, 0.0, 0.02, 0.1)}
        return s
    w = (torch.rand(n, generator=g, device="cuda") > 0.1).float()  # a tenth of the rows is padding
    w[:1] = 1.0
    # a mean over the rows; in f16 the weights carry the loss scale that keeps small gradients from underflow
    s["weights"] = w * 64 if case["dtype"] == "f16" else w / w.sum()
    if case["op"] == "ppo":
        rows = torch.arange(n, device="cuda")
        a = torch.empty(n, 1, dtype=torch.int64, device="cuda")
        step = max(1, (1 << 27) // v)
        for i in range(0, n, step):
            k = min(step, n - i)
            noise = torch.rand(k, v, generator=g, device="cuda").clamp_(1e-12).log_().neg_()
            a[i:i + k] = (s["x"][i:i + k].float().exp() / noise).argmax(1, keepdim=True)
        lp = _logprob_of(s["x"], a)[:, 0]
        s["actions"] = torch.where(w > 0, a[:, 0], -1 - rows % 2)  # padded rows hold no action
        s["old"] = lp + 0.15 * torch.randn(n, generator=g, device="cuda")
        s["adv"] = torch.randn(n, generator=g, device="cuda")
        s["ref"] = lp + 0.1 * torch.randn(n, generator=g, device="cuda") if case["ref"] else None
        s["par"] = {"temperature": 1.0, "clip_coef": 0.2, "clip_coef_high": 0.28, "ent_coef": 0.01, "kl_coef": 0.05 if case["ref"] else 0.0}
        return s
    k = case["k"]
    s["idx"] = torch.empty(n, k, dtype=torch.int64, device="cuda")
    s["top"] = torch.empty(n, k, dtype=torch.float32, device="cuda")
    s["lse"] = torch.empty(n, dtype=torch.float32, device="cuda") if case["lse"] else None
    s["par"] = {"temperature": 2.0}
    step = max(1, (1 << 27) // v)
    for i in range(0, n, step):
        r = s["x"][i:i + step].float()
        t = 0.8 * r + 0.8 * torch.randn(r.shape, generator=g, device="cuda")
        s["top"][i:i + step], s["idx"][i:i + step] = torch.topk(t, k, dim=1)
        if case["lse"]:
            s["lse"][i:i + step] = torch.logsumexp(t / 2.0, 1)
    cut = torch.randint(1, k + 1, (n, 1), generator=g, device="cuda")  # some teachers gave fewer
    short = (torch.rand(n, 1, generator=g, device="cuda") < 0.1) & (torch.arange(k, device="cuda") >= cut)
    s["idx"][short] = -1
    return s


def work(case):
    n, v, e = case["n"], case["v"], 4 if case["dtype"] == "f32" else 2
    if case["op"] == "sample":
        return {"bytes": n * v * e + 20 * n, "flops": 4 * n * v}
    both = 1 if case["form"] == "loss" else 2
    rows = n * 28 if case["op"] == "ppo" else n * (12 * case["k"] + 8)
    return {"bytes": n * v * e * both + rows, "flops": n * v * 5 * both}


def run(state):
    return (_own if own else _plain)(state)


def _own(s):
    import _rtpkg  # noqa: F401  registers the package
    from ppo_radiotherapy_amd import categorical as C

    c, x = s["case"], s["x"]
    if c["op"] == "sample":
        r = C.sample(x, s["u"], **s["par"])
        return {"action": r.action, "logprob": r.logprob, "kept_logprob": r.kept_logprob}
    if c["op"] == "ppo":
        args = (s["actions"], s["old"], s["adv"])
        kw = s["par"] | {"weights": s["weights"], "ref_logprobs": s["ref"]}
        loss, loss_grad = C.ppo_loss, C.ppo_loss_grad
    else:
        args = (s["idx"], s["top"])
        kw = s["par"] | {"weights": s["weights"], "teacher_lse": s["lse"]}
        loss, loss_grad = C.distill_loss, C.distill_loss_grad
    grad = None
    if c["form"] == "fused":
        r, grad = loss_grad(x, *args, **kw)
    elif c["form"] == "autograd":
        leaf = x.detach().requires_grad_()
        r = loss(leaf, *args, **kw)
        grad, = torch.autograd.grad(r.loss, leaf)
    else:
        with torch.no_grad():
            r = loss(x, *args, **kw)
    out = {"loss": r.loss.detach()}
    if c["op"] == "ppo":
        out |= {"logprob": r.logprob, "entropy": r.entropy, "stats": r.stats}
    else:
        out |= {"kl": r.kl}
    return out if grad is None else out | {"grad": grad}


def _plain(s):
    return {"sample": _plain_sample, "ppo": _plain_ppo, "distill": _plain_distill}[s["case"]["op"]](s)


def _plain_sample(s):
    # which action a number falls to is a border, so weights and sums are in 64 bits
    x, u, n, v = s["x"].float(), s["u"], s["case"]["n"], s["case"]["v"]
    par = {k: torch.as_tensor(p, device=x.device).expand(n).unsqueeze(1) for k, p in s["par"].items()}
    t = par["temperature"].double()
    greedy = ~(t > 0)
    t = torch.where(greedy, 1.0, t)
    m = x.amax(1, keepdim=True)
    d = x.double() - m.double()
    w = torch.where(x == -math.inf, 0.0, torch.exp(d / t) * UNIT).round().long()
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = torch.gather(w, 1, order)
    rank = torch.arange(v, device=x.device)
    keep = (rank < par["top_k"]) | (par["top_k"] <= 0)
    ws = torch.where(keep, ws, 0)
    total = ws.sum(1, keepdim=True)
    limit = torch.ceil(par["top_p"].double() * total.double()).long().clamp(min=1)
    keep &= (torch.cumsum(ws, 1) - ws < limit) | (par["top_p"] >= 1)
    keep = torch.zeros_like(keep).scatter_(1, order, keep)
    keep &= (d >= t * torch.log(par["min_p"].double().clamp(max=1.0))) | (par["min_p"] <= 0)
    kept = torch.cumsum(torch.where(keep, w, 0), 1)
    mass = kept[:, -1:]
    target = torch.minimum(torch.floor(u.double().unsqueeze(1) * mass.double()).long(), mass - 1)
    a = (kept <= target).sum(1, keepdim=True).clamp(max=v - 1)
    a = torch.where(greedy, x.argmax(1, keepdim=True), a)
    za = torch.gather(d, 1, a) / t
    full = torch.where(greedy, 0.0, za - torch.log(w.sum(1, keepdim=True).double() / UNIT))
    part = torch.where(greedy, 0.0, za - torch.log(mass.double() / UNIT))
    return {"action": a[:, 0], "logprob": full[:, 0].float(), "kept_logprob": part[:, 0].float()}


def _softmax_parts(x, temperature):
    """(x as numbers, row maximum, (x - max) / T, exp of it, its sum in 64 bits)."""
    # a row's log-probability stands next to the border of a clip; where rows are short they are many, and
    # 64 bits cost little
    f = x.double() if x.shape[1] <= NARROW else x.float()
    m = f.amax(1, keepdim=True)
    d = (f - m) / temperature
    e = torch.exp(d)
    return f, m, d, e, e.sum(1, keepdim=True, dtype=torch.float64)


def _plain_ppo(s):
    x, par, form = s["x"], s["par"], s["case"]["form"]
    t, low, high = par["temperature"], par["clip_coef"], par["clip_coef_high"]
    f, m, d, e, total = _softmax_parts(x, t)
    w = s["weights"].double().unsqueeze(1)
    a = s["actions"].unsqueeze(1)
    w = torch.where((a >= 0) & (a < x.shape[1]), w, 0.0)
    here = w != 0
    a = torch.where(here, a, 0)
    logs = torch.log(total)
    lp = (torch.gather(f, 1, a).double() - m.double()) / t - logs
    h = logs - (e * d).sum(1, keepdim=True, dtype=torch.float64) / total
    adv = s["adv"].double().unsqueeze(1)
    lr = lp - s["old"].double().unsqueeze(1)
    r = torch.exp(lr)
    one, two = -adv * r, -adv * r.clamp(1 - low, 1 + high)
    pg = torch.maximum(one, two)
    c = torch.where(one >= two, one, 0.0)
    kl = torch.zeros_like(lp)
    if s["ref"] is not None:
        away = s["ref"].double().unsqueeze(1) - lp
        kl = torch.exp(away) - away - 1
        c = c + par["kl_coef"] * (1 - torch.exp(away))
    clipped = ((r < 1 - low) | (r > 1 + high)).double()
    stats = torch.cat([pg, kl, h, -lr, (r - 1) - lr, clipped], 1)
    stats = torch.where(here, w * stats, 0.0).sum(0)
    loss = stats[0] + par["kl_coef"] * stats[1] - par["ent_coef"] * stats[2]
    out = {"loss": loss.float(), "logprob": torch.where(here, lp, 0.0)[:, 0].float(), "entropy": torch.where(here, h, 0.0)[:, 0].float(), "stats": stats.float()}
    if form == "loss":
        return out
    p = e.div_(total.to(e.dtype))
    wide = lambda y: y.to(e.dtype)  # noqa: E731
    grad = p * (d.sub_(wide(logs - h)).mul_(wide(par["ent_coef"] * w / t)).sub_(wide(c * w / t)))
    grad.scatter_add_(1, a, wide(c * w / t))
    return out | {"grad": torch.where(here, grad, 0.0).to(x.dtype)}


def _plain_distill(s):
    x, t, form = s["x"], s["par"]["temperature"], s["case"]["form"]
    f, m, d, e, total = _softmax_parts(x, t)
    w = s["weights"].double().unsqueeze(1)
    there = (s["idx"] >= 0) & (s["idx"] < x.shape[1])
    idx = torch.where(there, s["idx"], 0)
    top = torch.where(there, s["top"].double() / t, -math.inf)
    if s["lse"] is None:
        most = top.amax(1, keepdim=True)
        lse = most + torch.log(torch.exp(top - most).sum(1, keepdim=True))
    else:
        lse = s["lse"].double().unsqueeze(1)
    lq = top - lse
    q = torch.exp(lq)
    lp = (torch.gather(f, 1, idx).double() - m.double()) / t - torch.log(total)
    kl = torch.where(q > 0, q * (lq - lp), 0.0).sum(1, keepdim=True)
    kl = torch.where(w != 0, kl, 0.0)
    out = {"loss": (w * kl).sum().float(), "kl": kl[:, 0].float()}
    if form == "loss":
        return out
    grad = e.mul_((w / t * q.sum(1, keepdim=True) / total).to(e.dtype))
    grad.scatter_add_(1, idx, (-w / t * q).to(e.dtype))
    return out | {"grad": grad.to(x.dtype)}


def exact(case, seed):
    """The definitions in 64 bits, over chunks of rows: torch's own log_softmax, sorted sums of real numbers and autograd,
    where the plain forms have whole-number weights and written-out gradients."""
    s = prepare(case, seed)
    parts, step = [], max(1, (1 << 26) // case["v"])
    part = {"sample": _exact_sample, "ppo": _exact_ppo, "distill": _exact_distill}[case["op"]]
    for i in range(0, case["n"], step):
        parts.append(part(s, slice(i, i + step)))
    out = {}
    for k in parts[0]:
        v = [p[k] for p in parts]
        out[k] = sum(v) if k in ("loss", "stats") else torch.cat(v)
    return out


def _exact_sample(s, at):
    x = s["x"][at].double()
    n, v = x.shape
    par = {k: (p[at] if torch.is_tensor(p) else torch.full((n,), p, device=x.device)).double()[:, None] for k, p in s["par"].items()}
    t = par["temperature"].clamp(min=1e-300)
    cold = par["temperature"] <= 0
    z = torch.where(cold, x, x / t)
    order = z.argsort(dim=1, descending=True, stable=True)
    sp = z.softmax(1).gather(1, order)
    place = torch.arange(1, v + 1, device=x.device)
    off = (place > par["top_k"]) & (par["top_k"] > 0)
    sp = sp.masked_fill(off, 0)
    before = sp.cumsum(1) - sp
    gone = off | ((before >= par["top_p"] * sp.sum(1, keepdim=True)) & (par["top_p"] < 1))
    gone[:, 0] = False
    out = torch.empty_like(gone).scatter_(1, order, gone)
    out |= z.exp() < par["min_p"] * z.amax(1, keepdim=True).exp()
    lq = z.masked_fill(out, -math.inf).log_softmax(1)
    cum = lq.exp().cumsum(1)
    u = s["u"][at].double()[:, None] * cum[:, -1:]
    a = torch.searchsorted(cum, u, right=True).clamp(max=v - 1)
    a = torch.where(cold, order[:, :1], a)
    full, kept = z.log_softmax(1).gather(1, a), lq.gather(1, a)
    return {"action": a[:, 0], "logprob": torch.where(cold, 0.0, full)[:, 0], "kept_logprob": torch.where(cold, 0.0, kept)[:, 0]}


def _exact_ppo(s, at):
    par = s["par"]
    x = s["x"][at].double().requires_grad_()
    with torch.enable_grad():
        live = (s["weights"][at] != 0) & (s["actions"][at] >= 0)
        w = s["weights"][at].double()
        logp = (x / par["temperature"]).log_softmax(1)
        lp = logp.gather(1, s["actions"][at].clamp(min=0)[:, None])[:, 0]
        h = -(logp.exp() * logp).sum(1)
        lr = lp - s["old"][at].double()
        r, a = lr.exp(), s["adv"][at].double()
        lo, hi = 1 - par["clip_coef"], 1 + par["clip_coef_high"]
        pg = -torch.minimum(a * r, a * r.clamp(lo, hi))
        far = s["ref"][at].double() - lp if s["ref"] is not None else torch.zeros_like(lp)
        kl = far.exp() - far - 1
        rows = [pg, kl, h, -lr, r - 1 - lr, ((r < lo) | (r > hi)).double()]
        stats = torch.stack([(w * q)[live].sum() for q in rows])
        loss = stats[0] + par["kl_coef"] * stats[1] - par["ent_coef"] * stats[2]
        out = {"loss": loss.detach(), "logprob": lp.detach() * live, "entropy": h.detach() * live, "stats": stats.detach()}
        if s["case"]["form"] == "loss":
            return out
        return out | {"grad": torch.autograd.grad(loss, x)[0]}


def _exact_distill(s, at):
    t = s["par"]["temperature"]
    x = s["x"][at].double().requires_grad_()
    with torch.enable_grad():
        w, idx = s["weights"][at].double(), s["idx"][at]
        some = idx >= 0
        lt = (s["top"][at].double() / t).masked_fill(~some, -math.inf)
        lt = lt.log_softmax(1) if s["lse"] is None else lt - s["lse"][at].double()[:, None]
        lt, q = lt.masked_fill(~some, 0), lt.exp()
        lp = (x / t).log_softmax(1).gather(1, idx.clamp(min=0))
        kl = (q * (lt - lp)).sum(1)
        loss = (w * kl).sum()
        out = {"loss": loss.detach(), "kl": kl.detach() * (w != 0)}
        if s["case"]["form"] == "loss":
            return out
        return out | {"grad": torch.autograd.grad(loss, x)[0]}
