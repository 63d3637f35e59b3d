"""Cases of the post-training losses and of the balanced router, with their plain forms.

Four operators:

* ``distill``: distillation of a vocabulary's softmax from a teacher's top logits,
* ``policy``: clipped policy loss with a KL term on the chosen tokens,
* ``preference``: paired log-ratio loss over packed chosen / rejected sequences,
* ``router``: top-k routing with the balance loss and per-expert counts.

``run`` computes an operator in elementary torch operations, or with ``own`` through
``spec_ep.ops.loss`` and ``spec_ep.ops.router``. ``exact`` is the same from the
definitions in 64 bits. The preference loss sums log-probabilities of whole sequences
whose difference matters, so its plain form sums them in 64 bits.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# rows x vocabulary of the largest listed case: what a drawn case may cost at most
_MOST = 4096 * 151936


def listed():
    return [
        # distillation: a test-sized vocabulary, an odd vocabulary in 32 bits, and one
        # rank's training batch at the full vocabulary
        {"name": "distill 64x4096", "op": "distill", "T": 64, "V": 4096, "K": 8, "dtype": "bf16", "tau": 1.0},
        {"name": "distill 1000x50257 fp32", "op": "distill", "T": 1000, "V": 50257, "K": 20, "dtype": "fp32",
         "tau": 2.0},
        {"name": "distill 4096x151936", "op": "distill", "T": 4096, "V": 151936, "K": 64, "dtype": "bf16",
         "tau": 1.0},
        # policy: the few sampled tokens of a short rollout, an odd vocabulary, and a full
        # batch of prompts (not in the loss) and responses
        {"name": "policy 16x151936", "op": "policy", "T": 16, "V": 151936, "dtype": "bf16", "tau": 1.0,
         "kl": 0.0, "keep": 1.0},
        {"name": "policy 2049x32001", "op": "policy", "T": 2049, "V": 32001, "dtype": "bf16", "tau": 0.7,
         "kl": 0.05, "keep": 0.8},
        {"name": "policy 4096x151936", "op": "policy", "T": 4096, "V": 151936, "dtype": "bf16", "tau": 1.0,
         "kl": 0.05, "keep": 0.6},
        # preference: scoring a few short pairs without gradients, ragged pairs in 32
        # bits, and a packed training batch of pairs
        {"name": "preference 2 pairs, score", "op": "preference", "pairs": 2, "mean": 24, "V": 4096,
         "dtype": "bf16", "eps": 0.0, "train": False},
        {"name": "preference 13 pairs fp32", "op": "preference", "pairs": 13, "mean": 61, "V": 50257,
         "dtype": "fp32", "eps": 0.1, "train": True},
        {"name": "preference 8 pairs", "op": "preference", "pairs": 8, "mean": 250, "V": 151936,
         "dtype": "bf16", "eps": 0.0, "train": True},
        # router: the smallest preset, one rank's training batch, and a long packed batch
        # with padding and more experts
        {"name": "router 256x8", "op": "router", "T": 256, "E": 8, "k": 2, "dtype": "bf16", "keep": 1.0},
        {"name": "router 4096x128", "op": "router", "T": 4096, "E": 128, "k": 8, "dtype": "bf16", "keep": 1.0},
        {"name": "router 65537x256", "op": "router", "T": 65537, "E": 256, "k": 8, "dtype": "fp32", "keep": 0.9},
    ]


def _between(rng, low, high):
    """A whole number, spread over the logarithm of the range."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["distill", "policy", "preference", "router"])
    if op == "router":
        E = rng.choice([8, 13, 60, 64, 128, 160, 256, 384])
        return {"op": op, "T": _between(rng, 1, 65536 * 256 // max(E, 256)), "E": E, "k": rng.randint(1, min(E, 10)),
                "dtype": rng.choice(["bf16", "fp32"]), "keep": rng.choice([1.0, 0.9, 0.5])}
    dtype = rng.choice(["bf16", "bf16", "fp32", "fp16"])
    V = rng.choice([151936, 151936, _between(rng, 1000, 160000)])
    most = _MOST // V // (2 if dtype == "fp32" else 1)
    if op == "preference":
        pairs = rng.randint(1, 24)
        return {"op": op, "pairs": pairs, "mean": _between(rng, 4, max(5, most // (3 * pairs))), "V": V,
                "dtype": dtype, "eps": rng.choice([0.0, 0.1]), "train": rng.random() < 0.8}
    T = _between(rng, 1, min(most, 8192))
    tau = rng.choice([1.0, 1.0, 0.7, 2.0])
    if op == "distill":
        return {"op": op, "T": T, "V": V, "K": _between(rng, 1, 128), "dtype": dtype, "tau": tau}
    return {"op": op, "T": T, "V": V, "dtype": dtype, "tau": tau, "kl": rng.choice([0.0, 0.05]),
            "keep": rng.choice([1.0, 0.7, 0.4])}


def _lengths(case):
    """Ragged sequence lengths of a preference case, 0.4 to 1.6 times their mean."""
    return [max(2, int(case["mean"] * (0.4 + 1.2 * ((0.37 + 0.618034 * i) % 1.0)))) for i in range(2 * case["pairs"])]


def _logits(g, T, V, dtype, dev):
    return (torch.randn(T, V, generator=g, device=dev) * 2.0).to(dtype)


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dtype = _DTYPES[case["dtype"]]

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=dev)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def randint(n, *shape):
        return torch.randint(0, n, shape, generator=g, device=dev)

    if case["op"] == "router":
        T, E, k = case["T"], case["E"], case["k"]
        # router logits come from a bf16 projection; some experts are more popular
        x = (randn(T, E) + 0.5 * randn(E)).to(torch.bfloat16).to(dtype)
        valid = None if case["keep"] == 1.0 else rand(T) < case["keep"]
        return {"case": case, "x": x.requires_grad_(), "valid": valid, "dw": randn(T, k),
                "dloss": torch.full((), 0.01, device=dev)}
    V, dev_i32 = case["V"], torch.int32
    if case["op"] == "distill":
        T, K = case["T"], case["K"]
        z = _logits(g, T, V, dtype, dev)
        # the teacher's best tokens, without repeats, score well with the student too
        start, step = randint(V, T, 1), 1 + randint(max(1, V // K), T, 1)
        ids = (start + step * torch.arange(K, device=dev)) % V
        t = (6.0 + 2.5 * randn(T, K)).sort(-1, descending=True).values
        z.scatter_(1, ids, (t + 1.0 * randn(T, K)).to(dtype))
        given = torch.where(rand(T, 1) < 0.1, 1 + randint(K, T, 1), torch.full((T, 1), K, device=dev))
        ids = torch.where(torch.arange(K, device=dev) < given, ids, -1)  # some rows list fewer
        ids = torch.where(rand(T, 1) < (0.05 if T > 1 else 0.0), -1, ids)  # and some none: padding
        return {"case": case, "z": z.requires_grad_(), "ids": ids.to(dev_i32), "t": t}
    if case["op"] == "policy":
        T = case["T"]
        z = _logits(g, T, V, dtype, dev)
        a = randint(V, T)
        z[torch.arange(T, device=dev), a] = (9.0 + 2.0 * randn(T)).to(dtype)  # sampled: likely
        logp = torch.log_softmax(z.float() / case["tau"], -1)[torch.arange(T, device=dev), a]
        old = logp + 0.15 * randn(T)
        ref = logp + 0.3 * randn(T)
        adv = 0.25 + randn(T)
        if case["keep"] < 1.0:
            a = torch.where((rand(T) < case["keep"]) | (torch.arange(T, device=dev) == T - 1), a, -1)
        return {"case": case, "z": z.requires_grad_(), "a": a.to(dev_i32), "old": old, "adv": adv, "ref": ref}
    # preference: 2 * pairs packed sequences, chosen before rejected, each a prompt (not
    # in the loss) and a response
    n = 2 * case["pairs"]
    lens = torch.tensor(_lengths(case), device=dev)
    off = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), lens.cumsum(0)])
    T = sum(_lengths(case))
    z = _logits(g, T, V, dtype, dev)
    y = randint(V, T)
    z[torch.arange(T, device=dev), y] = (8.0 + 2.0 * randn(T)).to(dtype)
    ref = torch.log_softmax(z.float(), -1)[torch.arange(T, device=dev), y] + 0.1 * randn(T)
    seq = torch.bucketize(torch.arange(T, device=dev), off[1:], right=True)
    prompt = torch.arange(T, device=dev) - off[seq] < (lens[seq] // 4)
    y = torch.where(prompt, -1, y)
    return {"case": case, "z": z.requires_grad_(bool(case["train"])), "y": y.to(dev_i32), "off": off.to(dev_i32), "ref": ref,
            "n": n}


# ------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------
def _distill(s):
    z, ids, t, tau = s["z"].detach(), s["ids"].long(), s["t"], s["case"]["tau"]
    x = z.float() / tau
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    tot = e.sum(-1, keepdim=True)
    has = ids >= 0
    rows = has.any(-1)
    N = rows.sum().clamp_min(1)
    tm = torch.where(has, t / tau, -math.inf)
    top = torch.where(rows[:, None], tm.amax(-1, keepdim=True), 0.0)
    pe = (tm - top).exp()
    psum = torch.where(rows[:, None], pe.sum(-1, keepdim=True), 1.0)
    p = pe / psum
    at = ids.clamp_min(0)
    logq = x.gather(1, at) - m - tot.log()
    logp = torch.where(has, tm - top - psum.log(), 0.0)
    loss = torch.where(has, p * (logp - logq), 0.0).sum(-1) * tau * tau
    grad = e / tot
    grad.scatter_add_(1, at, -p)
    grad = grad * torch.where(rows, tau / N, 0.0)[:, None]
    return {"loss": loss.sum() / N, "grad": grad.to(z.dtype)}


def _policy(s):
    z, a, c = s["z"].detach(), s["a"].long(), s["case"]
    x = z.float() / c["tau"]
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    tot = e.sum(-1, keepdim=True)
    has = a >= 0
    N = has.sum().clamp_min(1)
    at = a.clamp_min(0)[:, None]
    logp = (x.gather(1, at) - m - tot.log())[:, 0]
    r = (logp - s["old"]).exp()
    adv = s["adv"]
    u, v = r * adv, r.clamp(0.8, 1.28) * adv
    d = s["ref"] - logp
    kl = d.exp() - d - 1.0
    loss = -torch.minimum(u, v) + c["kl"] * kl
    dl = torch.where(u <= v, -u, 0.0) + c["kl"] * (1.0 - d.exp())
    coef = torch.where(has, dl / (N * c["tau"]), 0.0)[:, None]
    grad = e / tot * -coef
    grad.scatter_add_(1, at, coef)
    zero = torch.zeros((), device=z.device)
    return {"loss": torch.where(has, loss, zero).sum() / N, "logp": torch.where(has, logp, zero),
            "kl": torch.where(has, kl, zero), "grad": grad.to(z.dtype)}


def _preference(s):
    z, y, off, c, n = s["z"].detach(), s["y"].long(), s["off"].long(), s["case"], s["n"]
    beta, T = 0.1, z.shape[0]
    x = z.float()
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    tot = e.sum(-1, keepdim=True)
    has = y >= 0
    at = y.clamp_min(0)[:, None]
    logp = torch.where(has, (x.gather(1, at) - m - tot.log())[:, 0], 0.0)
    seq = torch.bucketize(torch.arange(T, device=z.device), off[1:], right=True)
    ratio = torch.where(has, logp.double() - s["ref"].double(), 0.0)
    R = beta * torch.zeros(n, dtype=torch.float64, device=z.device).index_add_(0, seq, ratio)
    mg = R[0::2] - R[1::2]

    def softplus(v):
        return v.clamp_min(0.0) + (1.0 + (-v.abs()).exp()).log()

    loss = ((1.0 - c["eps"]) * softplus(-mg) + c["eps"] * softplus(mg)).mean()
    out = {"loss": loss.float(), "rewards": R.float(), "logp": logp}
    if c["train"]:
        dm = (c["eps"] / (1.0 + (-mg).exp()) - (1.0 - c["eps"]) / (1.0 + mg.exp())) * (beta / (n // 2))
        dR = torch.stack([dm, -dm], 1).reshape(-1).float()
        coef = torch.where(has, dR[seq], 0.0)[:, None]
        grad = e / tot * -coef
        grad.scatter_add_(1, at, coef)
        out["grad"] = grad.to(z.dtype)
    return out


def _router(s):
    x, k, E = s["x"].detach(), s["case"]["k"], s["case"]["E"]
    l = x.float()
    ex = (l - l.amax(-1, keepdim=True)).exp()
    p = ex / ex.sum(-1, keepdim=True)
    top = l.sort(dim=-1, descending=True, stable=True).indices[:, :k]  # ties: lowest index
    pw = p.gather(1, top)
    S = pw.sum(-1, keepdim=True)
    w = pw / S
    T = l.shape[0]
    valid = s["valid"] if s["valid"] is not None else torch.ones(T, dtype=torch.bool, device=x.device)
    N = valid.sum().clamp_min(1).float()
    counts = torch.zeros(E, dtype=torch.int32, device=x.device)
    counts.index_add_(0, top.reshape(-1), valid[:, None].expand(T, k).reshape(-1).int())
    mean = (p.double() * valid[:, None]).sum(0) / N.double()
    frac = counts.double() / (k * N.double())
    loss = (E * (frac * mean).sum()).float()
    # backward: dw through the renormalisation, and the balance loss through p
    dw = s["dw"]
    dp = (s["dloss"] * E * (frac.float() / N))[None, :] * valid[:, None]
    dp = dp.scatter_add(1, top, (dw - (dw * w).sum(-1, keepdim=True)) / S)
    dx = p * (dp - (p * dp).sum(-1, keepdim=True))
    return {"w": w, "e": top.int(), "loss": loss, "counts": counts, "grad": dx.to(x.dtype)}


def _own(s):
    from spec_ep.ops.loss import clipped_policy_loss, preference_loss, topk_distill_loss
    from spec_ep.ops.router import router_topk_balanced

    c = s["case"]
    if c["op"] == "distill":
        loss = topk_distill_loss(s["z"], s["ids"], s["t"], temperature=c["tau"])
        (grad,) = torch.autograd.grad(loss, s["z"])
        return {"loss": loss.detach(), "grad": grad}
    if c["op"] == "policy":
        loss, logp, kl = clipped_policy_loss(s["z"], s["a"], s["old"], s["adv"], ref_logp=s["ref"], clip_low=0.2,
                                             clip_high=0.28, kl_coef=c["kl"], temperature=c["tau"])
        (grad,) = torch.autograd.grad(loss, s["z"])
        return {"loss": loss.detach(), "logp": logp, "kl": kl, "grad": grad}
    if c["op"] == "preference":
        loss, rewards, logp = preference_loss(s["z"], s["y"], s["off"], s["ref"], beta=0.1, label_smoothing=c["eps"])
        out = {"loss": loss.detach(), "rewards": rewards, "logp": logp}
        if c["train"]:
            (out["grad"],) = torch.autograd.grad(loss, s["z"])
        return out
    w, e, loss, counts = router_topk_balanced(s["x"], c["k"], valid=s["valid"])
    (grad,) = torch.autograd.grad([w, loss], s["x"], [s["dw"], s["dloss"]])
    return {"w": w.detach(), "e": e, "loss": loss.detach(), "counts": counts, "grad": grad}


def run(state):
    if own:
        return _own(state)
    return {"distill": _distill, "policy": _policy, "preference": _preference, "router": _router}[state["case"]["op"]](
        state)


# ------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "router":
        T, E, k = case["T"], case["E"], case["k"]
        # logits in and gradient out; weights and ids out, their gradient in; mask; counts
        return {"bytes": T * (2 * E * size + 12 * k + (1 if case["keep"] < 1.0 else 0)) + 4 * E, "flops": 12 * T * E}
    V = case["V"]
    if case["op"] == "distill":
        T, K = case["T"], case["K"]
        return {"bytes": T * (2 * V * size + 8 * K), "flops": 8 * T * V}
    if case["op"] == "policy":
        T = case["T"]  # rows out of the loss need no reading, their gradient is written
        return {"bytes": int(T * ((1 + case["keep"]) * V * size + 24)), "flops": int(8 * T * case["keep"] * V)}
    T = sum(_lengths(case))
    on = sum(n - n // 4 for n in _lengths(case))  # a quarter of each sequence is prompt
    return {"bytes": V * size * (on + (T if case["train"] else 0)) + 12 * T, "flops": (8 if case["train"] else 4) * on * V}


# ------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------
def _rows(T, V):
    """Row ranges small enough for several 64-bit copies."""
    step = max(1, (1 << 27) // V)
    return [(i, min(T, i + step)) for i in range(0, T, step)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "router":
        return _exact_router(s)
    z = s["z"].detach()
    T, V = z.shape
    dev, f64 = z.device, torch.float64
    if case["op"] == "distill":
        tau = case["tau"]
        keep = s["ids"] >= 0
        N = max(int(keep.any(1).sum()), 1)
        loss, grad = torch.zeros((), dtype=f64, device=dev), torch.empty(T, V, dtype=f64, device=dev)
        for a, b in _rows(T, V):
            lq = torch.log_softmax(z[a:b].double() / tau, 1)
            P = torch.zeros(b - a, V, dtype=f64, device=dev)
            lt = (s["t"][a:b].double() / tau).masked_fill(~keep[a:b], -math.inf)
            lp = torch.log_softmax(lt, 1).nan_to_num(nan=-math.inf, neginf=-math.inf)
            k = s["ids"][a:b].long().clamp_min(0)
            P.scatter_add_(1, k, lp.exp())
            loss += torch.special.xlogy(lp.exp(), lp.exp()).sum() - (P * lq).sum()
            grad[a:b] = (lq.exp() - P) * keep[a:b].any(1, keepdim=True) * (tau / N)
        return {"loss": loss * tau * tau / N, "grad": grad}
    label = (s["a"] if case["op"] == "policy" else s["y"]).long()
    tau = case.get("tau", 1.0)
    on = label >= 0
    logp = torch.zeros(T, dtype=f64, device=dev)
    for a, b in _rows(T, V):
        lq = torch.log_softmax(z[a:b].double() / tau, 1)
        logp[a:b] = lq[torch.arange(b - a, device=dev), label[a:b].clamp_min(0)] * on[a:b]
    leaf = logp.clone().requires_grad_()
    if case["op"] == "policy":
        N = max(int(on.sum()), 1)
        ratio = torch.exp(leaf - s["old"].double())
        adv = s["adv"].double()
        gain = torch.minimum(ratio * adv, torch.clamp(ratio, 1 - 0.2, 1 + 0.28) * adv)
        d = s["ref"].double() - leaf
        kl = torch.special.expm1(d) - d
        loss = ((case["kl"] * kl - gain) * on).sum() / N
        out = {"loss": loss.detach(), "logp": logp, "kl": (kl * on).detach()}
    else:
        off = s["off"].tolist()
        R = 0.1 * torch.stack([((leaf - s["ref"].double()) * on)[off[i]:off[i + 1]].sum() for i in range(s["n"])])
        m = R[0::2] - R[1::2]
        ls = torch.nn.functional.logsigmoid
        loss = -((1 - case["eps"]) * ls(m) + case["eps"] * ls(-m)).mean()
        out = {"loss": loss.detach(), "rewards": R.detach(), "logp": logp}
        if not case["train"]:
            return out
    (dl,) = torch.autograd.grad(loss, leaf)
    dl = dl * on / tau
    grad = torch.empty(T, V, dtype=f64, device=dev)
    for a, b in _rows(T, V):
        q = torch.softmax(z[a:b].double() / tau, 1)
        q[torch.arange(b - a, device=dev), label[a:b].clamp_min(0)] -= 1.0
        grad[a:b] = -dl[a:b, None] * q
    return {**out, "grad": grad}


def _exact_router(s):
    x, k, E = s["x"].detach().double().requires_grad_(), s["case"]["k"], s["case"]["E"]
    T = x.shape[0]
    p = torch.softmax(x, 1)
    # the k largest, lower index first among equals: rank by (value, -index)
    key = x.detach().clone()
    idx = torch.arange(E, device=x.device).expand(T, E)
    chosen = []
    for _ in range(k):
        best = key.amax(1, keepdim=True)
        e = torch.where(key == best, idx, E).amin(1)
        chosen.append(e)
        key[torch.arange(T, device=x.device), e] = -math.inf
    e = torch.stack(chosen, 1)
    w = p.gather(1, e)
    w = w / w.sum(1, keepdim=True)
    valid = torch.ones(T, device=x.device).bool() if s["valid"] is None else s["valid"]
    N = max(int(valid.sum()), 1)
    counts = torch.bincount(e[valid].reshape(-1), minlength=E)
    loss = E * ((counts.double() / (k * N)) * (p[valid].sum(0) / N)).sum()
    (g,) = torch.autograd.grad([w, loss], x, [s["dw"].double(), s["dloss"].double()])
    return {"w": w.detach(), "e": e.int(), "loss": loss.detach(), "counts": counts.int(), "grad": g}
