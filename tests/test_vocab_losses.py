"""Losses over a vocabulary's logits against their definitions in 64 bits.

Tolerances. The kernels compute in fp32: a term 2^((z - max) c) is off by the rounding of
its argument (two roundings of a number below ~40: 40 * 2^-23 relative at the very most,
weighted by the term itself) and the hardware exponential's 2^-22; a sum of V terms over
512 threads adds V / 512 roundings of 2^-24. ``_lse_tol`` counts those. A log-probability
adds three roundings of its own size. A gradient A (q - P) is off by A q times the error of
lse, A times a few 2^-24, and one rounding to the logits' type (eps / 2).
"""
import math

import pytest
import torch

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _lse_tol(V):
    return 2.0**-24 * (V / 512 + 64)


def _close(got, want, rtol, atol):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    err = (got - want).abs() - (rtol * want.abs() + atol)
    assert torch.isfinite(got).all()
    assert err.max().item() <= 0, f"off by {err.max().item():.3g} more than allowed"


def _grad_close(got, want, z, coef):
    """coef: the largest |A| of the gradient A (q - P) of each row."""
    V = z.shape[1]
    tol = _lse_tol(V) + 8 * 2.0**-24
    half = torch.finfo(z.dtype).eps / 2
    tiny = torch.finfo(z.dtype).smallest_normal * torch.finfo(z.dtype).eps  # half a denormal step of fp16
    got, want = got.double(), want.double()
    err = (got - want).abs() - (want.abs() * (half + 2 * tol) + coef.double()[:, None] * tol + tiny)
    assert torch.isfinite(got).all()
    assert err.max().item() <= 0, f"off by {err.max().item():.3g} more than allowed"


def _logits(T, V, dtype, strided, seed, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(T, V, generator=g) * scale).to(DT[dtype])
    if strided:  # rows that start at odd places, in a wider buffer whose rest is NaN
        wide = torch.full((T, V + 5), math.nan, dtype=DT[dtype])
        wide[:, 3:3 + V] = z
        return wide.cuda()[:, 3:3 + V].requires_grad_(), g
    return z.cuda().requires_grad_(), g


# --------------------------------------------------------------------------- definitions
def distill_ref(z, ids, t, tau):
    z = z.detach().double()
    has = (ids >= 0) & (t != -math.inf)
    on = has.any(1)
    n = max(int(on.sum()), 1)
    loss, grad, coef = 0.0, torch.zeros_like(z), torch.zeros(z.shape[0], dtype=torch.float64, device=z.device)
    for r in range(z.shape[0]):
        if not on[r]:
            continue
        lq = torch.log_softmax(z[r] / tau, 0)
        k = has[r].nonzero()[:, 0]
        lp = torch.log_softmax(t[r, k].double() / tau, 0)
        i = ids[r, k].long()
        loss = loss + tau * tau * (lp.exp() * (lp - lq[i])).sum()
        P = torch.zeros_like(lq).index_add_(0, i, lp.exp())
        grad[r] = tau / n * (lq.exp() - P)
        coef[r] = tau / n
    return torch.as_tensor(loss) / n, grad, coef


def policy_ref(z, a, old, adv, ref, lo, hi, beta, tau, dtype=torch.float64):
    z = z.detach().to(dtype)
    on = a >= 0
    n = max(int(on.sum()), 1)
    rows = on.nonzero()[:, 0]
    lq = torch.log_softmax(z[rows] / tau, 1)
    lp = lq.gather(1, a[rows].long()[:, None])[:, 0].requires_grad_()
    r = (lp - old[rows].to(dtype)).exp()
    A = adv[rows].to(dtype)
    loss = -torch.minimum(r * A, r.clamp(1 - lo, 1 + hi) * A)
    kl = torch.zeros_like(lp)
    if ref is not None:
        d = ref[rows].to(dtype) - lp
        kl = torch.special.expm1(d) - d
        loss = loss + beta * kl
    loss = loss.sum() / n
    dl = torch.zeros_like(lp)
    if rows.numel():
        (dl,) = torch.autograd.grad(loss, lp, allow_unused=True)
    grad, coef = torch.zeros_like(z), torch.zeros(z.shape[0], dtype=dtype, device=z.device)
    q = lq.exp()
    q[torch.arange(rows.numel(), device=z.device), a[rows].long()] -= 1
    grad[rows] = -dl[:, None] / tau * q
    coef[rows] = dl.abs() / tau
    full = torch.zeros(z.shape[0], dtype=dtype, device=z.device)
    return loss.detach(), full.index_copy(0, rows, lp.detach()), full.index_copy(0, rows, kl.detach()), grad, coef


def preference_ref(z, y, off, ref, beta, eps):
    z = z.detach().double()
    o = off.tolist()
    t = torch.arange(z.shape[0], device=z.device)
    on = (y >= 0) & (t >= o[0]) & (t < o[-1])
    rows = on.nonzero()[:, 0]
    lq = torch.log_softmax(z[rows], 1)
    lp = torch.zeros(z.shape[0], dtype=torch.float64, device=z.device)
    lp[rows] = lq.gather(1, y[rows].long()[:, None])[:, 0]
    lp.requires_grad_()
    ratio = torch.where(on, lp - torch.where(on, ref, 0.0).double(), 0.0)
    R = beta * torch.stack([ratio[o[s]:o[s + 1]].sum() for s in range(len(o) - 1)])
    m = R[0::2] - R[1::2]
    ls = torch.nn.functional.logsigmoid
    loss = -((1 - eps) * ls(m) + eps * ls(-m)).mean()
    (dl,) = torch.autograd.grad(loss, lp)
    grad = torch.zeros_like(z)
    q = lq.exp()
    q[torch.arange(rows.numel(), device=z.device), y[rows].long()] -= 1
    grad[rows] = -dl[rows, None] * q
    return loss.detach(), R.detach(), lp.detach(), grad, dl.abs()


# ------------------------------------------------------------------------------- inputs
def _distill_inputs(T, V, K, dtype, strided, seed=0):
    z, g = _logits(T, V, dtype, strided, seed)
    ids = torch.randint(0, V, (T, K), generator=g)  # repeats are likely in small vocabularies
    t = 3 * torch.randn(T, K, generator=g)
    drop = torch.rand(T, K, generator=g) < 0.2
    ids[drop] = -1
    t[drop] = torch.tensor([math.nan, math.inf, -math.inf, 1e30])[torch.randint(0, 4, (int(drop.sum()),), generator=g)]
    if T > 2:
        ids[1] = -1  # a row without entries, over logits that hold anything
        t[2, 0] = -math.inf
        with torch.no_grad():
            z[1] = math.nan
    return z, ids.cuda(), t.cuda()


CASES = [(1, 1, 1), (1, 7, 3), (3, 8, 8), (5, 257, 2), (4, 4104, 64), (3, 50257, 300), (2, 151936, 16),
         (500, 300, 5), (330, 20011, 40), (2, 900001, 12)]


@pytest.mark.gpu
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,V,K", CASES)
def test_distill(T, V, K, dtype, strided):
    from spec_ep.ops.loss import topk_distill_loss

    for tau, i64 in ((1.0, False), (0.6, True)):
        z, ids, t = _distill_inputs(T, V, K, dtype, strided)
        want, grad, coef = distill_ref(z, ids, t, tau)
        loss = topk_distill_loss(z, ids if i64 else ids.int(), t, temperature=tau)
        (got,) = torch.autograd.grad(loss, z)
        # terms of the loss: tau^2 p (ln p - ln q), sums of p at most 1
        _close(loss, want, 4 * 2.0**-24, tau * tau * (2 * _lse_tol(V) + 64 / tau * 2.0**-24))
        assert got.dtype == z.dtype
        _grad_close(got, grad, z, coef)
        with torch.no_grad():  # no gradient buffer: the same loss
            again = topk_distill_loss(z, ids, t, temperature=tau, num_valid=int((coef > 0).sum()))
        _close(again, loss.detach(), 2.0**-23, 0.0)


def _policy_inputs(T, V, dtype, strided, seed=0, tau=1.0):
    z, g = _logits(T, V, dtype, strided, seed)
    a = torch.randint(0, V, (T,), generator=g).cuda()
    lp = torch.log_softmax(z.detach().float() / tau, 1).gather(1, a[:, None])[:, 0]
    old, ref = lp + 0.3 * torch.randn(T, generator=g).cuda(), lp + 0.5 * torch.randn(T, generator=g).cuda()
    adv = torch.randn(T, generator=g).cuda()
    if T > 2:
        a[1] = -1  # not in the loss: nothing of the row is looked at
        adv[2] = 0.0
        with torch.no_grad():
            z[1] = math.nan
        old[1], ref[1], adv[1] = math.nan, math.inf, math.nan
    return z, a, old, adv, ref


@pytest.mark.gpu
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,V", [(1, 1), (1, 9), (4, 8), (67, 257), (9, 4104), (5, 50257), (3, 151936), (700, 301), (331, 20011),
                                 (2, 900001)])
def test_policy(T, V, dtype, strided):
    from spec_ep.ops.loss import clipped_policy_loss

    for tau, beta, with_ref in ((1.0, 0.0, False), (0.8, 0.07, True), (1.0, 0.0, True)):
        z, a, old, adv, ref = _policy_inputs(T, V, dtype, strided, tau=tau)
        ref = ref if with_ref else None
        want, lp, kl, grad, coef = policy_ref(z, a, old, adv, ref, 0.1, 0.25, beta, tau)
        out = clipped_policy_loss(z, a.int(), old, adv, ref, 0.1, 0.25, beta, tau)
        (got,) = torch.autograd.grad(out.loss, z)
        e = _lse_tol(V) + 4 * 2.0**-24 * lp.abs().max().item()  # of a log-probability
        _close(out.logp, lp, 0.0, e)
        # kl = exp(d) - d - 1 with |d| < 3: slope below 20, and three roundings
        _close(out.kl, kl, 8 * 2.0**-24, 20 * e)
        _close(out.loss, want, 8 * 2.0**-24, 10 * e)  # slopes of r A and beta kl
        # A itself is off by its slope (r A, beta e^d) times e
        _grad_close(got, grad, z, coef + 20 * e / (_lse_tol(V) * tau * max(int((a >= 0).sum()), 1)))
        assert not got[a < 0].any() and not out.logp[a < 0].any() and not out.kl[a < 0].any()


def test_preference_reference_margin_sign():
    """CPU: the definition prefers the chosen sequence: its reward grows along -grad."""
    z = torch.zeros(4, 5)
    loss, R, lp, grad, _ = preference_ref(z, torch.tensor([1, 2, 3, 4]), torch.tensor([0, 2, 4]), torch.full((4,), -2.0),
                                          0.1, 0.0)
    assert grad[0, 1] < 0 and grad[2, 3] > 0 and loss > 0


@pytest.mark.gpu
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("off,tail,V", [([0, 1, 2], 0, 9), ([0, 3, 3, 10, 11], 0, 257), ([2, 9, 300, 301, 340], 6, 520),
                                        ([0, 5, 12], 1, 50257), ([0, 2, 3], 0, 151936), ([1, 50, 333, 400, 640], 9, 5003),
                                        ([0, 1, 2], 0, 900001)])
def test_preference(off, tail, V, dtype, strided):
    from spec_ep.ops.loss import preference_loss, token_logp

    T = off[-1] + tail
    for eps in (0.0, 0.2):
        z, g = _logits(T, V, dtype, strided, 3)
        y = torch.randint(0, V, (T,), generator=g)
        y[torch.rand(T, generator=g) < 0.3] = -1
        y[off[0]] = 0
        y, o = y.cuda(), torch.tensor(off, dtype=torch.int32).cuda()
        ref = torch.log_softmax(z.detach().float(), 1).gather(1, y.clamp_min(0)[:, None])[:, 0] + 0.1
        out_of_loss = y < 0
        out_of_loss[:off[0]] = True
        out_of_loss[off[-1]:] = True
        with torch.no_grad():
            z[out_of_loss] = math.nan
        ref[out_of_loss] = math.nan
        want, R, lp, grad, coef = preference_ref(z, y, o, ref, 0.3, eps)
        out = preference_loss(z, y.int(), o, ref, beta=0.3, label_smoothing=eps)
        (got,) = torch.autograd.grad(out.loss, z)
        e = _lse_tol(V) + 4 * 2.0**-24 * lp.abs().max().item()
        n = max(b - a for a, b in zip(off, off[1:]))
        _close(out.logp, lp, 0.0, e)
        _close(out.rewards, R, 2.0**-24, 0.3 * n * e)
        _close(out.loss, want, 2.0**-23, 2 * 0.3 * n * e)
        # the rows' factor is off by beta / pairs times the margin's error, slope at most 1/4
        _grad_close(got, grad, z, coef * (1 + 2 * 0.3 * n * e / _lse_tol(V)))
        assert not got[out_of_loss].any() and not out.logp[out_of_loss].any()
        inside = ~out_of_loss
        _close(token_logp(z.detach()[inside], y[inside]), lp[inside], 0.0, e)


@pytest.mark.gpu
def test_gradients_against_differences():
    """Central differences of the kernels' own losses along random directions. With h = 2^-6
    the loss's fp32 rounding (2^-23 of a loss below 8) gives 2^-23 * 8 / h < 1e-4 and the
    third derivative along a unit-size direction h^2 / 6 < 1e-4."""
    from spec_ep.ops.loss import clipped_policy_loss, preference_loss, topk_distill_loss

    T, V, h = 6, 131, 2.0**-6
    z, ids, t = _distill_inputs(T, V, 9, "fp32", False, seed=5)
    with torch.no_grad():
        z[1] = 0.0
    zp, a, old, adv, ref = _policy_inputs(T, V, "fp32", False, seed=6)
    with torch.no_grad():
        zp[1] = 0.0
    old = torch.where(a >= 0, torch.log_softmax(zp.detach(), 1).gather(1, a.clamp_min(0)[:, None])[:, 0] + 0.05, 0.0)
    ref = old + 0.2
    off = torch.tensor([0, 2, 6], dtype=torch.int32).cuda()
    fns = [(z, lambda x: topk_distill_loss(x, ids, t, temperature=1.5)),
           (zp, lambda x: clipped_policy_loss(x, a, old, adv, ref, kl_coef=0.1).loss),
           (zp, lambda x: preference_loss(x, a, off, ref, beta=0.5, label_smoothing=0.1).loss)]
    for x, f in fns:
        (g,) = torch.autograd.grad(f(x), x)
        gen = torch.Generator().manual_seed(9)
        for _ in range(4):
            d = torch.randn(T, V, generator=gen).cuda()
            d /= d.abs().amax()
            with torch.no_grad():
                diff = (f(x + h * d).double() - f(x - h * d).double()) / (2 * h)
            assert abs(diff.item() - (g.double() * d).sum().item()) < 3e-4


def _three(z, i):
    """Loss number i of logits z, on inputs made from z's shape."""
    from spec_ep.ops.loss import clipped_policy_loss, preference_loss, topk_distill_loss

    T, V = z.shape
    r = torch.arange(T, device=z.device)
    if i == 0:
        ids = (r[:, None] * 7 + torch.arange(5, device=z.device) * 11) % V
        return topk_distill_loss(z, ids, torch.linspace(2, 0, 5, device=z.device).expand(T, 5))
    y, old = (r * 13) % V, torch.full((T,), -5.0, device=z.device)
    if i == 1:
        return clipped_policy_loss(z, y, old, 0.5 - (r % 3).float(), old - 0.1, kl_coef=0.1, clip_high=9.0).loss
    return preference_loss(z, y, torch.tensor([0, T // 3, T], dtype=torch.int32, device=z.device), old).loss


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("i", [0, 1, 2])
def test_upstream_gradient_and_second_backward(i, dtype):
    """The gradient formed in the forward is scaled by the upstream gradient; a second
    backward through the same graph gets the same values and leaves the first's alone."""
    z, _ = _logits(33, 1003, dtype, False, 1)
    (one,) = torch.autograd.grad(_three(z, i), z)
    loss = _three(z, i)
    up = torch.tensor(-4.0, device="cuda")  # a power of two: exact on top of one rounding
    (a,) = torch.autograd.grad(loss, z, up, retain_graph=True)
    kept = a.clone()
    (b,) = torch.autograd.grad(loss, z, up, retain_graph=True)
    (c,) = torch.autograd.grad(loss, z, torch.tensor(1.0, device="cuda"))
    assert torch.equal(a, kept) and a.data_ptr() != b.data_ptr()
    if dtype != "fp16":  # fp16: denormal gradients round differently before and after scaling
        assert torch.equal(a, -4 * one)
    assert torch.equal(a, b) and torch.equal(c, one)
    assert one.any()


@pytest.mark.gpu
def test_fp16_gradient_under_a_loss_scale_keeps_small_values():
    """Unscaled, gradients of a long batch are below fp16's range; scaled ones are not, so
    they have to be formed from the scaled factor."""
    z, _ = _logits(64, 4096, "fp16", False, 2)
    up = torch.tensor(65536.0, device="cuda")
    for i in range(3):
        (g,) = torch.autograd.grad(_three(z, i), z, up)
        z64 = z.detach().float().requires_grad_()
        (w,) = torch.autograd.grad(_three(z64, i), z64, up)
        # both from the same fp32 factor: one rounding to fp16 and its denormal step apart.
        # fp16 rounds 65520 and more to infinity (its largest value is 65504, the next step
        # would be 65536), which a label's entry of up / N = 65536 / 64 times A can pass.
        over = w.abs() >= 65520
        assert torch.equal(g.isinf(), over) and torch.equal(g[over].sign().float(), w[over].sign())
        assert ((g.float() - w).abs() <= w.abs() * 2.0**-10 + 2.0**-24)[~over].all()


@pytest.mark.gpu
@pytest.mark.parametrize("i", [0, 1, 2])
def test_same_bits_on_every_run_and_on_another_stream(i):
    z, _ = _logits(50, 3001, "bf16", False, 4)
    loss = _three(z, i)
    (g,) = torch.autograd.grad(loss, z)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            l2 = _three(z, i)
            (g2,) = torch.autograd.grad(l2, z)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(loss, l2) and torch.equal(g, g2)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1000, 8000, 40001, 151936])
@pytest.mark.parametrize("i", [0, 1, 2])
def test_same_bits_over_many_long_rows(i, V):
    """Several rows per block, so that a row's sum begins while another's gradient is owed:
    where the sums are split must not depend on what has arrived."""
    z, _ = _logits(1300 if V < 100000 else 500, V, "bf16", False, 4)
    loss = _three(z, i)
    (g,) = torch.autograd.grad(loss, z)
    for _ in range(4):
        l2 = _three(z, i)
        (g2,) = torch.autograd.grad(l2, z)
        assert torch.equal(loss, l2) and torch.equal(g, g2)


@pytest.mark.gpu
@pytest.mark.parametrize("i", [0, 1, 2])
def test_two_captured_graphs_replay_with_new_inputs(i):
    """Forward and backward captured twice, replayed in turn over changed logits."""
    za, _ = _logits(20, 777, "bf16", False, 5)
    zb, _ = _logits(20, 777, "bf16", False, 6)
    off = torch.tensor([0, 6, 20], dtype=torch.int32, device="cuda")
    import spec_ep.ops.loss as L

    def one(z):
        if i < 2:
            return _three(z, i)
        r = torch.arange(20, device=z.device)
        return L.preference_loss(z, (r * 13) % 777, off, torch.full((20,), -5.0, device=z.device)).loss

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for z in (za, zb):
            torch.autograd.grad(one(z), z)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for z in (za, zb):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            loss = one(z)
            (grad,) = torch.autograd.grad(loss, z)
        graphs.append(gr)
        outs.append((loss, grad))
    for step in range(3):
        with torch.no_grad():
            za += 0.25
            zb.mul_(0.9)
        for gr in graphs:
            gr.replay()
        for z, (loss, grad) in zip((za, zb), outs):
            want = one(z)
            (wg,) = torch.autograd.grad(want, z)
            assert torch.equal(loss, want) and torch.equal(grad, wg)


@pytest.mark.gpu
def test_ids_outside_the_vocabulary_make_nan():
    from spec_ep.ops.loss import clipped_policy_loss, preference_loss, token_logp, topk_distill_loss

    z, _ = _logits(4, 100, "fp32", False, 7)
    for bad in (100, 2**31 - 1, 2**40):
        ids = torch.tensor([[1, 2], [3, bad], [-1, -1], [5, 5]]).cuda()
        loss = topk_distill_loss(z, ids, torch.zeros(4, 2).cuda())
        (g,) = torch.autograd.grad(loss, z)
        assert loss.isnan() and g[1].isnan().all() and g[[0, 2, 3]].isfinite().all()
        a = torch.tensor([1, bad, -1, 5]).cuda()
        out = clipped_policy_loss(z, a, torch.zeros(4).cuda(), torch.ones(4).cuda())
        (g,) = torch.autograd.grad(out.loss, z)
        assert out.loss.isnan() and out.logp[1].isnan() and g[1].isnan().all() and g[[0, 2, 3]].isfinite().all()
        assert token_logp(z, a)[1].isnan()
        out = preference_loss(z, a, torch.tensor([0, 1, 4], dtype=torch.int32).cuda(), torch.zeros(4).cuda())
        assert out.loss.isnan()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_extreme_logits(dtype):
    """Parts of the vocabulary at -inf or at the type's lowest value, whole rows at the
    lowest or the highest value, and a row with no finite logit (NaN, as its softmax)."""
    from spec_ep.ops.loss import topk_distill_loss

    T, V = 6, 2050
    z, _ = _logits(T, V, dtype, False, 8)
    lo, hi = torch.finfo(z.dtype).min, torch.finfo(z.dtype).max
    with torch.no_grad():
        z[0, 7:] = -math.inf
        z[1, :2000] = lo
        z[2] = lo
        z[3] = hi
        z[4, 1:] = -math.inf
        z[4, 0] = 0.0
    ids = torch.tensor([[0, 3, 3], [2001, 2002, -1], [4, 5, 6], [7, 2049, 9], [0, -1, -1], [1, 2, 3]]).cuda()
    t = torch.tensor([1.0, 0.5, -0.5]).expand(T, 3).cuda()
    want, grad, coef = distill_ref(z, ids, t, 1.0)
    loss = topk_distill_loss(z, ids, t)
    (g,) = torch.autograd.grad(loss, z)
    _close(loss, want, 4 * 2.0**-24, 2 * _lse_tol(V) + 64 * 2.0**-24)
    _grad_close(g, grad, z, coef)
    with torch.no_grad():
        z[5] = -math.inf
    loss = topk_distill_loss(z, ids, t)
    (g,) = torch.autograd.grad(loss, z)
    assert loss.isnan() and g[5].isnan().all() and g[:5].isfinite().all()


@pytest.mark.gpu
def test_nothing_in_the_loss():
    from spec_ep.ops.loss import clipped_policy_loss, preference_loss, topk_distill_loss

    for T in (0, 3):
        z = torch.full((T, 64), math.nan, device="cuda", requires_grad=True)
        none = torch.full((T,), -1, device="cuda")
        zero = torch.zeros(T, device="cuda")
        for loss in (topk_distill_loss(z, none[:, None], zero[:, None]), clipped_policy_loss(z, none, zero, zero).loss):
            (g,) = torch.autograd.grad(loss, z)
            assert loss.item() == 0 and g.shape == z.shape and not g.any()
        off = torch.tensor([0, T, T], dtype=torch.int32, device="cuda")
        out = preference_loss(z, none, off, zero)
        (g,) = torch.autograd.grad(out.loss, z)
        assert abs(out.loss.item() - math.log(2)) < 1e-6 and not g.any() and not out.rewards.any()


@pytest.mark.gpu
def test_offsets_beyond_the_rows_touch_nothing():
    from spec_ep.ops.loss import preference_loss

    z, _ = _logits(4, 64, "fp32", False, 1)
    y = torch.tensor([1, 2, 3, 4]).cuda()
    out = preference_loss(z, y, torch.tensor([-5, 2, 9000], dtype=torch.int32).cuda(), torch.zeros(4).cuda())
    same = preference_loss(z, y, torch.tensor([0, 2, 4], dtype=torch.int32).cuda(), torch.zeros(4).cuda())
    assert torch.equal(out.loss, same.loss) and torch.equal(out.rewards, same.rewards)


@pytest.mark.gpu
def test_row_offsets_pass_32_bits():
    """15000 rows of 151936 logits: the last rows lie beyond 2^31 elements."""
    from spec_ep.ops.loss import clipped_policy_loss, preference_loss

    T, V = 15000, 151936
    z = torch.zeros(T, V, dtype=torch.bfloat16, device="cuda")
    a = torch.full((T,), -1, device="cuda")
    a[-1] = 77
    z[-1, 77] = 4.0
    z.requires_grad_()
    q = math.exp(4) / (math.exp(4) + V - 1)
    out = clipped_policy_loss(z, a, torch.full((T,), math.log(q), device="cuda"), torch.ones(T, device="cuda"))
    (g,) = torch.autograd.grad(out.loss, z)
    assert abs(out.logp[-1].item() - math.log(q)) < 2 * _lse_tol(V) + 8 * 2.0**-24 * 12
    assert not g[:-1].any() and abs(g[-1, 77].item() + (1 - q)) < 2.0**-8
    del g
    off = torch.tensor([0, T - 1, T], dtype=torch.int32, device="cuda")
    out = preference_loss(z, a, off, torch.zeros(T, device="cuda"))
    (g,) = torch.autograd.grad(out.loss, z)
    assert not g[:-1].any() and g[-1, 77].item() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("tau", [1.0, 2.0])
def test_log_probabilities_have_no_mean_error(tau):
    """What all tokens of a sequence are off by alike adds up in its log-ratio. Single errors
    here: the output's rounding (|logp| < 16: at most 2^-21, 2^-21 / sqrt 3 = 2.8e-7 rms) and
    that of the row's sum (below 2e-7 rms), together 3.4e-7; over 8192 rows their mean stays
    below 4 * 3.4e-7 / sqrt(8192) = 1.5e-8, and the exponential's mean error is known to 1e-9."""
    from spec_ep.ops.loss import token_logp

    T, V = 8192, 4096
    g = torch.Generator("cuda").manual_seed(5)
    z = 2.0 * torch.randn(T, V, generator=g, device="cuda")
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    want = torch.log_softmax(z.double() / tau, 1).gather(1, y[:, None])[:, 0]
    off = token_logp(z, y.int(), tau).double() - want
    assert abs(off.mean().item()) < 2e-8


# -------------------------------------------------------------------------- refusals, CPU
def _refused(f, *a, match, **kw):
    with pytest.raises((RuntimeError, ValueError), match=match):
        f(*a, **kw)


def test_refusals():
    from spec_ep.ops.loss import clipped_policy_loss, preference_loss, token_logp, topk_distill_loss

    z, i, f = torch.zeros(4, 10), torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    k, t = i[:, None], f[:, None]
    off = torch.tensor([0, 2, 4], dtype=torch.int32)
    _refused(topk_distill_loss, z, k, t, match="CUDA")
    _refused(topk_distill_loss, z[0], k, t, match=r"\[T, V\]")
    _refused(topk_distill_loss, z.t().contiguous().t(), k, t, match="unit stride")
    _refused(topk_distill_loss, z.double(), k, t, match="bf16, fp16 or fp32")
    _refused(topk_distill_loss, z, k.float(), t, match="int32 or int64")
    _refused(topk_distill_loss, z, k[:3], t[:3], match="teacher_ids")
    _refused(topk_distill_loss, z, k, t.expand(4, 2), match="shape of teacher_ids")
    _refused(topk_distill_loss, z, k.expand(4, 1025), t.expand(4, 1025), match="teacher entries")
    _refused(topk_distill_loss, z, k[:, :0], t[:, :0], match="teacher entries")
    for tau in (0.0, -1.0, float("nan"), float("inf"), 1e-42, 1e25):
        _refused(topk_distill_loss, z, k, t, temperature=tau, match="temperature")
    _refused(topk_distill_loss, z, k, t, num_valid=-2, match="num_valid")
    _refused(clipped_policy_loss, z, i, f, f, match="CUDA")
    _refused(clipped_policy_loss, z, i[:3], f, f, match="actions")
    _refused(clipped_policy_loss, z, i, f[:3], f, match="old_logp")
    _refused(clipped_policy_loss, z, i, f, f[:2], match="advantages")
    _refused(clipped_policy_loss, z, i, f, f, f[:2], match="ref_logp")
    _refused(clipped_policy_loss, z, i, f, f, kl_coef=0.1, match="ref_logp")
    _refused(clipped_policy_loss, z, i, f, f, f, kl_coef=-0.1, match="kl_coef")
    _refused(clipped_policy_loss, z, i, f, f, clip_low=1.5, match="clip_low")
    _refused(clipped_policy_loss, z, i, f, f, clip_high=-0.5, match="clip_high")
    _refused(clipped_policy_loss, z[:, :0], i, f, f, match="vocabulary")
    _refused(token_logp, z, i, match="CUDA")
    _refused(token_logp, z, i.float(), match="int32 or int64")
    _refused(preference_loss, z, i, off, f, match="CUDA")
    _refused(preference_loss, z, i, off.long(), f, match="int32")
    _refused(preference_loss, z, i, off[:2], f, match="pairs")
    _refused(preference_loss, z, i, off, f[:3], match="ref_logp")
    _refused(preference_loss, z, i, off, f, beta=0.0, match="beta")
    _refused(preference_loss, z, i, off, f, label_smoothing=0.5, match="label_smoothing")


@pytest.mark.gpu
@pytest.mark.parametrize("i", [0, 1, 2])
def test_backward_twice_needs_a_kept_graph_and_gradients_are_not_differentiable(i):
    z, _ = _logits(33, 515, "bf16", False, 1)
    loss = _three(z, i)
    torch.autograd.grad(loss, z)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, z)
    (g,) = torch.autograd.grad(_three(z, i), z, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(g.float().sum(), z)


@pytest.mark.gpu
@pytest.mark.parametrize("i", [0, 1, 2])
def test_gradient_reaches_a_leaf_behind_other_operations(i):
    """z = w * x: the losses' gradient goes on through the product, twice into one .grad."""
    x, _ = _logits(33, 515, "fp32", False, 1)
    w = torch.full((515,), 1.5, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(_three((x.detach() * 1.5).requires_grad_(), i).sum() * 0 + _three(x * w, i), x)
    z = (x.detach() * 1.5).requires_grad_()
    (gz,) = torch.autograd.grad(_three(z, i), z)
    assert torch.equal(g, gz * 1.5)
    leaf = x.detach().clone().requires_grad_()
    for _ in range(2):
        _three(leaf, i).backward()
    (once,) = torch.autograd.grad(_three(leaf, i), leaf)
    assert torch.equal(leaf.grad, 2 * once)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 9000, 40001, 151936])
@pytest.mark.parametrize("pattern", ["runs", "scattered", "ends"])
def test_many_rows_out_of_the_loss(V, pattern):
    """Long runs of rows that are not in the loss between rows that are, over several rows
    per block: all losses equal those of the remaining rows alone."""
    from spec_ep.ops.loss import clipped_policy_loss, preference_loss, topk_distill_loss

    T = 1500 if V > 100000 else 3000
    g = torch.Generator(device="cuda").manual_seed(V)
    z = torch.randn(T, V, generator=g, device="cuda").bfloat16()
    r = torch.arange(T, device="cuda")
    on = {"runs": (r // 700) % 2 == 1, "scattered": torch.rand(T, generator=g, device="cuda") < 0.15,
          "ends": (r < 3) | (r >= T - 2)}[pattern]
    z[~on] = math.nan
    z.requires_grad_()
    zk = z.detach()[on].requires_grad_()
    n = int(on.sum())
    y = torch.where(on, (r * 17) % V, -1)
    old, adv = torch.full((T,), -9.0, device="cuda"), 1.0 + (r % 5).float()
    ids = torch.where(on[:, None], (r[:, None] * 31 + torch.arange(6, device="cuda") * 7) % V, -1)
    big = torch.where(on[:, None], (r[:, None] + torch.arange(300, device="cuda")) % V, -1)
    t6, t300 = torch.linspace(1, 0, 6, device="cuda"), torch.linspace(2, 0, 300, device="cuda")
    off, offk = ([0, T // 2, T], [0, int(on[:T // 2].sum()), n])
    cu = lambda o: torch.tensor(o, dtype=torch.int32, device="cuda")  # noqa: E731
    # d loss / d (a common error of all log-probabilities): the weights sum to 1; r A with every
    # A > 0; beta / 2 per row of either sequence
    cases = [(lambda q, s, o: topk_distill_loss(q, ids[s], t6.expand(q.shape[0], 6)), lambda v: 1.0),
             (lambda q, s, o: topk_distill_loss(q, big[s], t300.expand(q.shape[0], 300)), lambda v: 1.0),
             (lambda q, s, o: clipped_policy_loss(q, y[s], old[s], adv[s], clip_high=99.0).loss, abs),
             (lambda q, s, o: preference_loss(q, y[s], cu(o), old[s]).loss, lambda v: 0.1 * n)]
    for f, slope in cases:
        loss, kept = f(z, slice(None), off), f(zk, on, offk)
        (gz,), (gk,) = torch.autograd.grad(loss, z), torch.autograd.grad(kept, zk)
        # The same rows in another place: the sum over rows has another order (64 bits), and
        # with an odd vocabulary a row begins elsewhere in its 16 bytes, so the row's own
        # fp32 sum is grouped differently: both are within _lse_tol of the exact one.
        tol = 2.0**-22 * abs(kept.item()) + (V % 8 > 0) * 2 * _lse_tol(V) * slope(kept.item())
        assert abs(loss.item() - kept.item()) <= tol
        # (the preference loss's row factors come from that sum)
        assert (gz[on].float() - gk.float()).abs().max().item() <= 2.0**-7 * gk.abs().max().item()
        assert not gz[~on].any() and gz[on].isfinite().all()
        del gz, gk
        with torch.no_grad():
            assert abs(f(z, slice(None), off).item() - loss.item()) <= 2.0**-22 * abs(loss.item())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("i", [0, 1, 2])
def test_views_of_padded_logits(i, dtype):
    """Logits of an odd vocabulary in rows padded to a multiple of 64, rows that start at an
    odd place, far apart or expanded: the values of contiguous ones. Row sums are grouped by
    a row's place in its 16 bytes, so sums may differ by twice _lse_tol."""
    T, V = 300, 5007
    g = torch.Generator().manual_seed(i)
    z = torch.randn(T, V, generator=g).to(DT[dtype]).cuda()
    want = z.clone().requires_grad_()
    lw = _three(want, i)
    (gw,) = torch.autograd.grad(lw, want, torch.tensor(4.0, device="cuda"))

    def held(pad, first):
        wide = torch.full((T, V + pad), math.nan, device="cuda", dtype=DT[dtype])
        wide[:, first:first + V] = z
        return wide[:, first:first + V].requires_grad_()

    flat = torch.full((T * V + 9,), math.nan, device="cuda", dtype=DT[dtype])
    flat[3:3 + T * V] = z.reshape(-1)
    for q in (held(49, 0), held(49, 5), held(3000, 7), flat[3:3 + T * V].view(T, V).requires_grad_()):
        loss = _three(q, i)
        assert abs(loss.item() - lw.item()) <= 0.1 * T * 2 * _lse_tol(V) + 2.0**-22 * abs(lw.item())
        (gq,) = torch.autograd.grad(loss, q, torch.tensor(4.0, device="cuda"), retain_graph=True)
        assert gq.shape == (T, V) and gq.isfinite().all()
        assert (gq.float() - gw.float()).abs().max().item() <= 2.0**-7 * gw.abs().max().item()
        (again,) = torch.autograd.grad(loss, q, torch.tensor(4.0, device="cuda"))
        assert torch.equal(gq, again)
    one = z[:1].expand(T, V).detach().requires_grad_()
    loss = _three(one, i)
    (gq,) = torch.autograd.grad(loss, one)
    assert gq.shape == (T, V) and gq.isfinite().all()
