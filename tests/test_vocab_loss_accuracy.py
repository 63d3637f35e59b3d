"""How exact the vocabulary losses are where a sum over the vocabulary hides it: tokens of
probability near 1, and errors that all tokens share.

Errors counted: an exponential 2^a is off by the roundings of its argument (two of a number
below 16 + |a|) and the hardware's 2^-22; a row's sum adds the rounding of its partial sums
(``_lse_tol``).
"""
import math

import pytest
import torch

from test_vocab_losses import DT, _lse_tol


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("V", [300, 4104, 50257, 151936, 900001])
def test_tokens_of_probability_near_one(V, dtype):
    """ln q = -log(1 + rest / own term): its relative error is that of the rest's sum and of the
    two terms' exponents (arguments below 80), and it is never above 0. The same for 1 - q, the
    label's element of the gradient."""
    from spec_ep.ops.loss import clipped_policy_loss, preference_loss, token_logp, topk_distill_loss

    T = 12
    g = torch.Generator().manual_seed(V)
    z = (2 * torch.randn(T, V, generator=g)).to(DT[dtype])
    y = torch.randint(0, V, (T,), generator=g)
    y[0], y[1] = 0, V - 1
    r = torch.arange(T)
    z[r, y] = torch.linspace(18, 40, T).to(DT[dtype])
    z, y = z.cuda().requires_grad_(), y.cuda()
    rel = _lse_tol(V) + 2.0**-24 * 160
    for tau in (1.0, 0.8):
        z64 = z.detach().double() / tau
        rest = z64.scatter(1, y[:, None], -math.inf).logsumexp(1) - z64.gather(1, y[:, None])[:, 0]
        lp, miss = -torch.log1p(rest.exp()), torch.sigmoid(rest)
        for got in (token_logp(z, y, tau), clipped_policy_loss(z, y, lp.float(), torch.ones(T).cuda(), temperature=tau).logp):
            assert (got <= 0).all()
            assert ((got.double() - lp).abs() <= rel * lp.abs()).all()
        # A (q - 1) with A = -1 / (tau T) and a ratio of 1; one rounding to the logits' type
        half, tiny = torch.finfo(z.dtype).eps / 2, torch.finfo(z.dtype).smallest_normal * torch.finfo(z.dtype).eps
        out = clipped_policy_loss(z, y, lp.float(), torch.ones(T).cuda(), temperature=tau)
        (gz,) = torch.autograd.grad(out.loss, z)
        want = -miss / (tau * T)
        assert ((gz.double().gather(1, y[:, None])[:, 0] - want).abs() <= (rel + half + 2.0**-20) * want.abs() + tiny).all()
        # distillation: all of the teacher's weight on the token: tau^2 times the mean of -ln q
        loss = topk_distill_loss(z, y[:, None], torch.zeros(T, 1).cuda(), temperature=tau)
        want = -tau * tau * lp.mean()
        assert abs(loss.item() - want.item()) <= (rel + 2.0**-22) * want.item()
    off = torch.tensor([0, 5, T], dtype=torch.int32, device="cuda")
    out = preference_loss(z, y, off, torch.zeros(T, device="cuda"), beta=1.0)
    lp = -torch.log1p((z.detach().double().scatter(1, y[:, None], -math.inf).logsumexp(1)
                       - z.detach().double().gather(1, y[:, None])[:, 0]).exp())
    miss = 1 - lp.exp()
    assert ((out.logp.double() - lp).abs() <= rel * lp.abs()).all() and (out.logp <= 0).all()
    (gz,) = torch.autograd.grad(out.loss, z)
    m = (lp[:5].sum() - lp[5:].sum()).item()
    A = torch.where(torch.arange(T, device="cuda") < 5, 1.0, -1.0).double() / (1 + math.exp(m))
    miss = -torch.expm1(lp)
    tiny = torch.finfo(z.dtype).smallest_normal * torch.finfo(z.dtype).eps
    got = gz.double().gather(1, y[:, None])[:, 0]
    assert ((got + A * miss).abs() <= (rel + torch.finfo(z.dtype).eps / 2 + 2.0**-20) * (A * miss).abs() + tiny).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_the_only_token_has_probability_one(dtype):
    """A vocabulary of one, and rows whose other logits are all -inf: ln q is 0, exactly."""
    from spec_ep.ops.loss import token_logp

    for V in (1, 9, 4104, 900001):
        z = torch.full((7, V), -math.inf, dtype=DT[dtype], device="cuda")
        y = torch.tensor([0, V // 2, V - 1, 0, V // 3, V - 1, 0], device="cuda")
        z[torch.arange(7), y] = torch.tensor([0.0, 0.3, -7.7, 1e4, -1e4, 3.0, 11.1], device="cuda").to(DT[dtype])
        for tau in (1.0, 0.7):
            assert not token_logp(z, y, tau).any()


def _mean_error(z, y, tau, dtype=torch.float32):
    from spec_ep.ops.loss import token_logp

    z = z.to(dtype)
    want = torch.log_softmax(z.double() / tau, 1).gather(1, y[:, None])[:, 0]
    return abs((token_logp(z, y.int(), tau).double() - want).mean().item()), want


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1024, 4096, 20011])
@pytest.mark.parametrize("scale", [1.0, 2.0, 4.0])
@pytest.mark.parametrize("tau", [0.7, 1.0, 2.0])
def test_mean_error_over_tokens(tau, scale, V):
    """What all tokens of a sequence are off by alike adds up in its log-ratio. Single errors
    of a log-probability below 64: the output's rounding (at most 2^-19, 2^-19 / sqrt 3 = 1.1e-6
    rms; 2.8e-7 below 16) and that of a row's sum, at worst one term's (argument roundings
    2^-20 at most, ln 2 2^-20 / sqrt 3, and the hardware's 2^-22: 5e-7 rms). Their mean over
    8192 rows stays within 4 standard errors, and the exponential's mean error is known to 1e-9."""
    T = 8192
    g = torch.Generator("cuda").manual_seed(5)
    z = scale * torch.randn(T, V, generator=g, device="cuda")
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    err, want = _mean_error(z, y, tau)
    out = (2.0 ** (torch.log2(want.abs().clamp_min(1.0)).floor() - 24) / math.sqrt(3)).pow(2).mean().sqrt().item()
    share = torch.softmax(z.double() / tau, 1).pow(2).sum(1).mean().item()  # 1 / effective terms
    assert err < 4 * math.sqrt((out**2 + 2.5e-13 * share) / T) + 2e-9


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1024, 4096, 20011])
@pytest.mark.parametrize("tau", [0.7, 1.0])
def test_mean_error_where_another_token_has_the_weight(tau, V):
    """As above, with one logit far above the rest at a random place."""
    T = 8192
    g = torch.Generator("cuda").manual_seed(6)
    z = 2 * torch.randn(T, V, generator=g, device="cuda")
    top = torch.randint(0, V, (T,), generator=g, device="cuda")
    z[torch.arange(T), top] = 14 + 6 * torch.rand(T, generator=g, device="cuda")
    y = (top + torch.randint(1, V, (T,), generator=g, device="cuda")) % V
    err, want = _mean_error(z, y, tau)
    out = (2.0 ** (torch.log2(want.abs().clamp_min(1.0)).floor() - 24) / math.sqrt(3)).pow(2).mean().sqrt().item()
    assert err < 4 * math.sqrt((out**2 + 2.5e-13) / T) + 2e-9


@pytest.mark.gpu
def test_rows_without_spread():
    """Equal logits, and temperatures so high that all terms are nearly equal: the exponential's
    error is one number there instead of its mean, so the correction by the mean (5.05e-8) may
    remain as an error; beside it the output's rounding."""
    from spec_ep.ops.loss import token_logp

    for V in (9, 4096, 151936):
        y = torch.arange(7, device="cuda")
        bound = math.log(V) * 2.0**-24 + 5.1e-8 + 2.0**-24 * (V / 512 + 8)
        for value in (0.0, 3.0, -250.0, 1e6):
            z = torch.full((7, V), value, device="cuda")
            assert (token_logp(z, y).double() + math.log(V)).abs().max().item() <= bound
        z = torch.randn(7, V, device="cuda")
        want = torch.log_softmax(z.double() / 1e9, 1).gather(1, y[:, None])[:, 0]
        assert (token_logp(z, y, 1e9).double() - want).abs().max().item() <= bound + 2.0**-22
