"""Vocabulary losses over logits with finite mask values, against definitions in 64 bits.

Masks of -1e4 to -1e30 (and the types' lowest values), over parts of the vocabulary and over
whole rows, and rows at +1e10. Tolerances: those of test_vocab_losses (``_lse_tol``: argument
roundings, the hardware exponential and the sum). The exponents' constant in two parts of 12
and 24 bits adds 2^-36 of |z| log2(e) / tau, at most 2^-18 for |z| log2(e) / tau <= 2^17;
beyond that the difference from the row's largest logit is taken first.
"""
import math

import pytest
import torch

from test_vocab_losses import DT, _lse_tol, distill_ref, policy_ref, preference_ref

MASKS = [-1e4, -6e4, -1e5, -1e6, -1e9, -1e10, -1e20, -1e30, 1e10]


def _tol(V):
    return _lse_tol(V) + 2.0**-18


def _near(got, want, rtol, atol):
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all()
    over = ((got - want).abs() - (rtol * want.abs() + atol)).max().item()
    assert over <= 0, f"off by {over:.3g} more than allowed"


def _masked(V, dtype, value, seed=0):
    """Rows: ordinary; most of the vocabulary masked at its start, at its end, and all but
    two of it; everything masked; the highest logit of a masked row one step above it."""
    g = torch.Generator().manual_seed(seed)
    z = (2 * torch.randn(6, V, generator=g)).to(DT[dtype])
    value = torch.tensor(value).to(DT[dtype])
    z[1, :V - 40] = value
    z[2, 40:] = value
    z[3, :] = value
    z[3, [3, V - 2]] = torch.tensor([1.0, 0.5]).to(DT[dtype])
    z[4:] = value
    z[5, V // 2] = value.float() * (1 + math.copysign(2.0**-6, value.item()))
    y = torch.tensor([5, V - 7, 11, V - 2, 9, V // 2])
    return z.cuda().requires_grad_(), y.cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 4104, 50257, 151936, 900001])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("value", MASKS)
def test_finite_masks(value, dtype, V):
    from spec_ep.ops.loss import clipped_policy_loss, preference_loss, token_logp, topk_distill_loss

    if dtype == "fp16":
        value = max(value, -65504.0) if value < 0 else 6e4
    for tau in (1.0, 0.7):
        z, y = _masked(V, dtype, value)
        T = z.shape[0]
        tol, half = _tol(V), torch.finfo(z.dtype).eps / 2
        tiny = torch.finfo(z.dtype).smallest_normal * torch.finfo(z.dtype).eps
        ids = torch.stack([y, (y + 1) % V], 1)
        ids[:, 1] = torch.where(z.detach().gather(1, ids[:, 1:])[:, 0].float().abs() < 100, ids[:, 1], -1)
        t = torch.tensor([1.0, 0.0], device="cuda").expand(T, 2)
        want, grad, coef = distill_ref(z, ids, t, tau)
        loss = topk_distill_loss(z, ids, t, temperature=tau)
        # P from a logarithm, a quotient and an exponential: 4 roundings of numbers below 2, and
        # one of the result
        _near(loss, want, 16 * 2.0**-24, tau * tau * (2 * tol + 64 / tau * 2.0**-24))
        # the label's or an entry's element is a difference of two near A; others are A q
        _near(torch.autograd.grad(loss, z)[0], grad, half + 2 * tol + 8 * 2.0**-24, coef.double()[:, None] * tol + tiny)

        lp64 = torch.log_softmax(z.detach().double() / tau, 1).gather(1, y[:, None])[:, 0]
        _near(token_logp(z, y, tau), lp64, 4 * 2.0**-24, tol)
        y = torch.where(lp64 > -1000, y, -1)  # a ratio of probabilities needs some
        old, adv = (lp64 - 0.05).float(), torch.ones(T, device="cuda")
        want, lp, _, grad, coef = policy_ref(z, y, old, adv, None, 0.2, 0.2, 0.0, tau)
        out = clipped_policy_loss(z, y, old, adv, temperature=tau)
        e = tol + 4 * 2.0**-24 * lp.abs().max().item()
        _near(out.logp, lp, 4 * 2.0**-24, tol)
        _near(out.loss, want, 8 * 2.0**-24, 2 * e)
        _near(torch.autograd.grad(out.loss, z)[0], grad, half + 2 * tol + 8 * 2.0**-24 + 2 * e,
              coef.double()[:, None] * 2 * e + tiny)

    lp64 = torch.log_softmax(z.detach().double(), 1).gather(1, y.clamp_min(0)[:, None])[:, 0]
    y = torch.where(lp64 > -1000, y, -1)
    off = torch.tensor([0, 1, 3, 4, 6], dtype=torch.int32, device="cuda")
    ref = (lp64 - 0.1).float()
    want, R, lp, grad, coef = preference_ref(z, y, off, ref, 0.3, 0.1)
    out = preference_loss(z, y, off, ref, beta=0.3, label_smoothing=0.1)
    e = tol + 4 * 2.0**-24 * lp.abs().max().item()
    _near(out.logp, lp, 4 * 2.0**-24, tol)
    _near(out.rewards, R, 2.0**-24, 2 * 0.3 * e)
    _near(out.loss, want, 2.0**-23, 4 * 0.3 * e)
    # the rows' factor is off by beta / pairs times the margin's error, slope at most 1/4
    _near(torch.autograd.grad(out.loss, z)[0], grad, half + 2 * tol + 8 * 2.0**-24 + 4 * 0.3 * e,
          coef.double()[:, None] * (tol + 4 * 0.3 * e) + tiny)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("value", [-1e5, -1e10, -1e30])
def test_finite_masks_over_many_rows(value, dtype):
    """A restricted vocabulary (all but 64 neighbouring entries masked) in more rows than
    blocks: the log-probabilities are those of the 64 entries alone."""
    from spec_ep.ops.loss import token_logp

    for V in (1000, 8000, 40001):
        T = 1500
        g = torch.Generator().manual_seed(V)
        z = torch.full((T, V), value, dtype=DT[dtype])
        at = torch.randint(0, V - 64, (T,), generator=g)
        cols = at[:, None] + torch.arange(64)
        few = (2 * torch.randn(T, 64, generator=g)).to(DT[dtype])
        z.scatter_(1, cols, few)
        y = at + torch.randint(0, 64, (T,), generator=g)
        want = torch.log_softmax(few.double(), 1).gather(1, (y - at)[:, None])[:, 0].cuda()
        _near(token_logp(z.cuda(), y.cuda()), want, 0.0, _tol(V) + 4 * 2.0**-24 * 20)
