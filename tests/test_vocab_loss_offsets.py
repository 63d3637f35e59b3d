"""Gradients of the vocabulary losses over logits with a common offset.

Errors counted: an exponential 2^a is off by the roundings of its argument (two of a number
below 16 + |a|) and the hardware's 2^-22; a row's sum adds the rounding of its partial sums
(``_lse_tol``). With logits around an offset c, the exponents' constant in two parts adds
2^-36 of |c| log2(e) / tau twice (its own rounding and that of the product with its first part),
up to 2^17; beyond that the difference from the largest logit is taken first.
"""
import math

import pytest
import torch

from test_vocab_losses import _lse_tol, distill_ref, policy_ref, preference_ref


def _offset_tol(V, c, tau):
    M = abs(c) * math.log2(math.e) / tau
    return _lse_tol(V) + 2.0**-24 * 40 + (2 * M * 2.0**-36 if M <= 2.0**17 else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [515, 2050, 20011])
@pytest.mark.parametrize("c", [0.0, 1e3, -2e4, 8e4, 1e5, -3e6])
@pytest.mark.parametrize("tau", [1.0, 0.7])
def test_gradients_of_logits_with_an_offset(tau, c, V):
    """Dense elements A q to a relative tolerance (an absolute one would hide them below the
    label's), and rows of every gradient sum to 0."""
    from spec_ep.ops.loss import clipped_policy_loss, preference_loss, topk_distill_loss

    T = 8
    g = torch.Generator().manual_seed(3)
    z = (2 * torch.randn(T, V, generator=g) + c).cuda().requires_grad_()
    y = torch.randint(0, V, (T,), generator=g).cuda()
    ids = torch.randint(0, V, (T, 5), generator=g).cuda()
    t = torch.linspace(1, 0, 5).expand(T, 5).cuda()
    off = torch.tensor([0, 3, 8], dtype=torch.int32).cuda()
    lp = torch.log_softmax(z.detach().double(), 1).gather(1, y[:, None])[:, 0]
    old, adv = (torch.log_softmax(z.detach().double() / tau, 1).gather(1, y[:, None])[:, 0] - 0.1).float(), torch.ones(T).cuda()
    cases = [(topk_distill_loss(z, ids, t, temperature=tau), distill_ref(z, ids, t, tau)[1], ids, tau),
             (clipped_policy_loss(z, y, old, adv, temperature=tau).loss,
              policy_ref(z, y, old, adv, None, 0.2, 0.2, 0.0, tau)[3], y[:, None], tau),
             (preference_loss(z, y, off, lp.float() - 0.1).loss, preference_ref(z, y, off, lp.float() - 0.1, 0.1, 0.0)[3],
              y[:, None], 1.0)]
    for loss, want, own, tau_ in cases:
        tol = _offset_tol(V, c, tau_)
        (got,) = torch.autograd.grad(loss, z)
        got = got.double()
        dense = torch.ones_like(got, dtype=torch.bool).scatter_(1, own, False)
        # the rows' factor of the policy and preference losses is off by a log-probability's error
        rel = 2 * tol + 8 * 2.0**-24 + 16 * 2.0**-24
        err = ((got - want).abs() / want.abs())[dense].max().item()
        assert err <= rel, f"relative error {err:.3g} above {rel:.3g}"
        assert (got.sum(1).abs() <= rel * got.abs().sum(1)).all()
