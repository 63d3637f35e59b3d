"""Waits of the vocabulary losses that run out: a row is never announced to the warps that wait
for it, the limit is 2 ms. Every wait ends, loss and log-probability are NaN, the gradient of
the lost rows is NaN and never what its buffer held, and the next call is right."""
import math

import pytest
import torch

from test_vocab_losses import _logits, _three


def _stall(row, wait_ns=2000000):
    from spec_ep.ops._ext import load

    load().test_stall(row, wait_ns)


def test_limits_are_checked():
    for bad in ((-2, 0), (0, -1), (0, 3 * 10**9)):
        with pytest.raises(RuntimeError):
            _stall(*bad)
    _stall(-1, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T,V", [(700, 1000), (700, 20011), (20, 151936), (3, 50257), (330, 151936)])
@pytest.mark.parametrize("i", [0, 1, 2])
def test_a_row_that_never_comes(i, T, V, dtype):
    z, _ = _logits(T, V, dtype, False, 1)
    want = _three(z, i)
    (gw,) = torch.autograd.grad(want, z)
    for row in (0, T // 2, T - 1):
        _stall(row)
        try:
            loss = _three(z, i)
            torch.cuda.synchronize()
            (g,) = torch.autograd.grad(loss, z)
            torch.cuda.synchronize()
        finally:
            _stall(-1, 0)
        assert loss.isnan()
        assert g[row].isnan().all()
        lost = g.isnan().all(1)
        if i < 2:  # (the preference loss's factors are NaN for both sequences of the pair)
            assert torch.equal(g[~lost], gw[~lost])
        again = _three(z, i)
        assert torch.equal(again, want)
        assert torch.equal(torch.autograd.grad(again, z)[0], gw)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [4104, 151936])
@pytest.mark.parametrize("which", ["distill", "policy", "preference"])
def test_behind_the_lm_head_nothing_finite_is_left(which, V):
    """The gradient buffer is the logits: products of them must not pass for gradients."""
    from test_lm_head_upstream import _head, _lm_head_losses

    h, w, y = _head(V=V)
    f = _lm_head_losses(h, w, y)[which]
    want = f()
    row = int((y >= 0).nonzero()[7])
    _stall(row)
    try:
        loss = f()
        torch.cuda.synchronize()
    finally:
        _stall(-1, 0)
    dh, dw = torch.autograd.grad(loss, (h, w))
    assert loss.isnan() and dh[row].isnan().all() and dw.isnan().all()
    again = f()
    assert torch.equal(again, want)
    for g in torch.autograd.grad(again, (h, w)):
        assert g.isfinite().all()


@pytest.mark.gpu
def test_log_probabilities_without_a_gradient():
    from spec_ep.ops.loss import token_logp

    for T, V in ((9, 151936), (900, 5003)):
        z, _ = _logits(T, V, "bf16", False, 2)
        y = torch.arange(T, device="cuda")
        want = token_logp(z, y)
        _stall(4)
        try:
            got = token_logp(z, y)
            torch.cuda.synchronize()
        finally:
            _stall(-1, 0)
        assert math.isnan(got[4].item())
        ok = ~got.isnan()
        assert torch.equal(got[ok], want[ok])
        assert torch.equal(token_logp(z, y), want)
