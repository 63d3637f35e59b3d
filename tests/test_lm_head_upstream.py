"""Upstream factors of the losses behind the LM head."""
import pytest
import torch


def _head(T=192, H=256, V=4104):
    torch.manual_seed(1)
    h = (torch.randn(T, H, device="cuda") / 4).bfloat16().requires_grad_()
    w = (torch.randn(V, H, device="cuda") / 16).bfloat16().requires_grad_()
    r = torch.arange(T, device="cuda")
    return h, w, torch.where(r % 5 == 0, -1, (r * 37) % V)


def _lm_head_losses(h, w, y):
    from spec_ep.ops import loss as L

    T, V = h.shape[0], w.shape[0]
    ids = torch.where(y[:, None] >= 0, (y[:, None] + torch.arange(4, device="cuda") * 11) % V, -1)
    t = torch.linspace(2, 0, 4, device="cuda").expand(T, 4)
    old = torch.full((T,), -8.0, device="cuda")
    adv = 1.0 - (torch.arange(T, device="cuda") % 3)
    off = torch.tensor([0, 50, 90, 100, T], dtype=torch.int32, device="cuda")
    return {"distill": lambda: L.lm_head_distill(h, w, ids, t, temperature=1.5),
            "policy": lambda: L.lm_head_policy(h, w, y, old, adv, old - 0.2, kl_coef=0.1, clip_high=99.0).loss,
            "preference": lambda: L.lm_head_preference(h, w, y, off, old, beta=0.5).loss}


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["distill", "policy", "preference"])
@pytest.mark.parametrize("up", [1 / 3, 0.1, 1000.0, 1.0])
def test_upstream_factor_behind_the_lm_head(up, which):
    """A factor that bf16 does not hold reaches dh and dw in fp32. Each value of the gradient
    under a factor of 1, and under this one, was rounded to bf16 once before and once after the
    factor (and the preference loss's terms of dw once on h): 2^-8 each.

    As the ratio of both gradients those roundings average out, but not without limit: a bf16
    number has 128 mantissas, so a product with one fixed factor has 128 different relative
    errors, however many values there are. Each is uniform within half a step (2^-9 to 2^-8 of
    the value, 2^-8.5 / sqrt(3) rms), their mean 2^-8.5 / sqrt(3 * 128) = 1.4e-4 rms; 6 of those
    are 8.5e-4. A factor rounded to bf16 would show: 0.1 is 9.8e-4 off, 1/3 2e-3 (1000 and 1 are
    bf16 numbers)."""
    h, w, y = _head()
    f = _lm_head_losses(h, w, y)[which]
    one = torch.autograd.grad(f(), (h, w))
    got = torch.autograd.grad(f(), (h, w), torch.tensor(up, device="cuda"))
    for g, o in zip(got, one):
        g, o = g.double(), o.double()
        assert ((g - up * o).norm() / (up * o.norm())).item() < 2 * 2.0**-8
        assert abs((g * o).sum().item() / (o * o).sum().item() / up - 1) < 8.5e-4
