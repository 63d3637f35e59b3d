"""Forward-mode derivatives of the losses and of the balanced router are refused."""
import pytest
import torch

from test_lm_head_upstream import _head, _lm_head_losses


@pytest.mark.gpu
def test_forward_mode_is_refused():
    """A tangent on the logits, with or without requires_grad, is an error and never lost."""
    import torch.autograd.forward_ad as fwd

    from spec_ep.ops import loss as L
    from spec_ep.ops.router import router_topk_balanced

    T, V = 6, 64
    y, f = torch.arange(T, device="cuda"), torch.zeros(T, device="cuda")
    off = torch.tensor([0, 3, T], dtype=torch.int32, device="cuda")
    calls = [lambda x: L.topk_distill_loss(x, y[:, None], f[:, None]), lambda x: L.clipped_policy_loss(x, y, f, f),
             lambda x: L.preference_loss(x, y, off, f), lambda x: router_topk_balanced(x, 4)]
    for needs in (False, True):
        for call in calls:
            with fwd.dual_level():
                x = fwd.make_dual(torch.randn(T, V, device="cuda", requires_grad=needs), torch.ones(T, V, device="cuda"))
                with pytest.raises(RuntimeError, match="jvp|forward"):
                    call(x)
    h, w, labels = _head()
    h, w = h.detach(), w.detach()
    for which in ("distill", "policy", "preference"):
        for i in range(2):
            with fwd.dual_level():
                a = [h, w]
                a[i] = fwd.make_dual(a[i], torch.ones_like(a[i]))
                with pytest.raises(RuntimeError, match="jvp|forward"):
                    _lm_head_losses(*a, labels)[which]()
    # no tangent: as ever
    with fwd.dual_level():
        assert calls[0](torch.zeros(T, V, device="cuda")).isfinite()
        assert _lm_head_losses(h, w, labels)["policy"]().isfinite()
