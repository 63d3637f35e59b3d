"""The balance loss and the routing with and without gradients."""
import pytest
import torch


def _tiny(T=256):
    from spec_ep.models.config import get_config
    from spec_ep.models.qwen3_moe import Qwen3MoeForCausalLM
    from spec_ep.parallel.ep import ExpertParallel

    dev = torch.device("cuda", 0)
    cfg = get_config("tiny")
    ep = ExpertParallel(cfg.num_experts, cfg.top_k, cfg.hidden_size, max_tokens=T, device=dev)
    torch.manual_seed(0)
    return cfg, ep, Qwen3MoeForCausalLM(cfg, ep, device=dev)


@pytest.mark.gpu
def test_same_routing_with_and_without_gradients():
    """With the balance loss on, a pass under no_grad (a rollout's log-probabilities) routes
    with the same kernel as the training pass: the weights have the same bits."""
    import spec_ep.models.qwen3_moe as M

    cfg, ep, model = _tiny()
    model.set_balance_loss(0.25)
    ids = torch.randint(0, cfg.vocab_size, (256,), device="cuda")
    seen = []
    orig = M.ep_moe

    def spy(x, topk_e, topk_w, *a, **kw):
        seen.append((x.detach().clone(), topk_e.clone(), topk_w.detach().clone()))
        return orig(x, topk_e, topk_w, *a, **kw)

    M.ep_moe = spy
    try:
        model.hidden_states(ids)
        with torch.no_grad():
            model.hidden_states(ids)
    finally:
        M.ep_moe = orig
    assert len(seen) == 2 * cfg.num_layers
    x0, e0, w0 = seen[0]
    x1, e1, w1 = seen[cfg.num_layers]
    assert torch.equal(x0, x1)  # the same input of the first layer's router
    assert torch.equal(e0, e1) and torch.equal(w0, w1)
    ep.close()
