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


@pytest.mark.gpu
def test_padding_stays_out_of_the_balance_loss():
    """A batch [1, S] with padding behind it: counts and balance loss are those of the tokens
    before it (attention is causal, so they do not see the padding)."""
    cfg, ep, model = _tiny()
    model.set_balance_loss(0.25)
    S, n = 200, 137
    ids = torch.randint(0, cfg.vocab_size, (1, S), device="cuda")
    valid = torch.arange(S, device="cuda")[None] < n
    none = torch.full((1, S), -1, device="cuda")
    zero = torch.zeros(1, S, device="cuda")
    k = 3
    calls = [lambda v: model(ids, none.int(), 1, valid=v),
             lambda v: model.distill(ids, none[..., None].expand(1, S, k), zero[..., None].expand(1, S, k), valid=v),
             lambda v: model.policy(ids, none, zero, zero, zero, valid=v).loss]
    short = model(ids[:, :n], none[:, :n].int(), 1).item()
    counts = [layer.expert_counts.clone() for layer in model.layers]
    for f in calls:
        # 0 plus the balance loss: the same tokens through kernels of another row count, a
        # choice of equal scores apart; probabilities to the roundings of bf16
        assert f(valid).item() == pytest.approx(short, rel=2.0**-7)
        for layer, c in zip(model.layers, counts):
            assert layer.expert_counts.sum().item() == cfg.top_k * n
            assert (layer.expert_counts - c).abs().sum().item() <= 0.05 * cfg.top_k * n
        assert model.layers[0].expert_counts.sum().item() < cfg.top_k * S
        f(None)
        assert model.layers[0].expert_counts.sum().item() == cfg.top_k * S
    ep.close()
