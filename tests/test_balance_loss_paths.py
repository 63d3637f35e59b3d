"""The routers' balance loss on every way to a loss of the model, and the preference loss of the
model and in its trainer."""
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


def _pairs(cfg, lengths):
    torch.manual_seed(2)
    seqs = [torch.randint(0, cfg.vocab_size, (n,), device="cuda") for n in lengths]
    labels = [s.roll(-1) for s in seqs]
    for y in labels:
        y[-1] = -1
        y[:3] = -1
    return seqs, labels


@pytest.mark.gpu
def test_preference_of_the_model():
    """Each sequence through its own forward: the loss of the sequences' hidden states, plus the
    mean balance loss of all forwards' layers."""
    from spec_ep.ops.loss import lm_head_preference

    cfg, ep, model = _tiny()
    seqs, labels = _pairs(cfg, (40, 7, 33, 64))
    ref = [model.token_logp(s, y) - 0.1 for s, y in zip(seqs, labels)]
    off = torch.tensor([0, 40, 47, 80, 144], dtype=torch.int32, device="cuda")
    h = torch.cat([model.hidden_states(s) for s in seqs])
    want = lm_head_preference(h, model.lm_head, torch.cat(labels), off, torch.cat(ref), 0.3, 0.1)
    got = model.preference(seqs, labels, ref, beta=0.3, label_smoothing=0.1)
    assert torch.equal(got.rewards, want.rewards) and torch.equal(got.logp, want.logp)
    assert torch.equal(got.loss, want.loss)
    params = [model.lm_head, model.layers[0].w_qkv, model.layers[1].w_router]
    for a, b in zip(torch.autograd.grad(got.loss, params), torch.autograd.grad(want.loss, params)):
        assert ((a - b).float().norm() / b.float().norm()).item() < 2.0**-6  # fp32 atomics, bf16 roundings
    model.set_balance_loss(0.25)
    losses = []
    for s in seqs:  # each forward's own balance loss, from a loss that is otherwise known
        y = torch.full_like(s, -1).int()
        losses.append(model(s, y, 1).item())
    # with the balance loss on the router is another kernel (last bits of the weights), so the
    # hidden states are formed again
    h = torch.cat([model.hidden_states(s) for s in seqs])
    want = lm_head_preference(h, model.lm_head, torch.cat(labels), off, torch.cat(ref), 0.3, 0.1)
    with_balance = model.preference(seqs, labels, ref, beta=0.3, label_smoothing=0.1)
    assert with_balance.loss.item() == pytest.approx(want.loss.item() + sum(losses) / 4, rel=1e-5)
    (g,) = torch.autograd.grad(with_balance.loss, model.layers[1].w_router)
    assert g.isfinite().all()
    with pytest.raises(ValueError, match="pairs"):
        model.preference(seqs[:3], labels[:3], ref[:3])
    with pytest.raises(ValueError, match="labels"):
        model.preference(seqs, labels[:3], ref)
    with pytest.raises(ValueError, match="length"):
        model.preference(seqs, [y[1:] for y in labels], ref)
    ep.close()


@pytest.mark.gpu
def test_preference_in_the_trainer():
    from spec_ep.train import Trainer

    cfg, ep, model = _tiny()
    trainer = Trainer(model, lr=1e-3)
    model.set_balance_loss(0.01)
    seqs, labels = _pairs(cfg, (40, 7, 33, 64))
    ref = [model.token_logp(s, y) for s, y in zip(seqs, labels)]
    before = [p.detach().clone() for p in (model.layers[0].w_gu, model.lm_head)]
    for _ in range(2):
        assert trainer.step(lambda: model.preference(seqs, labels, ref).loss).isfinite()
    for b, p in zip(before, (model.layers[0].w_gu, model.lm_head)):
        assert not torch.equal(b, p)
    torch.cuda.synchronize()
    ep.check()
    ep.close()


@pytest.mark.gpu
def test_no_forward_leaves_its_graph_behind():
    cfg, ep, model = _tiny()
    model.set_balance_loss(0.25)
    ids = torch.randint(0, cfg.vocab_size, (64,), device="cuda")
    for f in (lambda: model(ids), lambda: model.hidden_states(ids),
              lambda: model(ids, ids.roll(-1).int(), 64)):
        f()
        for layer in model.layers:
            assert layer.balance_loss is None
    ep.close()
