"""The losses behind the LM head and in the model's training step, as they are used together."""
import math

import pytest
import torch


def _tiny(seed=0, T=256):
    from spec_ep.models.config import get_config
    from spec_ep.models.qwen3_moe import Qwen3MoeForCausalLM
    from spec_ep.parallel.ep import ExpertParallel

    dev = torch.device("cuda", 0)
    cfg = get_config("tiny")
    ep = ExpertParallel(cfg.num_experts, cfg.top_k, cfg.hidden_size, max_tokens=T, device=dev)
    torch.manual_seed(seed)
    return cfg, ep, Qwen3MoeForCausalLM(cfg, ep, device=dev)


def _head_inputs(T=192, H=256, V=4104):
    torch.manual_seed(1)
    h = (torch.randn(T, H, device="cuda") / 4).bfloat16().requires_grad_()
    w = (torch.randn(V, H, device="cuda") / 16).bfloat16().requires_grad_()
    r = torch.arange(T, device="cuda")
    y = torch.where(r % 5 == 0, -1, (r * 37) % V)
    return h, w, y


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["distill", "policy", "preference"])
def test_lm_head_forms_equal_the_losses_of_the_same_logits(which):
    """Loss bit for bit (the same kernel on the same bf16 logits); dh and dw against fp64
    products of the logits-level gradient. The GEMMs round once (2^-8 of a value and of
    the largest term, as bf16 sums go through fp32), the upstream factor and, for the
    preference loss, the factor on h and the unit gradient once more each."""
    from spec_ep.ops import loss as L
    from spec_ep.ops.linear import dense_fwd

    h, w, y = _head_inputs()
    T, V = h.shape[0], w.shape[0]
    z = dense_fwd(h.detach(), w.detach()).requires_grad_()
    old = L.token_logp(z, y) + 0.1
    assert torch.equal(old, L.lm_head_token_logp(h, w, y) + 0.1)
    off = torch.tensor([0, 50, 90, 100, T], dtype=torch.int32, device="cuda")
    ids = torch.where(y[:, None] >= 0, (y[:, None] + torch.arange(4, device="cuda") * 11) % V, -1)
    t = torch.linspace(2, 0, 4, device="cuda").expand(T, 4)
    adv = 1.0 - (torch.arange(T, device="cuda") % 3)
    f = {"distill": (lambda a, *p: L.topk_distill_loss(a, ids, t, temperature=1.5),
                     lambda: L.lm_head_distill(h, w, ids, t, temperature=1.5)),
         "policy": (lambda a, *p: L.clipped_policy_loss(a, y, old, adv, old - 0.2, kl_coef=0.1).loss,
                    lambda: L.lm_head_policy(h, w, y, old, adv, old - 0.2, kl_coef=0.1).loss),
         "preference": (lambda a, *p: L.preference_loss(a, y, off, old, beta=0.5).loss,
                        lambda: L.lm_head_preference(h, w, y, off, old, beta=0.5).loss)}[which]
    want, got = f[0](z), f[1]()
    assert torch.equal(want, got)
    up = torch.tensor(3.0, device="cuda")
    (gz,) = torch.autograd.grad(want, z, up)
    dh, dw = torch.autograd.grad(got, (h, w), up)
    for g, ref in ((dh, gz.double() @ w.double()), (dw, gz.double().t() @ h.double())):
        assert ((g.double() - ref).norm() / ref.norm()).item() < 4 * 2.0**-8
    with torch.no_grad():
        assert abs(f[1]().item() - want.item()) <= 2.0**-22 * abs(want.item())


@pytest.mark.gpu
def test_balance_loss_in_the_model():
    """The loss grows by coef times the mean of the layers' losses, the counts are those of
    the routing, and only gradients below the routers' logits change."""
    cfg, ep, model = _tiny()
    T = 256
    ids = torch.randint(0, cfg.vocab_size, (T,), device="cuda")
    labels = torch.cat([ids[1:], torch.full((1,), -1, device="cuda")]).int()
    seen = []
    for layer in model.layers:
        layer.routing_callback = lambda e: seen.append(e.clone())
    base = model(ids, labels, T - 1)
    model.set_balance_loss(0.25)
    seen.clear()
    loss = model(ids, labels, T - 1)
    for layer, e in zip(model.layers, seen):
        assert torch.equal(layer.expert_counts.long(), torch.bincount(e.reshape(-1).long(), minlength=cfg.num_experts))
        assert layer.balance_loss is None
    # counts and mean probabilities of a softmax router: at least about 1, at most E
    assert 0.25 * 0.9 < (loss - base).item() < 0.25 * cfg.num_experts
    (g0,) = torch.autograd.grad(base, model.layers[1].w_router, retain_graph=True)
    (g1,) = torch.autograd.grad(loss, model.layers[1].w_router, retain_graph=True)
    assert (g1 - g0).abs().max().item() > 0 and g1.isfinite().all()
    # the head's gradient does not see the routers' term
    (h0,) = torch.autograd.grad(base, model.final_norm)
    (h1,) = torch.autograd.grad(loss, model.final_norm)
    assert ((h0 - h1).abs().max() / h0.abs().max()).item() < 2.0**-6  # fp32 atomics, one bf16 rounding each
    model.set_balance_loss(0.0)
    assert model(ids, labels, T - 1).item() == pytest.approx(base.item(), rel=2.0**-12)
    with torch.no_grad():
        model.set_balance_loss(0.25)
        assert model(ids, labels, T - 1).item() == pytest.approx(base.item(), rel=2.0**-12)
    with pytest.raises(ValueError):
        model.set_balance_loss(-1.0)
    with pytest.raises(ValueError):
        model.set_balance_loss(math.nan)
    ep.close()


@pytest.mark.gpu
def test_training_steps_with_each_loss():
    """Trainer.step on the policy and the distillation loss with the balance loss: finite
    losses and metrics, parameters move, and a policy equal to its old self has ratio 1."""
    from spec_ep.train import Trainer

    cfg, ep, model = _tiny()
    trainer = Trainer(model, lr=1e-3)
    model.set_balance_loss(0.01)
    T = 256
    ids = torch.randint(0, cfg.vocab_size, (T,), device="cuda")
    actions = torch.where(torch.arange(T, device="cuda") < 100, -1, ids.roll(-1))
    old = model.token_logp(ids, actions)
    assert not old[:100].any() and (old[100:] < 0).all()
    adv = torch.randn(T, device="cuda")
    with torch.no_grad():
        out = model.policy(ids, actions, old, adv, old)
    # ratio 1: -mean(A), up to the two passes' rounding of the same bf16 logits
    assert out.loss.item() == pytest.approx(-adv[100:].mean().item(), abs=1e-5) and out.kl.abs().max().item() < 1e-9
    before = model.layers[0].w_router.detach().clone()
    last = []

    def policy_loss():
        last.append(model.policy(ids, actions, old, adv, old, kl_coef=0.05, clip_high=0.28))
        return last[-1].loss

    for _ in range(2):
        assert trainer.step(policy_loss).isfinite()
    assert last[-1].kl.isfinite().all() and last[-1].kl.max().item() > 0
    assert not torch.equal(before, model.layers[0].w_router)
    with torch.no_grad():
        teacher = model(ids).float().topk(8, -1)
    before = model.lm_head.detach().clone()
    for _ in range(2):
        assert trainer.step(lambda: model.distill(ids, teacher.indices, teacher.values)).isfinite()
    assert not torch.equal(before, model.lm_head)
    torch.cuda.synchronize()
    ep.check()
    ep.close()
