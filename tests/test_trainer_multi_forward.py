"""One optimizer step on a loss of several forward passes: every expert is updated once, with
the sum of the passes' gradients, after the last pass has used its weights."""
import pytest
import torch


class _Opt:
    def __init__(self):
        self.calls = []

    def apply_now(self, p, g):
        self.calls.append((p, g.clone()))

    def fused_wgrad(self, *a):
        raise AssertionError("fused update of a weight that other passes still use")


class _Trainer:
    expert_world, fuse_expert_optimizer, expert_dp_group = 1, True, None

    def __init__(self):
        self.opt, self.model = _Opt(), object()


def test_expert_updater_waits_for_the_last_pass():
    """CPU: the updater alone."""
    from spec_ep.train import _ExpertUpdater

    t = _Trainer()
    u = _ExpertUpdater(t)
    p, q = torch.zeros(3), torch.zeros(2)
    g1, g2, g3 = torch.tensor([1.0, 2.0, 3.0]), torch.tensor([4.0, 5.0, 6.0]), torch.ones(2)
    # one pass: fused, or at once
    u.begin()
    u.used(p)
    assert u.fused_for(p) == t.opt.fused_wgrad
    u(p, g1.clone())
    assert len(t.opt.calls) == 1 and torch.equal(t.opt.calls[0][1], g1)
    u.flush()
    # two passes of p, one of q; a discarded attempt before them does not count
    t.opt.calls.clear()
    u.begin()
    u.used(p)
    u.begin()
    u.used(p)
    u.used(q)
    u.used(p)
    assert u.fused_for(p) is None and u.fused_for(q) == t.opt.fused_wgrad
    u(p, g1.clone())
    assert not t.opt.calls
    u(q, g3)
    u(p, g2.clone())
    assert [c[0] is x for c, x in zip(t.opt.calls, (q, p))] == [True, True]
    assert torch.equal(t.opt.calls[1][1], g1 + g2)
    u.flush()
    assert len(t.opt.calls) == 2
    # a pass whose loss was not used: what the others left is applied at the end
    t.opt.calls.clear()
    u.begin()
    u.used(p)
    u.used(p)
    u(p, g2.clone())
    assert not t.opt.calls
    u.flush()
    assert len(t.opt.calls) == 1 and torch.equal(t.opt.calls[0][1], g2)
    # outside of a step: at once, as ever
    u.end()
    u.used(p)
    u.used(p)
    assert u.fused_for(p) == t.opt.fused_wgrad
    u(p, g1.clone())
    assert len(t.opt.calls) == 2


def _setup(state, fuse=None):
    from spec_ep.models.config import get_config
    from spec_ep.models.qwen3_moe import Qwen3MoeForCausalLM
    from spec_ep.parallel.ep import ExpertParallel
    from spec_ep.train import Trainer

    dev = torch.device("cuda", 0)
    cfg = get_config("tiny")
    ep = ExpertParallel(cfg.num_experts, cfg.top_k, cfg.hidden_size, max_tokens=256, device=dev)
    torch.manual_seed(0)
    model = Qwen3MoeForCausalLM(cfg, ep, device=dev)
    return cfg, ep, model, Trainer(model, lr=1e-3, expert_state=state, fuse_expert_optimizer=fuse)


@pytest.mark.gpu
@pytest.mark.parametrize("state,fuse", [("fp32", False), ("fp32", True), ("8bit", None)])
def test_step_over_two_forwards_updates_the_experts_once(state, fuse):
    """First moments after one step are (1 - b1) times the sum of both passes' gradients. The
    reference gradients go through bf16 (2 roundings of 2^-8 per value; 2^-7 of the norm),
    8-bit moments are off by 1 / 254 of their block's largest (which is below 4 times the
    norm's root mean square: 2% of the norm). A second update would leave 10% of one pass."""
    from spec_ep.ops.optim import decode_8bit

    cfg, ep, model, trainer = _setup(state, fuse)
    T = 200
    torch.manual_seed(1)
    ids = [torch.randint(0, cfg.vocab_size, (T,), device="cuda") for _ in range(2)]
    labels = [i.roll(-1).int() for i in ids]

    def loss_fn():
        return sum(model(i, y, T) for i, y in zip(ids, labels))

    model.set_grad_sink(None)
    loss_fn().backward()
    want = [p.grad.float() for p in trainer.experts]
    dense = [p.grad.float() for p in trainer.dense]
    trainer.opt.zero_grad()
    model.set_grad_sink(trainer.expert_updater)
    before = [p.detach().clone() for p in trainer.experts]
    assert trainer.step(loss_fn).isfinite()
    for p, g, b in zip(trainer.experts, want, before):
        st = trainer.opt.state[id(p)]
        m = st["m"] if state == "fp32" else decode_8bit(st["mq"], st["ms"], st["vq"], st["vs"])[0]
        m = m.reshape(g.shape).float() / (1 - trainer.opt.betas[0])
        assert ((m - g).norm() / g.norm()).item() < (2.0**-7 if state == "fp32" else 2.0**-7 + 0.02)
        assert not torch.equal(p, b)
    for p, g in zip(trainer.dense, dense):
        m = trainer.opt.state[id(p)]["m"].reshape(g.shape).float() / (1 - trainer.opt.betas[0])
        assert ((m - g).norm() / g.norm().clamp_min(1e-30)).item() < 2.0**-6  # fp32 atomics, bf16 gradients
    # a step of one forward keeps the fused path, and more steps work
    assert trainer.step(lambda: model(ids[0], labels[0], T)).isfinite()
    assert trainer.step(loss_fn).isfinite()
    torch.cuda.synchronize()
    ep.check()
    ep.close()
