"""Qwen3-MoE-shaped decoder on the sm_100a ops, with expert parallelism.

Per layer:
    h = RMSNorm(x)
    qkv = h @ W_qkv^T                              (one fused projection, tcgen05 GEMM)
    q, k, v = qk_norm_rope(qkv)                    (per-head RMSNorm + RoPE, one kernel)
    x = x + attn(q, k, v) @ W_o^T                  (causal GQA)
    h = RMSNorm(x)
    w, e = router_topk(h @ W_router^T)             (softmax / top-k / renorm kernel)
    x = x + MoE(h; e, w)                           (EP dispatch -> tcgen05 GEMMs -> combine;
                                                    the residual add is folded into the
                                                    source-side reduction)

Expert weights use the transformers layout (``gate_up_proj [E, 2I, H]``,
``down_proj [E, H, I]``) restricted to this rank's local experts; see
``spec_ep.integrations.hf_qwen`` for loading HF checkpoints.

Reference parity: the reference's model path runs HF Qwen3.5-MoE under DeepSpeed AutoEP,
forward only (scripts/ds_moe.py:26-61, :145-174); this module is the trainable
equivalent with the dispatch of src/rbd.py wired into the MoE block.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops.attention import causal_gqa_attention
from ..ops.linear import dense_fwd, linear
from ..ops.loss import (PolicyLoss, PreferenceLoss, lm_head_distill, lm_head_policy, lm_head_preference,
                        lm_head_token_logp, lm_head_xent)
from ..ops.norm import add_rms_norm, rms_norm, rms_norm_res
from ..ops.rope import qk_norm_rope
from ..ops.router import router_topk, router_topk_balanced
from ..parallel.ep import ExpertParallel, ep_moe
from .config import MoEModelConfig


def _normal(shape, std, device, dtype):
    return torch.empty(shape, device=device, dtype=dtype).normal_(0.0, std)


class Qwen3MoeLayer(nn.Module):
    def __init__(self, cfg: MoEModelConfig, ep: ExpertParallel, device, dtype=torch.bfloat16):
        super().__init__()
        H, D, I = cfg.hidden_size, cfg.head_dim, cfg.moe_intermediate_size
        std = cfg.initializer_range
        self.cfg, self.ep = cfg, ep
        self.input_norm = nn.Parameter(torch.ones(H, device=device, dtype=dtype))
        self.w_qkv = nn.Parameter(_normal((cfg.qkv_width, H), std, device, dtype))
        self.q_norm = nn.Parameter(torch.ones(D, device=device, dtype=dtype))
        self.k_norm = nn.Parameter(torch.ones(D, device=device, dtype=dtype))
        self.w_o = nn.Parameter(_normal((H, cfg.num_heads * D), std, device, dtype))
        self.post_norm = nn.Parameter(torch.ones(H, device=device, dtype=dtype))
        self.w_router = nn.Parameter(_normal((cfg.num_experts, H), std, device, dtype))
        G = ep.G
        self.w_gu = nn.Parameter(_normal((G, 2 * I, H), std, device, dtype))
        self.w_d = nn.Parameter(_normal((G, H, I), std, device, dtype))
        for p in (self.w_gu, self.w_d):
            p._sepx_expert = True
        self.grad_sink = None
        self.router_bias = None  # optional selection bias added to the probabilities
        self.router_logit_bias = None  # optional fp32 [E] bias added to the router logits (skew studies)
        self.routing_callback = None  # receives topk expert ids (routing capture)
        self.spec = None  # SpeculativeExperts (speculative replication, inference only)
        self.balance = False  # route with the balance loss, into the two below
        self.balance_loss = None  # this forward's loss, until the model has added it to its own
        self.expert_counts = None  # tokens of the last forward that chose each expert, [E] int32

    def forward(self, x, pos=None, valid=None):
        cfg = self.cfg
        spec = self.spec
        x_in = x
        if spec is not None:
            if torch.is_grad_enabled() and self.w_gu.requires_grad:
                raise RuntimeError("speculative expert replication is inference-only: run under torch.no_grad()")
            # predict this layer's experts from the incoming residual stream; the replica
            # fetch runs on a side stream while the attention below executes
            spec.speculate(x, self.post_norm, self.w_router, cfg.top_k, cfg.rms_norm_eps, cfg.norm_topk_prob,
                           self.router_bias, self.router_logit_bias)
        # the residual adds and the gradient sums of the residual stream ride in the norm
        # kernels (rms_norm_res, add_rms_norm)
        h, x = rms_norm_res(x, self.input_norm, cfg.rms_norm_eps)
        qkv = linear(h, self.w_qkv)
        q, k, v = qk_norm_rope(qkv, self.q_norm, self.k_norm, cfg.num_heads, cfg.num_kv_heads, cfg.rms_norm_eps,
                               cfg.rope_theta, pos)
        a = causal_gqa_attention(q, k, v)
        x, h = add_rms_norm(x, linear(a, self.w_o), self.post_norm, cfg.rms_norm_eps)
        logits = linear(h, self.w_router)
        if self.router_logit_bias is not None:
            logits = logits.float() + self.router_logit_bias
        if self.balance:  # without gradients too: a rollout routes with the training pass's bits
            topk_w, topk_e, loss, self.expert_counts = router_topk_balanced(
                logits, cfg.top_k, cfg.norm_topk_prob, self.router_bias, valid)
            self.balance_loss = loss if torch.is_grad_enabled() else None
        else:
            topk_w, topk_e = router_topk(logits.float(), cfg.top_k, cfg.norm_topk_prob, self.router_bias)
        if self.routing_callback is not None:
            self.routing_callback(topk_e)
        if spec is not None:
            spec.observe(x_in, topk_e)
            return ep_moe(h, topk_e, topk_w, spec.w_gu, spec.w_d, self.ep, None, residual=x, route=spec.tables())
        return ep_moe(h, topk_e, topk_w, self.w_gu, self.w_d, self.ep, self.grad_sink, residual=x)


class Qwen3MoeForCausalLM(nn.Module):
    """Decoder-only MoE LM; ``forward(input_ids, labels)`` returns the mean CE loss, ``distill``,
    ``policy`` and ``preference`` the losses of their names. ``set_balance_loss`` adds the
    routers' balance loss to each."""

    def __init__(self, cfg: MoEModelConfig, ep: ExpertParallel, device=None, dtype=torch.bfloat16):
        super().__init__()
        device = device or ep.device
        self.cfg, self.ep = cfg, ep
        self.balance_coef = 0.0
        self.embed = nn.Parameter(_normal((cfg.vocab_size, cfg.hidden_size), cfg.initializer_range, device, dtype))
        self.layers = nn.ModuleList([Qwen3MoeLayer(cfg, ep, device, dtype) for _ in range(cfg.num_layers)])
        self.final_norm = nn.Parameter(torch.ones(cfg.hidden_size, device=device, dtype=dtype))
        if cfg.tie_word_embeddings:
            self.lm_head = self.embed
        else:
            self.lm_head = nn.Parameter(_normal((cfg.vocab_size, cfg.hidden_size), cfg.initializer_range, device,
                                                dtype))

    def expert_parameters(self):
        return [p for p in self.parameters() if getattr(p, "_sepx_expert", False)]

    def dense_parameters(self):
        return [p for p in self.parameters() if not getattr(p, "_sepx_expert", False)]

    def set_grad_sink(self, sink):
        for layer in self.layers:
            layer.grad_sink = sink

    def set_balance_loss(self, coef: float):
        """Add ``coef`` times the layers' mean router balance loss to the losses that this model
        returns (0: off); a loss formed from ``hidden_states`` gets none. Tokens that a loss's
        ``valid`` (bool, one per token) leaves out, such as padding, do not count in it. Each
        layer then also keeps its last forward's ``expert_counts``."""
        if not coef >= 0.0:
            raise ValueError(f"the balance loss's coefficient must be >= 0, not {coef}")
        self.balance_coef = float(coef)
        for layer in self.layers:
            layer.balance = coef > 0.0

    def _hidden(self, input_ids, pos, valid=None):
        """Hidden states of one token stream, and the layers' balance losses (none without
        gradients, or where the loss is off)."""
        x = F.embedding(input_ids.view(-1), self.embed)
        valid = None if valid is None else valid.reshape(-1)
        balance = []
        for layer in self.layers:
            x = layer(x, pos, valid)
            if layer.balance_loss is not None:
                balance.append(layer.balance_loss)
                layer.balance_loss = None  # its graph lives as long as the loss's
        return rms_norm(x, self.final_norm, self.cfg.rms_norm_eps), balance

    def _with_balance(self, loss, balance):
        return loss + self.balance_coef * torch.stack(balance).mean() if balance else loss

    def hidden_states(self, input_ids, pos=None):
        return self._hidden(input_ids, pos)[0]

    def forward(self, input_ids, labels=None, num_valid=None, pos=None, valid=None):
        h, balance = self._hidden(input_ids, pos, valid)
        if labels is None:
            return dense_fwd(h, self.lm_head)
        return self._with_balance(lm_head_xent(h, self.lm_head, labels.view(-1), num_valid), balance)

    def distill(self, input_ids, teacher_ids, teacher_logits, temperature=1.0, num_valid=None, pos=None,
                valid=None):
        """Distillation loss of one token stream from a teacher's top logits ``[T, K]`` per
        token (see ``spec_ep.ops.loss.topk_distill_loss``)."""
        h, balance = self._hidden(input_ids, pos, valid)
        ids, t = (x.reshape(-1, x.shape[-1]) for x in (teacher_ids, teacher_logits))
        return self._with_balance(lm_head_distill(h, self.lm_head, ids, t, temperature, num_valid), balance)

    def policy(self, input_ids, actions, old_logp, advantages, ref_logp=None, pos=None, valid=None,
               **kw) -> PolicyLoss:
        """Clipped policy loss of one token stream: ``actions[t]`` is the token chosen after
        token ``t``, -1 where none was (see ``spec_ep.ops.loss.clipped_policy_loss``, whose
        other arguments go through ``kw``)."""
        h, balance = self._hidden(input_ids, pos, valid)
        actions, old_logp, advantages, ref_logp = (None if x is None else x.reshape(-1)
                                                   for x in (actions, old_logp, advantages, ref_logp))
        out = lm_head_policy(h, self.lm_head, actions, old_logp, advantages, ref_logp, **kw)
        return out._replace(loss=self._with_balance(out.loss, balance))

    def preference(self, sequences, labels, ref_logp, beta=0.1, label_smoothing=0.0) -> PreferenceLoss:
        """Paired preference loss of ``2 * pairs`` token sequences, the chosen one of each pair
        before the rejected one, each through a forward of its own (attention is causal over a
        whole token stream). ``labels[s]`` and ``ref_logp[s]`` belong to ``sequences[s]``: the
        next tokens, -1 where not in the loss, and the reference model's ``token_logp`` of them
        (see ``spec_ep.ops.loss.preference_loss``, which has the sequences one after another)."""
        if not sequences or len(sequences) % 2:
            raise ValueError(f"sequences must come in pairs, not {len(sequences)}")
        if len(labels) != len(sequences) or len(ref_logp) != len(sequences):
            raise ValueError("every sequence needs its labels and ref_logp")
        ends = [0]
        for s, y, r in zip(sequences, labels, ref_logp):
            if not s.numel() == y.numel() == r.numel():
                raise ValueError("a sequence, its labels and its ref_logp must have one length")
            ends.append(ends[-1] + s.numel())
        hs, balance = [], []
        for s in sequences:
            h, b = self._hidden(s, None)
            hs.append(h)
            balance += b
        off = torch.tensor(ends, dtype=torch.int32, device=hs[0].device)
        out = lm_head_preference(torch.cat(hs), self.lm_head, torch.cat([y.view(-1) for y in labels]), off,
                                 torch.cat([r.view(-1) for r in ref_logp]), beta, label_smoothing)
        return out._replace(loss=self._with_balance(out.loss, balance))

    @torch.no_grad()
    def token_logp(self, input_ids, labels, temperature=1.0, pos=None):
        """Log-probability of each label (0 where it is below 0): a rollout's ``old_logp``,
        or, from a reference model, the losses' ``ref_logp``."""
        return lm_head_token_logp(self.hidden_states(input_ids, pos), self.lm_head, labels.view(-1), temperature)
