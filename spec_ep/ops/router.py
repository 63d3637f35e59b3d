"""Router: softmax over experts, top-k, optional renormalisation (sm_100a kernel).

Matches transformers' Qwen3-MoE router (softmax in fp32, ``norm_topk_prob``). The
optional ``bias`` shifts only the *selection* scores (not the returned weights); the
synthetic-skew benchmarks use it to make expert popularity follow a Zipf law.

``router_topk_balanced`` is the same routing with the load-balance loss of the batch and
the per-expert token counts, in one pass over the logits each way (csrc/router_balance.cu).
"""
from __future__ import annotations

import torch

from ._ext import load


class _RouterTopK(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, renorm, bias):
        C = load()
        T, E = logits.shape
        topk_e = torch.empty(T, k, device=logits.device, dtype=torch.int32)
        topk_w = torch.empty(T, k, device=logits.device, dtype=torch.float32)
        probs = torch.empty(T, E, device=logits.device, dtype=torch.float32)
        C.router_topk(logits.contiguous(), bias, k, renorm, topk_e, topk_w, probs)
        ctx.save_for_backward(probs, topk_e)
        ctx.renorm = renorm
        ctx.mark_non_differentiable(topk_e)
        return topk_w, topk_e

    @staticmethod
    def backward(ctx, dw, _de):
        probs, topk_e = ctx.saved_tensors
        dlogits = torch.empty_like(probs)
        load().router_bwd(probs, topk_e, dw.contiguous().float(), ctx.renorm, dlogits)
        return dlogits, None, None, None


def router_topk(logits: torch.Tensor, k: int, renorm: bool = True, bias: torch.Tensor | None = None):
    """Returns (topk_w [T, k] fp32, topk_e [T, k] int32) from fp32 router logits."""
    return _RouterTopK.apply(logits.float(), k, renorm, bias)


def router_topk_reference(logits, k, renorm=True, bias=None):
    p = torch.softmax(logits.float(), -1)
    score = p if bias is None else p + bias
    idx = score.topk(k, -1).indices
    w = p.gather(-1, idx)
    if renorm:
        w = w / w.sum(-1, keepdim=True)
    return w, idx.int()


def router_topk_balanced(logits: torch.Tensor, k: int, renorm: bool = True, bias: torch.Tensor | None = None,
                         valid: torch.Tensor | None = None):
    """Top-k routing with a load-balance loss: ``(topk_w, topk_e, loss, counts)``.

    ``topk_w [T, k]`` fp32 and ``topk_e [T, k]`` int32 as in ``router_topk`` (``bias [E]``
    fp32 shifts the selection scores only). ``counts [E]`` int32 is the number of tokens
    that chose each expert, and ``loss = E * sum_e f_e * P_e`` with ``f_e`` the expert's
    share of the ``k`` choices and ``P_e`` its mean router probability: 1 when both are
    uniform. Gradients reach ``logits`` from ``topk_w`` and from ``loss``; the counts are
    constants in them.

    ``logits [T, E]`` bf16, fp16 or fp32 (any row stride), at most 512 experts and
    ``k <= 32``. ``valid [T]`` bool leaves tokens (padding) out of ``loss`` and ``counts``;
    they are routed all the same. With no token left the loss is 0. Among equal scores the
    lowest expert index is chosen; a NaN score is chosen before any number.
    """
    return tuple(load().router_balanced(logits, int(k), bool(renorm), bias, valid))


def router_topk_balanced_reference(logits, k, renorm=True, bias=None, valid=None):
    """The same in torch operations, in the logits' precision (fp32 at least)."""
    x = logits if logits.dtype == torch.float64 else logits.float()
    T, E = x.shape
    p = torch.softmax(x, -1)
    score = x.detach() if bias is None else p.detach() + bias
    e = score.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    w = p.gather(-1, e)
    if renorm:
        w = w / w.sum(-1, keepdim=True)
    on = torch.ones(T, dtype=torch.bool, device=x.device) if valid is None else valid
    n = max(int(on.sum()), 1)
    counts = torch.bincount(e[on].reshape(-1), minlength=E)
    loss = E * (counts.to(p.dtype) / (k * n) * p[on].sum(0) / n).sum()
    return w, e.int(), loss, counts.int()
