"""Language-model head + cross-entropy with a fused loss/gradient kernel.

The logits GEMM and both gradient GEMMs run on the tcgen05 GEMM (``spec_ep.ops.linear``;
the vocabulary's last 256-column tile is partial); the softmax cross-entropy and its
gradient run in one sm_100a kernel that overwrites the bf16 logits with
``(softmax - onehot) * scale`` so no fp32 copy of the [T, V] logits is ever stored.

Three objectives for training after the pre-training, on the kernels of
csrc/vocab_loss.cu, each over given logits and as an ``lm_head_*`` form that owns the
logits and overwrites them with their gradient:

* ``topk_distill_loss``: distillation from a teacher's top logits,
* ``clipped_policy_loss``: clipped policy ratio with a KL term to a reference model,
* ``preference_loss``: paired log-ratios of packed chosen / rejected sequences
  (``token_logp`` gives the reference model's side, and a rollout's).
"""
from __future__ import annotations

from typing import NamedTuple

import torch
import torch.autograd.forward_ad as fwd
from torch.autograd.function import once_differentiable

from ._ext import load
from .linear import dense_dgrad, dense_fwd, dense_wgrad


class _LMHeadXent(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, w, labels, num_valid):
        C = load()
        logits = dense_fwd(h, w)  # [T, V] bf16
        loss = torch.empty(h.shape[0], device=h.device, dtype=torch.float32)
        if num_valid is not None:
            scale = 1.0 / max(int(num_valid), 1)
            C.xent_fwd_bwd(logits, labels, scale, loss)
            ctx.dev_scale = None
            out = loss.sum() * scale
        else:
            C.xent_fwd_bwd(logits, labels, 1.0, loss)
            valid = (labels >= 0).sum().clamp_min(1).float()
            ctx.dev_scale = 1.0 / valid
            out = loss.sum() / valid
        ctx.save_for_backward(h, w, logits)
        return out

    @staticmethod
    def backward(ctx, g):
        h, w, dlogits = ctx.saved_tensors
        dh = dense_dgrad(dlogits, w)
        dw = dense_wgrad(dlogits, h)
        s = g if ctx.dev_scale is None else g * ctx.dev_scale
        return dh * s.to(dh.dtype), dw * s.to(dw.dtype), None, None


def lm_head_xent(h: torch.Tensor, w: torch.Tensor, labels: torch.Tensor, num_valid: int | None = None):
    """Mean next-token cross-entropy of ``h @ w.T`` against ``labels`` (int32, -1 = ignore).

    ``num_valid`` (labels >= 0, known on the host) lets the kernel apply the mean's
    scale directly; otherwise it is applied from a device-side count.
    """
    return _LMHeadXent.apply(h, w, labels.int().contiguous(), num_valid)


def lm_head_xent_reference(h, w, labels):
    logits = h.float() @ w.float().t()
    return torch.nn.functional.cross_entropy(logits, labels.long(), ignore_index=-1)


# ----------------------------------------------------------------------------------------
# losses after pre-training
# ----------------------------------------------------------------------------------------
def _valid(num_valid):
    """Rows in the loss for the kernels: -1 counts them on the device."""
    if num_valid is None:
        return -1
    if num_valid < 0:
        raise ValueError(f"num_valid must be >= 0, not {num_valid}")
    return int(num_valid)


def _f32(t):
    """An input that gets no gradient, in fp32."""
    return t.detach().float().contiguous()


def topk_distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                      temperature: float = 1.0, num_valid: int | None = None) -> torch.Tensor:
    """Distillation from a teacher's top logits: mean over rows of
    ``temperature^2 * KL(p || q)``, ``p`` the softmax of the row's listed teacher logits and
    ``q`` the softmax of all its ``logits``, both over ``temperature``.

    ``logits [T, V]`` bf16, fp16 or fp32 (any row stride); ``teacher_ids [T, K]`` int32 or
    int64 and ``teacher_logits [T, K]``, ``K <= 1024``. An id below 0, or a teacher logit of
    -inf, is no entry (what stands beside such an id is not looked at); a row without
    entries is not in the loss, its logits are not read and its gradient is 0. The same id
    twice counts with both weights. An id outside the vocabulary makes the loss NaN.
    ``num_valid`` (rows with an entry, if the host knows it) spares a count on the device.
    Gradients reach ``logits`` only, once through reverse mode; forward-mode tangents are refused.
    """
    return load().topk_distill(logits, teacher_ids.contiguous(), _f32(teacher_logits), float(temperature),
                               _valid(num_valid))


class PolicyLoss(NamedTuple):
    loss: torch.Tensor  # scalar
    logp: torch.Tensor  # [T] log-probability of each action (0 where there is none)
    kl: torch.Tensor    # [T] estimate of the KL to the reference model (0 without one)


def clipped_policy_loss(logits: torch.Tensor, actions: torch.Tensor, old_logp: torch.Tensor,
                        advantages: torch.Tensor, ref_logp: torch.Tensor | None = None, clip_low: float = 0.2,
                        clip_high: float = 0.2, kl_coef: float = 0.0, temperature: float = 1.0,
                        num_valid: int | None = None) -> PolicyLoss:
    """Clipped policy loss over tokens, with a KL term to a reference model.

    With ``logp`` the log-probability of the row's action under
    ``softmax(logits / temperature)`` and ``r = exp(logp - old_logp)``::

        loss = mean( -min(r * A, clip(r, 1 - clip_low, 1 + clip_high) * A)
                     + kl_coef * (exp(d) - d - 1) ),   d = ref_logp - logp

    The mean is over rows with an action; an action below 0 leaves its row (a prompt token)
    out: the row is not read and its gradient is 0. ``logits [T, V]`` bf16, fp16 or fp32
    (any row stride), ``actions [T]`` int32 or int64, the others ``[T]``. An action outside
    the vocabulary makes the loss NaN. ``num_valid`` (rows with an action, if the host
    knows it) spares a count on the device. Gradients reach ``logits`` only.
    """
    return PolicyLoss(*load().clipped_policy(logits, actions.contiguous(), _f32(old_logp), _f32(advantages),
                                             None if ref_logp is None else _f32(ref_logp), float(clip_low),
                                             float(clip_high), float(kl_coef), float(temperature),
                                             _valid(num_valid)))


def token_logp(logits: torch.Tensor, labels: torch.Tensor, temperature: float = 1.0) -> torch.Tensor:
    """Log-probability ``[T]`` (fp32) of each row's label under ``softmax(logits /
    temperature)``, 0 where the label is below 0. No gradient: the ``old_logp`` and
    ``ref_logp`` of the losses here."""
    return load().token_logp(logits.detach(), labels.contiguous(), float(temperature))


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor     # scalar
    rewards: torch.Tensor  # [2 * pairs] beta * (sum of logp - ref_logp) of each sequence
    logp: torch.Tensor     # [T] log-probability of each label (0 where there is none)


def preference_loss(logits: torch.Tensor, labels: torch.Tensor, seq_offsets: torch.Tensor, ref_logp: torch.Tensor,
                    beta: float = 0.1, label_smoothing: float = 0.0) -> PreferenceLoss:
    """Paired preference loss over packed sequences: sequence ``s`` is the rows
    ``seq_offsets[s] .. seq_offsets[s + 1]``, sequence ``2 i`` the chosen and ``2 i + 1`` the
    rejected one of pair ``i``. With ``R_s = beta * sum(logp - ref_logp)`` over its labels::

        m_i  = R_2i - R_2i+1
        loss = mean_i( -(1 - eps) * log sigmoid(m_i) - eps * log sigmoid(-m_i) )

    ``logits [T, V]`` bf16, fp16 or fp32 (any row stride), ``labels [T]`` int32 or int64
    (below 0: not in the loss, as a prompt's tokens), ``ref_logp [T]`` the reference model's
    log-probabilities of the same labels (``token_logp``), ``seq_offsets [2 * pairs + 1]``
    int32, not decreasing. Rows outside all sequences, and rows without a label, are not
    read and their gradient is 0. A label outside the vocabulary makes the loss NaN.
    Gradients reach ``logits`` only.
    """
    return PreferenceLoss(*load().preference(logits, labels.contiguous(), seq_offsets.contiguous(), _f32(ref_logp),
                                             float(beta), float(label_smoothing)))


# ----------------------------------------------------------------------------------------
# the same behind the LM head: ``h [T, H] @ w[V, H].T`` gives the logits, which are kept in
# bf16 and overwritten with their gradient
# ----------------------------------------------------------------------------------------
class _LMHead(torch.autograd.Function):
    """``kernel(logits, grad)`` returns ``(loss, row_scale, *aux)``: with ``row_scale [T]`` the
    gradient that it leaves is still to be multiplied by a factor per row."""

    @staticmethod
    def forward(ctx, h, w, kernel):
        logits = dense_fwd(h, w)
        loss, row_scale, *aux = kernel(logits, logits)
        ctx.save_for_backward(h, w, logits, row_scale)
        ctx.mark_non_differentiable(*aux)
        ctx.set_materialize_grads(False)
        return (loss, *aux)

    @staticmethod
    @once_differentiable
    def backward(ctx, up, *_):
        if up is None:
            return None, None, None
        h, w, dlogits, row_scale = ctx.saved_tensors
        dh = dense_dgrad(dlogits, w) if ctx.needs_input_grad[0] else None
        if row_scale is None:
            dw = dense_wgrad(dlogits, h) if ctx.needs_input_grad[1] else None
            for g in (dh, dw):
                if g is not None:
                    load().scale_grad(g, up)  # in place, by the fp32 factor; untouched where it is 1
            return dh, dw, None
        # the rows' factors go to the small side of each product: onto dh, and onto h, where
        # they cost one more rounding to bf16 (2^-9 of each term of a sum over tokens)
        s = (row_scale * up)[:, None]
        dw = dense_wgrad(dlogits, (h * s).to(h.dtype)) if ctx.needs_input_grad[1] else None
        return None if dh is None else (dh * s).to(h.dtype), dw, None


def _has_tangent(*ts):
    return fwd._current_level >= 0 and any(fwd.unpack_dual(t).tangent is not None for t in ts)


def _lm_head(h, w, kernel):
    # a forward-mode tangent too goes through autograd, which refuses it
    if (torch.is_grad_enabled() and (h.requires_grad or w.requires_grad)) or _has_tangent(h, w):
        return _LMHead.apply(h, w, kernel)
    loss, _, *aux = kernel(dense_fwd(h, w), None)
    return (loss, *aux)


def lm_head_distill(h: torch.Tensor, w: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                    temperature: float = 1.0, num_valid: int | None = None) -> torch.Tensor:
    """``topk_distill_loss`` of the logits ``h @ w.T``, with gradients for ``h`` and ``w``."""
    ids, t, n = teacher_ids.contiguous(), _f32(teacher_logits), _valid(num_valid)

    def kernel(logits, grad):
        return load().distill_loss(logits, ids, t, float(temperature), n, grad, None), None

    return _lm_head(h, w, kernel)[0]


def lm_head_policy(h: torch.Tensor, w: torch.Tensor, actions: torch.Tensor, old_logp: torch.Tensor,
                   advantages: torch.Tensor, ref_logp: torch.Tensor | None = None, clip_low: float = 0.2,
                   clip_high: float = 0.2, kl_coef: float = 0.0, temperature: float = 1.0,
                   num_valid: int | None = None) -> PolicyLoss:
    """``clipped_policy_loss`` of the logits ``h @ w.T``, with gradients for ``h`` and ``w``."""
    a, old, adv, n = actions.contiguous(), _f32(old_logp), _f32(advantages), _valid(num_valid)
    ref = None if ref_logp is None else _f32(ref_logp)

    def kernel(logits, grad):
        loss, logp, kl = load().policy_loss(logits, a, old, adv, ref, float(clip_low), float(clip_high),
                                            float(kl_coef), float(temperature), n, grad, None)
        return loss, None, logp, kl

    return PolicyLoss(*_lm_head(h, w, kernel))


def lm_head_preference(h: torch.Tensor, w: torch.Tensor, labels: torch.Tensor, seq_offsets: torch.Tensor,
                       ref_logp: torch.Tensor, beta: float = 0.1, label_smoothing: float = 0.0) -> PreferenceLoss:
    """``preference_loss`` of the logits ``h @ w.T``, with gradients for ``h`` and ``w``. The
    logits are read once: their gradient per unit of each row's factor is written in the
    forward, and the factors, known after the whole pair, join in the backward."""
    y, off, ref = labels.contiguous(), seq_offsets.contiguous(), _f32(ref_logp)

    def kernel(logits, grad):
        loss, rewards, logp, rows = load().preference_fwd(logits, y, off, ref, float(beta), float(label_smoothing),
                                                          grad)
        return loss, rows[2], rewards, logp

    return PreferenceLoss(*_lm_head(h, w, kernel))


def lm_head_token_logp(h: torch.Tensor, w: torch.Tensor, labels: torch.Tensor, temperature: float = 1.0):
    """``token_logp`` of the logits ``h @ w.T``."""
    return token_logp(dense_fwd(h.detach(), w.detach()), labels, temperature)
