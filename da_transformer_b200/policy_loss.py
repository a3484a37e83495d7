"""Losses that train a DAG model on rewards and on preferences.

* ``dag_policy_loss``: the clipped policy loss with a KL term over the vertices' tokens (and transitions),
  from the logits that ``dag_logsoftmax_gather_inplace`` and ``dag_match`` read;
* ``dag_preference_loss``: the loss of paired log ratios of sentence log-likelihoods, which ``dag_loss``
  returns, beside ``dag_loss_mean``.

Neither has a counterpart in the reference.  Both call the C ABI of ``libdat_b200.so``; there is no CPU or
PyTorch fallback.
"""
import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _native
from ._native import check, lib, ptr, require_cuda, require_same_device, stream_ptr
from .dag_loss import _status_word
from .graph_ops import _mask_bytes

__all__ = ["DagPolicyLossFunc", "dag_policy_loss", "DagPreferenceLossFunc", "dag_preference_loss"]

_PREFERENCE_KINDS = {"sigmoid": 0, "hinge": 1, "squared": 2}


class DagPolicyLossFunc(Function):
    @staticmethod
    def forward(ctx, word_ins_out, link_logp, tokens, old_logp, advantage, mask, ref_logits, ref_logp, kl_coef,
                clip_low, clip_high, grad_scale):
        if word_ins_out.dim() != 3:
            raise RuntimeError("word_ins_out dim != 3")
        bsz, prelen, vocab = word_ins_out.shape
        if vocab < 1:
            raise RuntimeError("word_ins_out has an empty vocabulary")
        dt = _native.dtype_code(word_ins_out.dtype)
        if not word_ins_out.is_contiguous():
            raise RuntimeError("word_ins_out is not contiguous")
        if tokens.shape != (bsz, prelen) or tokens.dtype != torch.long:
            raise RuntimeError("tokens should be a long tensor of shape [batch, prelen]")
        for name, t in (("old_logp", old_logp), ("link_logp", link_logp), ("ref_logp", ref_logp)):
            if t is not None and (t.shape != (bsz, prelen) or t.dtype != torch.float32):
                raise RuntimeError(f"{name} should be a float32 tensor of shape [batch, prelen]")
        if advantage.dtype != torch.float32 or advantage.shape not in ((bsz,), (bsz, prelen)):
            raise RuntimeError("advantage should be a float32 tensor of shape [batch] or [batch, prelen]")
        if mask is not None and mask.shape != (bsz, prelen):
            raise RuntimeError("mask should be [batch, prelen]")
        if ref_logits is not None:
            if ref_logp is not None:
                raise RuntimeError("give ref_logits (KL over the vocabulary) or ref_logp (KL estimate), not both")
            if ref_logits.shape != word_ins_out.shape or ref_logits.dtype != word_ins_out.dtype:
                raise RuntimeError("ref_logits should have the shape and dtype of word_ins_out")
            if not ref_logits.is_contiguous():
                raise RuntimeError("ref_logits is not contiguous")
        clip_low, clip_high = float(clip_low), float(clip_high)
        if not (clip_low >= 0 and clip_high >= 0):
            raise RuntimeError("clip_low and clip_high should not be negative")
        scale_tensor = None
        if isinstance(grad_scale, torch.Tensor):
            if grad_scale.numel() != 1 or grad_scale.dtype != torch.float32:
                raise RuntimeError("grad_scale should be a number or a float32 tensor with one element")
            scale_tensor = grad_scale
        require_cuda(word_ins_out, link_logp, tokens, old_logp, advantage, mask, ref_logits, ref_logp, scale_tensor)
        dev = word_ins_out.device
        require_same_device(dev, link_logp=link_logp, tokens=tokens, old_logp=old_logp, advantage=advantage, mask=mask,
                            ref_logits=ref_logits, ref_logp=ref_logp, grad_scale=scale_tensor)
        L = lib()
        need_logits, need_link = ctx.needs_input_grad[0], link_logp is not None and ctx.needs_input_grad[1]
        with torch.cuda.device(dev):
            tokens = tokens.contiguous()
            mask = _mask_bytes(mask)
            old_logp = old_logp.contiguous()
            link = None if link_logp is None else link_logp.contiguous()
            refp = None if ref_logp is None else ref_logp.contiguous()
            loss = torch.empty((), dtype=torch.float32, device=dev)
            stats = torch.empty(5, dtype=torch.float64, device=dev)
            logp = torch.empty(bsz, prelen, dtype=torch.float32, device=dev)
            kl = torch.empty(bsz, prelen, dtype=torch.float32, device=dev)
            state = (torch.empty(bsz * prelen, 4, dtype=torch.float32, device=dev)
                     if need_logits or need_link else None)
            grad = torch.empty_like(word_ins_out) if need_logits and grad_scale is not None else None
            ws = torch.empty(L.dat_policy_loss_workspace_bytes(bsz, prelen), dtype=torch.uint8, device=dev)
            check(L.dat_policy_loss(
                ptr(word_ins_out), ptr(ref_logits), dt, ptr(tokens), ptr(old_logp), ptr(advantage), advantage.stride(0),
                advantage.stride(1) if advantage.dim() == 2 else 0, ptr(link), ptr(refp), ptr(mask), float(kl_coef),
                clip_low, clip_high, ptr(scale_tensor), 1.0 if scale_tensor is not None or grad_scale is None else
                float(grad_scale), ptr(loss), ptr(stats), ptr(logp), ptr(kl), ptr(state), ptr(grad), ptr(ws),
                ptr(_status_word(dev)), bsz, prelen, vocab, stream_ptr(dev)), "policy_loss")
        ctx.mark_non_differentiable(logp, kl, stats)
        ctx.set_materialize_grads(False)
        if state is not None:
            ctx.save_for_backward(word_ins_out, ref_logits, tokens, mask, state, ws)
            ctx.grad, ctx.kl_coef = grad, float(kl_coef)
        return loss, logp, kl, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, grad_logp, grad_kl, grad_stats):
        none = (None,) * 12
        if grad_loss is None:
            return none
        word_ins_out, ref_logits, tokens, mask, state, ws = ctx.saved_tensors
        bsz, prelen, vocab = word_ins_out.shape
        dev = word_ins_out.device
        # the buffer that the forward wrote is given away once; a second backward makes its own
        grad, ctx.grad = ctx.grad, None
        with torch.cuda.device(dev):
            grad_loss = grad_loss.to(torch.float32).contiguous()
            written = grad is not None
            if not written and ctx.needs_input_grad[0]:
                grad = torch.empty_like(word_ins_out)
            link = torch.empty(bsz, prelen, dtype=torch.float32, device=dev) if ctx.needs_input_grad[1] else None
            check(lib().dat_policy_loss_backward(
                ptr(word_ins_out), ptr(ref_logits), _native.dtype_code(word_ins_out.dtype), ptr(tokens), ptr(mask),
                ctx.kl_coef, ptr(state), ptr(ws), ptr(grad_loss), int(written), ptr(grad), ptr(link), bsz, prelen,
                vocab, stream_ptr(dev)), "policy_loss_backward")
        return (grad, link) + none[2:]


def dag_policy_loss(word_ins_out, tokens, old_logp, advantage, mask=None, link_logp=None, ref_logits=None,
                    ref_logp=None, kl_coef=0.0, clip_low=0.2, clip_high=0.2, grad_scale=1.0):
    r"""Clipped policy loss with a KL term over the vertices of sampled paths::

        logp  = log_softmax(word_ins_out, -1).gather(-1, tokens) + link_logp
        ratio = exp(logp - old_logp)
        term  = -min(ratio * advantage, clamp(ratio, 1 - clip_low, 1 + clip_high) * advantage)
        kl    = (p * (log p - log q)).sum(-1)      with ref_logits (q = softmax(ref_logits)), or
                exp(u) - u - 1, u = ref_logp - logp     with ref_logp, or 0 with neither
        loss  = (term + kl_coef * kl)[mask].mean()                     # 0 where no vertex takes part

    word_ins_out [B,L,V] fp32/fp16/bf16 contiguous; tokens [B,L] int64, the token taken at each vertex;
    old_logp [B,L] fp32, its log-probability when it was sampled; advantage [B] or [B,L] fp32; mask [B,L]
    bool (True: the vertex is on the path; None: all are), nothing of the other vertices is looked at;
    link_logp [B,L] fp32, the log-probability of the transition that leaves the vertex (None: 0);
    ref_logits like word_ins_out; ref_logp [B,L] fp32, of the same step (transition included).
    Returns ``(loss, logp, kl, stats)``: the scalar, differentiable in ``word_ins_out`` and ``link_logp``, the
    vertices' log-probabilities and KL [B,L] fp32 (0 where masked), and the fp64 vector ``[sum term, sum kl,
    sum ratio, n clipped, n vertices]`` that ``dist.all_reduce_stats`` can sum over ranks.

    The gradient of the logits is written by the forward, while a row is in the cache, for a loss whose own
    gradient is ``grad_scale`` (a number, or a one-element fp32 tensor such as a loss scale); the backward
    computes it again where another gradient arrives.  ``grad_scale=None`` leaves it to the backward (the
    logits are then read twice, and nothing of their size is held in between).  ``word_ins_out`` is not
    changed.  A token outside the vocabulary makes its row NaN and sets bit 4 of ``last_status()``."""
    return DagPolicyLossFunc.apply(word_ins_out, link_logp, tokens, old_logp, advantage, mask, ref_logits, ref_logp,
                                   kl_coef, clip_low, clip_high, grad_scale)


class DagPreferenceLossFunc(Function):
    @staticmethod
    def forward(ctx, chosen, rejected, reference_chosen, reference_rejected, chosen_length, rejected_length, beta,
                kind, label_smoothing):
        if chosen.dim() != 1 or rejected.shape != chosen.shape:
            raise RuntimeError("chosen and rejected must be [pairs]")
        pairs = chosen.numel()
        for name, t in (("chosen", chosen), ("rejected", rejected), ("reference_chosen", reference_chosen),
                        ("reference_rejected", reference_rejected)):
            if t is not None and (t.shape != chosen.shape or t.dtype != torch.float32):
                raise RuntimeError(f"{name} should be a float32 tensor of shape [pairs]")
        for name, t in (("chosen_length", chosen_length), ("rejected_length", rejected_length)):
            if t is not None and (t.shape != chosen.shape or t.dtype != torch.long):
                raise RuntimeError(f"{name} should be a long tensor of shape [pairs]")
        if (reference_chosen is None) != (reference_rejected is None):
            raise RuntimeError("reference_chosen and reference_rejected are given together")
        if (chosen_length is None) != (rejected_length is None):
            raise RuntimeError("chosen_length and rejected_length are given together")
        if kind not in _PREFERENCE_KINDS:
            raise RuntimeError(f"unknown kind {kind!r} (one of {', '.join(_PREFERENCE_KINDS)})")
        if not 0.0 <= label_smoothing <= 1.0:
            raise RuntimeError("label_smoothing should be in [0, 1]")
        others = dict(rejected=rejected, reference_chosen=reference_chosen, reference_rejected=reference_rejected,
                      chosen_length=chosen_length, rejected_length=rejected_length)
        require_cuda(chosen, *others.values())
        dev = chosen.device
        require_same_device(dev, **others)
        with torch.cuda.device(dev):
            flat = [None if t is None else t.contiguous() for t in (chosen, *others.values())]
            loss = torch.empty((), dtype=torch.float32, device=dev)
            rewards = torch.empty(2, pairs, dtype=torch.float32, device=dev)
            stats = torch.empty(6, dtype=torch.float64, device=dev)
            need_grad = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
            slope = torch.empty(2, pairs, dtype=torch.float32, device=dev) if need_grad else None
            check(lib().dat_preference_loss(*(ptr(t) for t in flat), float(beta), float(label_smoothing),
                                            _PREFERENCE_KINDS[kind], ptr(loss), ptr(rewards), ptr(stats), ptr(slope),
                                            ptr(_status_word(dev)), pairs, stream_ptr(dev)), "preference_loss")
        ctx.mark_non_differentiable(rewards, stats)
        ctx.set_materialize_grads(False)
        if need_grad:
            ctx.save_for_backward(slope)
        return loss, rewards, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, grad_rewards, grad_stats):
        none = (None,) * 9
        if grad_loss is None:
            return none
        (slope,) = ctx.saved_tensors
        grads = slope * grad_loss
        return (grads[0], grads[1]) + none[2:]


def dag_preference_loss(chosen, rejected, reference_chosen=None, reference_rejected=None, beta=0.1, kind="sigmoid",
                        label_smoothing=0.0, chosen_length=None, rejected_length=None):
    r"""Preference loss of pairs of sentences from their log-likelihoods::

        reward = beta * (log_likelihood - reference) / length          # reference 0, length 1 where not given
        h = reward_chosen - reward_rejected;  e = label_smoothing
        sigmoid:  -(1-e) * logsigmoid(h) - e * logsigmoid(-h)
        hinge:     (1-e) * relu(1 - h) + e * relu(1 + h)
        squared:   (1-e) * (h - 1/2)**2 + e * (h + 1/2)**2

    and the mean over all pairs, in one launch.  chosen, rejected [B] fp32 are what ``dag_loss`` returns for the
    preferred and the rejected sentences; reference_* [B] fp32 the same under a reference model (no gradient);
    *_length [B] int64.  Like ``dag_loss_mean`` a sentence whose log-likelihood is inf or nan counts as
    invalid: its pair adds 0 to the mean and gets no gradient (so does a pair with a length below 1, which also
    sets bit 1 of ``last_status()``).  Returns ``(loss, rewards, stats)``: the scalar, differentiable in
    ``chosen`` and ``rejected``; the rewards [2,B] fp32; the fp64 vector ``[sum of the losses, sum of the chosen
    rewards, of the rejected ones, n with h > 0, n pairs, n invalid]``."""
    return DagPreferenceLossFunc.apply(chosen, rejected, reference_chosen, reference_rejected, chosen_length,
                                       rejected_length, beta, kind, label_smoothing)
