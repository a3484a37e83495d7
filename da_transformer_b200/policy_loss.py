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
from ._native import address, check, lib, require_device, stream_address
from .dag_loss import _status_word
from .graph_ops import _mask_bytes

__all__ = ["DagPolicyLossFunc", "dag_policy_loss", "DagPreferenceLossFunc", "dag_preference_loss"]

_PREFERENCE_KINDS = {"sigmoid": 0, "hinge": 1, "squared": 2}


def _check_policy(word_ins_out, link_logp, tokens, old_logp, advantage, mask, ref_logits, ref_logp, grad_scale):
    if word_ins_out.dim() != 3:
        raise RuntimeError("word_ins_out dim != 3")
    bsz, prelen, vocab = word_ins_out.shape
    if vocab < 1:
        raise RuntimeError("word_ins_out has an empty vocabulary")
    if vocab >= 2 ** 30 or bsz * prelen >= 2 ** 31:
        raise RuntimeError("dag_policy_loss takes vocabularies below 2^30 and less than 2^31 vertices")
    if not word_ins_out.is_contiguous():
        raise RuntimeError("word_ins_out is not contiguous")
    shape = (bsz, prelen)
    if tokens.shape != shape or tokens.dtype is not torch.long:
        raise RuntimeError("tokens should be a long tensor of shape [batch, prelen]")
    for name, t in (("old_logp", old_logp), ("link_logp", link_logp), ("ref_logp", ref_logp)):
        if t is not None and (t.shape != shape or t.dtype is not torch.float32):
            raise RuntimeError(f"{name} should be a float32 tensor of shape [batch, prelen]")
    if advantage.dtype is not torch.float32 or (advantage.shape != shape and advantage.shape != (bsz,)):
        raise RuntimeError("advantage should be a float32 tensor of shape [batch] or [batch, prelen]")
    if mask is not None and mask.shape != shape:
        raise RuntimeError("mask should be [batch, prelen]")
    if ref_logits is not None:
        if ref_logp is not None:
            raise RuntimeError("give ref_logits (KL over the vocabulary) or ref_logp (KL estimate), not both")
        if ref_logits.shape != word_ins_out.shape or ref_logits.dtype is not word_ins_out.dtype:
            raise RuntimeError("ref_logits should have the shape and dtype of word_ins_out")
        if not ref_logits.is_contiguous():
            raise RuntimeError("ref_logits is not contiguous")
    if grad_scale is not None and (grad_scale.numel() != 1 or grad_scale.dtype is not torch.float32):
        raise RuntimeError("grad_scale should be a number or a float32 tensor with one element")
    require_device(word_ins_out.device, link_logp=link_logp, tokens=tokens, old_logp=old_logp, advantage=advantage,
                   mask=mask, ref_logits=ref_logits, ref_logp=ref_logp, grad_scale=grad_scale)


class DagPolicyLossFunc(Function):
    """``dag_policy_loss``.  ``rest``: its other arguments, in their order."""

    @staticmethod
    def forward(ctx, word_ins_out, link_logp, rest):
        (tokens, old_logp, advantage, mask, ref_logits, ref_logp, kl_coef, clip_low, clip_high, grad_scale) = rest
        dt = _native.dtype_code(word_ins_out.dtype)
        clip_low, clip_high, kl_coef = float(clip_low), float(clip_high), float(kl_coef)
        if not (clip_low >= 0 and clip_high >= 0):
            raise RuntimeError("clip_low and clip_high should not be negative")
        scale_tensor = grad_scale if isinstance(grad_scale, torch.Tensor) else None
        _check_policy(word_ins_out, link_logp, tokens, old_logp, advantage, mask, ref_logits, ref_logp, scale_tensor)
        scale = 1.0 if scale_tensor is not None or grad_scale is None else float(grad_scale)
        bsz, prelen, vocab = word_ins_out.shape
        dev = word_ins_out.device
        L = lib()
        need_logits, need_link = ctx.needs_input_grad[0], link_logp is not None and ctx.needs_input_grad[1]
        with torch.cuda.device(dev):
            stream = stream_address(dev)
            tokens = tokens.contiguous()
            mask = _mask_bytes(mask)
            old_logp = old_logp.contiguous()
            link = None if link_logp is None else link_logp.contiguous()
            refp = None if ref_logp is None else ref_logp.contiguous()
            loss = torch.empty((), dtype=torch.float32, device=dev)
            stats = torch.empty(5, dtype=torch.float64, device=dev)
            logp, kl = torch.empty_like(old_logp), torch.empty_like(old_logp)
            need_grad = need_logits or need_link
            grad = torch.empty_like(word_ins_out) if need_logits and grad_scale is not None else None
            # the state of the rows (32 bytes each) for the backward, then the workspace
            at = bsz * prelen * 32 if need_grad else 0
            ws = torch.empty(at + L.dat_policy_loss_workspace_bytes(bsz, prelen), dtype=torch.uint8, device=dev)
            check(L.dat_policy_loss(
                word_ins_out.data_ptr(), address(ref_logits), dt, tokens.data_ptr(), old_logp.data_ptr(),
                advantage.data_ptr(), advantage.stride(0), advantage.stride(1) if advantage.dim() == 2 else 0,
                address(link), address(refp), address(mask), kl_coef, clip_low, clip_high, address(scale_tensor), scale,
                loss.data_ptr(), stats.data_ptr(), logp.data_ptr(), kl.data_ptr(), ws.data_ptr() if at else 0, address(grad),
                ws.data_ptr() + at, _status_word(dev).data_ptr(), bsz, prelen, vocab, stream), "policy_loss")
        ctx.mark_non_differentiable(logp, kl, stats)
        ctx.set_materialize_grads(False)
        if need_grad:
            ctx.save_for_backward(word_ins_out, ref_logits, tokens, mask)
            ctx.ws = ws               # the library's own, nobody else holds it
            ctx.grad, ctx.kl_coef = grad, kl_coef
            # a graph that holds the backward alone would find the buffer as it was left after the last replay
            ctx.capture = 0 if grad is None else L.dat_stream_capture_id(stream)
        return loss, logp, kl, stats

    @staticmethod
    def backward(ctx, grad_loss, *unused):
        # as for the links: the marking wrapper only for whoever differentiates again
        return _policy_backward_once(ctx, grad_loss) if torch.is_grad_enabled() else _policy_backward(ctx, grad_loss)


def _policy_backward(ctx, grad_loss):
    if grad_loss is None:
        return None, None, None
    word_ins_out, ref_logits, tokens, mask = ctx.saved_tensors
    ws = ctx.ws.data_ptr()
    bsz, prelen, vocab = word_ins_out.shape
    dev = word_ins_out.device
    # the buffer that the forward wrote is given away once; a second backward makes its own
    grad, ctx.grad = ctx.grad, None
    with torch.cuda.device(dev):
        grad_loss = grad_loss.to(torch.float32).contiguous()
        stream = stream_address(dev)
        written = grad is not None and lib().dat_stream_capture_id(stream) == ctx.capture
        if not written:
            grad = None
        if not written and ctx.needs_input_grad[0]:
            grad = torch.empty_like(word_ins_out)
        link = torch.empty(bsz, prelen, dtype=torch.float32, device=dev) if ctx.needs_input_grad[1] else None
        check(lib().dat_policy_loss_backward(
            word_ins_out.data_ptr(), address(ref_logits), _native.dtype_code(word_ins_out.dtype), tokens.data_ptr(),
            address(mask), ctx.kl_coef, ws, ws + bsz * prelen * 32, grad_loss.data_ptr(), int(written),
            address(grad), address(link), bsz, prelen, vocab, stream), "policy_loss_backward")
    return grad, link, None


_policy_backward_once = once_differentiable(_policy_backward)


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
    return DagPolicyLossFunc.apply(word_ins_out, link_logp, (tokens, old_logp, advantage, mask, ref_logits, ref_logp,
                                                             kl_coef, clip_low, clip_high, grad_scale))


def _check_preference(chosen, rejected, reference_chosen, reference_rejected, chosen_length, rejected_length, kind,
                      label_smoothing):
    shape = chosen.shape
    if len(shape) != 1 or rejected.shape != shape:
        raise RuntimeError("chosen and rejected must be [pairs]")
    for name, t in (("chosen", chosen), ("rejected", rejected), ("reference_chosen", reference_chosen),
                    ("reference_rejected", reference_rejected)):
        if t is not None and (t.dtype is not torch.float32 or t.shape != shape):
            raise RuntimeError(f"{name} should be a float32 tensor of shape [pairs]")
    for name, t in (("chosen_length", chosen_length), ("rejected_length", rejected_length)):
        if t is not None and (t.dtype is not torch.long or t.shape != shape):
            raise RuntimeError(f"{name} should be a long tensor of shape [pairs]")
    if (reference_chosen is None) != (reference_rejected is None):
        raise RuntimeError("reference_chosen and reference_rejected are given together")
    if (chosen_length is None) != (rejected_length is None):
        raise RuntimeError("chosen_length and rejected_length are given together")
    if kind not in _PREFERENCE_KINDS:
        raise RuntimeError(f"unknown kind {kind!r} (one of {', '.join(_PREFERENCE_KINDS)})")
    if not 0.0 <= label_smoothing <= 1.0:
        raise RuntimeError("label_smoothing should be in [0, 1]")
    require_device(chosen.device, rejected=rejected, reference_chosen=reference_chosen,
                   reference_rejected=reference_rejected, chosen_length=chosen_length, rejected_length=rejected_length)


class DagPreferenceLossFunc(Function):
    """``dag_preference_loss``.  ``rest``: its other arguments, in their order."""

    @staticmethod
    def forward(ctx, chosen, rejected, rest):
        (reference_chosen, reference_rejected, chosen_length, rejected_length, beta, kind, label_smoothing) = rest
        _check_preference(chosen, rejected, reference_chosen, reference_rejected, chosen_length, rejected_length, kind,
                          label_smoothing)
        pairs, dev = chosen.size(0), chosen.device
        need_grad = True in ctx.needs_input_grad
        with torch.cuda.device(dev):
            flat = [None if t is None else t.contiguous() for t in (chosen, rejected, reference_chosen, reference_rejected,
                                                                    chosen_length, rejected_length)]
            loss = torch.empty((), dtype=torch.float32, device=dev)
            rewards = torch.empty(2, pairs, dtype=torch.float32, device=dev)
            stats = torch.empty(6, dtype=torch.float64, device=dev)
            slope = torch.empty_like(rewards) if need_grad else None
            check(lib().dat_preference_loss(*map(address, flat), float(beta), float(label_smoothing),
                                            _PREFERENCE_KINDS[kind], loss.data_ptr(), rewards.data_ptr(),
                                            stats.data_ptr(), address(slope), _status_word(dev).data_ptr(), pairs,
                                            stream_address(dev)), "preference_loss")
        ctx.mark_non_differentiable(rewards, stats)
        ctx.set_materialize_grads(False)
        ctx.slope = slope     # d loss / d (chosen, rejected): the library's own, nobody else holds it
        return loss, rewards, stats

    @staticmethod
    def backward(ctx, grad_loss, *unused):
        return _preference_backward_once(ctx, grad_loss) if torch.is_grad_enabled() else _preference_backward(ctx, grad_loss)


def _preference_backward(ctx, grad_loss):
    if grad_loss is None:
        return None, None, None
    chosen, rejected = (ctx.slope * grad_loss).unbind()
    return chosen, rejected, None


_preference_backward_once = once_differentiable(_preference_backward)


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
    return DagPreferenceLossFunc.apply(chosen, rejected, (reference_chosen, reference_rejected, chosen_length,
                                                          rejected_length, beta, kind, label_smoothing))
