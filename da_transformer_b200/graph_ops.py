"""Producers and consumers of the transition matrix on either side of the three custom ops:

* ``dag_links_from_heads``: the tail of ``GlatDecomposedLink.extract_links``
  (fs_plugins/models/glat_decomposed_with_link.py:380-404), which turns per-head transition scores
  into the band ``links`` that ``dag_loss`` reads, forward and backward;
* ``dag_node_passing_prob`` and ``dag_viterbi_decode``: the decode-side dynamic programmes on the
  square transition matrix (``_analyze_graph`` :559-569, ``inference_viterbi`` :720-777).

All call the C ABI of ``libdat_b200.so``; there is no CPU or PyTorch fallback.
"""
import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ._native import address, check, lib, ptr, require_cuda, require_device, stream_address, stream_ptr
from .dag_loss import _status_word

__all__ = ["DagLinksFromHeadsFunc", "DagBiasedLinksFunc", "dag_links_from_heads", "dag_relative_buckets",
           "dag_node_passing_prob", "dag_viterbi_decode"]


def _mask_u8(mask):
    if mask is None:
        return None
    return (mask if mask.dtype == torch.uint8 else mask.to(torch.uint8)).contiguous()


def _mask_bytes(mask):
    """The mask as uint8, without a copy where it is a bool tensor."""
    if mask is None:
        return None
    if mask.dtype == torch.bool:
        return mask.contiguous().view(torch.uint8)
    return _mask_u8(mask)


class DagLinksFromHeadsFunc(Function):
    @staticmethod
    def forward(ctx, log_multi_content, log_gates, nonpad_mask, bound_end, max_transition_length):
        require_cuda(log_multi_content, log_gates, nonpad_mask, bound_end)
        if log_multi_content.dim() != 4 or log_multi_content.size(1) != log_multi_content.size(2):
            raise RuntimeError("log_multi_content should be [batch, prelen, prelen, heads]")
        bsz, prelen, _, heads = log_multi_content.shape
        if log_gates.shape != (bsz, prelen, heads):
            raise RuntimeError("log_gates should be [batch, prelen, heads]")
        if log_multi_content.dtype != torch.float32 or log_gates.dtype != torch.float32:
            raise RuntimeError("dag_links_from_heads is implemented for float32 (the reference computes the "
                               "training links in float32 too)")
        content = log_multi_content.contiguous()
        gates = log_gates.contiguous()
        translen = min(int(max_transition_length), prelen - 1)
        if translen < 1:
            raise RuntimeError("max_transition_length must be at least 1 and prelen at least 2")
        nonpad = _mask_u8(nonpad_mask)
        if nonpad is not None and nonpad.shape != (bsz, prelen):
            raise RuntimeError("nonpad_mask should be [batch, prelen]")
        if bound_end is not None:
            if bound_end.shape != (bsz, prelen) or bound_end.dtype != torch.long:
                raise RuntimeError("bound_end should be a long tensor of shape [batch, prelen]")
            bound_end = bound_end.contiguous()
        dev = content.device
        need_grad = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        with torch.cuda.device(dev):
            links = torch.empty(bsz, prelen, translen, dtype=torch.float32, device=dev)
            head_lse = torch.empty(bsz, prelen, heads, dtype=torch.float32, device=dev) if need_grad else None
            check(lib().dat_links_from_heads(ptr(content), ptr(gates), ptr(bound_end), ptr(nonpad), ptr(links),
                                             ptr(head_lse), bsz, prelen, heads, translen, stream_ptr(dev)),
                  "links_from_heads")
        if need_grad:
            ctx.save_for_backward(content, gates, links, head_lse, nonpad, bound_end)
        return links

    @staticmethod
    def backward(ctx, grad_links):
        content, gates, links, head_lse, nonpad, bound_end = ctx.saved_tensors
        bsz, prelen, _, heads = content.shape
        translen = links.size(2)
        grad_links = grad_links.to(torch.float32).contiguous()
        dev = content.device
        with torch.cuda.device(dev):
            grad_content = torch.empty_like(content)
            grad_gates = torch.empty_like(gates)
            check(lib().dat_links_from_heads_backward(
                ptr(grad_links), ptr(content), ptr(gates), ptr(links), ptr(head_lse), ptr(bound_end),
                ptr(nonpad), ptr(grad_content), ptr(grad_gates), bsz, prelen, heads, translen,
                stream_ptr(dev)), "links_from_heads_backward")
        return grad_content, grad_gates, None, None, None


def _check_biased_links(content, gates, table, buckets, nonpad_mask, bound_end, translen):
    if content.dim() != 4 or content.size(1) != content.size(2):
        raise RuntimeError("log_multi_content should be [batch, prelen, prelen, heads]")
    bsz, prelen, _, heads = content.shape
    if gates.shape != (bsz, prelen, heads):
        raise RuntimeError("log_gates should be [batch, prelen, heads]")
    if table.dim() != 2 or table.size(0) < 1 or table.size(1) != heads:
        raise RuntimeError("relative_bias should be [num_buckets, heads]")
    for name, t in (("log_multi_content", content), ("log_gates", gates), ("relative_bias", table)):
        if t.dtype is not torch.float32:
            raise RuntimeError(f"dag_links_from_heads is implemented for float32 ({name} is {t.dtype})")
    if translen < 1:
        raise RuntimeError("max_transition_length must be at least 1 and prelen at least 2")
    if buckets.dim() != 1 or buckets.dtype is not torch.long or buckets.size(0) < translen:
        raise RuntimeError(f"relative_buckets should be a long tensor with at least {translen} distances")
    if nonpad_mask is not None and nonpad_mask.shape != (bsz, prelen):
        raise RuntimeError("nonpad_mask should be [batch, prelen]")
    if bound_end is not None and (bound_end.shape != (bsz, prelen) or bound_end.dtype is not torch.long):
        raise RuntimeError("bound_end should be a long tensor of shape [batch, prelen]")
    require_device(content.device, log_gates=gates, relative_bias=table, relative_buckets=buckets,
                   nonpad_mask=nonpad_mask, bound_end=bound_end)


class DagBiasedLinksFunc(Function):
    """``dag_links_from_heads`` with a learned relative position bias.  ``rest``: (relative_buckets, nonpad_mask,
    bound_end, max_transition_length)."""

    @staticmethod
    def forward(ctx, log_multi_content, log_gates, relative_bias, rest):
        relative_buckets, nonpad_mask, bound_end, max_transition_length = rest
        translen = min(int(max_transition_length), log_multi_content.size(1) - 1) if log_multi_content.dim() > 1 else 0
        _check_biased_links(log_multi_content, log_gates, relative_bias, relative_buckets, nonpad_mask, bound_end, translen)
        bsz, prelen, _, heads = log_multi_content.shape
        dev = log_multi_content.device
        need_grad = True in ctx.needs_input_grad
        with torch.cuda.device(dev):
            content, gates, table = log_multi_content.contiguous(), log_gates.contiguous(), relative_bias.contiguous()
            buckets = relative_buckets.contiguous()
            nonpad = _mask_bytes(nonpad_mask)
            if bound_end is not None:
                bound_end = bound_end.contiguous()
            links = content.new_empty((bsz, prelen, translen))
            head_lse = torch.empty_like(gates) if need_grad else None
            spans = None if nonpad is None else torch.empty(max(bsz, 1), 2, dtype=torch.int32, device=dev)
            check(lib().dat_links_from_heads_biased(
                content.data_ptr(), gates.data_ptr(), table.data_ptr(), buckets.data_ptr(), table.size(0),
                address(bound_end), address(nonpad), links.data_ptr(), address(head_lse), address(spans),
                _status_word(dev).data_ptr(), bsz, prelen, heads, translen, stream_address(dev)),
                "links_from_heads (biased)")
        if need_grad:
            ctx.save_for_backward(content, gates, table, buckets, links, head_lse, nonpad, bound_end, spans)
        return links

    @staticmethod
    def backward(ctx, grad_links):
        # the wrapper that marks the gradients costs a good part of a small backward and is only wanted by
        # whoever differentiates again
        return _biased_links_backward_once(ctx, grad_links) if torch.is_grad_enabled() else _biased_links_backward(ctx, grad_links)


def _biased_links_backward(ctx, grad_links):
    content, gates, table, buckets, links, head_lse, nonpad, bound_end, spans = ctx.saved_tensors
    bsz, prelen, _, heads = content.shape
    translen = links.size(2)
    dev = content.device
    L = lib()
    with torch.cuda.device(dev):
        grad_links = grad_links.to(torch.float32).contiguous()
        grad_content, grad_gates = torch.empty_like(content), torch.empty_like(gates)
        grad_table = ws = None
        if ctx.needs_input_grad[2]:
            grad_table = torch.empty_like(table)
            ws = torch.empty(max(L.dat_links_bias_workspace_bytes(bsz, prelen, heads, translen), 1),
                             dtype=torch.uint8, device=dev)
        check(L.dat_links_from_heads_biased_backward(
            grad_links.data_ptr(), content.data_ptr(), gates.data_ptr(), table.data_ptr(), buckets.data_ptr(),
            table.size(0), links.data_ptr(), head_lse.data_ptr(), address(bound_end), address(nonpad), address(spans),
            grad_content.data_ptr(), grad_gates.data_ptr(), address(grad_table), address(ws),
            _status_word(dev).data_ptr(), bsz, prelen, heads, translen, stream_address(dev)),
            "links_from_heads_backward (biased)")
    return grad_content, grad_gates, grad_table, None


_biased_links_backward_once = once_differentiable(_biased_links_backward)


def dag_relative_buckets(num_distances, num_buckets, max_distance=128, device=None):
    r"""Bucket of each distance ``1..num_distances`` between two vertices, for ``dag_links_from_heads``.

    The first half of the buckets holds one distance each, the others grow geometrically up to
    ``max_distance``, and the last one holds every distance beyond it.  Computed in whole numbers, so no
    distance next to a border depends on a rounded logarithm.  Returns int64 [num_distances]."""
    num_distances, num_buckets, max_distance = int(num_distances), int(num_buckets), int(max_distance)
    exact = num_buckets // 2
    if num_distances < 1 or num_buckets < 1 or max_distance <= exact:
        raise RuntimeError("dag_relative_buckets needs num_distances >= 1, num_buckets >= 1 and "
                           "max_distance > num_buckets // 2")
    grown = num_buckets - exact
    start = max(exact, 1)
    out, k = [], 0
    for d in range(num_distances):        # d = 0 is the distance 1
        if d < exact:
            out.append(d)
            continue
        # bucket exact + k begins where d >= start * (max_distance / start) ** (k / grown)
        while k + 1 < grown and d ** grown >= start ** (grown - k - 1) * max_distance ** (k + 1):
            k += 1
        out.append(exact + k)
    return torch.tensor(out, dtype=torch.long, device=device)


def dag_links_from_heads(log_multi_content, log_gates, nonpad_mask=None, bound_end=None,
                         max_transition_length=99999, relative_bias=None, relative_buckets=None):
    r"""Band links from per-head transition scores (glat_decomposed_with_link.py:380-404, the
    finite ``max_transition_length`` branch)::

        extract, nouse = model.extract_valid_links(log_multi_content, valid_mask)     # [B,L,K,H]
        extract = F.log_softmax(extract.masked_fill(nouse, -inf), dim=2).masked_fill(nouse, -inf)
        links   = logsumexp(extract + log_gates.unsqueeze(2), dim=-1)                   # [B,L,K]

    log_multi_content [B,L,L,H] fp32, log_gates [B,L,H] fp32.  The valid successors of a vertex are
    the later vertices inside the band that ``nonpad_mask`` ([B,L] bool, ``prev_output_tokens != pad``)
    allows, or, while decoding, those up to ``bound_end`` ([B,L] int64).  Returns links [B,L,K] fp32
    with K = min(max_transition_length, L-1).  Differentiable in the first two arguments.

    ``relative_bias`` [num_buckets,H] fp32 is a learned bias of the distance between two vertices:
    ``relative_bias[relative_buckets[j-i-1]]`` is added to the scores of the transition i -> j
    (``relative_buckets``: int64, one bucket for each distance 1..K or more, see ``dag_relative_buckets``).
    Differentiable in it too; the gradient is summed in a fixed order.  A bucket outside the table forbids
    the transitions of its distance and sets bit 4 of ``last_status()``.  With a bias, NaN or +inf at a valid
    successor makes the links and gradients of its vertex NaN; masked places may hold anything."""
    if (relative_bias is None) != (relative_buckets is None):
        raise RuntimeError("relative_bias and relative_buckets are given together")
    if relative_bias is not None:
        return DagBiasedLinksFunc.apply(log_multi_content, log_gates, relative_bias,
                                        (relative_buckets, nonpad_mask, bound_end, max_transition_length))
    return DagLinksFromHeadsFunc.apply(log_multi_content, log_gates, nonpad_mask, bound_end,
                                       max_transition_length)


@torch.no_grad()
def dag_node_passing_prob(links):
    r"""Probability that a path from vertex 0 visits each vertex (``_analyze_graph``,
    glat_decomposed_with_link.py:559-569).  links [B,L,L] fp32 square, -inf on and below the diagonal.
    Returns [B,L] fp32."""
    require_cuda(links)
    if links.dim() != 3 or links.size(1) != links.size(2) or links.dtype != torch.float32:
        raise RuntimeError("links should be a float32 tensor of shape [batch, prelen, prelen]")
    links = links.contiguous()
    bsz, prelen, _ = links.shape
    dev = links.device
    with torch.cuda.device(dev):
        out = torch.empty(bsz, prelen, dtype=torch.float32, device=dev)
        check(lib().dat_node_passing_prob(ptr(links), ptr(out), bsz, prelen, stream_ptr(dev)), "node_passing_prob")
    return out


@torch.no_grad()
def dag_viterbi_decode(links, output_logits_normalized, output_length, max_length, joint=False,
                       viterbibeta=1.0, pad_index=1):
    r"""``inference_viterbi`` (glat_decomposed_with_link.py:720-777) on the device.

    links [B,L,L] fp32 square log-probabilities (left untouched), output_logits_normalized [B,L,V]
    (its maximum and arg-max over V are taken with torch), or a pair ``(unreduced_logits [B,L] fp32,
    unreduced_tokens [B,L] int64)``; output_length [B] int64; ``max_length`` is the reference's
    ``int(2 * L / decode_upsample_scale)``.  Returns ``(tokens [B,max_length] padded with pad_index,
    lengths [B], vertices [B,max_length] of the chosen path, -1 padded, scores [B])``."""
    if isinstance(output_logits_normalized, (tuple, list)):
        unreduced_logits, unreduced_tokens = output_logits_normalized
    else:
        unreduced_logits, unreduced_tokens = output_logits_normalized.max(dim=-1)
    require_cuda(links, unreduced_logits, unreduced_tokens, output_length)
    if links.dim() != 3 or links.size(1) != links.size(2) or links.dtype != torch.float32:
        raise RuntimeError("links should be a float32 tensor of shape [batch, prelen, prelen]")
    bsz, prelen, _ = links.shape
    if unreduced_logits.shape != (bsz, prelen) or unreduced_tokens.shape != (bsz, prelen):
        raise RuntimeError("token scores should be [batch, prelen]")
    if output_length.dtype != torch.long or unreduced_tokens.dtype != torch.long:
        raise RuntimeError("length should be long")
    links = links.contiguous()
    logit = unreduced_logits.to(torch.float32).contiguous()
    toks = unreduced_tokens.contiguous()
    ol = output_length.contiguous()
    max_length = int(max_length)
    dev = links.device
    L = lib()
    with torch.cuda.device(dev):
        ws = torch.empty(max(L.dat_viterbi_decode_workspace_bytes(bsz, prelen, max_length), 1),
                         dtype=torch.uint8, device=dev)
        tokens = torch.empty(bsz, max_length, dtype=torch.long, device=dev)
        verts = torch.empty(bsz, max_length, dtype=torch.long, device=dev)
        lengths = torch.empty(bsz, dtype=torch.long, device=dev)
        scores = torch.empty(bsz, dtype=torch.float32, device=dev)
        check(L.dat_viterbi_decode(ptr(links), ptr(logit), ptr(toks), ptr(ol), ptr(ws), ptr(tokens), ptr(lengths),
                                   ptr(verts), ptr(scores), ptr(_status_word(dev)), bsz, prelen, max_length,
                                   int(bool(joint)), float(viterbibeta), int(pad_index), stream_ptr(dev)),
              "viterbi_decode")
    return tokens, lengths, verts, scores
