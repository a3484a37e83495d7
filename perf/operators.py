"""Cases, plain forms and 64-bit results of the operators that train a DAG model on preferences and rewards.

Three operators:

* ``links``: the transition matrix from per-head scores with a learned relative position bias by buckets of
  the distance between two vertices (``dag_links_from_heads(..., relative_bias=, relative_buckets=)``),
  forward for decoding, forward and backward for training;
* ``policy``: the clipped policy loss with a KL term over the vertices' tokens (``dag_policy_loss``),
  forward and backward from the logits;
* ``preference``: the loss of paired log ratios of sentence likelihoods (``dag_preference_loss``), forward
  and backward.

``run`` computes the plain form, or with ``own`` the package's operators.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
NEG_INF = float("-inf")
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
CLIP_LOW, CLIP_HIGH = 0.2, 0.25
KL_COEF = 0.05


# ------------------------------------------------------------------------------------------------ the cases

def listed():
    return [
        # one short graph while decoding: the successors end at bound_end, no gradient; latency counts
        dict(name="links decode 1x64x8", op="links", B=1, L=64, H=8, K=63, buckets=32, train=False),
        # a training batch of 64 graphs of 512 vertices (8x upsampling of up to 64 source tokens), full band
        dict(name="links train 64x512x8", op="links", B=64, L=512, H=8, K=511, buckets=32, train=True),
        # long graphs with a band: max_transition_length 256 of 1024 vertices
        dict(name="links train 16x1024x8 band", op="links", B=16, L=1024, H=8, K=256, buckets=64, train=True),
        # odd sizes and a head count that is no multiple of four
        dict(name="links train 5x333x6", op="links", B=5, L=333, H=6, K=332, buckets=20, train=True),
        # one vertex: what a loop over single decisions pays
        dict(name="policy 1x1x32000", op="policy", B=1, L=1, V=32000, T=1, dtype="bf16", kl="estimate", link=False),
        # the small training batch: 20 of 160 vertices are on the sampled path, fp32 logits
        dict(name="policy 8x160x1000", op="policy", B=8, L=160, V=1000, T=20, dtype="fp32", kl="estimate", link=True),
        # the translation batch: 64 of 512 vertices on the path, KL to a reference model over the vocabulary
        dict(name="policy 64x512x42000 path", op="policy", B=64, L=512, V=42000, T=64, dtype="fp16", kl="full", link=True),
        # every vertex takes part (path vertices gathered beforehand), KL over the vocabulary: the largest
        dict(name="policy 32x1024x32000 full", op="policy", B=32, L=1024, V=32000, T=1024, dtype="bf16", kl="full", link=False),
        # an odd vocabulary, whose rows do not start on 16-byte boundaries, every vertex, KL estimate
        dict(name="policy 7x333x30523", op="policy", B=7, L=333, V=30523, T=333, dtype="bf16", kl="estimate", link=True),
        # a batch of 64 pairs of sentences against a reference model
        dict(name="preference 64", op="preference", B=64, kind="sigmoid", smoothing=0.0, lengths=False, reference=True),
        # 512 pairs, likelihoods per token, smoothed labels
        dict(name="preference 512 per token", op="preference", B=512, kind="sigmoid", smoothing=0.1, lengths=True, reference=True),
        # many small sentences, squared loss, no reference model
        dict(name="preference 4099 squared", op="preference", B=4099, kind="squared", smoothing=0.0, lengths=True, reference=False),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["links", "links", "policy", "policy", "policy", "preference"])
    if op == "links":
        L = _spread(rng, 2, 1024)
        H = rng.choice([1, 2, 3, 4, 6, 8, 8, 12, 16])
        B = _spread(rng, 1, max(1, min(64, 64 * 512 * 512 * 8 // (L * L * H))))
        K = L - 1 if rng.random() < 0.6 else _spread(rng, 1, L - 1)
        return dict(op=op, B=B, L=L, H=H, K=K, buckets=_spread(rng, 2, 64), train=rng.random() < 0.8)
    if op == "policy":
        V = _spread(rng, 500, 64000)
        dtype = rng.choice(["fp32", "fp16", "bf16", "bf16"])
        rows = _spread(rng, 1, min(32768, 32768 * 32000 // V // (2 if dtype == "fp32" else 1)))
        B = _spread(rng, 1, min(64, rows))
        L = max(1, rows // B)
        T = L if rng.random() < 0.4 else _spread(rng, 1, L)
        return dict(op=op, B=B, L=L, V=V, T=T, dtype=dtype, kl=rng.choice(["none", "estimate", "full", "full"]),
                    link=rng.random() < 0.5)
    return dict(op=op, B=_spread(rng, 1, 4099), kind=rng.choice(["sigmoid", "sigmoid", "hinge", "squared"]),
                smoothing=rng.choice([0.0, 0.1]), lengths=rng.random() < 0.5, reference=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------ inputs

def _lengths(case):
    """Vertices of each graph: from the full length down to half of it, the same for every seed."""
    B, L = case["B"], case["L"]
    return [max(2, L - (b * L) // (2 * B)) for b in range(B)]


def _bucket_map(K, buckets, max_distance=128):
    """Bucket of each distance 1..K: the first half of the buckets holds one distance each, the others grow
    geometrically up to max_distance and the last one holds all beyond it.  Whole-number arithmetic, so that
    no distance next to a border depends on a rounded logarithm."""
    first = buckets // 2
    more = buckets - first
    top = max(max_distance, first + 1)
    out = []
    for d in range(K):
        if d < first:
            out.append(d)
            continue
        k = 0
        while k + 1 < more and d ** more >= max(first, 1) ** (more - k - 1) * top ** (k + 1):
            k += 1
        out.append(first + k)
    return out


def _prepare_links(case, gen):
    B, L, H, K = case["B"], case["L"], case["H"], case["K"]
    n = torch.tensor(_lengths(case), device=DEV)
    ar = torch.arange(L, device=DEV)
    s = dict(op="links", K=K, train=case["train"],
             content=torch.randn(B, L, L, H, generator=gen, device=DEV) * 1.5,
             gates=torch.log_softmax(torch.randn(B, L, H, generator=gen, device=DEV), -1),
             bias=torch.randn(case["buckets"], H, generator=gen, device=DEV) * 0.5,
             buckets=torch.tensor(_bucket_map(K, case["buckets"]), device=DEV), nonpad=None, bound_end=None)
    if case["train"]:
        s["nonpad"] = ar.view(1, L) < n.view(B, 1)
        s["grad"] = torch.randn(B, L, K, generator=gen, device=DEV) * 0.01
        for k in ("content", "gates", "bias"):
            s[k].requires_grad_()
    else:
        s["bound_end"] = (n - 1).view(B, 1).expand(B, L).contiguous()
    return s


def _prepare_policy(case, gen):
    B, L, V, T = case["B"], case["L"], case["V"], case["T"]
    dtype = DTYPES[case["dtype"]]
    x = torch.randn(B, L, V, generator=gen, device=DEV, dtype=dtype).mul_(2)
    tokens = torch.randint(0, V, (B, L), generator=gen, device=DEV)
    # sampled tokens are likely ones: their logits stand above the rest
    x.scatter_add_(-1, tokens.unsqueeze(-1), torch.full((B, L, 1), 8.0, device=DEV, dtype=dtype))
    s = dict(op="policy", logits=x, tokens=tokens, mask=None, link=None, ref_logp=None, ref_logits=None,
             kl_coef=0.0 if case["kl"] == "none" else KL_COEF)
    if T < L:
        order = torch.rand(B, L, generator=gen, device=DEV).argsort(-1)
        s["mask"] = torch.zeros(B, L, dtype=torch.bool, device=DEV).scatter_(1, order[:, :T], True)
    logp = torch.stack([x[b].gather(-1, tokens[b].unsqueeze(-1)).squeeze(-1).float()
                        - torch.logsumexp(x[b].float(), -1) for b in range(B)])
    if case["link"]:
        s["link"] = -torch.rand(B, L, generator=gen, device=DEV) * 5
        logp = logp + s["link"]
    # the log ratio to the policy that sampled; on which side of a clip bound a ratio within the rounding of a
    # 32-bit log-probability falls is nobody's to say, so none is left there
    move = torch.randn(B, L, generator=gen, device=DEV) * 0.2
    for edge in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
        move = torch.where((move - edge).abs() < 1e-3, move + 4e-3, move)
    s["old"] = logp - move
    s["advantage"] = torch.randn(B, generator=gen, device=DEV) if case["link"] else torch.randn(B, L, generator=gen, device=DEV)
    if case["kl"] == "estimate":
        s["ref_logp"] = logp + torch.randn(B, L, generator=gen, device=DEV) * 0.4
    elif case["kl"] == "full":
        y = torch.randn(B, L, V, generator=gen, device=DEV, dtype=dtype).mul_(0.5)
        s["ref_logits"] = y.add_(x, alpha=0.9)
    x.requires_grad_()
    if s["link"] is not None:
        s["link"].requires_grad_()
    return s


def _prepare_preference(case, gen):
    B = case["B"]
    tl = torch.randint(8, 65, (2, B), generator=gen, device=DEV)
    base = -tl * (4 + 4 * torch.rand(2, B, generator=gen, device=DEV))   # sentence log-likelihoods
    moved = base + torch.randn(2, B, generator=gen, device=DEV) * 6
    if B > 8:
        moved[1, 5] = NEG_INF     # a rejected sentence that has no path through its graph
    s = dict(op="preference", kind=case["kind"], smoothing=case["smoothing"], beta=2.0 if case["lengths"] else 0.1,
             chosen=moved[0].contiguous().requires_grad_(), rejected=moved[1].contiguous().requires_grad_(),
             ref=None, lengths=None)
    if case["reference"]:
        s["ref"] = (base[0].contiguous(), base[1].contiguous())
    if case["lengths"]:
        s["lengths"] = (tl[0].contiguous(), tl[1].contiguous())
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    return {"links": _prepare_links, "policy": _prepare_policy, "preference": _prepare_preference}[case["op"]](case, gen)


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    if own:
        return {"links": _own_links, "policy": _own_policy, "preference": _own_preference}[state["op"]](state)
    with torch.no_grad():
        return {"links": _plain_links, "policy": _plain_policy, "preference": _plain_preference}[state["op"]](state)


def _own_links(s):
    import da_transformer_b200 as dat

    if not s["train"]:
        return dat.dag_links_from_heads(s["content"], s["gates"], bound_end=s["bound_end"], max_transition_length=s["K"],
                                        relative_bias=s["bias"], relative_buckets=s["buckets"])
    links = dat.dag_links_from_heads(s["content"], s["gates"], nonpad_mask=s["nonpad"], max_transition_length=s["K"],
                                     relative_bias=s["bias"], relative_buckets=s["buckets"])
    return (links.detach(),) + torch.autograd.grad(links, (s["content"], s["gates"], s["bias"]), s["grad"])


def _own_policy(s):
    import da_transformer_b200 as dat

    loss, logp, kl, stats = dat.dag_policy_loss(
        s["logits"], s["tokens"], s["old"], s["advantage"], mask=s["mask"], link_logp=s["link"],
        ref_logits=s["ref_logits"], ref_logp=s["ref_logp"], kl_coef=s["kl_coef"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH)
    leaves = [t for t in (s["logits"], s["link"]) if t is not None]
    return (loss.detach(), logp, kl, stats.float()) + torch.autograd.grad(loss, leaves)


def _own_preference(s):
    import da_transformer_b200 as dat

    refs = s["ref"] or (None, None)
    lens = s["lengths"] or (None, None)
    loss, rewards, stats = dat.dag_preference_loss(
        s["chosen"], s["rejected"], refs[0], refs[1], beta=s["beta"], kind=s["kind"], label_smoothing=s["smoothing"],
        chosen_length=lens[0], rejected_length=lens[1])
    return (loss.detach(), rewards, stats) + torch.autograd.grad(loss, (s["chosen"], s["rejected"]))


def _plain_links(s):
    c, K = s["content"], s["K"]
    B, L, _, H = c.shape
    ar = torch.arange(L, device=c.device)
    dist = (ar.view(1, L) - ar.view(L, 1) - 1)
    valid = ((dist >= 0) & (dist < K)).view(1, L, L)
    if s["nonpad"] is not None:
        valid = valid & s["nonpad"].view(B, 1, L)
    else:
        valid = valid & (ar.view(1, 1, L) <= s["bound_end"].unsqueeze(2))
    dist = dist.clamp(0, K - 1)
    dead = ~valid.unsqueeze(-1)
    z = (c + s["bias"][s["buckets"]][dist]).masked_fill(dead, NEG_INF)
    m = z.amax(2, keepdim=True)
    m = torch.where(m == NEG_INF, torch.zeros_like(m), m)
    e = (z - m).exp()
    total = e.sum(2, keepdim=True)
    lse = torch.where(total > 0, m + total.log(), torch.zeros_like(m))
    soft = e / torch.where(total > 0, total, torch.ones_like(total))
    t = z - lse + s["gates"].unsqueeze(2)
    mh = t.amax(3, keepdim=True)
    mh = torch.where(mh == NEG_INF, torch.zeros_like(mh), mh)
    eh = (t - mh).exp()
    th = eh.sum(3, keepdim=True)
    square = (mh + th.log()).squeeze(3)
    share = eh / torch.where(th > 0, th, torch.ones_like(th))
    # row i, distance d of the band is column i + d + 1 of the square
    col = ar.view(L, 1) + torch.arange(K, device=c.device).view(1, K) + 1
    out = col >= L
    col = col.clamp(max=L - 1)
    links = square.gather(2, col.expand(B, L, K)).masked_fill(out, NEG_INF)
    if not s["train"]:
        return links
    g = s["grad"].gather(2, dist.expand(B, L, L)).masked_fill(~valid, 0).unsqueeze(-1)
    gp = g * share
    grad_gates = gp.sum(2)
    grad_content = gp - soft * grad_gates.unsqueeze(2)
    by_distance = grad_content.gather(2, col.view(1, L, K, 1).expand(B, L, K, H)).masked_fill(out.view(1, L, K, 1), 0)
    by_distance = by_distance.sum((0, 1), dtype=torch.float64)
    onehot = (s["buckets"].view(1, K) == torch.arange(s["bias"].shape[0], device=c.device).view(-1, 1)).double()
    return links, grad_content, grad_gates, (onehot @ by_distance).float()


def _plain_policy(s):
    x = s["logits"].float()
    dtype = s["logits"].dtype
    tok = s["tokens"].unsqueeze(-1)
    act = torch.ones_like(s["tokens"], dtype=torch.bool) if s["mask"] is None else s["mask"]
    n = act.sum().clamp(min=1).double()
    m = x.amax(-1, keepdim=True)
    p = (x - m).exp()
    total = p.sum(-1, keepdim=True, dtype=torch.float64)
    logp = ((x.gather(-1, tok) - m).double() - total.log()).squeeze(-1)
    if s["link"] is not None:
        logp = logp + s["link"].double()
    adv = (s["advantage"] if s["advantage"].dim() == 2 else s["advantage"].unsqueeze(1)).double()
    ratio = (logp - s["old"].double()).exp()
    clipped = ((adv > 0) & (ratio > 1 + CLIP_HIGH)) | ((adv < 0) & (ratio < 1 - CLIP_LOW))
    term = -torch.minimum(ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv)
    coef = torch.where(clipped, torch.zeros_like(ratio), -adv * ratio)
    kl = torch.zeros_like(logp)
    p = p / total.float()
    if s["ref_logp"] is not None:
        u = s["ref_logp"].double() - logp
        kl = u.exp() - u - 1
        coef = coef + s["kl_coef"] * (1 - u.exp())
    coef = torch.where(act, coef, torch.zeros_like(coef)) / n
    grad = p * (-coef).float().unsqueeze(-1)
    if s["ref_logits"] is not None:
        y = s["ref_logits"].float()
        my = y.amax(-1, keepdim=True)
        log_ty = (y - my).exp().sum(-1, keepdim=True, dtype=torch.float64).log()
        y = x - y
        shift = (m - my).double() + total.log() - log_ty
        klk = (p * y).sum(-1, keepdim=True, dtype=torch.float64) - shift
        kl = klk.squeeze(-1)
        w = (act.double() * (s["kl_coef"] / n)).float().unsqueeze(-1)
        grad += w * p * (y - (shift + klk).float())
    grad.scatter_add_(-1, tok, coef.float().unsqueeze(-1))
    zero = torch.zeros_like(logp)
    logp, kl, ratio, term = (torch.where(act, t, zero) for t in (logp, kl, ratio, term))
    loss = (term + s["kl_coef"] * kl).sum() / n
    stats = torch.stack([term.sum(), kl.sum(), ratio.sum(), (clipped & act).sum().double(), act.sum().double()])
    res = (loss.float(), logp.float(), kl.float(), stats.float(), grad.to(dtype))
    return res if s["link"] is None else res + (coef.float(),)


def _plain_preference(s):
    pair = torch.stack([s["chosen"], s["rejected"]]).double()
    if s["ref"] is not None:
        pair = pair - torch.stack(s["ref"]).double()
    scale = torch.full_like(pair, s["beta"])
    if s["lengths"] is not None:
        scale = scale / torch.stack(s["lengths"]).double()
    good = pair.isfinite().all(0)
    reward = torch.where(good, pair * scale, torch.zeros_like(pair))
    h = reward[0] - reward[1]
    eps = s["smoothing"]
    if s["kind"] == "sigmoid":
        small = (-h.abs()).exp()
        soft = torch.log1p(small)
        down, up = soft + (-h).clamp(min=0), soft + h.clamp(min=0)     # -log sigmoid(h), -log sigmoid(-h)
        sig = torch.where(h >= 0, 1 / (1 + small), small / (1 + small))
        term, slope = (1 - eps) * down + eps * up, sig - (1 - eps)
    elif s["kind"] == "hinge":
        term = (1 - eps) * (1 - h).clamp(min=0) + eps * (1 + h).clamp(min=0)
        slope = eps * (h > -1).double() - (1 - eps) * (h < 1).double()
    else:
        term = (1 - eps) * (h - 0.5).square() + eps * (h + 0.5).square()
        slope = 2 * (h - 0.5) + 2 * eps
    n = h.numel()
    zero = torch.zeros_like(h)
    term, slope = torch.where(good, term, zero), torch.where(good, slope, zero)
    loss = term.sum() / n
    stats = torch.stack([term.sum(), reward[0].sum(), reward[1].sum(), ((h > 0) & good).sum().double(),
                         torch.full_like(loss, n), (~good).sum().double()])
    return loss.float(), reward.float(), stats, (slope * scale[0] / n).float(), (-slope * scale[1] / n).float()


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    if case["op"] == "links":
        B, L, H, K = case["B"], case["L"], case["H"], case["K"]
        # valid transitions: i < j < n, j - i <= K
        pairs = 0
        for n in _lengths(case):
            k = min(K, n - 1)
            pairs += k * n - k * (k + 1) // 2
        read = 4 * H * (pairs + B * L)
        if not case["train"]:
            return {"bytes": read + 4 * B * L * K + 8 * B * L, "flops": 10 * pairs * H}
        # the scores and the band's gradient in; the band, the dense gradient of the scores and the gates' out
        return {"bytes": read + 4 * pairs + 4 * B * L * K + 4 * B * L * L * H + 4 * B * L * H, "flops": 24 * pairs * H}
    if case["op"] == "policy":
        B, L, V, T = case["B"], case["L"], case["V"], case["T"]
        size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
        full = case["kl"] == "full"
        return {"bytes": size * V * (B * T * (2 if full else 1) + B * L) + 40 * B * L, "flops": B * T * V * (20 if full else 9)}
    return {"bytes": 4 * case["B"] * (4 + 2 * case["reference"] + 4 * case["lengths"]) + 56, "flops": 60 * case["B"]}


# ------------------------------------------------------------------------------------------------ 64 bits, from the definition

def exact(case, seed):
    s = prepare(case, seed)
    return {"links": _exact_links, "policy": _exact_policy, "preference": _exact_preference}[case["op"]](s)


def _exact_links(s):
    """Sentence by sentence in the band layout, differentiated by torch."""
    B, L, _, H = s["content"].shape
    K = s["K"]
    i = torch.arange(L, device=DEV).view(L, 1)
    j = i + 1 + torch.arange(K, device=DEV).view(1, K)
    inside = j < L
    j = j.clamp(max=L - 1)
    bias = s["bias"].detach().double().requires_grad_()
    links, grads = [], []
    for b in range(B):
        ok = inside & (s["nonpad"][b][j] if s["nonpad"] is not None else j <= s["bound_end"][b].view(L, 1))
        content = s["content"][b].detach().double().requires_grad_()
        gates = s["gates"][b].detach().double().requires_grad_()
        band = content[i, j] + bias[s["buckets"]]                              # [L, K, H]
        alive = ok.any(1)
        band = band[alive].masked_fill(~ok[alive].unsqueeze(-1), NEG_INF)
        z = torch.log_softmax(band, 1) + gates[alive].unsqueeze(1)
        some = torch.logsumexp(z[ok[alive]], -1)                               # one value for each valid transition
        out = torch.full((L, K), NEG_INF, device=DEV, dtype=torch.float64)
        out[ok] = some.detach()
        links.append(out)
        if s["train"]:
            g = s["grad"][b].double()[ok]
            if some.numel():
                grads.append(torch.autograd.grad(some, (content, gates, bias), g))
            else:
                grads.append((torch.zeros_like(content), torch.zeros_like(gates), torch.zeros_like(bias)))
    links = torch.stack(links)
    if not s["train"]:
        return links
    gc, gg, gb = zip(*grads)
    return links, torch.stack(gc), torch.stack(gg), torch.stack(gb).sum(0)


def _exact_policy(s):
    """A few hundred rows at a time, differentiated by torch."""
    B, L, V = s["logits"].shape
    flat = lambda t: None if t is None else t.detach().reshape(B * L, *t.shape[2:])  # noqa: E731
    adv = s["advantage"]
    adv = flat((adv if adv.dim() == 2 else adv.unsqueeze(1).expand(B, L)).double())
    x, tok, old, link, ref, refx = (flat(s[k]) for k in ("logits", "tokens", "old", "link", "ref_logp", "ref_logits"))
    act = torch.ones(B * L, dtype=torch.bool, device=DEV) if s["mask"] is None else flat(s["mask"])
    n = max(1, int(act.sum()))
    grad = torch.zeros(B * L, V, dtype=torch.float64, device=DEV)
    rows = {k: torch.zeros(B * L, dtype=torch.float64, device=DEV) for k in ("logp", "kl", "term", "ratio", "clip", "link")}
    for r in torch.nonzero(act).squeeze(1).split(512):
        xr = x[r].double().requires_grad_()
        lk = (torch.zeros(len(r), device=DEV) if link is None else link[r]).double().requires_grad_()
        every = torch.log_softmax(xr, -1)
        logp = every.gather(1, tok[r].unsqueeze(1)).squeeze(1) + lk
        ratio = torch.exp(logp - old[r].double())
        held = torch.clamp(ratio, 1 - CLIP_LOW, 1 + CLIP_HIGH)
        term = -torch.min(ratio * adv[r], held * adv[r])
        kl = torch.zeros_like(term)
        if ref is not None:
            u = ref[r].double() - logp
            kl = torch.expm1(u) - u
        elif refx is not None:
            kl = (every.exp() * (every - torch.log_softmax(refx[r].double(), -1))).sum(-1)
        grad[r], rows["link"][r] = torch.autograd.grad((term + s["kl_coef"] * kl).sum() / n, (xr, lk))
        for k, v in (("logp", logp), ("kl", kl), ("term", term), ("ratio", ratio)):
            rows[k][r] = v.detach()
        rows["clip"][r] = (held.detach() * adv[r] < ratio.detach() * adv[r]).double()
    loss = (rows["term"] + s["kl_coef"] * rows["kl"]).sum() / n
    stats = torch.stack([rows["term"].sum(), rows["kl"].sum(), rows["ratio"].sum(), rows["clip"].sum(),
                         torch.tensor(float(act.sum()), device=DEV, dtype=torch.float64)])
    res = (loss, rows["logp"].view(B, L), rows["kl"].view(B, L), stats, grad.view(B, L, V))
    return res if s["link"] is None else res + (rows["link"].view(B, L),)


def _exact_preference(s):
    """In numpy, pair by pair as vectors."""
    host = lambda t: t.detach().cpu().numpy().astype(np.float64)  # noqa: E731
    c, r = host(s["chosen"]), host(s["rejected"])
    if s["ref"] is not None:
        c, r = c - host(s["ref"][0]), r - host(s["ref"][1])
    kc, kr = np.full(len(c), s["beta"]), np.full(len(c), s["beta"])
    if s["lengths"] is not None:
        kc, kr = kc / host(s["lengths"][0]), kr / host(s["lengths"][1])
    good = np.isfinite(c) & np.isfinite(r)
    c, r = np.where(good, c, 0) * kc, np.where(good, r, 0) * kr
    h, e = c - r, s["smoothing"]
    if s["kind"] == "sigmoid":
        term = (1 - e) * np.logaddexp(0, -h) + e * np.logaddexp(0, h)
        slope = np.exp(-np.logaddexp(0, -h)) - (1 - e)
    elif s["kind"] == "hinge":
        term = (1 - e) * np.maximum(0, 1 - h) + e * np.maximum(0, 1 + h)
        slope = e * (h > -1) - (1 - e) * (h < 1)
    else:
        term = (1 - e) * (h - 0.5) ** 2 + e * (h + 0.5) ** 2
        slope = 2 * ((1 - e) * (h - 0.5) + e * (h + 0.5))
    term, slope = np.where(good, term, 0), np.where(good, slope, 0)
    stats = np.array([term.sum(), c.sum(), r.sum(), ((h > 0) & good).sum(), len(h), (~good).sum()], dtype=np.float64)
    return np.float64(term.sum() / len(h)), np.stack([c, r]), stats, slope * kc / len(h), -slope * kr / len(h)
