"""``dag_policy_loss`` and ``dag_preference_loss`` against plain torch in 64 bits, their refusals, and a training
step that uses them together with the links' bias and ``dag_loss``."""
import itertools
import math

import numpy as np
import pytest
import torch

import da_transformer_b200 as dat
from da_transformer_b200 import torch_twins, workloads
from util import assert_rel, assert_rel_quantized

DEV = "cuda:0"
NEG_INF = float("-inf")
NAN = float("nan")
U = 2.0 ** -24          # half a step of fp32 relative to the value


# ------------------------------------------------------------------------------------------------ policy: oracle

def policy_oracle(x, tokens, old, adv, mask=None, link=None, ref_logits=None, ref_logp=None, kl_coef=0.0, lo=0.2, hi=0.2):
    """(loss, logp, kl, stats, d loss / d x, d loss / d link) in 64 bits on the CPU."""
    B, L, V = x.shape
    c = lambda t: None if t is None else t.detach().cpu()  # noqa: E731
    x, tokens, old, adv, mask, link, ref_logits, ref_logp = map(c, (x, tokens, old, adv, mask, link, ref_logits, ref_logp))
    act = torch.ones(B, L, dtype=torch.bool) if mask is None else mask.bool()
    adv = (adv if adv.dim() == 2 else adv.view(B, 1).expand(B, L)).double()[act]
    xa = x[act].double().requires_grad_()
    la = (torch.zeros(B, L) if link is None else link)[act].double().requires_grad_()
    every = torch.log_softmax(xa, -1)
    lp = every.gather(1, tokens[act].unsqueeze(1)).squeeze(1) + la
    r = (lp - old[act].double()).exp()
    held = r.clamp(1 - lo, 1 + hi)
    term = -torch.where(r * adv < held * adv, r * adv, held * adv)
    kl = torch.zeros_like(term)
    if ref_logits is not None:
        logq = torch.log_softmax(ref_logits[act].double(), -1)
        p = every.exp()
        kl = (p * torch.where(p > 0, every - logq, torch.zeros_like(p))).sum(-1)
    elif ref_logp is not None:
        u = ref_logp[act].double() - lp
        kl = torch.expm1(u) - u
    n = max(1, int(act.sum()))
    loss = (term + kl_coef * kl).sum() / n
    gx, gl = torch.autograd.grad(loss, (xa, la))
    clipped = ((adv > 0) & (r > 1 + hi)) | ((adv < 0) & (r < 1 - lo))
    full = lambda t: torch.zeros((B, L) + t.shape[1:], dtype=torch.float64).index_put((act,), t.detach().double())  # noqa: E731
    stats = [float(t.detach().sum()) for t in (term, kl, r, clipped, act)]
    return float(loss.detach()), full(lp).numpy(), full(kl).numpy(), np.array(stats), full(gx).numpy(), full(gl).numpy()


def policy_inputs(B, L, V, dtype, seed=0, link=False, ref=None, mask=None, adv_rows=True):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, L, V, generator=gen) * 2).to(dtype)
    tokens = torch.randint(0, V, (B, L), generator=gen)
    kw = dict(tokens=tokens)
    lp = torch.log_softmax(x.double(), -1).gather(-1, tokens.unsqueeze(-1)).squeeze(-1)
    if link:
        kw["link"] = -torch.rand(B, L, generator=gen) * 4
        lp = lp + kw["link"]
    move = torch.randn(B, L, generator=gen) * 0.3
    for edge in (math.log(0.8), math.log(1.2)):    # no ratio within rounding of a clip bound
        move = torch.where((move - edge).abs() < 1e-3, move + 3e-3, move)
    kw["old"] = (lp - move).float()
    kw["adv"] = torch.randn(B, L, generator=gen) if adv_rows else torch.randn(B, generator=gen)
    if ref == "full":
        kw["ref_logits"] = (x.float() * 0.8 + torch.randn(B, L, V, generator=gen)).to(dtype)
    elif ref == "estimate":
        kw["ref_logp"] = (lp + torch.randn(B, L, generator=gen) * 0.5).float()
    if mask is not None:
        kw["mask"] = torch.rand(B, L, generator=gen) < mask
    return x.to(DEV), {k: v.to(DEV) for k, v in kw.items()}


def policy_call(x, tokens, old, adv, mask=None, link=None, ref_logits=None, ref_logp=None, kl_coef=0.0, lo=0.2, hi=0.2,
                **kw):
    return dat.dag_policy_loss(x, tokens, old, adv, mask=mask, link_logp=link, ref_logits=ref_logits, ref_logp=ref_logp,
                               kl_coef=kl_coef, clip_low=lo, clip_high=hi, **kw)


def row_tolerance(V):
    """How far a log-sum-exp over V logits may be off: each term of the sum is rounded by ex2 (2 U) and by the
    difference and product in its argument (2 U times |x - max| log2 e, below 16 where e^(x - max) counts), and
    passes at most V / 256 additions of a thread, 13 of the reductions and 3 rescalings."""
    return U * (V / 256 + 13 + 3 + 2 + 2 * 16)


def check_policy(got, want, dtype, V, kw, kl_coef=0.0, d_max=0.0):
    loss, logp, kl, stats, gx, gl = got
    wloss, wlogp, wkl, wstats, wgx, wgl = want
    act = np.ones(wlogp.shape, bool) if kw.get("mask") is None else kw["mask"].cpu().numpy().astype(bool)
    tol = row_tolerance(V)
    a = logp.cpu().numpy().astype(np.float64)
    assert (np.abs(a - wlogp) <= tol + 2 * U * np.abs(wlogp)).all()
    k = kl.cpu().numpy().astype(np.float64)
    # two log-sum-exps and the mean of d = x - y (relative to its first value) with the sum's rounding
    klt = 2 * tol + tol * d_max + 2 * U * np.abs(wkl) + (0 if kw.get("ref_logp") is None else tol * (1 + np.abs(wkl)))
    assert (np.abs(k - wkl) <= klt).all()
    assert not a[~act].any() and not k[~act].any()
    adv = kw["adv"].cpu().numpy().astype(np.float64)
    adv = adv if adv.ndim == 2 else adv[:, None] * np.ones_like(wlogp)
    ratio = np.exp(wlogp - kw["old"].cpu().numpy())
    n = max(1, act.sum())
    dr = np.where(act, ratio * (tol + 2 * U), 0)      # off by as much as the log-probability, and stored in 32 bits
    dterm = dr * np.abs(np.where(act, adv, 0)) + U * np.abs(np.where(act, ratio * adv, 0))
    dloss = (dterm.sum() + abs(kl_coef) * np.where(act, klt, 0).sum()) / n + 2 * U * abs(wloss)
    assert abs(float(loss) - wloss) <= dloss
    s = stats.cpu().numpy()
    assert s[3] == wstats[3] and s[4] == wstats[4]
    assert abs(s[0] - wstats[0]) <= dterm.sum() + 1e-12 * abs(wstats[0])
    assert abs(s[1] - wstats[1]) <= np.where(act, klt, 0).sum() + 1e-12 * abs(wstats[1])
    assert abs(s[2] - wstats[2]) <= dr.sum() + 1e-12 * abs(wstats[2])
    if gx is not None:
        g = gx.float().cpu().numpy()
        assert not g[~act].any()
        if dtype == torch.float32:
            assert_rel(g, wgx, 1e-4, "gradient of the logits")
        else:
            assert_rel_quantized(g, wgx, 1e-4, str(dtype).split(".")[1], "gradient of the logits")
    if gl is not None:
        assert_rel(gl.cpu().numpy(), wgl, 1e-4, "gradient of the link log-probabilities")


def run_policy(x, kw, kl_coef=0.0, scale=None, **more):
    x = x.detach().clone().requires_grad_()
    link = kw.get("link")
    k = dict(kw)
    if link is not None:
        link = k["link"] = link.detach().clone().requires_grad_()
    loss, logp, kl, stats = policy_call(x, kl_coef=kl_coef, **k, **more)
    leaves = [x] if link is None else [x, link]
    grads = torch.autograd.grad(loss if scale is None else loss * scale, leaves)
    return loss.detach(), logp, kl, stats, grads[0], grads[1] if link is not None else None


def d_range(x, kw):
    if kw.get("ref_logits") is None:
        return 0.0
    d = x.double() - kw["ref_logits"].double()
    d = d - d[..., :1]
    return float(d[d.isfinite()].abs().max())


# ------------------------------------------------------------------------------------------------ CPU: refusals

def test_policy_refusals_come_before_any_device_work():
    B, L, V = 2, 3, 8
    x, tok, f = torch.zeros(B, L, V), torch.zeros(B, L, dtype=torch.long), torch.zeros(B, L)

    def call(x=x, tok=tok, old=f, adv=f, **kw):
        return dat.dag_policy_loss(x, tok, old, adv, **kw)

    for kw, text in ((dict(x=x[0]), "dim"), (dict(x=x.double()), "dtype"), (dict(x=x.transpose(0, 1)), "contiguous"),
                     (dict(x=x[..., :0]), "vocabulary"), (dict(tok=tok.int()), "tokens"), (dict(tok=tok[:, :2]), "tokens"),
                     (dict(old=f.half()), "old_logp"), (dict(old=f[:1]), "old_logp"), (dict(adv=torch.zeros(L)), "advantage"),
                     (dict(adv=f.double()), "advantage"), (dict(mask=torch.ones(B)), "mask"),
                     (dict(link_logp=f[:, :1]), "link_logp"), (dict(ref_logp=f.double()), "ref_logp"),
                     (dict(ref_logits=x.half()), "ref_logits"), (dict(ref_logits=x[:, :2]), "ref_logits"),
                     (dict(ref_logits=torch.zeros(L, B, V).transpose(0, 1)), "contiguous"),
                     (dict(ref_logits=x, ref_logp=f), "not both"), (dict(clip_low=-0.1), "negative"),
                     (dict(clip_high=NAN), "negative"), (dict(grad_scale=torch.ones(2)), "grad_scale"),
                     (dict(grad_scale=torch.ones(1, dtype=torch.float64)), "grad_scale")):
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_preference_refusals_come_before_any_device_work():
    f, n = torch.zeros(4), torch.ones(4, dtype=torch.long)
    for args, kw, text in (((f.view(2, 2), f), {}, "pairs"), ((f, f[:3]), {}, "pairs"), ((f, f.double()), {}, "float32"),
                           ((f, f, f), {}, "together"), ((f, f, f, f[:3]), {}, "reference_rejected"),
                           ((f, f), dict(chosen_length=n), "together"),
                           ((f, f), dict(chosen_length=n, rejected_length=n.int()), "long"),
                           ((f, f), dict(kind="other"), "kind"), ((f, f), dict(label_smoothing=1.5), "smoothing"),
                           ((f, f), dict(label_smoothing=NAN), "smoothing")):
        with pytest.raises(RuntimeError, match=text):
            dat.dag_preference_loss(*args, **kw)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="GPU"):
            dat.dag_preference_loss(f, f)


def test_entry_points_refuse_bad_arguments():
    lib = dat._native.lib()
    none = [None] * 4
    assert lib.dat_preference_loss(*none, None, None, 0.1, 0.0, 0, None, None, None, None, None, 3, None) == 1
    assert lib.dat_policy_loss(*none[:2], 0, *none[:3], 0, 0, *none[:3], 0.0, 0.2, 0.2, None, 1.0, *none, *none, 1, 1, 0,
                               None) == 1 and b"vocab=0" in lib.dat_last_error()
    assert lib.dat_links_from_heads_biased(*none, 0, *none, None, None, 1, 4, 4, 3, None) == 1
    assert b"num_buckets=0" in lib.dat_last_error()


# ------------------------------------------------------------------------------------------------ GPU: policy

SIZES = [(1, 20, 9001), (40, 5, 8192), (1, 2, 128000), (2, 90, 20011), (1, 1, 1), (1, 1, 2), (2, 3, 7), (1, 2, 255), (3, 5, 1000), (2, 130, 513), (1, 4, 4099), (1, 3, 32000), (2, 2, 30523),
         (5, 60, 64), (1, 2, 64001)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,L,V", SIZES)
def test_policy_against_64_bits(B, L, V, dtype):
    for ref, link, mask in itertools.product((None, "estimate", "full"), (False, True), (None, 0.4)):
        x, kw = policy_inputs(B, L, V, dtype, seed=V + 3 * L, link=link, ref=ref, mask=mask, adv_rows=link)
        coef = 0.0 if ref is None else 0.3
        got = run_policy(x, kw, kl_coef=coef)
        want = policy_oracle(x, kl_coef=coef, **kw)
        check_policy(got, want, dtype, V, kw, kl_coef=coef, d_max=d_range(x, kw))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [777, 9001])
@pytest.mark.parametrize("ref", [None, "estimate", "full"])
def test_policy_scales_of_the_loss(ref, V):
    """Whatever gradient reaches the loss, expected or not, the logits' gradient is rounded once."""
    x, kw = policy_inputs(2, 9, V, torch.float16, seed=4, link=True, ref=ref, mask=0.7)
    base = policy_oracle(x, kl_coef=0.1, **kw)
    for expected, scale in ((1.0, None), (1.0, 1024.0), (1024.0, 1024.0), (None, 1.0), (None, 1024.0), (2.0, None),
                            (torch.tensor(1024.0, device=DEV), 1024.0), (torch.tensor([8.0], device=DEV), 0.5)):
        got = run_policy(x, kw, kl_coef=0.1, scale=scale, grad_scale=expected)
        by = 1.0 if scale is None else scale
        assert_rel_quantized(got[4].float().cpu().numpy(), base[4] * by, 1e-4, "float16")
        assert_rel(got[5].cpu().numpy(), base[5] * by, 1e-4)


@pytest.mark.gpu
def test_policy_second_backward_has_its_own_buffer():
    x, kw = policy_inputs(2, 5, 300, torch.float32, seed=6, ref="full")
    x = x.requires_grad_()
    loss = policy_call(x, kl_coef=0.2, **kw)[0]
    first, = torch.autograd.grad(loss, x, retain_graph=True)
    keep = first.clone()
    second, = torch.autograd.grad(loss * 3, x, retain_graph=True)
    third, = torch.autograd.grad(loss, x)
    assert torch.equal(first, keep) and first.data_ptr() != second.data_ptr()
    assert_rel(second.cpu().numpy(), 3 * keep.double().cpu().numpy(), 1e-6)
    assert_rel(third.cpu().numpy(), keep.double().cpu().numpy(), 1e-6)
    loss = policy_call(x, kl_coef=0.2, **kw)[0]
    with pytest.raises(RuntimeError, match="once_differentiable|twice|does not require grad"):
        g, = torch.autograd.grad(loss, x, create_graph=True)
        g.sum().backward()
    loss = policy_call(x, kl_coef=0.2, **kw)[0]
    with torch.no_grad():
        x.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        loss.backward()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [700, 9001, 40000])
@pytest.mark.parametrize("ref", [None, "full"])
def test_policy_logits_far_apart(V, ref):
    """The token's logit 200 below the largest in both models (a ratio of probabilities that 32 bits do not hold), a
    row of which a single logit carries all, and logits of +-1e4."""
    x, kw = policy_inputs(2, 6, V, torch.float32, seed=V, ref=ref)
    b, l = torch.arange(2, device=DEV).view(2, 1), torch.arange(6, device=DEV).view(1, 6)
    tok = kw["tokens"]
    x[b, l, (tok + 1) % V] += torch.tensor([0., 60., 100., 200., 1000., 1e4], device=DEV)
    x[1, 5] *= 100
    if ref:
        kw["ref_logits"] = x * 0.9 + 0.5 * torch.randn(2, 6, V, generator=torch.Generator().manual_seed(1)).to(DEV)
    lp = torch.log_softmax(x.double(), -1).gather(-1, tok.unsqueeze(-1)).squeeze(-1)
    kw["old"] = (lp - 0.05).float()
    got = run_policy(x, kw, kl_coef=0.1)
    want = policy_oracle(x, kl_coef=0.1, **kw)
    # log-probabilities near -1e4 carry 5e-4 in 32 bits, and the ratio with them; the gradient is as far off as the
    # ratio, and the exponents of the logits that count are below 16
    a, w = got[1].cpu().numpy().astype(np.float64), want[1]
    tol = row_tolerance(V) + 4 * U * np.abs(w)
    assert (np.abs(a - w) <= tol).all()
    d = d_range(x, kw)
    assert (np.abs(got[2].cpu().numpy() - want[2]) <= 4 * row_tolerance(V) * (1 + d)).all()
    off = np.abs(got[4].cpu().numpy() - want[4])
    assert (off <= (3 * tol.max() + 4 * row_tolerance(V) * (1 + d)) / 12 * 3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [9001, 33000, 70001])
def test_policy_forbidden_tokens_in_long_rows(V, dtype):
    """-inf in both models, in every row and in the first rows only; a reference that has them alone; a token that is
    forbidden itself (its log-probability is -inf, and no number of its row but the loss's is asked for)."""
    x, kw = policy_inputs(1, 12, V, dtype, seed=V, ref="full", link=True)
    gen = torch.Generator().manual_seed(2)
    ban = (torch.rand(V, generator=gen) < 0.2).to(DEV)
    ban[kw["tokens"].unique()] = False
    for rows in (slice(0, 12), slice(0, 3), slice(7, 8)):
        xx, k = x.clone(), {n: t.clone() for n, t in kw.items()}
        xx[:, rows, ban] = NEG_INF
        k["ref_logits"][:, rows, ban] = NEG_INF
        lp = torch.log_softmax(xx.double(), -1).gather(-1, k["tokens"].unsqueeze(-1)).squeeze(-1) + k["link"].double()
        k["old"] = (lp - 0.1).float()
        got = run_policy(xx, k, kl_coef=0.2)
        check_policy(got, policy_oracle(xx, kl_coef=0.2, **k), dtype, V, k, kl_coef=0.2, d_max=d_range(xx, k))
    # every second logit of the policy forbidden, the reference free: finite
    xx = x.clone()
    keep = torch.zeros(V, dtype=torch.bool, device=DEV)
    keep[::2] = True
    keep[kw["tokens"].unique()] = True
    xx[..., ~keep] = NEG_INF
    lp = torch.log_softmax(xx.double(), -1).gather(-1, kw["tokens"].unsqueeze(-1)).squeeze(-1) + kw["link"].double()
    k = {**kw, "old": (lp - 0.1).float()}
    check_policy(run_policy(xx, k, kl_coef=0.2), policy_oracle(xx, kl_coef=0.2, **k), dtype, V, k, kl_coef=0.2,
                 d_max=d_range(xx, k))
    # the token itself forbidden
    xx = x.clone()
    xx[0, 4, kw["tokens"][0, 4]] = NEG_INF
    loss, logp, kl, stats, gx, gl = run_policy(xx, {**kw, "old": kw["old"].clone()}, kl_coef=0.2)
    assert float(logp[0, 4]) == NEG_INF and logp[0, 5:].isfinite().all() and logp[0, :4].isfinite().all()
    rest = [n for n in range(12) if n != 4]
    want = policy_oracle(x, kl_coef=0.2, **kw)
    assert_rel(logp[0, rest].cpu().numpy(), want[1][0, rest], 1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [5000, 9003, 30000, 64000])
def test_policy_rows_of_a_long_batch(V, dtype):
    """More rows than CTAs, a mask that leaves some CTAs nothing, every kind of KL: each row by itself as in a call
    of its own rows (one thread's order of sums apart)."""
    B, L = 3, 200
    for ref in (None, "estimate", "full"):
        x, kw = policy_inputs(B, L, V, dtype, seed=V, ref=ref, mask=0.3)
        kw["mask"][1] = False
        got = run_policy(x, kw, kl_coef=0.1)
        rows = kw["mask"].nonzero()[::7]
        pick = lambda t: t[rows[:, 0], rows[:, 1]].unsqueeze(0).contiguous()  # noqa: E731
        small = {n: pick(t) for n, t in kw.items() if n != "mask"}
        want = policy_oracle(pick(x), kl_coef=0.1, **small)
        share = len(rows) / int(kw["mask"].sum())       # the mean is over more rows here
        sub = (got[0], pick(got[1]), pick(got[2]), got[3], pick(got[4]), None)
        tol = row_tolerance(V)
        assert (np.abs(sub[1].cpu().numpy() - want[1]) <= tol + 2 * U * np.abs(want[1])).all()
        g, w = sub[4].float().cpu().numpy(), want[4] * share
        if dtype == torch.float32:
            assert_rel(g, w, 1e-4)
        else:
            assert_rel_quantized(g, w, 1e-4, str(dtype).split(".")[1])
        assert not got[4][~kw["mask"]].any() and float(got[3][4]) == int(kw["mask"].sum())
        again = run_policy(x, kw, kl_coef=0.1)
        for a, b in zip(got[:5], again[:5]):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [130, 10001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_policy_masked_vertices_may_hold_anything(dtype, V):
    x, kw = policy_inputs(3, 90, V, dtype, seed=7, link=True, ref="full", mask=0.5)
    want = run_policy(x, kw, kl_coef=0.1)
    off = ~kw["mask"]
    for value in (NAN, float("inf"), NEG_INF, torch.finfo(dtype).min):
        xd, k = x.clone(), {n: t.clone() for n, t in kw.items()}
        for t in (xd, k["old"], k["adv"], k["link"], k["ref_logits"]):
            t[off] = value
        k["tokens"][off] = -5
        dat.last_status(DEV)
        for a, b in zip(run_policy(xd, k, kl_coef=0.1), want):
            assert torch.equal(a, b)
        assert not dat.last_status(DEV) & 4


@pytest.mark.gpu
def test_policy_without_active_vertices_and_empty_batches():
    x, kw = policy_inputs(2, 4, 33, torch.bfloat16, seed=8, link=True, ref="estimate")
    kw["mask"] = torch.zeros(2, 4, dtype=torch.bool, device=DEV)
    loss, logp, kl, stats, gx, gl = run_policy(x, kw, kl_coef=0.1)
    for t in (loss, logp, kl, stats, gx, gl):
        assert not t.any()
    x, kw = policy_inputs(2, 4, 33, torch.bfloat16, seed=8, link=True, ref="full")
    for s in (slice(0, 0), slice(None)):
        k = {n: (t[s] if s.stop == 0 else t[:, :0]) for n, t in kw.items()}
        loss, logp, kl, stats, gx, gl = run_policy((x[s] if s.stop == 0 else x[:, :0]).contiguous(),
                                                   {n: t.contiguous() for n, t in k.items()}, kl_coef=0.1)
        assert float(loss) == 0 and not stats.any() and logp.numel() == gx.numel() == gl.numel() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_policy_forbidden_tokens_and_shifted_references(dtype):
    """Logits of -inf in both models (tokens that generation bans), a constant between the models' logits, and a
    policy that puts nothing where the reference puts something."""
    x, kw = policy_inputs(2, 7, 900, dtype, seed=9, ref="full")
    gen = torch.Generator().manual_seed(1)
    ban = (torch.rand(900, generator=gen) < 0.3).to(DEV)
    ban[0] = True                                # also the value that d is taken relative to
    ban[kw["tokens"].unique()] = False
    x[..., ban] = NEG_INF
    kw["ref_logits"] = kw["ref_logits"] + 64
    kw["ref_logits"][0, :, ban] = NEG_INF
    only = torch.log_softmax(x.double(), -1).gather(-1, kw["tokens"].unsqueeze(-1)).squeeze(-1)
    kw["old"] = (only - 0.1).float()
    got = run_policy(x, kw, kl_coef=0.2)
    want = policy_oracle(x, kl_coef=0.2, **kw)
    d = (x.double() - kw["ref_logits"].double())
    d = d[d.isfinite()]
    check_policy(got, want, dtype, 900, kw, kl_coef=0.2, d_max=float(d.abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [40, 9001])
def test_policy_token_outside_the_vocabulary(V):
    x, kw = policy_inputs(2, 3, V, torch.float32, seed=10)
    kw["tokens"][0, 1], kw["tokens"][1, 2] = V, -1
    dat.last_status(DEV)
    loss, logp, _, _, gx, _ = run_policy(x, kw)
    assert dat.last_status(DEV) & 4
    assert math.isnan(float(loss)) and logp.isnan().nonzero().tolist() == [[0, 1], [1, 2]]
    assert gx.isnan().all(-1).nonzero().tolist() == [[0, 1], [1, 2]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [64, 333, 9001])
def test_policy_strides_and_alignment(dtype, V):
    x, kw = policy_inputs(3, 4, V, dtype, seed=11, link=True, ref="full", adv_rows=True)
    kw["mask"] = torch.tensor([1, 0, 1, 1], device=DEV, dtype=torch.bool).expand(3, 4)
    want = policy_oracle(x, kl_coef=0.2, **kw)

    def off(t):
        return torch.empty(t.numel() + 1, device=DEV, dtype=t.dtype)[1:].view(t.shape).copy_(t)

    def strided(t):
        return torch.empty(4, 3, 2, device=DEV, dtype=t.dtype)[..., 0].t().copy_(t)

    k = {n: (t if n in ("mask", "ref_logits") else strided(t)) for n, t in kw.items()}
    for xx, yy in ((x, kw["ref_logits"]), (off(x), kw["ref_logits"]), (x, off(kw["ref_logits"])), (off(x), off(kw["ref_logits"]))):
        xx = xx.detach().requires_grad_()       # no clone: the address is what is tested
        link = k["link"].detach().requires_grad_()
        loss, logp, kl, stats = policy_call(xx, kl_coef=0.2, **{**k, "ref_logits": yy, "link": link})
        check_policy((loss.detach(), logp, kl, stats, *torch.autograd.grad(loss, (xx, link))), want, dtype, V, kw,
                     kl_coef=0.2, d_max=d_range(x, kw))
    one = kw["adv"][:, :1].clone()              # an advantage of each sentence, as [B], as [B,1] expanded
    res = [run_policy(x, {**kw, "adv": a}, kl_coef=0.2) for a in (one.squeeze(1), one.expand(3, 4))]
    for a, b in zip(*res):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_policy_gradient_only_where_it_is_asked_for():
    x, kw = policy_inputs(2, 6, 120, torch.float32, seed=12, link=True, ref="estimate")
    want = run_policy(x, kw, kl_coef=0.1)
    with torch.no_grad():
        for a, b in zip(policy_call(x, kl_coef=0.1, **kw), want[:4]):
            assert torch.equal(a, b)
    link = kw["link"].clone().requires_grad_()
    loss = policy_call(x, kl_coef=0.1, **{**kw, "link": link})[0]
    assert torch.equal(torch.autograd.grad(loss, link)[0], want[5])
    leaf = x.clone().requires_grad_()
    loss, logp, kl, stats = policy_call(leaf, kl_coef=0.1, **kw)
    assert not (logp.requires_grad or kl.requires_grad or stats.requires_grad)
    loss.backward()
    assert torch.equal(leaf.grad, want[4])


@pytest.mark.gpu
@pytest.mark.parametrize("ref", [None, "estimate", "full"])
def test_policy_gradient_against_differences(ref):
    x, kw = policy_inputs(1, 6, 50, torch.float32, seed=13, link=True, ref=ref)
    got = run_policy(x, kw, kl_coef=0.5)
    gen = torch.Generator().manual_seed(5)
    eps = 1e-2
    for leaf, grad in ((x, got[4]), (kw["link"], got[5])):
        step = torch.randn(leaf.shape, generator=gen).to(DEV)
        step = step / step.norm()
        value = []
        for s in (eps, -eps):
            k = dict(kw)
            xx = x
            if leaf is x:
                xx = x + s * step
            else:
                k["link"] = k["link"] + s * step
            value.append(float(policy_call(xx, kl_coef=0.5, **k)[0]))
        slope = (value[0] - value[1]) / (2 * eps)
        # losses of about 1, each off by 1e-6, over 2 eps; eps^2 times third derivatives of order one
        assert abs(slope - float((step.double() * grad.double()).sum())) < 5e-4


@pytest.mark.gpu
def test_policy_many_rows_repeat_and_sum_in_a_fixed_order():
    """More rows than one chunk of the sums, the last chunk partly filled."""
    for L in (1, 255, 256, 257, 700, 5000):
        x, kw = policy_inputs(1, L, 17, torch.float32, seed=L, ref="estimate", mask=0.6)
        a, b = run_policy(x, kw, kl_coef=0.1), run_policy(x, kw, kl_coef=0.1)
        for u, v in zip(a[:5], b[:5]):
            assert torch.equal(u, v)
        check_policy(a, policy_oracle(x, kl_coef=0.1, **kw), torch.float32, 17, kw, kl_coef=0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [500, 20000])
def test_policy_on_streams_and_in_graphs(V):
    x, kw = policy_inputs(2, 40, V, torch.bfloat16, seed=14, link=True, ref="full", mask=0.5)
    want = run_policy(x, kw, kl_coef=0.1)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_policy(x, kw, kl_coef=0.1)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    stat = {n: t.clone() for n, t in kw.items()}
    xs = torch.zeros_like(x).requires_grad_()
    stat["link"].requires_grad_()

    def step():
        loss, logp, kl, st = policy_call(xs, kl_coef=0.1, **stat)
        return (loss.detach(), logp, kl, st) + torch.autograd.grad(loss, (xs, stat["link"]))

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):    # two graphs, replayed in turn: neither may hold what the other needs
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    with torch.no_grad():
        xs.copy_(x)
    for graph, out in graphs + graphs[:1]:
        graph.replay()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    other = policy_inputs(2, 40, V, torch.bfloat16, seed=15, link=True, ref="full", mask=0.5)
    with torch.no_grad():
        xs.copy_(other[0])
        for n, t in other[1].items():
            stat[n].copy_(t)
    graphs[0][0].replay()
    for a, b in zip(graphs[0][1], run_policy(*other, kl_coef=0.1)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_policy_offsets_beyond_32_bits():
    """More than 2^31 logits; the active vertices are the last ones."""
    B, L, V = 3, 23000, 32000
    x = torch.zeros(B, L, V, device=DEV, dtype=torch.bfloat16)
    small, kw = policy_inputs(1, 4, V, torch.bfloat16, seed=16)
    x[-1, -4:] = small[0]
    x.requires_grad_()
    mask = torch.zeros(B, L, dtype=torch.bool, device=DEV)
    mask[-1, -4:] = True
    full = {}
    for n, t in kw.items():
        full[n] = torch.zeros(B, L, dtype=t.dtype, device=DEV)
        full[n][-1, -4:] = t[0]
    loss, logp, kl, stats = policy_call(x, mask=mask, **full)
    g, = torch.autograd.grad(loss, x)
    want = policy_oracle(small, **kw)
    check_policy((loss.detach(), logp[-1:, -4:], kl[-1:, -4:], stats, g[-1:, -4:], None), want, torch.bfloat16, V, kw)
    assert not logp[:-1].any() and not g[:-1].any() and not g[-1, :-4].any()


# ------------------------------------------------------------------------------------------------ GPU: preference

def preference_oracle(c, r, rc=None, rr=None, beta=0.1, kind="sigmoid", label_smoothing=0.0, chosen_length=None,
                      rejected_length=None):
    v = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    c, r = v(c).requires_grad_(), v(r).requires_grad_()
    a, b = (c, r) if rc is None else (c - v(rc), r - v(rr))
    if chosen_length is not None:
        a, b = a / v(chosen_length), b / v(rejected_length)
    good = a.isfinite() & b.isfinite()
    if chosen_length is not None:
        good &= (v(chosen_length) >= 1) & (v(rejected_length) >= 1)
    a, b = a[good] * beta, b[good] * beta
    h, e = a - b, label_smoothing
    f = torch.nn.functional
    term = {"sigmoid": lambda: -(1 - e) * f.logsigmoid(h) - e * f.logsigmoid(-h),
            "hinge": lambda: (1 - e) * f.relu(1 - h) + e * f.relu(1 + h),
            "squared": lambda: (1 - e) * (h - 0.5) ** 2 + e * (h + 0.5) ** 2}[kind]()
    n = max(1, len(c))
    loss = term.sum() / n
    gc, gr = torch.autograd.grad(loss, (c, r), allow_unused=True) if len(h) else (None, None)
    z = lambda g: torch.zeros_like(c) if g is None else torch.nan_to_num(g)  # noqa: E731
    rewards = torch.zeros(2, len(c), dtype=torch.float64)
    rewards[0, good], rewards[1, good] = a.detach(), b.detach()
    a, b, term, loss = (t.detach() for t in (a, b, term, loss))
    stats = [float(term.sum()), float(a.sum()), float(b.sum()), int((h > 0).sum()), len(c), int((~good).sum())]
    return float(loss), rewards.numpy(), np.array(stats), z(gc).detach().numpy(), z(gr).detach().numpy()


def preference_inputs(n, seed=0):
    gen = torch.Generator().manual_seed(seed)
    tl = torch.randint(2, 65, (2, n), generator=gen)
    base = -tl * (4 + 5 * torch.rand(2, n, generator=gen))
    pol = base + torch.randn(2, n, generator=gen) * 8
    return [t.to(DEV) for t in (pol[0], pol[1], base[0], base[1], tl[0], tl[1])]


def check_preference(args, kw):
    c, r = (t.detach().clone().requires_grad_() for t in args[:2])
    loss, rewards, stats = dat.dag_preference_loss(c, r, *args[2:], **kw)
    got = torch.autograd.grad(loss, (c, r))
    want = preference_oracle(*args, **kw)
    # everything is put together in 64 bits and rounded once (the gradients twice: the kernel's and the product's)
    assert abs(float(loss.detach()) - want[0]) <= 1.01 * U * abs(want[0])
    assert (np.abs(rewards.cpu().numpy() - want[1]) <= 1.01 * U * np.abs(want[1])).all()
    s = stats.cpu().numpy()
    assert np.array_equal(s[3:], want[2][3:])
    scale = np.array([abs(want[2][0]), np.abs(want[1][0]).sum(), np.abs(want[1][1]).sum()])
    assert (np.abs(s[:3] - want[2][:3]) <= 1e-12 * (1 + scale)).all()
    for a, b in zip(got, want[3:]):
        assert (np.abs(a.cpu().numpy() - b) <= 2.02 * U * np.abs(b) + 1e-30).all()
    return loss, rewards, stats, got


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "squared"])
@pytest.mark.parametrize("n", [1, 2, 31, 512, 513, 4096, 4099, 20001])
def test_preference_against_64_bits(n, kind):
    pc, pr, rc, rr, lc, lr = preference_inputs(n, seed=n)
    for e in (0.0, 0.1, 0.5, 1.0):
        check_preference((pc, pr, rc, rr), dict(kind=kind, label_smoothing=e, beta=0.1))
        check_preference((pc, pr), dict(kind=kind, label_smoothing=e, beta=2.0, chosen_length=lc, rejected_length=lr))
        check_preference((pc, pr, rc, rr), dict(kind=kind, label_smoothing=e, beta=2.0, chosen_length=lc, rejected_length=lr))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "squared"])
def test_preference_invalid_pairs_and_extreme_margins(kind):
    pc, pr, rc, rr, lc, lr = preference_inputs(64, seed=3)
    pc[3], pr[5], rc[7], rr[9], pc[11] = NEG_INF, NAN, float("inf"), NAN, NAN
    pr[11] = NEG_INF
    pc[20], pc[21], pr[22] = 1e30, -3e38, -1e4
    if kind == "squared":      # whose loss leaves 32 bits at such margins
        pc[20], pc[21] = 1e4, -1e4
    check_preference((pc, pr, rc, rr), dict(kind=kind, label_smoothing=0.1))
    check_preference((pc, pr, rc, rr), dict(kind=kind, beta=-1.0))
    dat.last_status(DEV)
    lc[0], lr[1], lc[2] = 0, -3, -(2 ** 62)
    check_preference((pc, pr, rc, rr), dict(kind=kind, chosen_length=lc, rejected_length=lr))
    assert dat.last_status(DEV) & 1
    pc[:] = NEG_INF
    loss, rewards, stats, grads = check_preference((pc, pr), dict(kind=kind))
    assert float(loss) == 0 and stats.tolist() == [0, 0, 0, 0, 64, 64] and not grads[0].any() and not grads[1].any()


@pytest.mark.gpu
def test_preference_empty_strided_and_one_sided():
    e = torch.zeros(0, device=DEV)
    loss, rewards, stats = dat.dag_preference_loss(e.requires_grad_(), e.detach())
    assert float(loss) == 0 and rewards.shape == (2, 0) and not stats.any()
    assert torch.autograd.grad(loss, e)[0].shape == (0,)
    pc, pr, rc, rr, lc, lr = preference_inputs(40, seed=5)
    both = torch.stack([pc, pr], 1).requires_grad_()      # interleaved, as one batch of pairs gives them
    want = check_preference((pc, pr, rc, rr), dict(chosen_length=lc, rejected_length=lr))
    refs, lens = torch.stack([rc, rr], 1), torch.stack([lc, lr], 1)
    loss, rewards, stats = dat.dag_preference_loss(both[:, 0], both[:, 1], refs[:, 0], refs[:, 1],
                                                   chosen_length=lens[:, 0], rejected_length=lens[:, 1])
    assert torch.equal(loss, want[0]) and torch.equal(rewards, want[1])
    g, = torch.autograd.grad(loss, both)
    assert torch.equal(g[:, 0], want[3][0]) and torch.equal(g[:, 1], want[3][1])
    leaf = pr.clone().requires_grad_()
    loss, _, _ = dat.dag_preference_loss(pc, leaf, rc, rr, chosen_length=lc, rejected_length=lr)
    assert torch.equal(torch.autograd.grad(loss, leaf)[0], want[3][1])
    same = pc.clone().requires_grad_()                    # the same sentence twice
    loss, _, stats = dat.dag_preference_loss(same, same)
    assert abs(float(loss) - math.log(2)) <= U and stats[3] == 0
    assert not torch.autograd.grad(loss, same)[0].any()


@pytest.mark.gpu
def test_preference_gradient_against_differences_and_in_graphs():
    pc, pr, rc, rr, lc, lr = preference_inputs(16, seed=6)
    for kind in ("sigmoid", "squared"):
        c = pc.clone().requires_grad_()
        loss = dat.dag_preference_loss(c, pr, rc, rr, kind=kind)[0]
        g, = torch.autograd.grad(loss, c)
        eps = 0.25
        for k in range(0, 16, 5):
            v = []
            for s in (eps, -eps):
                moved = pc.clone()
                moved[k] += s
                v.append(float(dat.dag_preference_loss(moved, pr, rc, rr, kind=kind)[2][0]) / 16)   # the 64-bit sum
            # third derivative below 0.1 beta^3 / 16, and moved - pc is exact to 2^-24 * 600 / eps
            assert abs((v[0] - v[1]) / (2 * eps) - float(g[k])) <= 1e-5 + 3e-4 * abs(float(g[k]))
    stat = [torch.zeros_like(t) for t in (pc, pr)]
    for s in stat:
        s.requires_grad_()

    def step():
        loss, rewards, stats = dat.dag_preference_loss(*stat, rc, rr, chosen_length=lc, rejected_length=lr)
        return (loss.detach(), rewards, stats) + torch.autograd.grad(loss, stat)

    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        stat[0].copy_(pc)
        stat[1].copy_(pr)
    graph.replay()
    got = [t.clone() for t in out]
    for a, b in zip(got, step()):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ GPU: together

@pytest.mark.gpu
def test_training_step_of_links_likelihoods_and_both_losses():
    """Scores and a learned bias -> links -> dag_loss of preferred and rejected sentences -> preference loss, and
    the policy loss of the vertices on a path, whose transitions are entries of the links: one backward into the
    logits, the scores, the gates and the bias, against the same in 64 bits on the CPU."""
    P, L, T, V, H = 3, 26, 6, 60, 4
    K = L - 1
    gen = torch.Generator().manual_seed(21)
    batch = workloads.small_batch(seed=7, B=P, L=L, T=T, V=V, ragged=False)
    logits = batch.logits
    content = torch.randn(P, L, L, H, generator=gen)
    gates = torch.log_softmax(torch.randn(P, L, H, generator=gen), -1)
    table = torch.randn(8, H, generator=gen) * 0.5
    bk = dat.dag_relative_buckets(K, 8, 32)
    targets = [torch.randint(4, V, (P, T), generator=gen) for _ in range(2)]
    ol, tl = torch.full((P,), L), torch.full((P,), T)
    path = torch.stack([torch.cat([torch.zeros(1, dtype=torch.long),
                                   torch.sort(torch.randperm(L - 2, generator=gen)[:T - 2] + 1).values,
                                   torch.tensor([L - 1])]) for _ in range(P)])
    mask = torch.zeros(P, L, dtype=torch.bool).scatter_(1, path, True)
    hop = torch.zeros(P, L, dtype=torch.long).scatter_(1, path[:, :-1], path[:, 1:] - path[:, :-1] - 1)   # band index
    leaves = mask.scatter(1, path[:, -1:], False)             # vertices that a transition leaves
    tokens = torch.randint(0, V, (P, L), generator=gen)
    adv = torch.randn(P, generator=gen)
    refs = -torch.rand(2, P, generator=gen) * 10 - 30
    old = -torch.rand(P, L, generator=gen) - 6.5
    ref_logits = logits + 0.3 * torch.randn(P, L, V, generator=gen)

    # 64 bits
    x, c, g, t = (v.double().requires_grad_() for v in (logits, content, gates, table))
    i = torch.arange(L).view(L, 1)
    j = i + 1 + torch.arange(K).view(1, K)
    ok = j < L
    z = (c[:, i, j.clamp(max=L - 1)] + t[bk])[:, :-1].masked_fill(~ok[:-1].view(1, L - 1, K, 1), NEG_INF)
    z = torch.log_softmax(z, 2)
    band = torch.full((P, L, K), NEG_INF, dtype=torch.float64)
    val = torch.logsumexp((z + g[:, :-1].unsqueeze(2))[ok[:-1].expand(P, L - 1, K)], -1)
    band = band.index_put(torch.nonzero(ok.expand(P, L, K), as_tuple=True), val)
    square = torch.full((P, L, L), NEG_INF, dtype=torch.float64)
    b0, i0, d0 = torch.nonzero(ok.expand(P, L, K), as_tuple=True)
    square = square.index_put((b0, i0, i0 + d0 + 1), val)
    every = torch.log_softmax(x, -1)
    like = []
    for tg in targets:
        match = every.gather(-1, tg.unsqueeze(1).expand(-1, L, -1)).transpose(1, 2)
        like.append(torch_twins.torch_dag_loss(match, square, ol, tl))
    r = [0.1 * (a - ref.double()) for a, ref in zip(like, refs)]
    pref = -torch.nn.functional.logsigmoid(r[0] - r[1]).mean()
    link = torch.where(leaves, band.gather(2, hop.unsqueeze(2)).squeeze(2), torch.zeros(P, L, dtype=torch.float64))
    lp = every.gather(-1, tokens.unsqueeze(-1)).squeeze(-1) + link
    ratio = (lp - old.double()).exp()
    a = adv.double().view(P, 1)
    term = -torch.minimum(ratio * a, ratio.clamp(0.8, 1.2) * a)
    kl = (every.exp() * (every - torch.log_softmax(ref_logits.double(), -1))).sum(-1)
    want_loss = pref + (term + 0.05 * kl)[mask].mean()
    want = torch.autograd.grad(want_loss, (x, c, g, t))

    # the library
    to = lambda v: v.to(DEV)  # noqa: E731
    x, c, g, t = (v.to(DEV).requires_grad_() for v in (logits, content, gates, table))
    links = dat.dag_links_from_heads(c, g, relative_bias=t, relative_buckets=to(bk))
    like = []
    for tg in targets:
        match = dat.dag_match(x.clone(), to(tg))[1]
        like.append(dat.dag_loss(match, links, to(ol), to(tl)))
    pref, _, pstats = dat.dag_preference_loss(like[0], like[1], to(refs[0]), to(refs[1]))
    link = torch.where(to(leaves), links.gather(2, to(hop).unsqueeze(2)).squeeze(2), torch.zeros((), device=DEV))
    pol, _, _, stats = dat.dag_policy_loss(x, to(tokens), to(old), to(adv), mask=to(mask), link_logp=link,
                                           ref_logits=to(ref_logits), kl_coef=0.05)
    loss = pref + pol
    got = torch.autograd.grad(loss, (x, c, g, t))
    assert abs(float(loss.detach()) - float(want_loss.detach())) <= 1e-5 * abs(float(want_loss))
    assert pstats[4] == P and pstats[5] == 0 and int(stats[4]) == int(mask.sum())
    for name, u, v in zip(("logits", "scores", "gates", "bias"), got, want):
        assert_rel(u.cpu().numpy(), v.numpy(), 1e-4, name)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [500, 30000])
@pytest.mark.parametrize("step", [0.004, -0.02, 0.3, -0.45])
def test_estimated_kl_of_small_steps_near_a_far_log_probability(V, step):
    """Equal logits: every exponential is 1 and the sum V, without a rounding, so that the log-probability is -log V and
    all that is left is how the row's numbers are put together.  The logarithm of V's mantissa (below 0.7) may be off by
    two units of its last place, 2^-23, and u is rounded once, 2^-25 of 1: less than 2^-22 that the KL takes times
    e^u - 1; the KL itself is a product of about ten rounded
    factors, each 2^-24 of it, and u enters it twice.  (A log-probability rounded to 32 bits is off by 2^-22 and more.)"""
    logits = torch.full((1, 4, V), 0.75, dtype=torch.bfloat16, device=DEV)
    ref = torch.full((1, 4), -math.log(V) + step, dtype=torch.float32, device=DEV)
    old = torch.full((1, 4), -math.log(V), dtype=torch.float32, device=DEV)
    tokens = torch.tensor([[0, 1, V // 2, V - 1]], device=DEV)
    _, logp, kl, _ = dat.dag_policy_loss(logits, tokens, old, torch.ones(1, 4, device=DEV), ref_logp=ref, kl_coef=0.1)
    u = ref.double() + math.log(V)
    want = torch.expm1(u) - u
    assert ((logp.double() + math.log(V)).abs() <= 2.0 ** -23 + 2.0 ** -24 * math.log(V)).all()
    assert ((kl.double() - want).abs() <= torch.expm1(u).abs() * 2.0 ** -22 + 16 * 2.0 ** -24 * want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 9000])
def test_policy_backward_in_a_graph_of_its_own(V):
    """The forward runs once, its backward is captured alone and replayed with changing gradients of the loss; in
    between the gradient is written over, as an optimiser's zeroing does."""
    x, kw = policy_inputs(2, 20, V, torch.bfloat16, seed=21, link=True, ref="full", mask=0.5)
    up = torch.ones((), device=DEV)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = x.clone().requires_grad_()
        loss = policy_call(leaf, kl_coef=0.1, **kw)[0]
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            grad, = torch.autograd.grad(loss, leaf, up)
    torch.cuda.current_stream().wait_stream(side)
    for scale in (1.0, 4.0, 1.0, 1.0, 0.5):
        up.fill_(scale)
        graph.replay()
        want = run_policy(x, kw, kl_coef=0.1, scale=scale, grad_scale=None)[4]   # the same kernel, in the backward
        assert torch.equal(grad, want), scale
        grad.zero_()


@pytest.mark.gpu
def test_policy_link_gradient_of_masked_vertices_stays_zero():
    x, kw = policy_inputs(2, 20, 300, torch.float32, seed=22, link=True, mask=0.5)
    link = kw.pop("link").clone().requires_grad_()
    loss = policy_call(x, link=link, **kw)[0]
    grad, = torch.autograd.grad(loss, link, torch.full((), math.inf, device=DEV))
    assert (grad[~kw["mask"]] == 0).all()
