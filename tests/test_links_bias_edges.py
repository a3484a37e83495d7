"""Biased links (``dag_links_from_heads(..., relative_bias=...)``) at the edges of their definition: vertices with one
successor, gates of any size, values that are no numbers, and sizes that leave the shared memory.

Every test runs the three forms of the kernels: a warp per vertex (the ordinary sizes), a CTA per vertex (here by a table
of more than 2048 numbers) and the kernels of the links without a bias (here by more than 32 heads, or by such a table
and a head count that is no multiple of four)."""
import numpy as np
import pytest
import torch

import da_transformer_b200 as dat
from test_links_bias import make, oracle
from util import assert_rel

DEV = "cuda:0"
NEG_INF = float("-inf")
NAN = float("nan")
U = 2.0 ** -24          # half a step of fp32 relative to the value

# heads, buckets of the table: a warp per vertex (exact and filled-up groups of heads), a CTA per vertex, the others
FORMS = [(1, 8), (2, 8), (4, 8), (5, 8), (6, 8), (8, 8), (12, 8), (16, 8), (32, 8), (4, 600), (8, 300), (16, 200), (32, 100),
         (1, 600), (5, 300), (12, 200), (40, 8), (128, 8)]


def run(content, gates, table, bk, K, grad, **mask):
    """links and the gradients of scores, gates and table, on the CPU in 64 bits."""
    leaves = [t.detach().clone().requires_grad_() for t in (content, gates, table)]
    links = dat.dag_links_from_heads(leaves[0], leaves[1], max_transition_length=K, relative_bias=leaves[2],
                                     relative_buckets=bk, **mask)
    grads = torch.autograd.grad(links, leaves, grad)
    return [t.detach().double().cpu().numpy() for t in (links, *grads)]


def some_buckets(K, n, seed=1):
    return torch.randint(0, n, (K,), generator=torch.Generator().manual_seed(seed)).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0.0, 50.0, 1000.0])
@pytest.mark.parametrize("H,buckets", FORMS)
def test_one_successor(H, buckets, offset):
    """A softmax over one element is 1 whatever the score: the gradient of the scores and of the table is 0, the link the
    log-sum-exp of the gates, and with one head whose gate is 0 the link is 0.

    The log-sum-exp: each exponential is off by 2^-22 of itself, their sum by 2^-24 in each of its log2(H) + 2 steps
    (2^-20 for all at most), its logarithm by 2^-22, the result by half a step."""
    B, L = 3, 20
    content, gates, table, grad, _, _ = make(B, L, H, L - 1, buckets=buckets, seed=H)
    if H == 1:
        gates.zero_()
    content += offset
    ar = torch.arange(L, device=DEV)
    last = (ar == L - 1).expand(B, L)                                   # all vertices reach the last one alone
    two = ar.view(1, L) < torch.tensor([2, 1, L], device=DEV).view(B, 1)   # graphs of two, one and L vertices
    cases = [(1, {}), (1, dict(nonpad_mask=two)), (L - 1, dict(bound_end=(ar + 1).expand(B, L).contiguous())),
             (L - 1, dict(nonpad_mask=last)), (3, dict(nonpad_mask=last))]
    if H <= 8:
        cases.append((1, dict(bound_end=(ar + 1).expand(B, L).contiguous())))
    for K, mask in cases:
        bk, g = some_buckets(K, buckets), grad[..., :K].contiguous()
        links, gc, gg, gt = run(content, gates, table, bk, K, g, **mask)
        fin = np.isfinite(links)
        assert fin.sum(2).max() == 1 and fin.any()
        assert not gc.any() and not gt.any(), (K, list(mask), np.abs(gc).max(), np.abs(gt).max())
        want = torch.logsumexp(gates.double(), -1).cpu().numpy()[..., None] * np.ones_like(links)
        assert (np.abs(links - want)[fin] <= (0 if H == 1 else 2.0 ** -20 + U * np.abs(want[fin]))).all()
        assert (links[~fin] == NEG_INF).all()
        share = torch.softmax(gates.double(), -1).cpu().numpy()
        at = np.where(fin, g.double().cpu().numpy(), 0).sum(2)[..., None]
        assert (np.abs(gg - at * share) <= 2.0 ** -19 * np.abs(at)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H,buckets", [(1, 8), (6, 8), (8, 8), (8, 300), (5, 300), (40, 8)])
def test_last_but_one_vertex_of_a_training_graph(H, buckets):
    """Padded graphs: the last but one vertex of each has a single successor, scores near 1000."""
    B, L = 4, 30
    content, gates, table, grad, _, nonpad = make(B, L, H, L - 1, buckets=buckets, seed=2)
    _, gc, _, _ = run(content + 1000, gates, table, some_buckets(L - 1, buckets), L - 1, grad, nonpad_mask=nonpad)
    for b, n in enumerate(nonpad.sum(1).tolist()):
        assert not gc[b, n - 2].any() and gc[b, n - 3].any()


def against_64_bits(content, gates, table, bk, K, grad, size, links_off=0.0, **mask):
    """size: the largest number that scores, gates and links are put together from; each is rounded a few times in 32
    bits, which a probability carries as a factor."""
    got = run(content, gates, table, bk, K, grad, **mask)
    want = oracle(content, gates, table, bk, K, grad=grad, **mask)
    fin = np.isfinite(want[0])
    assert np.array_equal(got[0][~fin], want[0][~fin])
    tol = 8 * U * size + 2e-6
    assert np.abs(got[0][fin] - want[0][fin]).max() <= tol + links_off
    rows = content.shape[0] * content.shape[1]
    for name, a, b, terms in zip(("scores", "gates", "table"), got[1:], want[1:], (1, rows ** 0.5, rows)):
        off = np.abs(a - b).max()
        assert off <= 4 * tol * float(grad.abs().max()) * terms + 1e-4 * np.abs(b).max(), (name, off)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("H,buckets", FORMS)
@pytest.mark.parametrize("kind", ["all", "one", "far"])
def test_gates_above_zero(H, buckets, kind):
    """log_gates may be any numbers: +100 for all heads of a vertex, for one of them, +3000 and -3000."""
    B, L = 2, 24
    content, gates, table, grad, _, nonpad = make(B, L, H, L - 1, buckets=buckets, seed=H + 1)
    if kind == "all":
        gates[:, ::2] += 100
    elif kind == "one":
        gates[:, ::2, 0] = 100
        gates[:, 1::2, -1] = 100
    else:
        gates[:, ::2, 0] = 3000
        gates[:, 1::3] = -3000
    got = against_64_bits(content, gates, table, some_buckets(L - 1, buckets), L - 1, grad, float(gates.abs().max()) + 10,
                          nonpad_mask=nonpad)
    assert np.isfinite(got[1]).all() and np.isfinite(got[2]).all() and np.isfinite(got[3]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H,buckets", [f for f in FORMS if f[0] >= 2])
@pytest.mark.parametrize("gap,gate,other", [(55, -45, -70), (58, -48, -54), (59, -35, -60), (50, -50, -69), (59, -66, -90)])
def test_rare_head_far_above_its_nearest_score(H, buckets, gap, gate, other):
    """A head that is rarely taken, whose score of one successor is far above the nearest successor's, while the other
    heads all but exclude that successor: the rare head's share is nearly all of the link."""
    B, L = 2, 9
    content, gates, table, grad, _, _ = make(B, L, H, L - 1, buckets=buckets, seed=H + 2)
    gates = torch.log_softmax(gates, -1)
    content *= 0.1
    table *= 0.1
    gates[:, :, H // 2] = gate
    far = 4                                         # successor 5 of the vertices before it
    content[:, :far, far + 1] += other
    content[:, :far, far + 1, H // 2] += gap - other
    got = against_64_bits(content, gates, table, some_buckets(L - 1, buckets), L - 1, grad, 100.0)
    assert (np.abs(got[0][:, 0, far] - gate) < 3).all() or other > gate - 4


@pytest.mark.gpu
@pytest.mark.parametrize("H,buckets", FORMS)
@pytest.mark.parametrize("value", [NAN, float("inf")])
def test_valid_scores_that_are_no_numbers_show(H, buckets, value):
    """A score of NaN or +inf at a valid successor makes the softmax of its head NaN, and with it every link of the vertex;
    nothing of another vertex changes.  A sentence with holes, one without a mask, one with a single vertex left."""
    B, L = 3, 33
    content, gates, table, grad, _, _ = make(B, L, H, L - 1, buckets=buckets, seed=H + 3)
    nonpad = torch.rand(B, L, generator=torch.Generator().manual_seed(5)).to(DEV) < 0.6
    nonpad[1] = True
    nonpad[0, 1], nonpad[0, 3], nonpad[0, 9], nonpad[0, 12], nonpad[0, 20] = True, False, False, True, True
    bk = some_buckets(L - 1, buckets)
    bad = ((0, 2, 12, 0), (0, 5, 20, H - 1), (1, 0, 1, H // 2), (1, 7, L - 1, 0))
    clean = run(content, gates, table, bk, L - 1, grad, nonpad_mask=nonpad)
    for at in bad:
        content[at] = value
    content[0, 2, 3], content[0, 5, 9] = NAN, value                        # masked ones, of no account
    links, gc, gg, gt = run(content, gates, table, bk, L - 1, grad, nonpad_mask=nonpad)
    hit = np.zeros((B, L), bool)
    for b, i, _, _ in bad:
        hit[b, i] = True
    ok = np.isfinite(clean[0])
    assert np.isnan(links[hit][ok[hit]]).all() and (links[hit][~ok[hit]] == NEG_INF).all()
    assert np.array_equal(links[~hit], clean[0][~hit])
    dense = np.zeros((B, L, L), bool)
    b, i, d = np.nonzero(ok)
    dense[b, i, i + d + 1] = True
    assert np.isnan(gc[hit][dense[hit]]).all() and not gc[hit][~dense[hit]].any()
    assert np.array_equal(gc[~hit], clean[1][~hit]) and np.array_equal(gg[~hit], clean[2][~hit])
    assert np.isnan(gg[hit]).all()
    reached = np.unique(bk.cpu().numpy()[(ok & hit[..., None]).any((0, 1))])
    assert np.isnan(gt[reached]).all()
    others = np.setdiff1d(np.arange(buckets), reached)
    assert np.array_equal(gt[others], clean[3][others])


@pytest.mark.gpu
@pytest.mark.parametrize("H,buckets", FORMS)
def test_distances_without_a_bucket_may_hold_anything(H, buckets):
    """The scores of a distance whose bucket lies outside the table are as good as masked."""
    B, L = 2, 40
    content, gates, table, grad, _, nonpad = make(B, L, H, L - 1, buckets=buckets, seed=H + 4)
    bk = some_buckets(L - 1, buckets)
    bk[0], bk[5], bk[17] = -1, buckets, 2 ** 40
    content[1, 2, 5, H // 2], content[0, 8, 10, 0] = NAN, NAN              # valid ones: these vertices are NaN where they reach
    want = run(content, gates, table, bk, L - 1, grad, nonpad_mask=nonpad)
    assert (want[0][:, :, [0, 5, 17]] == NEG_INF).all()
    for b, i in ((1, 2), (0, 8)):
        ok = want[0][b, i] != NEG_INF
        assert np.isnan(want[0][b, i][ok]).all() and np.isnan(want[1][b, i, i + 1:][ok[:L - 1 - i]]).all()
        assert not want[1][b, i, i + 1:][~ok[:L - 1 - i]].any()
    d = torch.arange(L, device=DEV).view(1, L) - torch.arange(L, device=DEV).view(L, 1) - 1
    out = (d == 0) | (d == 5) | (d == 17)
    for value in (NAN, float("inf"), NEG_INF, torch.finfo(torch.float32).max):
        dirty = torch.where(out.view(1, L, L, 1), torch.full((), value, device=DEV), content)
        g = torch.where(torch.from_numpy(want[0] != NEG_INF).to(DEV), grad, torch.full((), value, device=DEV))
        for a, b in zip(run(dirty, gates, table, bk, L - 1, g, nonpad_mask=nonpad), want):
            assert np.array_equal(a, b, equal_nan=True), value
    dat.last_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("H,buckets", FORMS)
def test_bias_of_minus_infinity(H, buckets):
    """A bias of -inf is a score of -inf (a head without a finite score takes no part, for which the definition has no number),
    and a score that is no number stays none beside it."""
    B, L = 2, 26
    content, gates, table, grad, _, nonpad = make(B, L, H, L - 1, buckets=buckets, seed=H + 5)
    bk = some_buckets(L - 1, buckets)
    table[int(bk[3])] = NEG_INF
    table[int(bk[7]), H // 2] = NEG_INF
    links, gc, gg, gt = run(content, gates, table, bk, L - 1, grad, nonpad_mask=nonpad)
    # in 64 bits, in the probability domain
    c, g, t = (x.double().cpu() for x in (content, gates, table))
    i = torch.arange(L).view(L, 1)
    j = i + 1 + torch.arange(L - 1).view(1, L - 1)
    ok = (j < L) & nonpad.cpu()[:, j.clamp(max=L - 1)]
    e = (c[:, i, j.clamp(max=L - 1)] + t[bk.cpu()]).exp() * ok.unsqueeze(-1)
    tot = e.sum(2, keepdim=True)
    soft = e / torch.where(tot > 0, tot, torch.ones_like(tot))
    w = soft * g.exp().unsqueeze(2)
    p = w.sum(3, keepdim=True)
    gp = grad.double().cpu().unsqueeze(-1) * w / torch.where(p > 0, p, torch.ones_like(p))
    S = gp.sum(2)
    dc = gp - soft * S.unsqueeze(2)
    assert_rel(links, p.squeeze(3).log().numpy(), 1e-5, "links")
    dense = torch.zeros(B, L, 2 * L, H, dtype=torch.float64)
    dense[:, i, j] = dc
    assert_rel(gc, dense[:, :, :L].numpy(), 1e-4, "gradient of content")
    assert_rel(gg, S.numpy(), 1e-4, "gradient of gates")
    dt = torch.zeros(t.shape, dtype=torch.float64).index_add_(0, bk.cpu(), dc.sum((0, 1)))
    assert_rel(gt, dt.numpy(), 1e-4, "gradient of table")
    content[0, 2, 2 + 1 + 3, 0] = NAN
    links = run(content, gates, table, bk, L - 1, grad, nonpad_mask=nonpad)[0]
    assert np.isnan(links[0, 2, :L - 3]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H", [6, 8])
def test_spans_of_the_call_before_are_not_seen(H):
    """The kernel that reads the sentences' spans begins while the one that writes them may still run, into memory that held
    the spans of the call before: calls with masks in turn, none waited for."""
    B, L = 40, 48
    content, gates, table, grad, _, _ = make(B, L, H, L - 1, seed=5)
    bk = some_buckets(L - 1, 8)
    gen = torch.Generator().manual_seed(6)
    masks = [(torch.rand(B, L, generator=gen) < p).to(DEV) for p in (0.1, 0.5, 0.9, 2.0)]
    masks.append(torch.zeros(B, L, dtype=torch.bool, device=DEV))
    call = lambda m: dat.dag_links_from_heads(content, gates, nonpad_mask=m, relative_bias=table, relative_buckets=bk)  # noqa: E731
    want = []
    for m in masks:
        torch.cuda.synchronize()
        want.append(call(m))
        torch.cuda.synchronize()
    leaves = [t.detach().clone().requires_grad_() for t in (content, gates, table)]
    first = None
    for n in range(60):
        m = n % len(masks)
        assert torch.equal(call(masks[m]), want[m])
        links = dat.dag_links_from_heads(leaves[0], leaves[1], nonpad_mask=masks[1], relative_bias=leaves[2], relative_buckets=bk)
        got = torch.autograd.grad(links, leaves, grad)
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,H,K", [(1, 448, 128, 447), (1, 460, 128, 459), (1, 900, 100, 40), (1, 470, 127, 469)])
def test_rows_beside_the_shared_memory(B, L, H, K):
    """Rows that fit the forward's shared memory and not the backward's, rows that fit neither, and long graphs whose band is
    short."""
    content, gates, table, grad, bk, nonpad = make(B, L, H, K, seed=H)
    against_64_bits(content, gates, table, bk, K, grad, 16.0, nonpad_mask=nonpad)


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,H,K", [(1, 448, 127, 447), (1, 470, 127, 469), (1, 900, 101, 40)])
def test_rows_beside_the_shared_memory_without_a_bias(B, L, H, K):
    content, gates, table, grad, bk, nonpad = make(B, L, H, K, seed=H)
    leaves = [t.detach().clone().requires_grad_() for t in (content, gates)]
    links = dat.dag_links_from_heads(*leaves, nonpad_mask=nonpad, max_transition_length=K)
    got = torch.autograd.grad(links, leaves, torch.where(links.isfinite(), grad, 0))
    want = oracle(content, gates, torch.zeros_like(table), bk, K, nonpad_mask=nonpad, grad=grad)
    fin = np.isfinite(want[0])
    a = links.detach().cpu().numpy()
    assert np.array_equal(a[~fin], want[0][~fin]) and np.abs(a[fin] - want[0][fin]).max() <= 1e-5 * np.abs(want[0][fin]).max()
    for u, v in zip(got, want[1:3]):
        assert np.abs(u.cpu().numpy() - v).max() <= 1e-4 * np.abs(v).max()


@pytest.mark.gpu
def test_a_bias_wherever_the_links_work_without_one():
    """2048 vertices and 32 heads, every transition: the links without a bias of the scores with the bias added."""
    B, L, H, K = 1, 2048, 32, 2047
    gen = torch.Generator(device=DEV).manual_seed(4)
    content = torch.randn(B, L, L, H, generator=gen, device=DEV)
    gates = torch.log_softmax(torch.randn(B, L, H, generator=gen, device=DEV), -1)
    table = torch.randn(16, H, generator=gen, device=DEV) * 0.5
    grad = torch.randn(B, L, K, generator=gen, device=DEV)
    bk = dat.dag_relative_buckets(K, 16, 512, device=DEV)
    leaves = [t.detach().clone().requires_grad_() for t in (content, gates, table)]
    links = dat.dag_links_from_heads(leaves[0], leaves[1], relative_bias=leaves[2], relative_buckets=bk)
    got = torch.autograd.grad(links, leaves, grad)
    i = torch.arange(L, device=DEV)
    d = (i.view(1, L) - i.view(L, 1) - 1).clamp(0, K - 1)
    both = content.clone()
    for n in range(0, L, 64):
        both[0, n:n + 64] += table[bk[d[n:n + 64]]]
    plain = [both.requires_grad_(), gates.clone().requires_grad_()]
    other = dat.dag_links_from_heads(*plain)
    want = torch.autograd.grad(other, plain, grad)
    fin = other.isfinite()
    assert torch.equal(links.isfinite(), fin)
    assert float((links - other)[fin].detach().abs().max()) <= 1e-5 * float(other[fin].detach().abs().max())
    for a, b in zip(got, want):
        assert float((a - b).abs().max()) <= 1e-4 * float(b.abs().max())
    by = torch.stack([torch.diagonal(want[0][0], d + 1, 0, 1).double().sum(-1) for d in range(K)])
    dt = torch.zeros(16, H, dtype=torch.float64, device=DEV).index_add_(0, bk, by)
    assert float((got[2] - dt).abs().max()) <= 1e-4 * float(dt.abs().max())


@pytest.mark.gpu
def test_workspace_has_no_more_bands_than_ctas_that_run_at_once():
    """Partial sums of the table's gradient: a band for each CTA.  At most two to an SM with a warp per vertex; a CTA per
    vertex keeps three rows of scores in shared memory (227 KB); none for head counts that neither takes."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    size = dat._native.lib().dat_links_bias_workspace_bytes
    for B, L, H, K in ((64, 512, 8, 511), (8, 1024, 16, 1023), (16, 1024, 8, 256), (64, 300, 3, 299), (4, 440, 128, 439), (4, 100, 40, 99)):
        band, sums = 4 * K * H, 8 * K * H
        bands = 0 if H > 32 else 2 * sms
        if H in (4, 8, 16, 32):
            bands = max(bands, sms * min(16, 232448 // (3 * band)))
        assert sums <= size(B, L, H, K) <= sums + bands * band + 64, (B, L, H, K)


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,H,K", [(2, 400, 8, 380), (2, 400, 8, 383), (2, 400, 8, 386), (3, 360, 8, 340), (2, 640, 4, 630),
                                     (2, 200, 16, 195)])
def test_rows_that_all_but_fill_their_ring(B, L, H, K):
    """A ring with no room for the next row beside the longest: its copy begins when the row before has been worked off."""
    content, gates, table, grad, bk, nonpad = make(B, L, H, K, buckets=32, seed=K)
    against_64_bits(content, gates, table, bk, K, grad, 16.0, nonpad_mask=nonpad)
