"""Band links with a learned relative position bias (``dag_links_from_heads(..., relative_bias=...)``).

The oracle is plain torch in 64 bits, sentence by sentence over the band, differentiated by autograd.
Tolerances are those the library states for fp32 results: values 1e-5 and gradients 1e-4 of the largest.  A
gradient is a difference G (p - soft) of two probabilities, each of which carries the rounding of an exponent
below 16 in 32 bits and of the exponential, 32 * 2^-24 = 2e-6: where a vertex has one successor the two are
equal, and what is left of the difference is at most 4e-6 of G (summed over the vertices in the table's).  A
link is the logarithm of such a probability, off by 2e-6 by itself where the vertex has one successor (link 0)."""
import numpy as np
import pytest
import torch

import da_transformer_b200 as dat
from util import assert_rel

DEV = "cuda:0"
NEG_INF = float("-inf")


def assert_links(got, want):
    got = got.detach().cpu().numpy()
    fin = np.isfinite(want)
    assert np.array_equal(got[~fin], want[~fin])
    if fin.any():
        assert np.abs(got[fin] - want[fin]).max() <= 1e-5 * np.abs(want[fin]).max() + 2e-6


def assert_grads(got, want, grad):
    top = float(grad.abs().max())
    rows = want[1].shape[0] * want[1].shape[1]
    for name, a, b, terms in zip(("content", "gates", "table"), got, want, (1, 1, rows if grad.shape[2] == 1 else rows ** 0.5)):
        off = np.abs(a.cpu().numpy() - b).max()
        assert off <= 1e-4 * np.abs(b).max() + 4e-6 * top * terms, f"gradient of {name}: {off}"


def oracle(content, gates, table, buckets, K, nonpad_mask=None, bound_end=None, grad=None):
    """links [B,L,K] and, with grad, the gradients of content, gates and table, in 64 bits."""
    content, gates, table = (t.detach().double().cpu().requires_grad_() for t in (content, gates, table))
    buckets = buckets.cpu()[:K]
    B, L, _, _ = content.shape
    i = torch.arange(L).view(L, 1)
    j = i + 1 + torch.arange(K).view(1, K)
    inside = (j < L) & ((buckets >= 0) & (buckets < table.shape[0])).view(1, K)
    j = j.clamp(max=L - 1)
    out = []
    for b in range(B):
        ok = inside.clone()
        if nonpad_mask is not None:
            ok &= nonpad_mask.cpu()[b].bool()[j]
        if bound_end is not None:
            ok &= j <= bound_end.cpu()[b].view(L, 1)
        z = content[b][i, j] + table[buckets.clamp(0, table.shape[0] - 1)]
        alive = ok.any(1)
        full = torch.full((L, K), NEG_INF, dtype=torch.float64)
        if alive.any():
            z = torch.log_softmax(z[alive].masked_fill(~ok[alive].unsqueeze(-1), NEG_INF), 1) + gates[b][alive].unsqueeze(1)
            full = full.index_put(torch.nonzero(ok, as_tuple=True), torch.logsumexp(z[ok[alive]], -1))
        out.append(full)
    links = torch.stack(out)
    if grad is None:
        return links.detach().numpy()
    g = torch.where(links.detach().isfinite(), grad.double().cpu(), 0)
    fin = links.isfinite()
    value = (links[fin] * g[fin]).sum()
    grads = (torch.autograd.grad(value, (content, gates, table), allow_unused=True) if value.requires_grad
             else (None, None, None))
    grads = [torch.zeros_like(t) if x is None else x for x, t in zip(grads, (content, gates, table))]
    return (links.detach().numpy(), *(x.numpy() for x in grads))


def make(B, L, H, K, buckets=8, seed=0, device=DEV):
    gen = torch.Generator().manual_seed(seed)
    content = torch.randn(B, L, L, H, generator=gen) * 1.5
    gates = torch.log_softmax(torch.randn(B, L, H, generator=gen), -1)
    table = torch.randn(buckets, H, generator=gen) * 0.7
    grad = torch.randn(B, L, K, generator=gen)
    bk = dat.dag_relative_buckets(K, buckets, max_distance=max(16, buckets))
    n = torch.tensor([max(1, L - (b * L) // B) for b in range(B)])
    nonpad = torch.arange(L).view(1, L) < n.view(B, 1)
    return [t.to(device) for t in (content, gates, table, grad, bk, nonpad)]


def check(content, gates, table, grad, bk, K, **mask):
    leaves = [t.detach().clone().requires_grad_() for t in (content, gates, table)]
    links = dat.dag_links_from_heads(leaves[0], leaves[1], max_transition_length=K, relative_bias=leaves[2],
                                     relative_buckets=bk, **mask)
    got = torch.autograd.grad(links, leaves, grad)
    want = oracle(content, gates, table, bk, K, grad=grad, **mask)
    assert_links(links, want[0])
    assert_grads(got, want[1:], grad)
    with torch.no_grad():   # the same values without a gradient
        again = dat.dag_links_from_heads(content, gates, max_transition_length=K, relative_bias=table,
                                         relative_buckets=bk, **mask)
    assert torch.equal(again, links.detach())
    return links, got


# ------------------------------------------------------------------------------------------------ CPU

def test_relative_buckets():
    b = dat.dag_relative_buckets(200, 32, 128)
    assert b.dtype == torch.long and b[:16].tolist() == list(range(16))
    assert (b[1:] >= b[:-1]).all() and int(b.max()) == 31 and int(b[-1]) == 31
    # bucket 16 + k begins at 16 * 8 ** (k / 16): whole powers of two are borders
    assert int(b[32]) == 16 + 16 // 3 and int(b[127]) == 31
    assert dat.dag_relative_buckets(64, 4, 32).tolist()[:9] == [0, 1, 2, 2, 2, 2, 2, 2, 3]   # 8 = 2 * 16 ** (1/2)
    assert dat.dag_relative_buckets(5, 1, 8).tolist() == [0] * 5
    for bad in ((0, 4, 8), (5, 0, 8), (5, 8, 4)):
        with pytest.raises(RuntimeError):
            dat.dag_relative_buckets(*bad)


def test_refusals_come_before_any_device_work():
    content, gates, table, _, bk, nonpad = make(2, 6, 3, 5, device="cpu")

    def call(c=content, g=gates, t=table, k=bk, **kw):
        return dat.dag_links_from_heads(c, g, relative_bias=t, relative_buckets=k, **kw)

    for kw, text in ((dict(t=None), "together"), (dict(k=None), "together"), (dict(c=content[:, :5]), "prelen, prelen"),
                     (dict(g=gates[..., :2]), "log_gates"), (dict(t=table[:, :2]), "num_buckets"),
                     (dict(t=table[:0]), "num_buckets"), (dict(t=table.half()), "float32"),
                     (dict(c=content.double()), "float32"), (dict(k=bk[:4]), "at least 5"),
                     (dict(k=bk.int()), "long"), (dict(nonpad_mask=nonpad[:, :5]), "nonpad_mask"),
                     (dict(bound_end=torch.zeros(2, 6)), "bound_end"), (dict(max_transition_length=0), "at least 1"),
                     (dict(c=content[:, :1, :1], g=gates[:, :1]), "at least 2")):
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="GPU"):
            call()


# ------------------------------------------------------------------------------------------------ GPU

SHAPES = [(2, 400, 8, 399), (1, 514, 8, 512), (1, 513, 8, 512), (1, 1026, 4, 1025), (1, 1025, 4, 1024), (3, 140, 32, 128),
          (2, 131, 32, 130), (7, 4, 4, 3), (150, 5, 8, 4), (9, 61, 16, 60), (1, 2, 1, 1), (2, 5, 8, 4), (3, 33, 8, 32), (2, 64, 4, 63), (2, 70, 16, 20), (1, 40, 32, 39), (3, 37, 6, 36),
          (2, 50, 3, 7), (1, 129, 12, 128), (2, 300, 8, 299), (1, 520, 4, 519), (1, 600, 16, 450), (2, 30, 128, 29),
          (5, 18, 2, 1), (1, 9, 5, 8), (1, 260, 32, 259), (1, 1100, 4, 1099),
          (3, 71, 1, 70), (1, 700, 1, 699), (1, 1100, 2, 1030), (1, 400, 3, 390), (2, 90, 7, 89), (1, 512, 12, 511),
          (1, 300, 10, 257), (2, 40, 20, 39), (1, 150, 29, 149), (1, 410, 16, 390), (1, 1030, 6, 1029), (2, 9, 31, 2),
          (1, 140, 24, 130), (1, 300, 18, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,H,K", SHAPES)
def test_against_64_bits_with_padding(B, L, H, K):
    content, gates, table, grad, bk, nonpad = make(B, L, H, K, seed=L + H)
    check(content, gates, table, grad, bk, K, nonpad_mask=nonpad)


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,H,K", [(2, 33, 8, 32), (3, 37, 6, 12), (1, 2, 4, 1)])
def test_against_64_bits_without_mask_and_with_bound(B, L, H, K):
    content, gates, table, grad, bk, _ = make(B, L, H, K, seed=5)
    check(content, gates, table, grad, bk, K)
    gen = torch.Generator().manual_seed(1)
    bound = torch.randint(-1, L + 3, (B, L), generator=gen).to(DEV)   # also past the graph and before the vertex
    check(content, gates, table, grad, bk, K, bound_end=bound)


@pytest.mark.gpu
@pytest.mark.parametrize("H,L,K", [(8, 90, 89), (4, 200, 60), (16, 65, 64), (3, 40, 39), (8, 700, 699), (12, 90, 89), (5, 50, 30)])
def test_masks_with_holes(H, L, K):
    """Padding inside a sentence and before it, a sentence without a vertex, one with a single one."""
    B = 6
    content, gates, table, grad, bk, _ = make(B, L, H, K, seed=H * L)
    gen = torch.Generator().manual_seed(7)
    mask = torch.rand(B, L, generator=gen) < 0.6
    mask[1, :L // 2] = False
    mask[2] = False
    mask[3] = False
    mask[3, L - 2] = True
    mask[4] = True
    mask[4, 1] = False            # the nearest successor of vertex 0 alone
    for form in (mask.to(DEV), mask.to(DEV).to(torch.uint8) * 5):
        check(content, gates, table, grad, bk, K, nonpad_mask=form)


@pytest.mark.gpu
@pytest.mark.parametrize("H,L", [(8, 50), (6, 50), (16, 40), (8, 600), (12, 40), (3, 300)])
@pytest.mark.parametrize("scale", [30.0, 200.0])
def test_scores_far_apart(H, L, scale):
    """Scores hundreds apart: the nearest successor's is far below the largest, and links reach -1000, which 32-bit
    probabilities do not.  Against the log-domain oracle; the values are rounded where scores and bias are added
    (2^-24 of the score) and where the exponent is taken apart, a few 2^-24 of 1500."""
    K = L - 1
    content, gates, table, grad, bk, nonpad = make(2, L, H, K, seed=3)
    content = content * scale
    leaves = [t.detach().clone().requires_grad_() for t in (content, gates, table)]
    links = dat.dag_links_from_heads(leaves[0], leaves[1], nonpad_mask=nonpad, relative_bias=leaves[2], relative_buckets=bk)
    got = torch.autograd.grad(links, leaves, grad)
    want = oracle(content, gates, table, bk, K, nonpad_mask=nonpad, grad=grad)
    fin = np.isfinite(want[0])
    a = links.detach().cpu().numpy()
    assert np.array_equal(np.isfinite(a), fin)
    top = float(content.abs().max()) * 1.5
    assert np.abs(a[fin] - want[0][fin]).max() <= 8 * 2.0 ** -24 * top + 2e-6
    # a probability off by as much as its logarithm
    for name, u, v in zip(("content", "gates"), got, want[1:3]):
        assert np.abs(u.cpu().numpy() - v).max() <= 3 * 8 * 2.0 ** -24 * top * float(grad.abs().max()) + 4e-6, name


@pytest.mark.gpu
@pytest.mark.parametrize("H,L", [(8, 60), (4, 33), (16, 50), (5, 40), (8, 640)])
def test_gates_far_apart(H, L):
    """Heads that a vertex all but never takes (gates of -70 to -300) are the only ones to reach some successors: there
    their share is 1 however small their probability, and what they lose through the softmax is as large."""
    K = L - 1
    content, gates, table, grad, bk, nonpad = make(2, L, H, K, seed=L)
    gates[:, ::2, 1] = -70
    gates[:, ::3, 2] = -300
    content[:, :, 3::4] -= 500                  # no head reaches these ...
    content[:, :, 3::4, 1:3] += 500             # ... but the rare ones
    leaves = [t.detach().clone().requires_grad_() for t in (content, gates, table)]
    links = dat.dag_links_from_heads(leaves[0], leaves[1], nonpad_mask=nonpad, relative_bias=leaves[2], relative_buckets=bk)
    got = torch.autograd.grad(links, leaves, grad)
    want = oracle(content, gates, table, bk, K, nonpad_mask=nonpad, grad=grad)
    fin = np.isfinite(want[0])
    a = links.detach().cpu().numpy()
    # a score of 500 is rounded by 2^-24 of it, a few times over
    assert np.abs(a[fin] - want[0][fin]).max() <= 8 * 2.0 ** -24 * 800
    for name, u, v in zip(("content", "gates"), got, want[1:3]):
        top = np.abs(v).max()
        assert np.abs(u.cpu().numpy() - v).max() <= 3 * 8 * 2.0 ** -24 * 800 * max(top, float(grad.abs().max())), name


@pytest.mark.gpu
def test_large_tables_take_the_other_kernels():
    """A table that does not fit beside the rows (more than 2048 numbers)."""
    content, gates, table, grad, _, nonpad = make(2, 40, 8, 39, buckets=300, seed=5)
    gen = torch.Generator().manual_seed(3)
    bk = torch.randint(0, 300, (39,), generator=gen).to(DEV)
    check(content, gates, table, grad, bk, 39, nonpad_mask=nonpad)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [37, 38, 39])
def test_band_gradient_on_any_address(K):
    """The band's gradient is copied in 16-byte pieces: rows that start anywhere, and a tensor that does."""
    content, gates, table, grad, bk, nonpad = make(5, 40, 8, K, seed=K)
    want = check(content, gates, table, grad, bk, K, nonpad_mask=nonpad)[1]
    for shift in (1, 2, 3):
        moved = torch.empty(grad.numel() + shift, device=DEV)[shift:].view(grad.shape).copy_(grad)
        leaves = [t.detach().clone().requires_grad_() for t in (content, gates, table)]
        links = dat.dag_links_from_heads(leaves[0], leaves[1], nonpad_mask=nonpad, max_transition_length=K,
                                         relative_bias=leaves[2], relative_buckets=bk)
        for a, b in zip(torch.autograd.grad(links, leaves, moved), want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("H", [8, 6])
def test_masked_places_may_hold_anything(H):
    B, L, K = 2, 40, 39
    content, gates, table, grad, bk, nonpad = make(B, L, H, K, seed=9)
    ok = nonpad.view(B, 1, L) & (torch.arange(L, device=DEV).view(1, L, 1) < torch.arange(L, device=DEV).view(1, 1, L))
    want = check(content, gates, table, grad, bk, K, nonpad_mask=nonpad)
    for value in (float("nan"), float("inf"), NEG_INF, torch.finfo(torch.float32).min):
        dirty = torch.where(ok.unsqueeze(-1), content, torch.tensor(value, device=DEV))
        # the band's places behind the last vertex of a short sentence hold anything in the gradient too
        g = torch.where(want[0].isfinite(), grad, torch.tensor(value, device=DEV))
        leaves = [t.detach().clone().requires_grad_() for t in (dirty, gates, table)]
        links = dat.dag_links_from_heads(leaves[0], leaves[1], nonpad_mask=nonpad, relative_bias=leaves[2], relative_buckets=bk)
        assert torch.equal(links, want[0])
        for a, b in zip(torch.autograd.grad(links, leaves, g), want[1]):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_scores_of_minus_infinity_take_no_part():
    B, L, H, K = 2, 24, 8, 23
    content, gates, table, grad, bk, _ = make(B, L, H, K, seed=11)
    content[0, 3, 5] = NEG_INF             # one transition of all heads
    content[0, 4, :, 2] = NEG_INF          # one head of a vertex
    content[1, 7] = NEG_INF                # a vertex without successors
    gates[1, 9, 0] = NEG_INF               # a head that a vertex never takes
    leaves = [t.detach().clone().requires_grad_() for t in (content, gates, table)]
    links = dat.dag_links_from_heads(leaves[0], leaves[1], relative_bias=leaves[2], relative_buckets=bk)
    got = torch.autograd.grad(links, leaves, grad)
    # the same in 64 bits, in the probability domain
    c, g, t = (x.double().cpu() for x in (content, gates, table))
    i = torch.arange(L).view(L, 1)
    j = i + 1 + torch.arange(K).view(1, K)
    e = (c[:, i, j.clamp(max=L - 1)] + t[bk.cpu()]).exp() * (j < L).view(1, L, K, 1)
    tot = e.sum(2, keepdim=True)
    soft = e / torch.where(tot > 0, tot, torch.ones_like(tot))
    w = soft * g.exp().unsqueeze(2)
    p = w.sum(3, keepdim=True)
    share = w / torch.where(p > 0, p, torch.ones_like(p))
    gp = grad.double().cpu().unsqueeze(-1) * share
    S = gp.sum(2)
    dc = gp - soft * S.unsqueeze(2)
    assert_rel(links.detach().cpu().numpy(), p.squeeze(3).log().numpy(), 1e-5, "links")
    dense = torch.zeros(B, L, L + K, H, dtype=torch.float64)
    dense[:, i, j] = dc
    assert_rel(got[0].cpu().numpy(), dense[:, :, :L].numpy(), 1e-4, "gradient of content")
    assert_rel(got[1].cpu().numpy(), S.numpy(), 1e-4, "gradient of gates")
    dt = torch.zeros(t.shape, dtype=torch.float64).index_add_(0, bk.cpu(), dc.sum((0, 1)))
    assert_rel(got[2].cpu().numpy(), dt.numpy(), 1e-4, "gradient of table")


@pytest.mark.gpu
@pytest.mark.parametrize("H", [4, 5])
def test_buckets_outside_the_table_forbid_their_distances(H):
    content, gates, table, grad, bk, nonpad = make(2, 20, H, 19, seed=3)
    bk[4], bk[11] = -1, table.shape[0]
    dat.last_status(DEV)
    check(content, gates, table, grad, bk, 19, nonpad_mask=nonpad)
    assert dat.last_status(DEV) & 4
    bk[4], bk[11] = 0, 1
    check(content, gates, table, grad, bk, 19, nonpad_mask=nonpad)
    assert not dat.last_status(DEV) & 4


@pytest.mark.gpu
def test_buckets_in_any_order_and_a_longer_map():
    content, gates, table, grad, _, nonpad = make(2, 30, 8, 29, seed=4)
    gen = torch.Generator().manual_seed(2)
    bk = torch.randint(0, table.shape[0], (80,), generator=gen).to(DEV)
    check(content, gates, table, grad, bk, 29, nonpad_mask=nonpad)
    check(content, gates, table, grad[..., :10].contiguous(), bk[::2], 10, nonpad_mask=nonpad)   # a strided map


@pytest.mark.gpu
def test_strided_and_misaligned_inputs():
    B, L, H, K = 2, 26, 8, 25
    content, gates, table, grad, bk, nonpad = make(B, L, H, K, seed=6)
    want = check(content, gates, table, grad, bk, K, nonpad_mask=nonpad)

    def off(t):   # the same values one element behind a 16-byte boundary
        u = torch.empty(t.numel() + 1, device=DEV, dtype=t.dtype)[1:].view(t.shape)
        return u.copy_(t)

    for c, g, t in ((off(content), off(gates), off(table)), (content, gates, off(table)),
                    (content.permute(3, 1, 2, 0).contiguous().permute(3, 1, 2, 0), gates, table)):
        leaves = [x.requires_grad_() for x in (c, g, t)]
        links = dat.dag_links_from_heads(leaves[0], leaves[1], nonpad_mask=nonpad.to(torch.uint8) * 3,
                                         relative_bias=leaves[2], relative_buckets=bk)
        assert_rel(links.detach().cpu().numpy(), want[0].detach().cpu().numpy(), 1e-5, "links")
        for a, b in zip(torch.autograd.grad(links, leaves, off(grad)), want[1]):
            assert_rel(a.cpu().numpy(), b.cpu().numpy(), 1e-4, "gradient")


@pytest.mark.gpu
def test_zero_table_gives_the_links_without_a_bias():
    content, gates, table, _, bk, nonpad = make(3, 45, 8, 44, seed=8)
    got = dat.dag_links_from_heads(content, gates, nonpad_mask=nonpad, relative_bias=torch.zeros_like(table), relative_buckets=bk)
    plain = dat.dag_links_from_heads(content, gates, nonpad_mask=nonpad)
    assert_rel(got.cpu().numpy(), plain.cpu().numpy(), 1e-5, "links")


@pytest.mark.gpu
def test_gradients_against_differences():
    B, L, H, K = 1, 14, 4, 13
    content, gates, table, grad, bk, nonpad = make(B, L, H, K, seed=12)
    fin = dat.dag_links_from_heads(content, gates, relative_bias=table, relative_buckets=bk).isfinite()

    def value(c, g, t):
        links = dat.dag_links_from_heads(c, g, relative_bias=t, relative_buckets=bk)
        return float((links[fin].double() * grad[fin].double()).sum())

    leaves = [t.detach().clone().requires_grad_() for t in (content, gates, table)]
    links = dat.dag_links_from_heads(leaves[0], leaves[1], relative_bias=leaves[2], relative_buckets=bk)
    got = torch.autograd.grad(links, leaves, torch.where(fin, grad, torch.zeros_like(grad)))
    gen = torch.Generator().manual_seed(3)
    eps = 2e-2
    for k in range(3):
        step = torch.randn(leaves[k].shape, generator=gen).to(DEV)
        step = step / step.norm()
        up, down = ([x + s * eps * step if n == k else x for n, x in enumerate((content, gates, table))] for s in (1, -1))
        slope = (value(*up) - value(*down)) / (2 * eps)
        # 91 links of magnitude < 16 with 1e-6 each, over 2 eps: < 5e-3; the third derivative's eps^2/6 is below that
        assert abs(slope - float((got[k].double() * step.double()).sum())) < 1e-2


@pytest.mark.gpu
def test_repeats_bit_for_bit_on_streams_and_in_graphs():
    content, gates, table, grad, bk, nonpad = make(4, 120, 8, 119, seed=13)

    def step(c, g, t, gr):
        links = dat.dag_links_from_heads(c, g, nonpad_mask=nonpad, relative_bias=t, relative_buckets=bk)
        return (links.detach(),) + torch.autograd.grad(links, (c, g, t), gr)

    leaves = [t.detach().clone().requires_grad_() for t in (content, gates, table)]
    want = step(*leaves, grad)
    for a, b in zip(want, step(*leaves, grad)):
        assert torch.equal(a, b)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [t.detach().clone().requires_grad_() for t in (content, gates, table)]
        got = step(*other, grad)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    # captured with leaves of its own, replayed on new values
    stat = [torch.zeros_like(t).requires_grad_() for t in (content, gates, table)]
    with torch.cuda.stream(side):
        step(*stat, grad)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*stat, grad)
    with torch.no_grad():
        for s, t in zip(stat, (content, gates, table)):
            s.copy_(t)
    graph.replay()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_only_what_needs_a_gradient_and_an_empty_batch():
    content, gates, table, grad, bk, nonpad = make(2, 16, 8, 15, seed=14)
    want = check(content, gates, table, grad, bk, 15, nonpad_mask=nonpad)[1]
    for k in range(3):
        leaves = [t.detach().clone().requires_grad_(n == k) for n, t in enumerate((content, gates, table))]
        links = dat.dag_links_from_heads(leaves[0], leaves[1], nonpad_mask=nonpad, relative_bias=leaves[2], relative_buckets=bk)
        (got,) = torch.autograd.grad(links, leaves[k:k + 1], grad)
        assert torch.equal(got, want[k])
    with pytest.raises(RuntimeError, match="once_differentiable|twice|does not require grad"):
        t = table.clone().requires_grad_()
        links = dat.dag_links_from_heads(content, gates, relative_bias=t, relative_buckets=bk)
        (g,) = torch.autograd.grad(links[:, 0].sum(), t, create_graph=True)
        g.sum().backward()
    t = table.clone().requires_grad_()
    links = dat.dag_links_from_heads(content[:0], gates[:0], relative_bias=t, relative_buckets=bk)
    assert links.shape == (0, 16, 15)
    (g,) = torch.autograd.grad(links.sum(), t)
    assert torch.equal(g, torch.zeros_like(t))


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 scores: the last sentence must be found and written."""
    B, L, H, K = 65, 1024, 32, 100
    content = torch.zeros(B, L, L, H, device=DEV)
    gates = torch.full((B, L, H), -float(np.log(H)), device=DEV)
    small = make(1, L, H, K, buckets=16, seed=15)
    content[-1], gates[-1] = small[0][0], small[1][0]
    table, bk = small[2].requires_grad_(), small[4]
    content.requires_grad_()
    links = dat.dag_links_from_heads(content, gates, max_transition_length=K, relative_bias=table, relative_buckets=bk)
    grad = torch.zeros(B, L, K, device=DEV)
    grad[-1] = small[3][0]
    gc, gt = torch.autograd.grad(links, (content, table), grad)
    assert not gc[:-1].any()
    want = oracle(small[0], small[1], small[2], bk, K, grad=small[3])
    assert_rel(links[-1:].detach().cpu().numpy(), want[0], 1e-5, "links")
    assert_rel(gc[-1:].cpu().numpy(), want[1], 1e-4, "gradient of content")
    assert_rel(gt.cpu().numpy(), want[3], 1e-4, "gradient of table")
