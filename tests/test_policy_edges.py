"""``dag_policy_loss`` at the edges of its numerics, against plain torch in 64 bits, row by row."""
import math

import numpy as np
import pytest
import torch

from test_policy_preference import policy_call, policy_inputs, policy_oracle, row_tolerance, run_policy

DEV = "cuda:0"
U = 2.0 ** -24          # half a step of fp32 relative to the value
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def kl_in_64_bits(x, y):
    """The KL of softmax(x) to softmax(y) as a sum of terms that are not negative: sum p (e^-u - 1 + u) with u = log p - log q
    does not cancel."""
    p, q = torch.log_softmax(x.double(), -1), torch.log_softmax(y.double(), -1)
    u = p - q
    return (p.exp() * torch.where(u.abs() < 1e-2, u * u * (0.5 - u / 6 + u * u / 24 - u ** 3 / 120), torch.expm1(-u) + u)).sum(-1)


def check_kl(x, y, kw, V, name):
    """Each term of the sum is off by as much as its probability (row_tolerance, with an exponent below 16) and by a few
    roundings of its own, and none is negative: the KL is off by that part of itself."""
    loss, logp, kl, stats = policy_call(x, kl_coef=0.1, **{**kw, "ref_logits": y})
    want = kl_in_64_bits(x, y)
    off = (kl.double() - want).abs()
    assert (off <= 2 * row_tolerance(V) * want).all(), (name, float((off / want.clamp(min=1e-300)).max()), float(want.min()))
    assert abs(float(stats[1]) - float(want.sum())) <= 2 * row_tolerance(V) * float(want.sum())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,V", [(1, 3, 1000), (2, 100, 1500), (1, 2, 9001), (2, 250, 5003), (1, 3, 32000), (1, 160, 30001),
                                   (1, 1, 128000)])
def test_kl_of_a_reference_close_to_the_policy(B, L, V, dtype):
    """Where training with a reference model starts: logits that differ by a thousandth to a tenth, by a constant beside,
    or not at all."""
    x, kw = policy_inputs(B, L, V, dtype, seed=V)
    noise = torch.randn(B, L, V, generator=torch.Generator().manual_seed(3)).to(DEV)
    for size in (1e-3, 1e-2, 1e-1, 0.3, 1.0):
        check_kl(x, (x.float() + size * noise).to(dtype), kw, V, size)
    if dtype == torch.float32:
        check_kl(x, x + 0.01 * noise + 2, kw, V, "constant")
    same = policy_call(x, kl_coef=0.1, **{**kw, "ref_logits": x.clone()})
    assert not same[2].any() and float(same[3][1]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("V", [2, 3, 50, 9001])
def test_kl_is_not_negative(V):
    """One token carries all but nothing of the row: KLs of 1e-25 to 1, below what the sums resolve."""
    x, kw = policy_inputs(1, 3000 if V < 100 else 300, V, torch.float32, seed=V + 9)
    x = x.scatter_add(-1, kw["tokens"].unsqueeze(-1), torch.full_like(kw["old"], 25.0).unsqueeze(-1))
    size = 10.0 ** torch.linspace(-5, 0.5, x.shape[1], device=DEV).view(1, -1, 1)
    y = x + size * torch.randn(x.shape, generator=torch.Generator().manual_seed(13)).to(DEV)
    kl = policy_call(x, kl_coef=0.1, **{**kw, "ref_logits": y})[2]
    want = kl_in_64_bits(x, y)
    assert (kl >= 0).all()
    # The KL lies with the other tokens, whose exponents reach 25 log2 e = 36: the exponential of one is off by 2 U, by U of its
    # argument in the difference and by U of it in the product, U (2 + 2 * 36) in all.  A term e e^-u - e + e u carries that
    # (e^-u + 1) / phi(u) times, below 6 for |u| >= 1 (5.2 at -1); the sums add as in row_tolerance.  A KL of 1/16 and more is
    # a difference of log-sum-exps and of the mean of d, of row_tolerance each.  64-bit sums near 1 leave 1e-15.
    d = float((x - y).abs().max())
    bound = U * (V / 256 + 16 + 6 * 74) * want + torch.where(want >= 0.06, row_tolerance(V) * (2 + d), 0)
    assert ((kl.double() - want).abs() <= bound + 1e-15).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1000, 9001, 30001, 100000])
def test_kl_of_models_that_differ_at_the_token(V, dtype):
    """The token's own logit far from the reference's, at tokens of any probability, and all others close."""
    x, kw = policy_inputs(1, 8, V, dtype, seed=V + 1)
    tok = kw["tokens"].unsqueeze(-1)
    noise = torch.randn(1, 8, V, generator=torch.Generator().manual_seed(4)).to(DEV)
    y = (x.float() + 0.05 * noise).to(dtype)
    up = torch.tensor([3.0, -3.0, 0.5, -0.5, 6.0, -6.0, 1.0, 0.1], device=DEV).view(1, 8, 1)
    y = y.scatter(-1, tok, (x.float().gather(-1, tok) + up).to(dtype))
    check_kl(x, y, kw, V, "token")


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1000, 9001, 30001])
def test_gradient_of_a_reference_close_to_the_policy(V):
    """The gradient of the KL alone (no advantage): p (d - E d)."""
    x, kw = policy_inputs(1, 6, V, torch.float32, seed=V + 2)
    kw["adv"].zero_()
    kw["ref_logits"] = x + 0.01 * torch.randn(1, 6, V, generator=torch.Generator().manual_seed(5)).to(DEV)
    got, want = run_policy(x, kw, kl_coef=1.0)[4].double().cpu().numpy(), policy_oracle(x, kl_coef=1.0, **kw)[4]
    # d is a difference of logits below 16, rounded there, and d - E d is about 0.03 at most
    for a, b in zip(got[0], want[0]):
        assert np.abs(a - b).max() <= 1e-3 * np.abs(b).max()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [700, 9001, 40000])
@pytest.mark.parametrize("ref", [False, True])
def test_small_gradients_of_unlikely_tokens(V, ref):
    """A token whose log-probability is -41 to -69 (in the reference model too) and a coefficient of 1e-13: the gradient of
    the likely logits is c p, whatever the sums are taken relative to."""
    x, kw = policy_inputs(1, 8, V, torch.float32, seed=V + 3)
    tok = kw["tokens"].unsqueeze(-1)
    low = x.amax(-1, keepdim=True) - torch.tensor([30., 41., 43., 50., 60., 66., 68., 75.], device=DEV).view(1, 8, 1)
    x = x.scatter(-1, tok, low)
    if ref:
        kw["ref_logits"] = x * 0.95 + 0.1 * torch.randn(1, 8, V, generator=torch.Generator().manual_seed(6)).to(DEV)
    kw["old"] = (torch.log_softmax(x.double(), -1).gather(-1, tok).squeeze(-1) - 0.05).float()
    kw["adv"] = torch.full_like(kw["adv"], 1e-13)
    coef = 1e-13 if ref else 0.0
    got, want = run_policy(x, kw, kl_coef=coef)[4].double().cpu().numpy(), policy_oracle(x, kl_coef=coef, **kw)[4]
    # log-probabilities near -70 are rounded by 2^-24 of them twice, the ratio with them
    for a, b in zip(got[0], want[0]):
        assert np.abs(a - b).max() <= (1e-4 + 300 * U) * np.abs(b).max()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [700, 9001, 40000])
@pytest.mark.parametrize("ref", [False, True])
def test_logits_far_apart_row_by_row(V, ref):
    """The token's logit 60 to 200 below the largest, which no sum relative to it holds in 32 bits: each row against bounds
    of its own numbers, far below its own gradient."""
    rows = [0.0, 60.0, 80.0, 100.0, 150.0, 200.0]
    x, kw = policy_inputs(1, len(rows), V, torch.float32, seed=V + 4)
    tok = kw["tokens"].unsqueeze(-1)
    top = (tok + 1) % V
    x = x.scatter_add(-1, top, torch.tensor(rows, device=DEV).view(1, -1, 1))
    if ref:
        kw["ref_logits"] = x * 0.9 + 0.5 * torch.randn(1, len(rows), V, generator=torch.Generator().manual_seed(7)).to(DEV)
    every = torch.log_softmax(x.double(), -1)
    kw["old"] = (every.gather(-1, tok).squeeze(-1) - 0.05).float()
    kw["adv"] = torch.linspace(0.5, 2, len(rows), device=DEV).view(1, -1)
    beta = 0.1 if ref else 0.0
    got = run_policy(x, kw, kl_coef=beta)
    want = policy_oracle(x, kl_coef=beta, **kw)
    p = every.exp()[0].cpu().numpy()
    d = (x.double() - kw["ref_logits"].double())[0].cpu().numpy() if ref else np.zeros_like(p)
    tol = row_tolerance(V)
    for n in range(len(rows)):
        lp, kl, g = float(got[1][0, n]), float(got[2][0, n]), got[4][0, n].double().cpu().numpy()
        wlp, wkl, wg = want[1][0, n], want[2][0, n], want[4][0, n]
        near = p[n] > 1e-12                                   # the logits that carry the row
        reach = np.abs(d[n] - d[n][near].mean())[near].max()   # how far their d are apart
        far = np.abs(d[n]).max()                              # what d is rounded at
        assert abs(lp - wlp) <= tol + 3 * U * abs(wlp)
        if ref:
            bound = 2 * tol * (1 + reach) + 4 * U * far
            assert abs(kl - wkl) <= bound
            assert bound < 0.05 * want[2].max()
        # the ratio is off by as much as the log-probability; the coefficient is below 2 of 1/N, p off by the exponent's part
        ratio = 2 * (tol + 4 * U * (abs(wlp) + abs(float(kw["old"][0, n]))))
        bound = (ratio + 2 * tol + beta * (2 * tol * (1 + reach) + 4 * U * far)) / len(rows)
        assert bound < 0.05 * np.abs(wg).max()
        assert np.abs(g - wg).max() <= bound, (n, np.abs(g - wg).max(), bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1001, 9001, 40000])
def test_close_reference_with_forbidden_tokens(V, dtype):
    """Tokens that both models forbid, and tokens that the policy alone forbids, to which the reference gives little: the KL
    counts what the reference has there."""
    x, kw = policy_inputs(2, 6, V, dtype, seed=V + 5)
    y = (x.float() + 0.05 * torch.randn(2, 6, V, generator=torch.Generator().manual_seed(8)).to(DEV)).to(dtype)
    gen = torch.Generator().manual_seed(9)
    ban = (torch.rand(V, generator=gen) < 0.2).to(DEV)
    ban[kw["tokens"].unique()] = False
    for alone in (False, True):
        xx, yy = x.clone(), y.clone()
        xx[..., ban] = float("-inf")
        yy[..., ban] = float("-inf")
        if alone:
            some = ban.nonzero()[:40, 0]
            yy[1][..., some] = y[1][..., some] - 9
        kw["old"] = (torch.log_softmax(xx.double(), -1).gather(-1, kw["tokens"].unsqueeze(-1)).squeeze(-1) - 0.1).float()
        loss, _, kl, stats = policy_call(xx, kl_coef=0.1, **{**kw, "ref_logits": yy})
        p, q = torch.log_softmax(xx.double(), -1), torch.log_softmax(yy.double(), -1)
        u = torch.where(p > float("-inf"), p - q, 0)
        # sum p (e^-u - 1 + u), plus what the reference has where the policy has nothing
        want = (p.exp() * torch.where(u.abs() < 1e-2, u * u * (0.5 - u / 6 + u * u / 24 - u ** 3 / 120), torch.expm1(-u) + u)).sum(-1)
        want += torch.where(p > float("-inf"), 0, q.exp()).sum(-1)
        assert float(want.max()) < 0.05 and float(want.min()) > 1e-4
        assert ((kl.double() - want).abs() <= 2 * row_tolerance(V) * want).all(), float(((kl.double() - want).abs() / want).max())


@pytest.mark.gpu
@pytest.mark.parametrize("V", [900, 9001])
def test_sums_and_loss_take_the_close_rows_as_they_are_returned(V):
    """Some rows close, some not, some masked: the loss and the sums are those of the returned KL; twice the same bits."""
    B, L = 3, 70
    x, kw = policy_inputs(B, L, V, torch.float32, seed=V + 6, link=True, mask=0.6)
    noise = torch.randn(B, L, V, generator=torch.Generator().manual_seed(10)).to(DEV)
    size = 10.0 ** torch.linspace(-4, 0, L, device=DEV).view(1, L, 1)
    kw["ref_logits"] = x + size * noise
    got = run_policy(x, kw, kl_coef=0.7)
    again = run_policy(x, kw, kl_coef=0.7)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    loss, _, kl, stats = got[:4]
    n = int(kw["mask"].sum())
    want = kl_in_64_bits(x, kw["ref_logits"])
    on = kw["mask"]
    assert ((kl.double() - want)[on].abs() <= 2 * row_tolerance(V) * want[on]).all() and not kl[~on].any()
    # the sum is of 64-bit numbers that are returned rounded once
    assert abs(float(stats[1]) - float(kl.double().sum())) <= 1.01 * U * float(kl.double().sum())
    total = (float(stats[0]) + 0.7 * float(stats[1])) / n
    assert abs(float(loss) - total) <= 2 * U * abs(total) + 1e-9 * 0.7
    assert int(stats[4]) == n


@pytest.mark.gpu
def test_close_rows_of_a_long_batch():
    """More rows than the CTAs look at together (256 each): they come back for the rest, with close ones among them."""
    B, L, V = 2, 110000, 4100
    gen = torch.Generator(device=DEV).manual_seed(11)
    x = torch.randn(B, L, V, generator=gen, device=DEV, dtype=torch.bfloat16).mul_(2)
    y = torch.randn(B, L, V, generator=gen, device=DEV, dtype=torch.bfloat16).mul_(0.05).add_(x)
    far = torch.arange(L, device=DEV) % 3 == 1
    for b in range(B):
        y[b, far] *= 0.5
    tokens = torch.randint(0, V, (B, L), generator=gen, device=DEV)
    zero = torch.zeros(B, L, device=DEV)
    mask = torch.rand(B, L, generator=gen, device=DEV) < 0.8
    with torch.no_grad():
        loss, logp, kl, stats = policy_call(x, tokens, zero - 8, zero + 1, mask=mask, ref_logits=y, kl_coef=0.1)
    assert not kl[~mask].any()
    at = torch.cat([torch.arange(0, L, 997, device=DEV), torch.arange(L - 50, L, device=DEV)])
    for b in range(B):
        want = kl_in_64_bits(x[b, at], y[b, at])
        on = mask[b, at]
        assert ((kl[b, at].double() - want)[on].abs() <= 2 * row_tolerance(V) * want[on]).all()
    assert abs(float(stats[1]) - float(kl.double().sum())) <= 1.01 * U * float(kl.double().sum())


@pytest.mark.gpu
@pytest.mark.parametrize("V", [500, 20000])
def test_close_rows_on_streams_and_in_graphs(V):
    x, kw = policy_inputs(2, 40, V, torch.bfloat16, seed=14, link=True, mask=0.5)
    kw["ref_logits"] = (x.float() + 0.05 * torch.randn(2, 40, V, generator=torch.Generator().manual_seed(12)).to(DEV)).to(x.dtype)
    want = run_policy(x, kw, kl_coef=0.1)
    stat = {n: t.clone() for n, t in kw.items()}
    xs = torch.zeros_like(x).requires_grad_()
    stat["link"].requires_grad_()

    def step():
        loss, logp, kl, st = policy_call(xs, kl_coef=0.1, **stat)
        return (loss.detach(), logp, kl, st) + torch.autograd.grad(loss, (xs, stat["link"]))

    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        for a, b in zip(run_policy(x, kw, kl_coef=0.1), want):
            assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
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
