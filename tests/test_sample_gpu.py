"""Sampling on the B200 against a plain float64 restatement of its definition.

The kept set and the running masses are computed in float64 from the row's
fp32 scaled logits. A token is right when it is in the kept set and u times
the kept mass lies in its interval of the running mass, within 2e-6 of the
mass: the kernel's weights are fp32 exponentials (2^-22) of fp32 differences
of magnitude below 32 (2^-20), and errors of the terms average out in sums.
Boundaries of top-p are placed in the middle of a token's interval, so that
no rounding can move them; logprob has the same 2e-6, plus fp32 rounding of
values up to 32 (2^-19).
"""
import numpy as np
import pytest
import torch

from tokengate_b200 import _lib, ops

pytestmark = pytest.mark.gpu


def weights(x, t):
    z = (x.astype(np.float32) / np.float32(t)).astype(np.float32)
    return np.exp((z - z.max()).astype(np.float64))


def kept_set(x, t, k, p, m):
    """Indices kept of one row, ascending, and every weight."""
    x = np.where(np.isnan(x), -np.inf, x)
    w = weights(x, t)
    order = np.lexsort((np.arange(len(x)), -x.astype(np.float64)))
    order = order[np.isfinite(x[order])]
    if k > 0:
        order = order[:k]
    if p < 1:
        cum = np.cumsum(w[order])
        order = order[:int((cum < p * cum[-1]).sum()) + 1]
    return np.sort(order[w[order] >= min(m, 1.0)]), w


def check_rows(x, u, t, k, p, m, token, logprob):
    for b in range(len(x)):
        if t[b] <= 0:
            assert token[b] == int(np.argmax(np.where(np.isnan(x[b]), -np.inf, x[b]))) and logprob[b] == 0.0, b
            continue
        keep, w = kept_set(x[b], t[b], k[b], p[b], m[b])
        cum = np.cumsum(w[keep])
        at = np.searchsorted(keep, token[b])
        assert at < len(keep) and keep[at] == token[b], (b, token[b], len(keep))
        goal, slack = u[b] * cum[-1], 2e-6 * cum[-1]
        assert cum[at] - w[token[b]] - slack <= goal <= cum[at] + slack, (b, at, goal, cum[at], w[token[b]])
        assert abs(logprob[b] - np.log(w[token[b]] / cum[-1])) <= 2e-6 + 2 ** -19 * 2, b


def run(cuda, x, u, t, k=None, p=None, m=None):
    B = len(x)
    f = lambda v, dt: None if v is None else torch.as_tensor(np.broadcast_to(v, (B,)).copy(), dtype=dt, device=cuda)  # noqa: E731
    tok, lp = ops.sample_tokens(x.to(cuda), f(u, torch.float32), f(t, torch.float32), top_k=f(k, torch.int32),
                                top_p=f(p, torch.float32), min_p=f(m, torch.float32))
    bc = lambda v, d: np.broadcast_to(d if v is None else v, (B,)).astype(np.float32)  # noqa: E731
    check_rows(x.float().numpy(), bc(u, 0), bc(t, 1), np.broadcast_to(0 if k is None else k, (B,)), bc(p, 1), bc(m, 0),
               tok.cpu().numpy(), lp.cpu().numpy())
    return tok.cpu(), lp.cpu()


def middle_p(x, t, k, n):
    """A top-p whose boundary is the middle of the n-th kept token's interval."""
    keep, w = kept_set(x, t, k, 1.0, 0.0)
    o = keep[np.lexsort((keep, -x[keep].astype(np.float64)))]
    cum = np.cumsum(w[o])
    n = min(n, len(o) - 1)
    return float((cum[n] - 0.5 * w[o[n]]) / cum[-1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,V", [(1, 151936), (3, 1001), (2, 1), (5, 2), (1, 33), (20, 4097), (2, 32000), (70, 9000), (1, 300001)])
def test_no_truncation_and_each_rule(cuda, dtype, B, V):
    g = torch.Generator().manual_seed(V + B)
    x = (torch.randn(B, V, generator=g) * 2.5).to(dtype)
    u = torch.rand(B, generator=g).numpy()
    t = 0.5 + torch.rand(B, generator=g).numpy()
    run(cuda, x, u, t)
    run(cuda, x, u, t, k=np.arange(B) % 60 + 1)
    run(cuda, x, u, t, m=0.07)
    xf = x.float().numpy()
    for n in (0, 3, 200, V // 3):
        run(cuda, x, u, t, p=np.array([middle_p(xf[b], t[b], 0, n) for b in range(B)], dtype=np.float32))
    ks = np.array([5, 40, 1000])[np.arange(B) % 3]
    run(cuda, x, u, t, k=ks, p=np.array([middle_p(xf[b], t[b], ks[b], ks[b] // 2) for b in range(B)], dtype=np.float32), m=0.001)


@pytest.mark.parametrize("spread", [0.0, 1e-4, 0.02, 0.3, 8.0, 300.0])
def test_flat_and_peaked(cuda, spread):
    """All logits equal, all in one bucket, and ranges beyond the buckets."""
    g = torch.Generator().manual_seed(11)
    for dtype in (torch.bfloat16, torch.float32):
        x = (torch.randn(4, 20000, generator=g) * spread - 3.0).to(dtype)
        u = np.array([0.0, 0.25, 0.6, 0.999], dtype=np.float32)
        xf = x.float().numpy()
        run(cuda, x, u, 1.0)
        run(cuda, x, u, 1.0, k=777)
        run(cuda, x, u, 0.7, p=np.array([middle_p(xf[b], 0.7, 0, 9000 if spread < 1 else 5) for b in range(4)], dtype=np.float32))
        run(cuda, x, u, 0.7, k=500, p=np.array([middle_p(xf[b], 0.7, 500, 250) for b in range(4)], dtype=np.float32))


@pytest.mark.parametrize("B,V,spread", [(1, 151936, 0.3), (2, 151936, 0.05), (1, 524288, 1.0), (150, 3000, 0.3), (64, 40000, 0.2)])
def test_long_and_flat_rows(cuda, B, V, spread):
    """Boundary buckets of thousands of logits (lists of a block, of all blocks, none), and the longest row."""
    g = torch.Generator().manual_seed(V + B)
    for dtype in (torch.bfloat16, torch.float32):
        x = (torch.randn(B, V, generator=g) * spread).to(dtype)
        u, xf = torch.rand(B, generator=g).numpy(), x.float().numpy()
        pick = lambda n: np.array([middle_p(xf[b], 1.0, 0, n) for b in range(B)], dtype=np.float32)  # noqa: E731
        run(cuda, x, u, 1.0, p=pick(V // 2))
        run(cuda, x, u, 1.0, k=V // 3)
        if B == 1:
            run(cuda, x, u, 1.0, k=V // 3, p=np.array([middle_p(xf[0], 1.0, V // 3, V // 9)], dtype=np.float32), m=0.2)


@pytest.mark.parametrize("shift", [0.0, 1e-3, -1e-3])
@pytest.mark.parametrize("V", [8191, 65528])
def test_masses_away_from_the_buckets_middles(cuda, V, shift):
    """Levels of equal mass at the edges of the buckets (powers of two), or just beside them: whatever
    guesses a bucket's mass from its count is wrong by the same sign everywhere."""
    levels = int(np.log2(V + 8)) - 3
    x = np.concatenate([np.full(8 << j, -j * np.log(2) + (shift if j else 0.0)) for j in range(levels)])
    rng = np.random.default_rng(5)
    x = torch.tensor(rng.permutation(x)[None], dtype=torch.float32)
    for k in (0, V // 3):
        for n in (3, 8, 100, 1000, 3000, V // 4):
            p = middle_p(x[0].numpy(), 1.0, k, n)
            run(cuda, x.expand(6, -1).contiguous(), rng.random(6), 1.0, k=k, p=p)


@pytest.mark.parametrize("k", [2, 31, 32, 33, 200, 255, 256, 257, 300])
def test_few_logits_at_their_limit(cuda, k):
    """As many logits down to the k-th's bucket as one block orders by counting, one fewer and one more: k
    isolated logits, the others far below."""
    g = torch.Generator().manual_seed(k)
    for V in (5000, 60000):
        x = torch.full((3, V), -40.0) - torch.rand(3, V, generator=g)
        for b in range(3):
            x[b, torch.randperm(V, generator=g)[:k]] = 2 * torch.randn(k, generator=g)
        u = np.array([0.1, 0.5, 0.95], dtype=np.float32)
        xf = x.numpy()
        run(cuda, x, u, 1.0, k=k)
        run(cuda, x, u, 1.0, k=max(k - 1, 2), p=np.array([middle_p(xf[b], 1.0, max(k - 1, 2), k // 2) for b in range(3)], dtype=np.float32))
        run(cuda, x, u, 1.0, k=k + 5, m=0.01)


def test_ties_go_to_the_lowest_index(cuda):
    x = torch.zeros(6, 5000)
    x[:, 100::700] = 2.0                      # 7 ties at the top
    k = np.array([1, 3, 7, 8, 9, 4999])
    for u in (0.0, 0.5, 0.9999):
        tok, _ = run(cuda, x, u, 1.0, k=k)
        assert tok[0] == 100 and tok[1] in (100, 800, 1500)
    # nine kept: the seven and the two lowest of the rest
    tok, _ = run(cuda, x[:1], 0.0, 1.0, k=9)
    assert tok[0] == 0
    # greedy
    tok, lp = run(cuda, x, 0.7, 0.0, k=50, p=0.2)
    assert (tok == 100).all() and (lp == 0).all()


def test_hard_logits(cuda):
    inf, nan = float("inf"), float("nan")
    x = torch.full((9, 1500), -inf)
    x[0, 700] = -5.0                          # one token left
    x[1, 3], x[1, 1499] = 1.0, 1.0
    x[2] = torch.randn(1500)
    x[2, 5] = nan
    x[2, 6] = 30.0
    x[4] = torch.finfo(torch.float32).min     # the type's lowest: finite, so uniform
    x[5, 10] = x[5, 20] = inf                 # infinities share the mass
    x[6, 0], x[6, 1] = 3e38, -3e38
    x[7] = torch.linspace(-200, 0, 1500)      # a far tail
    x[8] = nan
    u = torch.full((9,), 0.75, device=cuda)
    tok, lp = ops.sample_tokens(x.to(cuda), u, 1.0)
    tok, lp = tok.cpu(), lp.cpu()
    assert tok[0] == 700 and lp[0] == 0
    assert tok[1] == 1499 and abs(lp[1] + np.log(2)) < 1e-6
    assert tok[2] == 6
    assert tok[3] == 0 and torch.isnan(lp[3]) and tok[8] == 0 and torch.isnan(lp[8])    # nothing to choose from
    assert tok[4] == 1125 and abs(lp[4] + np.log(1500)) < 1e-5
    assert tok[5] == 20 and abs(lp[5] + np.log(2)) < 1e-6
    assert tok[6] == 0
    for kw in (dict(top_k=100), dict(top_p=0.9), dict(min_p=0.3), dict(top_k=2, top_p=0.99), dict(temperature=1e-30)):
        kw.setdefault("temperature", 1.0)
        tk, l2 = ops.sample_tokens(x.to(cuda), u, **kw)
        tk = tk.cpu()
        assert tk[0] == 700 and tk[2] == 6 and tk[3] == 0 and tk[8] == 0 and tk[6] == 0, kw
        assert torch.isnan(l2.cpu()[[3, 8]]).all()


@pytest.mark.parametrize("B,V", [(1, 1), (1, 301), (3, 1101), (1, 50257), (2, 50258), (1, 9999), (40, 513)])
def test_extreme_temperatures_of_odd_rows(cuda, B, V):
    """Temperatures outside the range in which quotients are products, on rows that do not fill their last four:
    an infinite one and 1e30 make every token alike, 1e-30 leaves the largest, here exactly 0. Tokens are of the row."""
    g = torch.Generator().manual_seed(V)
    u = ((torch.randint(0, V, (B,), generator=g) + 0.5) / V).numpy()
    u[-1] = (V - 0.5) / V                      # the row's last token
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.randn(B, V, generator=g).to(dtype)
        for t in (float("inf"), 1e30):
            tok, lp = run(cuda, x, u, t)
            assert (tok == torch.as_tensor(np.floor(u * V)).long()).all()
            assert (lp + np.log(V)).abs().max() <= 1e-5
            run(cuda, x, u, t, k=V // 2 + 1)
            run(cuda, x, u, t, m=0.5)
            if V > 8:
                xf = x.float().numpy()
                run(cuda, x, u, t, p=np.array([middle_p(xf[b], t, 0, V // 2) for b in range(B)], dtype=np.float32))
        x = -1 - x.abs()
        top = torch.randint(0, V, (B,), generator=g)
        x[torch.arange(B), top] = 0
        for kw in (dict(), dict(k=5), dict(p=0.9), dict(m=0.2)):
            tok, lp = run(cuda, x, u, 1e-30, **kw)
            assert torch.equal(tok, top) and (lp == 0).all(), kw


@pytest.mark.parametrize("t", [6e-7, 5e-8, 2e-8, 1e-8, 3e-9, 1e-12, 7e-15, 1e-17])
def test_small_temperatures_beside_the_lowest_logits(cuda, t):
    """Logits of the type's lowest value have no weight at any temperature, beside one that is larger than the rest."""
    g = torch.Generator().manual_seed(20)
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.randn(3, 2001, generator=g).clamp(max=3.0).to(dtype)
        x[:, ::3] = torch.finfo(dtype).min
        x[1, x[1] > -1] = -1.0
        x[:, 1000] = torch.tensor([8.0, -1e-3, 1e15]).to(dtype)
        for kw in (dict(), dict(k=40), dict(p=0.9), dict(m=0.1)):
            tok, lp = run(cuda, x, np.array([0.0, 0.4, 0.999], dtype=np.float32), t, **kw)
            assert (tok == 1000).all() and (lp == 0).all(), kw


@pytest.mark.parametrize("V", [300, 700, 1000, 1500, 2047, 9000])
def test_boundary_among_the_lowest_logits(cuda, V):
    """A top-k and a top-p that end among logits of the type's lowest value, which an infinite temperature makes
    as likely as the others: by index, behind all the others."""
    g = torch.Generator().manual_seed(V)
    for top in (1.0, 0.99, 0.5000001, 1.5, -0.25):     # keys of any low bits
        x = torch.full((2, V), torch.finfo(torch.float32).min)
        for b in range(2):
            x[b, torch.randperm(V, generator=g)[:V // 3]] = top - torch.rand(V // 3, generator=g)
            x[b, V // 2 + b] = top
        u = np.array([0.3, 0.999], dtype=np.float32)
        run(cuda, x, u, float("inf"), k=V // 2)
        run(cuda, x, u, float("inf"), p=middle_p(x[0].numpy(), float("inf"), 0, V // 2))
        run(cuda, x, u, float("inf"), k=V - 3, p=middle_p(x[0].numpy(), float("inf"), V - 3, V // 2))


def test_edges_of_the_parameters(cuda):
    g = torch.Generator().manual_seed(12)
    x = torch.randn(3, 3000, generator=g) * 2
    top = x.argmax(1)
    for kw in (dict(top_p=0.0), dict(top_p=-1.0), dict(min_p=1.0), dict(min_p=2.0), dict(top_k=1), dict(temperature=-1.0),
               dict(temperature=float("nan"))):
        kw.setdefault("temperature", 1.0)
        tok, lp = ops.sample_tokens(x.to(cuda), torch.full((3,), 0.9, device=cuda), **kw)
        assert torch.equal(tok.cpu(), top) and (lp == 0).all(), kw
    for u in (0.0, -1.0, float("nan")):       # the first kept index; u of 1 the last
        tok, _ = ops.sample_tokens(x.to(cuda), torch.full((3,), u, device=cuda), 1.0, top_k=10)
        assert torch.equal(tok.cpu(), x.topk(10).indices.min(1).values)
    tok, _ = ops.sample_tokens(x.to(cuda), torch.ones(3, device=cuda), 1.0, top_k=10)
    assert torch.equal(tok.cpu(), x.topk(10).indices.max(1).values)
    same = [ops.sample_tokens(x.to(cuda), torch.full((3,), 0.3, device=cuda), 1.0, **kw)[0]
            for kw in (dict(), dict(top_k=0), dict(top_k=-4), dict(top_k=3000), dict(top_k=10 ** 9), dict(top_p=1.0), dict(min_p=0.0))]
    assert all(torch.equal(same[0], s) for s in same)


def test_rows_with_a_stride_and_outputs_given(cuda):
    g = torch.Generator().manual_seed(13)
    big = (torch.randn(4, 2 * 1003, generator=g) * 2).bfloat16().to(cuda)
    x = big[:, 5:1006]                         # rows that start off any vector boundary
    u = torch.rand(4, generator=g).to(cuda)
    token, lp = torch.empty(4, dtype=torch.int64, device=cuda), torch.empty(4, device=cuda)
    a = ops.sample_tokens(x, u, 0.8, top_k=30, token=token, logprob=lp)
    assert a[0] is token and a[1] is lp
    b = ops.sample_tokens(x.contiguous(), u, 0.8, top_k=30)
    assert torch.equal(token, b[0]) and torch.equal(lp, b[1])


def test_frequencies(cuda):
    """4096 draws of one row follow its distribution: chi-square over 20 tokens, far below its 1e-6 quantile."""
    g = torch.Generator().manual_seed(14)
    x = torch.randn(1, 500, generator=g) * 2
    u = torch.rand(4096, generator=g)
    tok, _ = ops.sample_tokens(x.expand(4096, -1).contiguous().to(cuda), u.to(cuda), 1.0, top_k=20)
    keep, w = kept_set(x[0].numpy(), 1.0, 20, 1.0, 0.0)
    want = 4096 * w[keep] / w[keep].sum()
    seen = np.array([(tok.cpu().numpy() == i).sum() for i in keep])
    assert seen.sum() == 4096 and ((seen - want) ** 2 / want).sum() < 70


def test_refusals(cuda):
    x, u = torch.zeros(2, 10, device=cuda), torch.zeros(2, device=cuda)
    for bad in (x.half(), x[0], x.t(), x.cpu()):
        with pytest.raises(ValueError):
            ops.sample_tokens(bad, u)
    with pytest.raises(ValueError):
        ops.sample_tokens(x, None)
    with pytest.raises(ValueError):
        ops.sample_tokens(x, u[:1])
    with pytest.raises(ValueError):
        ops.sample_tokens(x, u, temperature=None)
    with pytest.raises(ValueError):
        ops.sample_tokens(x, u, top_k=torch.zeros(2, device=cuda))          # int32 wanted
    with pytest.raises(ValueError):
        ops.sample_tokens(x, u, token=torch.zeros(2, dtype=torch.int32, device=cuda))
    with pytest.raises(_lib.TokenGateUnsupportedError):
        ops.sample_tokens(torch.zeros(1, (1 << 19) + 1, device=cuda), u[:1])
    assert ops.sample_tokens(x[:0], u[:0])[0].shape == (0,)
