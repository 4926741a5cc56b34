"""Token log probabilities on the device (nst_token_logprobs_fwd / _bwd) against float64 (oracle/kernel_emulation.py).

Tolerances, u = 2^-24.  The sums S and T run over V terms spread over at least 256 partial sums, so their rounding is below (V / 256 + 16) u
of the sum of magnitudes; a term exp(x - m) carries the rounding of its exponent, at most 3 u |x - m| <= 3 u (|x| + |m|), weighted by the term
itself, and 4 u of the function.  Hence
    |lse err|     <= u (V / 256 + 40 + 3 (H + 8) + 2 |lse| + |m|)          (sum |d| e^d / S is at most the entropy plus log S)
    |logp err|    <= that + u (|x| + |lse| + |logp|)
    |entropy err| <= u (V / 256 + 48) (2 + 3 H + 2 log V)
The gradient p (a + b (log p + H)): log p is off by u (|x| + |lse|) and two roundings, so p by that relative; bf16 adds 2^-8 of the value.
"""
import math

import pytest
import torch

from oracle import kernel_emulation as E

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


@pytest.fixture(scope="module")
def K():
    from neurst_amd import kernels
    return kernels


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make_logits(rows, V, dtype, kind, seed=0):
    g = gen(seed)
    x = torch.randn(rows, V, generator=g) * 2.5
    if kind == "ties":            # a handful of different values: almost every alternative ties with many others
        x = torch.randint(-3, 4, (rows, V), generator=g).float()
    elif kind == "equal":
        x = torch.full((rows, V), 0.5)
    elif kind == "few":           # all but three symbols ruled out by the lowest value
        x = torch.full((rows, V), -1e9)
        for r in range(rows):
            x[r, torch.randperm(V, generator=g)[:3]] = torch.randn(min(3, V), generator=g)[:3]
    elif kind == "inf":           # half of the symbols ruled out by minus infinity
        x[torch.rand(rows, V, generator=g) < 0.5] = -math.inf
        x[:, V // 2] = 1.0
    elif kind == "sorted":        # all the large values in one place
        x = x.sort(dim=-1, descending=True).values
    elif kind == "peaked":
        x[:, V // 3] = 80.0
    elif kind == "signed zero":
        x = torch.where(torch.rand(rows, V, generator=g) < 0.5, torch.tensor(0.0), torch.tensor(-0.0))
    return x.to(dtype)


def assert_forward(K, x, tokens, top_n, xd=None):
    rows, V = x.shape
    want = E.token_logprobs(x.double(), tokens, top_n)
    got = K.token_logprobs(x.to(DEV) if xd is None else xd, tokens.to(DEV), top_n)
    x64 = x.double()
    lse64 = torch.logsumexp(x64, -1)
    lp = x64 - lse64[:, None]
    p = lp.exp()
    H = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    m = x64.amax(-1).abs()
    t_lse = U * (V / 256 + 40 + 3 * (H + 8) + 2 * lse64.abs() + m)
    logp, entropy, lse, top_logp, top_ids = (t.cpu() for t in got)
    assert ((lse.double() - lse64).abs() <= t_lse).all(), float(((lse.double() - lse64).abs() / t_lse).max())
    assert ((entropy.double() - H).abs() <= U * (V / 256 + 48) * (2 + 3 * H + 2 * math.log(V))).all()
    given = (tokens >= 0) & (tokens < V)
    xt = x64.gather(1, tokens.clamp(0, V - 1)[:, None])[:, 0]
    lt = torch.where(given, xt - lse64, torch.zeros_like(xt))
    assert (logp[~given] == 0).all()
    fin = given & torch.isfinite(xt)
    assert torch.equal(logp[given & ~torch.isfinite(xt)].double(), lt[given & ~torch.isfinite(xt)])
    assert ((logp.double() - lt).abs()[fin] <= (t_lse + U * (xt.abs() + lse64.abs() + lt.abs()))[fin]).all()
    assert top_ids.dtype == torch.int64 and torch.equal(top_ids, want[4])
    if top_n:
        tv = x64.gather(1, top_ids)
        ok = torch.isfinite(tv)
        tl = tv - lse64[:, None]
        assert torch.equal(top_logp[~ok].double(), tl[~ok])
        assert ((top_logp.double() - tl).abs()[ok] <= (t_lse[:, None] + U * (tv.abs() + lse64.abs()[:, None] + tl.abs()))[ok]).all()
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (2, 63), (5, 255), (4, 256), (7, 1000), (3, 2049), (128, 8008), (2, 32001), (1, 70000),
                                    (3, 130000), (300, 511)])
def test_forward_over_sizes(K, rows, V, dtype):
    x = make_logits(rows, V, dtype, "plain", seed=V)
    tokens = torch.randint(0, V, (rows,), generator=gen(1))
    for top_n in (0, 1, 6, 20, 64):
        if top_n <= V:
            assert_forward(K, x, tokens, top_n)


@pytest.mark.parametrize("kind", ["plain", "ties", "equal", "sorted", "few"])
@pytest.mark.parametrize("rows,V", [(1, 16384), (1, 16385), (1, 32768), (1, 32769), (3, 33001), (2, 45000), (130, 32801), (1, 1 << 20)])
def test_alternatives_joined_from_parts(K, rows, V, kind):
    """Rows cut into 2 .. 64 parts, fewer and more than the alternatives that are asked for."""
    x = make_logits(rows, V, torch.float32, kind, seed=V)
    for top_n in (1, 3, 10, 31, 50, 64):
        assert_forward(K, x, torch.zeros(rows, dtype=torch.int64), top_n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["ties", "equal", "few", "inf", "sorted", "peaked", "signed zero"])
@pytest.mark.parametrize("V", [70, 3001, 40000])
def test_forward_over_distributions(K, V, kind, dtype):
    x = make_logits(3, V, dtype, kind, seed=5)
    tokens = torch.tensor([0, V - 1, V // 2])
    for top_n in (1, 5, 64):
        assert_forward(K, x, tokens, top_n)


def test_tokens_outside_the_vocabulary_are_padding(K):
    x = make_logits(6, 50, torch.float32, "plain")
    assert_forward(K, x, torch.tensor([-1, 50, 3, -2 ** 40, 2 ** 40, 49]), 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_unaligned_logits(K, dtype):
    rows, V = 5, 1003
    big = torch.zeros(rows, V + 30, dtype=dtype, device=DEV)
    x = make_logits(rows, V, dtype, "plain", seed=2)
    for off in (0, 1, 8):
        view = big[:, off:off + V]
        view.copy_(x)
        assert_forward(K, x, torch.arange(rows), 7, xd=view)
    same = x[:1].to(DEV).expand(rows, V)                       # one row for all
    assert_forward(K, x[:1].expand(rows, V), torch.arange(rows), 4, xd=same)
    every = big[::2]
    every.copy_(torch.cat([x, torch.zeros(rows, 30, dtype=dtype)], 1)[::2])
    assert_forward(K, x[::2], torch.arange(3), 4, xd=every[:, :V])


def test_rows_with_nan_and_rows_of_minus_infinity(K):
    x = make_logits(4, 3000, torch.float32, "plain", seed=3)
    x[1, 77] = math.nan
    x[2] = -math.inf
    x[3, 5] = math.inf
    logp, ent, lse, top_logp, ids = (t.cpu() for t in K.token_logprobs(x.to(DEV), torch.tensor([1, 1, 1, 1], device=DEV), 4))
    assert torch.isfinite(logp[0]) and torch.isfinite(ent[0])
    assert torch.isnan(logp[1:]).all() and torch.isnan(lse[1:3]).all() and torch.isnan(ent[1:]).all()
    assert int(ids[1, 0]) == 77 and ids[2].tolist() == [0, 1, 2, 3] and int(ids[3, 0]) == 5
    assert torch.equal(ids[0], torch.sort(x[0], descending=True, stable=True).indices[:4])


# ------------------------------------------------------------------------------------------------ gradient
def assert_backward(K, x, tokens, a, b, out=None):
    rows, V = x.shape
    xd, td = x.to(DEV), tokens.to(DEV)
    _, ent, lse, _, _ = K.token_logprobs(xd, td)
    g = K.token_logprobs_bwd(xd, td, lse, ent, None if a is None else a.to(DEV), None if b is None else b.to(DEV), out=out(xd) if out else None)
    assert g.dtype == x.dtype and g.shape == x.shape
    l64, h64 = lse.cpu().double()[:, None], ent.cpu().double()[:, None]
    given = (tokens >= 0) & (tokens < V)
    a64 = torch.zeros(rows, 1, dtype=torch.float64) if a is None else torch.where(given, a.double(), torch.zeros(rows, dtype=torch.float64))[:, None]
    b64 = torch.zeros(rows, 1, dtype=torch.float64) if b is None else b.double()[:, None]
    x64 = x.double()
    lp = x64 - l64
    p = lp.exp()
    safe = torch.where(p > 0, lp, torch.zeros_like(lp))
    want = -p * (a64 + b64 * (safe + h64))
    hot = torch.zeros_like(p)
    hot[torch.arange(rows)[given], tokens[given]] = 1.0
    want = want + hot * a64
    x0 = torch.where(torch.isfinite(x64), x64, torch.zeros_like(x64))
    rel = U * (x0.abs() + l64.abs() + 3 * safe.abs() + 16)
    mag = p * (a64.abs() + b64.abs() * (safe.abs() + h64.abs() + 1))
    half = 2.0 ** -8 if x.dtype == torch.bfloat16 else U
    # a probability below 2^-126 is flushed to 0, which is off by less than 2^-126, and that factor times |a + b (log p + H)| in the
    # product; a product that falls below 2^-126 itself is flushed as well: another 2^-126
    flushed = 2.0 ** -126 * (1 + a64.abs() + b64.abs() * (safe.abs() + h64.abs()))
    tol = 4 * rel * mag + 2 * U * hot * a64.abs() + half * want.abs() + flushed
    err = (g.cpu().double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())
    return g


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 7), (2, 256), (130, 1001), (4, 8008), (2, 70001)])
def test_gradient_against_the_formula(K, rows, V, dtype):
    x = make_logits(rows, V, dtype, "plain", seed=V)
    tokens = torch.randint(0, V, (rows,), generator=gen(1))
    if rows > 2:
        tokens[1] = -1
    a, b = torch.randn(rows, generator=gen(2)), torch.randn(rows, generator=gen(3)) * 0.1
    assert_backward(K, x, tokens, a, b)
    assert_backward(K, x, tokens, a, None)
    assert_backward(K, x, tokens, None, b)
    assert_backward(K, x, tokens, a, b, out=lambda xd: xd)                     # in place
    assert_backward(K, x, tokens, a, b, out=lambda xd: torch.zeros(rows, V + 5, dtype=dtype, device=DEV)[:, 3:3 + V])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["few", "inf", "peaked", "equal"])
def test_gradient_over_distributions(K, kind, dtype):
    x = make_logits(4, 3001, dtype, kind, seed=4)
    a, b = torch.randn(4, generator=gen(2)), torch.randn(4, generator=gen(3))
    assert_backward(K, x, torch.tensor([5, 3000, -1, 1500]), a, b)


def test_gradient_against_differences(K):
    """d(sum w logp + c H) along random directions by central differences of the float64 forward; f32 kernels.  The difference's own error
    at h = 1e-4 is h^2 times a third derivative of order one: 1e-7 of the gradient's size here, far below the bound."""
    x = make_logits(5, 300, torch.float32, "plain", seed=9)
    tokens = torch.tensor([0, 299, 7, -1, 20])
    w, c = torch.randn(5, generator=gen(2)), torch.randn(5, generator=gen(3))
    xd = x.to(DEV)
    _, ent, lse, _, _ = K.token_logprobs(xd, tokens.to(DEV))
    g = K.token_logprobs_bwd(xd, tokens.to(DEV), lse, ent, w.to(DEV), c.to(DEV)).cpu().double()

    def value(y):
        lp = torch.log_softmax(y, -1)
        t = torch.where(tokens >= 0, lp.gather(1, tokens.clamp_min(0)[:, None])[:, 0], torch.zeros(5, dtype=torch.float64))
        return float((w.double() * t).sum() - (c.double() * (lp.exp() * lp).sum(-1)).sum())
    for s in range(5):
        d = torch.randn(5, 300, generator=gen(100 + s)).double()
        want = (value(x.double() + 1e-4 * d) - value(x.double() - 1e-4 * d)) / 2e-4
        assert abs(float((g * d).sum()) - want) <= 1e-4 * float((g.abs() * d.abs()).sum())


def test_captured_forward_and_gradient(K):
    rows, V = 6, 50000
    x = torch.zeros(rows, V, device=DEV)
    tokens = torch.arange(rows, device=DEV)
    a, b = torch.randn(rows, generator=gen(2)).to(DEV), torch.randn(rows, generator=gen(3)).to(DEV)

    def both():
        out = K.token_logprobs(x, tokens, 5)
        return (*out, K.token_logprobs_bwd(x, tokens, out[2], out[1], a, b))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = both()
    for i in range(5):
        x.copy_(make_logits(rows, V, torch.float32, "plain", seed=i))
        graph.replay()
        want = both()
        torch.cuda.synchronize()
        for p, q in zip(got, want):
            assert torch.equal(p, q), i


def test_calls_with_nothing_in_them(K):
    x, tokens = torch.zeros(0, 30, device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV)
    logp, entropy, lse, top_logp, top_ids = K.token_logprobs(x, tokens, 3)
    assert logp.shape == entropy.shape == lse.shape == (0,) and top_logp.shape == top_ids.shape == (0, 3)
    assert K.token_logprobs_bwd(x, tokens, lse, entropy, logp, entropy).shape == (0, 30)


# ------------------------------------------------------------------------------------------------ masks and offsets
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [-1e9, -1e36, float(torch.finfo(torch.bfloat16).min), float(torch.finfo(torch.float32).min), -math.inf])
@pytest.mark.parametrize("rows,V", [(1, 3000), (1, 40000), (4, 40000), (130, 40000), (1, 128000), (4, 128000), (130, 128000)])
def test_parts_of_nothing_but_ruled_out_symbols(K, rows, V, mask, dtype):
    """A short list is allowed, everything else has a large finite mask: whole parts of a row hold nothing else.  They add exactly nothing --
    to the entropy and to the gradient that takes it, too."""
    g = gen(V + rows)
    x = torch.full((rows, V), mask)
    for r in range(rows):
        x[r, torch.randperm(V, generator=g)[:20]] = torch.randn(20, generator=g) * 2
    x = x.to(dtype)
    tokens = x.argmax(-1)
    assert_forward(K, x, tokens, 6)
    assert_backward(K, x, tokens, torch.randn(rows, generator=g), torch.randn(rows, generator=g))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0.0, 1000.0, -1000.0, 20000.0])
@pytest.mark.parametrize("rows,V", [(7, 1000), (128, 8008), (2, 40000), (4, 128000)])
def test_log_probabilities_keep_their_bits_under_an_offset(K, rows, V, offset, dtype):
    """log p = (x - m) - log S: what all logits have in common drops out exactly, so the bound has no |lse| in it.
        x - m: u |x - m|;    log S: the sum and its terms as in the bound of lse, the logarithm's 4 u log S;    the result: u |log p|
    (x - m of logits within a factor of two of each other is exact; under a large offset they all are.)"""
    x = (make_logits(rows, V, torch.float32, "plain", seed=V) + offset).to(dtype)
    tokens = torch.randint(0, V, (rows,), generator=gen(1))
    logp, _, _, top_logp, top_ids = (t.cpu() for t in K.token_logprobs(x.to(DEV), tokens.to(DEV), 20))
    x64 = x.double()
    d = x64 - x64.amax(-1, keepdim=True)
    log_s = torch.logsumexp(d, -1)
    p = (d - log_s[:, None]).exp()
    H = -(p * (d - log_s[:, None])).sum(-1)
    t_log_s = U * (V / 256 + 40 + 3 * (H + 8) + 4 * log_s)
    for ids, got in ((tokens[:, None], logp[:, None]), (top_ids, top_logp)):
        at = d.gather(1, ids)
        want = at - log_s[:, None]
        assert ((got.double() - want).abs() <= t_log_s[:, None] + U * (at.abs() + want.abs())).all()
