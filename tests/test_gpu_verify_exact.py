"""verify_drafts at the borders of its decisions: draws and acceptances that
arithmetic of fewer than 64 bits would get wrong, against the definition in
64 bits."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

from dracort_b200 import paged_ops as P  # noqa: E402

DEV = torch.device("cuda", 0)


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def peaked(vocab, g):
    x = torch.randn(vocab, generator=g, device=DEV) * 2
    x[torch.randint(0, vocab, (4,), generator=g, device=DEV)] += torch.tensor([9.0, 8.0, 7.0, 6.0], device=DEV)
    return x


def softmax64(x, t):
    w = torch.exp((x.double() - x.double().max()) / t)
    return w / w.sum()


def cumulative(weights):
    c = weights.cumsum(0)
    return c / c[-1]


def draws_between(c, other, count, gap=1e-10):
    """Up to `count` fp32 numbers u, spread over the tokens, that lie between the cumulative weights c and `other` of
    a token, further than `gap` (100 times the error that fp64 sums of 10^5 weights may have) from both."""
    u = ((c + other) / 2).float()
    lo, hi = torch.minimum(c, other), torch.maximum(c, other)
    at = ((u.double() > lo + gap) & (u.double() < hi - gap) & (u < 1)).nonzero()[:, 0]
    at = at[torch.linspace(0, len(at) - 1, min(count, len(at)), device=DEV).long()] if len(at) else at
    return u[at]


@pytest.mark.parametrize("form", ["plain", "certain draft", "draft_probs"])
@pytest.mark.parametrize("temperature", [0.6, 0.7, 0.8, 0.9, 1.1, 1.3])
def test_draws_are_those_of_the_temperature_given(temperature, form):
    """Draws that the temperature rounded to fp32 would answer with the next token or the one before."""
    g = gen(int(temperature * 10))
    vocab = 128000
    x = peaked(vocab, g)
    q = softmax64(x + 0.5 * torch.randn(vocab, generator=g, device=DEV), temperature).float()
    rounded = float(torch.tensor(temperature, dtype=torch.float32))
    p = softmax64(x, temperature)
    rare = int(p.argmin())
    draft = int((q.double() - 2 * p).argmax())  # q > p there: rejected by a number near one

    def left(p):
        if form == "plain":
            return p
        if form == "certain draft":
            return torch.where(torch.arange(vocab, device=DEV) == rare, 0.0, p)
        return (p - q.double()).clamp_min(0.0)

    c = cumulative(left(p))
    u = draws_between(c, cumulative(left(softmax64(x, rounded))), 64)
    assert len(u) >= 16
    rows = 1 if form == "plain" else 2
    n = len(u) * rows
    count, tokens = P.verify_drafts(
        x.expand(n, -1), torch.arange(0, n + 1, rows, dtype=torch.int32, device=DEV),
        i32([rare if form == "certain draft" else draft] * n), torch.full((n,), 0.75, device=DEV), u,
        draft_probs=q.expand(n, -1) if form == "draft_probs" else None, temperature=temperature, max_rows=rows)
    want = torch.searchsorted(c, u.double(), right=True)
    assert not count.any()
    assert torch.equal(tokens[:, 0].long(), want)


def test_temperatures_below_the_limit_are_refused():
    """1e-46 is zero in fp32, which would be greedy."""
    x = torch.zeros(1, 5, device=DEV)
    for t in (1e-46, 1e-31, 1.1e30, float("nan"), -0.5):
        with pytest.raises(ValueError, match="temperature"):
            P.verify_drafts(x, i32([0, 1]), i32([0]), x[0, :1], x[0, :1], temperature=t)
    for t in (0.0, 1e-30, 1e30):
        P.verify_drafts(x, i32([0, 1]), i32([0]), x[0, :1], x[0, :1], temperature=t)


def neighbours(p):
    """The largest fp32 number below p (float64) and the smallest that is not."""
    f = p.float()
    lo = torch.where(f.double() < p, f, torch.nextafter(f, torch.zeros_like(f)))
    return lo, torch.nextafter(lo, torch.ones_like(lo))


def clear(p, lo, hi):
    """Both neighbours are further from p than fp64 sums of 10^5 weights are off (1e-12 of it)."""
    return ((p - lo.double()) > 1e-11 * p) & ((hi.double() - p) > 1e-11 * p)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [7, 3001, 128000])
@pytest.mark.parametrize("temperature", [0.7, 1.0])
def test_certain_drafts_are_decided_by_the_numbers_next_to_their_probability(temperature, vocab, dtype):
    g = gen(vocab)
    x = peaked(vocab, g).to(dtype)
    p = softmax64(x, temperature)
    lo, hi = neighbours(p)
    some = (clear(p, lo, hi) & (hi < 1)).nonzero()[:, 0]
    some = some[p[some].argsort(descending=True)][:400]  # the likely ones
    some = torch.cat([some, (p > 0).nonzero()[:1, 0]])
    n = len(some)
    starts = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=DEV)
    drafts = some.to(torch.int32).repeat_interleave(2)
    half = torch.full((n,), 0.5, device=DEV)
    for u, want in ((lo, 1), (hi, 0)):
        count, tokens = P.verify_drafts(x.expand(2 * n, -1), starts, drafts, u[some].repeat_interleave(2), half,
                                        temperature=temperature, max_rows=2)
        assert torch.equal(count[:-1], torch.full_like(count[:-1], want))
        assert bool(((tokens[:-1, 0].long() == some[:-1]) == bool(want)).all())


@pytest.mark.parametrize("temperature", [0.7, 1.0])
def test_drafts_with_probabilities_are_decided_by_the_numbers_next_to_the_border(temperature):
    g = gen(5)
    vocab, n = 32000, 300
    x = peaked(vocab, g)
    p = softmax64(x, temperature)
    some = p.argsort(descending=True)[:n]
    q = torch.zeros(n, vocab, device=DEV)
    q[torch.arange(n, device=DEV), some] = (p[some] * (1 + torch.rand(n, generator=g, device=DEV, dtype=torch.float64))).float()
    qx = q[torch.arange(n, device=DEV), some].double()
    lo, hi = neighbours(p[some] / qx)  # u q < p
    sure = clear(p[some] / qx, lo, hi)
    assert int(sure.sum()) > n * 0.9
    starts = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=DEV)
    for u, want in ((lo, 1), (hi, 0)):
        count, _ = P.verify_drafts(x.expand(2 * n, -1), starts, some.to(torch.int32).repeat_interleave(2),
                                   u.repeat_interleave(2), torch.full((n,), 0.5, device=DEV),
                                   draft_probs=q.repeat_interleave(2, 0), temperature=temperature, max_rows=2)
        assert bool((count[sure] == want).all())


@pytest.mark.parametrize("stop", [0, 31, 32, 40, 63, 64, 97, 99])
def test_a_chain_of_close_decisions_ends_at_the_first_that_is_not_taken(stop):
    """100 rows: every draft's number is the one just below its probability, but that of row `stop` (99: the last)."""
    g = gen(stop)
    vocab, rows = 5000, 100
    x = torch.randn(rows, vocab, generator=g, device=DEV) * 3
    p = torch.softmax(x.double(), -1)
    drafts = x.argmax(-1)
    px = p.gather(1, drafts[:, None])[:, 0]
    lo, hi = neighbours(px)
    sure = clear(px, lo, hi)
    u = torch.where(sure, lo, lo * 0.9)  # (a number that fp64 cannot tell apart moves away)
    u[stop] = torch.where(sure[stop], hi[stop], hi[stop] * 1.1)
    count, tokens = P.verify_drafts(x, i32([0, rows]), drafts.to(torch.int32), u, torch.full((1,), 0.5, device=DEV),
                                    max_rows=rows)
    assert count.tolist() == [min(stop, rows - 1)]
    assert torch.equal(tokens[0, :stop].long(), drafts[:stop]) and bool((tokens[0, stop + 1:] == -1).all())


def test_drafts_of_no_weight_and_numbers_of_zero():
    """u = 0 takes every draft of positive probability, and none of probability zero."""
    x = torch.zeros(6, 50, device=DEV)
    x[:, 3] = -200.0  # 1e-87 of the weight: zero in fp32
    x[:, 4] = -float("inf")
    x[:, 5] = float("nan")
    starts, u = i32([0, 2, 4, 6]), torch.zeros(6, device=DEV)
    count, _ = P.verify_drafts(x, starts, i32([3, 0, 4, 0, 5, 0]), u, u[:3], max_rows=2)
    assert count.tolist() == [1, 0, 0]


@pytest.mark.parametrize("seqs", [20, 21, 22, 23, 37, 38])
def test_as_many_sequences_as_clusters_of_either_size(seqs):
    """Around the number of sequences from which they get fewer blocks each: the same tokens as one by one."""
    g = gen(seqs)
    vocab = 20011
    x = torch.stack([peaked(vocab, g) for _ in range(2 * seqs)])
    q = torch.softmax(x + 0.5 * torch.randn(2 * seqs, vocab, generator=g, device=DEV), -1)
    d = torch.multinomial(q, 1, generator=g)[:, 0].to(torch.int32)
    au, su = torch.rand(2 * seqs, generator=g, device=DEV), torch.rand(seqs, generator=g, device=DEV)
    starts = torch.arange(0, 2 * seqs + 1, 2, dtype=torch.int32, device=DEV)
    count, tokens = P.verify_drafts(x, starts, d, au, su, draft_probs=q, temperature=0.9, max_rows=2)
    for s in range(seqs):
        r = slice(2 * s, 2 * s + 2)
        c, t = P.verify_drafts(x[r], i32([0, 2]), d[r], au[r], su[s:s + 1], draft_probs=q[r], temperature=0.9, max_rows=2)
        assert torch.equal(count[s:s + 1], c) and torch.equal(tokens[s:s + 1], t)


def test_temperatures_of_other_number_types():
    x = peaked(1000, gen(1)).expand(64, -1)
    u = torch.linspace(0, 0.99, 64, device=DEV)
    args = (x, torch.arange(65, dtype=torch.int32, device=DEV), i32([0] * 64), u, u)
    want = P.verify_drafts(*args, temperature=2.0, max_rows=1)
    for t in (2, np.float32(2), np.float64(2), torch.tensor(2.0)):
        got = P.verify_drafts(*args, temperature=t, max_rows=1)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
