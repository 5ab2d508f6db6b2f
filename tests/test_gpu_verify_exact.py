"""verify_drafts at the borders of its decisions: draws and acceptances that
arithmetic of fewer than 64 bits would get wrong, against the definition in
64 bits."""

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
