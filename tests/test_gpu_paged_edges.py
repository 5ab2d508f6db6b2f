"""The serving operators over the paged cache at the ends of their ranges."""

import ctypes
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

import test_gpu_paged as T  # noqa: E402
from dracort_b200 import _native as N  # noqa: E402
from dracort_b200 import gguf_executor as X  # noqa: E402
from dracort_b200 import paged_ops as P  # noqa: E402

DEV = torch.device("cuda", 0)
F32, BF16 = torch.float32, torch.bfloat16


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("tokens,dtype", [(1, F32), (1, BF16), (256, BF16)])
def test_the_longest_sequence(tokens, dtype):
    """0x7FFF0000 positions on two pages that the table repeats: values of 1 in the first nine tenths and 2 behind
    them, all scores equal.  The sums are whole numbers that fp32 holds; 2^-8 is the output's rounding."""
    page, hd, length = 1024, 32, 0x7FFF0000
    k, v = P.kv_cache("bf16", 2, 1, page, hd, DEV)
    v[0], v[1] = 1.0, 2.0
    pages = length // page
    table = torch.zeros((1, pages), dtype=torch.int32, device=DEV)
    table[:, pages * 9 // 10:] = 1
    want = 1 + (pages - pages * 9 // 10) / pages
    out = P.attention_paged(torch.zeros(tokens, 1, hd, dtype=dtype, device=DEV), k, v, table, i32([0, tokens]),
                            i32([length]), max_q=tokens, max_kv=length)
    assert P.attention_paged_status() == 0
    assert float((out.double() - want).abs().max()) <= want * 2.0 ** -8


@pytest.mark.parametrize("heads,kv", [(8, 8), (8, 2), (6, 1), (40, 2)])
@pytest.mark.parametrize("cache", ["bf16", "q8_0"])
def test_chunks_among_many_steps(cache, heads, kv):
    """Chunks that are split, at several places among 90 sequences of a token or none, some at the least length that
    the long chunks' kernel takes; run again, the same numbers."""
    least = 64 // (heads // kv) + 1
    new = [1, 0, 1, 1] * 22 + [1, 1]
    new[0], new[30], new[31], new[60], new[89] = least, 290, least, least - 1, 150
    past = [(s * 131) % 700 for s in range(90)]
    past[0], past[30], past[31], past[89] = 3000, 2500, 4000, 2000
    b = T.batch(new, past, heads, kv, 64, 64, cache, BF16, seed=41)
    out = torch.full_like(b[0], float("nan"))
    P.attention_paged(*b, max_q=290, max_kv=4000 + least, out=out)
    T.check(*b, out)
    for _ in range(3):
        assert torch.equal(P.attention_paged(*b, max_q=290, max_kv=4000 + least), out)


def set_status(value):
    """The device's status word, as a kernel whose wait ran out leaves it."""
    old = ctypes.c_int(-1)
    torch.cuda.synchronize()
    N.check(N.load().draco_attention_paged_status(value, ctypes.byref(old)))
    return old.value


def test_status_outlives_workspaces_and_replays():
    """An error is reported once, after the workspace of its call was replaced by a larger one, and after replays of
    a graph whose workspace is zeroed by each."""
    small = T.batch([1], [300], 8, 2, 64, 64, "bf16", BF16, seed=42)
    large = T.batch([300], [3000], 8, 2, 64, 64, "bf16", BF16, seed=43)
    want = P.attention_paged(*large)
    P.attention_paged_status()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        P.attention_paged(*small, max_q=1, max_kv=301)
        key = (0, st.cuda_stream)
        first = P._workspaces[key]
        P._workspaces[key] = first[:N.PAGED_WORKSPACE_HEAD].clone()  # (the kept ones begin at 1 MB)
        assert set_status(N.DRACO_ERR_TIMEOUT) == 0
        out = P.attention_paged(*large)
        assert P._workspaces[key].numel() > first.numel()
    assert P.attention_paged_status() == N.DRACO_ERR_TIMEOUT
    assert P.attention_paged_status() == 0
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = P.attention_paged(*large)
    graph.replay()
    assert set_status(N.DRACO_ERR_TIMEOUT) == 0
    graph.replay()
    assert P.attention_paged_status() == N.DRACO_ERR_TIMEOUT
    assert P.attention_paged_status() == 0
    assert torch.equal(out, want)


def test_every_workspace_with_an_error_is_made_ready_again():
    b = T.batch([1, 1], [4000, 3000], 8, 2, 128, 64, "q8_0", BF16, seed=44)
    want = P.attention_paged(*b, max_q=1, max_kv=4001)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            P.attention_paged(*b, max_q=1, max_kv=4001)
            ws = P._workspaces[(0, st.cuda_stream)]
            if i != 1:  # counters that an aborted merge left, and the status
                ws[:N.PAGED_WORKSPACE_HEAD].view(torch.int32)[:64] = 3
                ws[N.PAGED_WORKSPACE_STATUS:N.PAGED_WORKSPACE_STATUS + 4].view(torch.int32).fill_(5 + i)
    assert P.attention_paged_status() in (5, 7)
    assert P.attention_paged_status() == 0
    for st in streams:
        with torch.cuda.stream(st):
            assert torch.equal(P.attention_paged(*b, max_q=1, max_kv=4001), want)


@pytest.mark.parametrize("others", [1, 2])
def test_drafted_generation_in_a_full_pool(others, monkeypatch):
    """Four pages, one or two of them another sequence's, the rest just what the generation takes: drafts (wrong ones,
    whose pages come back) ask for no page that the tokens do not come to need, so the tokens are those without
    drafts; one token more than the pool holds is refused, as it is without drafts."""
    name = str(Path(__file__).resolve().parent / "golden" / "tiny_llama_decode.gguf")
    page = 2 * 2 * 4 * 16 * 32 * 2  # 2 layers of keys and values, 4 heads of 32, 16 positions of bf16
    be = X.GPUExecutionBackend(name, 3, "bf16", 4 * page, page_size=16, q6k_order="d_first")
    prompt, held = [5, 9, 5, 9, 5], 16 * (4 - others)
    count = held + 1 - len(prompt)  # (the last token is not cached)
    free = be.generate_speculative(prompt, count, num_drafts=0)
    s = be.new_sequence()
    be.forward_step(s, [1] * (16 * others), 0)
    drafted = []
    monkeypatch.setattr(X, "ngram_drafts", lambda ids, n, ngram: drafted.append(n) or [
        (t + 1) % be.config.vocab_size for t in free[len(ids):len(ids) + max(n, 0)]])
    assert be.generate_speculative(prompt, count, num_drafts=20) == free
    assert max(drafted) == 20 and drafted[-1] == 0
    for num_drafts in (0, 20):
        with pytest.raises(RuntimeError, match="free pages"):
            be.generate_speculative(prompt, count + 1, num_drafts=num_drafts)
    be.end_sequence(s)
    assert sorted(be._free_pages) == [0, 1, 2, 3]


@pytest.mark.parametrize("size", [1e3, 1e7, 1e9, 1e14, 1e20, 1e28])
@pytest.mark.parametrize("cache", ["bf16", "q8_0"])
@pytest.mark.parametrize("dtype,new", [(F32, 3), (BF16, 3), (BF16, 40)])
def test_scores_of_any_size(dtype, new, cache, size):
    """Scores far past 2^24, whose roundings are whole units: all weight on the largest score where it leads by a
    thousandth (fp32 sums of 64 products are off by less than 64 2^-24 of their largest).  Its value is then off by
    the output's rounding, and for bf16 activations by those of P (the sum is of unrounded ones) and of V: 2^-8 + 2^-8
    over bf16 pages, 2^-8 + 2 2^-11 over Q8_0."""
    b = T.batch([new], [300], 4, 2, 64, 16, cache, dtype, seed=45)
    q = (b[0].float() * size).to(dtype)
    out = P.attention_paged(q, *b[1:], max_q=new, max_kv=300 + new)
    k, v = (T.R.sequence(T.R.values(c), b[3][0], 300 + new, c.shape[0]).repeat_interleave(2, 0) for c in b[1:3])
    s = q.double().transpose(0, 1) @ k.transpose(1, 2) / 8
    s.masked_fill_(torch.ones(new, 300 + new, dtype=torch.bool, device=DEV).triu(301), -float("inf"))
    top, at = s.topk(2, -1)
    lead = top[..., 0] - top[..., 1] > 1e-3 * top[..., 0].abs() + 40
    assert float(lead.double().mean()) > 0.5
    want = v.gather(1, at[..., :1].expand(-1, -1, 64))
    got = out.double().transpose(0, 1)
    assert torch.isfinite(got).all()
    tol = 2.0 ** -20 if dtype is F32 else (2.0 ** -7 if cache == "bf16" else 2.0 ** -8 + 2.0 ** -10) * (1 + 2.0 ** -8)
    assert float(((got - want).abs() / want.abs().clamp_min(1e-6))[lead].max()) <= tol


@pytest.mark.parametrize("cache", ["bf16", "q8_0"])
@pytest.mark.parametrize("dtype,new", [(F32, 3), (BF16, 3), (BF16, 40)])
def test_rows_beside_rows_of_huge_scores(dtype, new, cache):
    """Rows of ordinary and of huge scores in one tile, tokens that see nothing, a key that is not finite."""
    b = T.batch([new], [300], 4, 2, 64, 16, cache, dtype, seed=46)
    q = b[0].clone()
    q[1::3] *= 1e9
    out = P.attention_paged(q, *b[1:], max_q=new, max_kv=300 + new)
    want, bound = T.R.attention(*b[:4], b[4].tolist(), b[5].tolist())
    rows = torch.arange(new, device=DEV) % 3 != 1
    assert torch.isfinite(out).all()
    assert float(((out.double() - want).abs() / bound)[rows].max()) <= 1
    few = i32([new - 2])  # two tokens see nothing
    out = P.attention_paged(q, *b[1:5], few, max_q=new, max_kv=300 + new)
    assert not out[:2].any() and torch.isfinite(out).all()
    page, off = int(b[3][0, 100 // 16]), 100 % 16
    if cache == "bf16":
        b[1][page, 0, off] = float("nan")
    else:
        T.R.q8_parts(b[1])[1][page, 0, off] = float("nan")
    out = P.attention_paged(q, *b[1:], max_q=new, max_kv=300 + new)
    assert torch.isnan(out[:, :2]).all() and torch.isfinite(out[:, 2:]).all()
