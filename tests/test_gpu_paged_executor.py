"""GPUExecutionBackend over the paged cache (kv_append + attention_paged) and
its drafted generation (verify_drafts), on the fixtures of the decode step.

The reference is the decode oracle whose cached keys and values are rounded as
the cache rounds them.  Its bar is the decode step's (logits within 2e-3
relative L2) and what a rounding that falls the other way can add: a cached
value is off by one step at most then, 2^-7 of the value in bf16 and 1/127 of
its block's largest in Q8_0, by half of that in the mean of roundings that all
fall the wrong way.  A greedy token's logit is within the errors of the two
logits compared (each at most the relative L2 error times the row's norm) of
the largest."""

from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

import paged_reference as R  # noqa: E402
from dracort_b200 import gguf_executor as X  # noqa: E402
from dracort_b200 import paged_ops as P  # noqa: E402
from dracort_b200.format.gguf_file import GGUFFile  # noqa: E402
from oracle.llama_decode import OracleLlama  # noqa: E402

HERE = Path(__file__).resolve().parent / "golden"
TOL = {"bf16": 2e-3 + 2.0 ** -8, "q8_0": 2e-3 + 1.0 / 127}


class RoundedOracle(OracleLlama):
    cache_type = "bf16"

    def _attention(self, s, layer, q, k, v, causal):
        k, v = (R.cached_values(torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)),
                                self.cache_type).float().numpy() for x in (k, v))
        return super()._attention(s, layer, q, k, v, causal)


@pytest.fixture(scope="module", params=[("tiny_llama_decode", "bf16"), ("tiny_llama_decode", "q8_0"),
                                        ("tiny_qwen2_decode", "q8_0"), ("tiny_fused_decode", "bf16")],
                ids=lambda p: f"{p[0]}-{p[1]}")
def pair(request):
    name, kind = request.param
    be = X.GPUExecutionBackend(str(HERE / f"{name}.gguf"), 3, kind, page_size=16, q6k_order="d_first")
    gf = GGUFFile(str(HERE / f"{name}.gguf"))
    try:
        orc = RoundedOracle(gf, q6k_order="d_first")
    finally:
        gf.close()
    orc.cache_type = kind
    return be, orc, TOL[kind]


def rel(a, b):
    return float(np.linalg.norm(a - b) / np.linalg.norm(b))


def all_free(be):
    return sorted(be._free_pages) == list(range(be.k_cache[0].shape[0])) and len(be._free) == be.max_num_seqs


def assert_greedy(orc, ids, prompt_len, tol):
    so = orc.new_sequence()
    logits = orc.forward_step(so, np.array(ids[:-1]), 0, return_all_positions=True)
    orc.end_sequence(so)
    for p in range(prompt_len, len(ids)):
        row = logits[p - 1]
        assert row[ids[p]] >= row.max() - 2 * tol * np.linalg.norm(row)


def test_prompt_chunks_and_decode_steps(pair):
    """50 tokens (chunks of 32 and 18 over four pages), then decode steps; run
    three times, so that the passes are eager, captured and replayed."""
    be, orc, tol = pair
    rng = np.random.default_rng(7)
    for _ in range(3):
        ids = rng.integers(0, be.config.vocab_size, 56)
        so, s = orc.new_sequence(), be.new_sequence()
        assert rel(be.forward_step(s, ids[:50], 0, return_all_positions=True),
                   orc.forward_step(so, ids[:50], 0, return_all_positions=True)) < tol
        for p in range(50, 56):
            assert rel(be.forward_step(s, ids[p:p + 1], p), orc.forward_step(so, ids[p:p + 1], p)) < tol
        assert len(be._pages[s]) == 4
        be.end_sequence(s)
        orc.end_sequence(so)
    assert all_free(be)


def test_batch_decode_of_sequences_in_any_order(pair):
    be, orc, tol = pair
    rng = np.random.default_rng(8)
    lengths = [3, 31, 16]
    seqs, refs = [be.new_sequence() for _ in lengths], [orc.new_sequence() for _ in lengths]
    for s, so, n in zip(seqs, refs, lengths):
        ids = rng.integers(0, be.config.vocab_size, n)
        be.forward_step(s, ids, 0)
        orc.forward_step(so, ids, 0)
    for step in range(4):
        order = rng.permutation(3)
        toks = rng.integers(0, be.config.vocab_size, 3)
        got = be.forward_batch_decode([seqs[i] for i in order], toks, [lengths[i] + step for i in order])
        want = np.stack([orc.forward_step(refs[i], toks[j:j + 1], lengths[i] + step) for j, i in enumerate(order)])
        assert rel(got, want) < tol
    for s in seqs:
        be.end_sequence(s)
    assert all_free(be)


def test_truncated_sequences_rewrite_their_positions_and_free_pages(pair):
    be, orc, tol = pair
    rng = np.random.default_rng(9)
    a, b = rng.integers(0, be.config.vocab_size, 40), rng.integers(0, be.config.vocab_size, 12)
    s, other, so = be.new_sequence(), be.new_sequence(), orc.new_sequence()
    be.forward_step(s, a, 0)
    be.truncate_sequence(s, 17)
    assert len(be._pages[s]) == 2
    be.forward_step(other, b, 0)  # takes the page that was freed last
    orc.forward_step(so, a[:17], 0)
    assert rel(be.forward_step(s, b, 17, return_all_positions=True),
               orc.forward_step(so, b, 17, return_all_positions=True)) < tol
    be.truncate_sequence(s, 0)
    assert be._pages[s] == []
    be.end_sequence(s)
    be.end_sequence(other)
    assert all_free(be)


def test_greedy_generation_with_and_without_drafts(pair, monkeypatch):
    be, orc, tol = pair
    prompt = [5, 9, 5, 9, 5, 9, 5]
    plain = be.generate_greedy(prompt, 20)
    assert_greedy(orc, plain, len(prompt), tol)
    ids = be.generate_speculative(prompt, 20, num_drafts=3)
    assert ids[:7] == prompt and len(ids) == 27
    assert_greedy(orc, ids, len(prompt), tol)
    # drafts that are right are taken: four tokens a pass
    calls = []
    run = be._verified
    monkeypatch.setattr(be, "_verified", lambda *a: calls.append(a) or run(*a))
    monkeypatch.setattr(X, "ngram_drafts", lambda seen, count, ngram: ids[len(seen):len(seen) + min(count, 3)])
    again = be.generate_speculative(prompt, 20, num_drafts=3)
    assert_greedy(orc, again, len(prompt), tol)
    if again == ids:
        assert len(calls) == 5
    # drafts that are wrong are not
    wrong = [(t + 1) % be.config.vocab_size for t in ids]
    monkeypatch.setattr(X, "ngram_drafts", lambda seen, count, ngram: wrong[len(seen):len(seen) + min(count, 3)])
    assert_greedy(orc, be.generate_speculative(prompt, 20, num_drafts=3), len(prompt), tol)
    assert all_free(be)


def test_sampled_generation_repeats_by_its_seed(pair):
    be, _, _ = pair
    prompt = [1, 2, 3, 1, 2]
    a = be.generate_speculative(prompt, 30, num_drafts=5, temperature=0.8, seed=3)
    assert a == be.generate_speculative(prompt, 30, num_drafts=5, temperature=0.8, seed=3)
    assert len(a) == 35 and all(0 <= t < be.config.vocab_size for t in a)
    assert be.generate_speculative(prompt, 0) == prompt
    assert len(be.generate_speculative([7], 5, num_drafts=0)) == 6
    for bad in (dict(num_drafts=32), dict(num_drafts=-1), dict(ngram=0), dict(temperature=-1.0)):
        with pytest.raises(ValueError):
            be.generate_speculative(prompt, 3, **bad)
    with pytest.raises(ValueError, match="no token"):
        be.generate_speculative([], 3)
    with pytest.raises(ValueError, match="capacity"):
        be.generate_speculative(prompt, be.capacity)
    assert all_free(be)


def test_drafted_generation_over_the_fp32_cache():
    be = X.GPUExecutionBackend(str(HERE / "tiny_llama_decode.gguf"), q6k_order="d_first")
    gf = GGUFFile(str(HERE / "tiny_llama_decode.gguf"))
    try:
        orc = OracleLlama(gf, q6k_order="d_first")
    finally:
        gf.close()
    ids = be.generate_speculative([5, 9, 5, 9, 5], 20, num_drafts=4)
    assert len(ids) == 25
    assert_greedy(orc, ids, 5, 2e-3)


def test_pool_that_runs_out_refuses_and_recovers():
    name = str(HERE / "tiny_llama_decode.gguf")
    page = 2 * 2 * 4 * 16 * 32 * 2  # 2 layers of keys and values, 4 heads of 32, 16 positions of bf16
    be = X.GPUExecutionBackend(name, 4, "bf16", 3 * page, page_size=16, q6k_order="d_first")
    assert be.capacity == 48 and be.k_cache[0].shape[0] == 3
    a, b = be.new_sequence(), be.new_sequence()
    be.forward_step(a, np.arange(20), 0)
    first = be.forward_step(b, np.arange(16), 0)
    with pytest.raises(RuntimeError, match="free pages"):
        be.forward_step(b, np.array([3]), 16)
    with pytest.raises(RuntimeError, match="free pages"):
        be.forward_batch_decode([a, b], [1, 2], [20, 16])
    assert be._len[a] == 20 and be._len[b] == 16
    be.end_sequence(a)
    be.forward_step(b, np.array([3]), 16)
    be.truncate_sequence(b, 0)
    assert rel(be.forward_step(b, np.arange(16), 0), first) < 1e-6  # the same pass again
    be.end_sequence(b)
    assert all_free(be)


def test_launches_per_layer():
    be = X.GPUExecutionBackend(str(HERE / "tiny_llama_decode.gguf"), 1, "q8_0", q6k_order="d_first")
    assert be.launches_per_layer == 6  # four GEMV steps, the append, the attention
    assert P.attention_paged_status(be._buffers(1)["attn_ws"]) == 0
