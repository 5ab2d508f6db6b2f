"""The serving operators over the paged cache (dracort_b200.paged_ops) on the
GPU against their 64-bit statements (paged_reference): appending (bit-exact),
reading back, attention of new tokens, verification of drafts."""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

import paged_reference as R  # noqa: E402
from dracort_b200 import paged_ops as P  # noqa: E402

DEV = torch.device("cuda", 0)
F32, BF16 = torch.float32, torch.bfloat16


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def randn(*shape, g, dtype=F32):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def make_cache(cache, pages, kv, page, hd, g):
    k, v = P.kv_cache(cache, pages, kv, page, hd, DEV)
    for c in (k, v):
        R.fill(c, randn(pages, kv, page, hd, g=g))
    return k, v


def tables(hd, n):
    ang = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)
    return ang.cos().float(), ang.sin().float()


def bits(x):
    return x.view(torch.int32 if x.dtype == F32 else torch.int16)


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------
APPEND = [  # heads, kv_heads, head_dim, page
    (8, 4, 32, 16), (4, 4, 64, 32), (6, 2, 96, 16), (32, 8, 128, 64), (5, 1, 128, 1024), (3, 3, 256, 128)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cache", ["bf16", "q8_0"])
@pytest.mark.parametrize("heads,kv,hd,page", APPEND)
def test_append_is_bit_exact_and_touches_nothing_else(heads, kv, hd, page, cache, dtype):
    g = gen(heads * hd + page)
    seqs, width = 3, 3
    pages = seqs * width + 2
    kc, vc = make_cache(cache, pages, kv, page, hd, g)
    table = torch.randperm(pages, generator=g, device=DEV)[:seqs * width].reshape(seqs, width).to(torch.int32)
    pos = [0, 1, page - 1, page, 2 * page + 5, 3 * page - 1, 7, 15]
    seq = [0, 0, 0, 1, 1, 2, 2, 1]
    n = len(pos)
    q, k, v = (randn(n, h, hd, g=g, dtype=dtype) for h in (heads, kv, kv))
    k[:, :, 3] *= 100
    cos, sin = tables(hd, 3 * page)
    before = (kc.clone(), vc.clone())
    out = P.kv_append(q, k, v, kc, vc, table, i32(seq), i32(pos), cos, sin)
    at = torch.tensor(pos, device=DEV)
    want_q = R.rotate(q, cos[at], sin[at])
    assert torch.equal(bits(out), bits(want_q.to(F32).to(dtype)))
    rows = table[torch.tensor(seq, device=DEV), at // page].long()
    off = at % page
    for c, old, x in ((kc, before[0], R.rotate(k, cos[at], sin[at])), (vc, before[1], v.double())):
        want = R.cached_values(x, cache)
        assert torch.equal(R.values(c)[rows, :, off], want)
        mask = torch.ones((pages, kv, page), dtype=torch.bool, device=DEV)
        mask[rows, :, off] = False
        new, was = (R.q8_parts(t) if cache == "q8_0" else (t,) for t in (c, old))
        for a, b in zip(new, was):
            assert torch.equal(a[mask], b[mask])
    rk, rv = P.kv_read(kc, vc, table, i32(seq), i32(pos), hd, F32)
    assert torch.equal(rk.double(), R.values(kc)[rows, :, off]) and torch.equal(rv.double(), R.values(vc)[rows, :, off])
    bk, _ = P.kv_read(kc, vc, table, i32(seq), i32(pos), hd, BF16)
    assert torch.equal(bk, rk.to(BF16))


def test_append_of_a_long_batch():
    """More rows than one wave of blocks: several rows per thread."""
    g = gen(1)
    heads, kv, hd, page, n = 32, 8, 128, 64, 1500
    kc, vc = make_cache("q8_0", 30, kv, page, hd, g)
    table = torch.arange(30, device=DEV, dtype=torch.int32)[None]
    q, k, v = (randn(n, h, hd, g=g, dtype=BF16) for h in (heads, kv, kv))
    cos, sin = tables(hd, n)
    pos = torch.randperm(n, generator=g, device=DEV).to(torch.int32)
    out = P.kv_append(q, k, v, kc, vc, table, torch.zeros_like(pos), pos, cos, sin)
    at = pos.long()
    assert torch.equal(out, R.rotate(q, cos[at], sin[at]).to(F32).to(BF16))
    rk, rv = P.kv_read(kc, vc, table, torch.zeros_like(pos), pos, hd)
    assert torch.equal(rk.double(), R.cached_values(R.rotate(k, cos[at], sin[at]), "q8_0"))
    assert torch.equal(rv.double(), R.cached_values(v, "q8_0"))


@pytest.mark.parametrize("cache", ["bf16", "q8_0"])
def test_append_in_place_from_a_fused_projection_without_rotation(cache):
    g = gen(2)
    heads, kv, hd, n = 4, 2, 64, 5
    fused = randn(n, heads + 2 * kv, hd, g=g)
    q, k, v = fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:]
    copy = fused.clone()
    kc, vc = make_cache(cache, 2, kv, 16, hd, g)
    table, seq, pos = i32([[1, 0]]), i32([0] * n), i32(list(range(14, 14 + n)))
    assert P.kv_append(q, k, v, kc, vc, table, seq, pos, q_out=q) is q
    assert torch.equal(fused, copy)  # nothing to rotate
    rk, rv = P.kv_read(kc, vc, table, seq, pos, hd)
    assert torch.equal(rk.double(), R.cached_values(copy[:, heads:heads + kv], cache))
    assert torch.equal(rv.double(), R.cached_values(copy[:, heads + kv:], cache))
    cos, sin = tables(hd, 32)
    P.kv_append(q, k, v, kc, vc, table, seq, pos, cos, sin, q_out=q)
    want = R.rotate(copy[:, :heads], cos[pos.long()], sin[pos.long()])
    assert torch.equal(fused[:, :heads].double(), want) and torch.equal(fused[:, heads:], copy[:, heads:])
    assert P.kv_append(None, k, v, kc, vc, table, seq, pos, cos, sin) is None


def test_tokens_outside_write_nothing_and_read_as_zeros():
    g = gen(3)
    kv, hd, page = 2, 64, 16
    kc, vc = make_cache("q8_0", 3, kv, page, hd, g)
    table = i32([[0, 1], [2, 3], [-1, 1]])  # page 3 and page -1 are outside
    seq, pos = i32([-1, 3, 0, 0, 1, 2]), i32([0, 0, -1, 32, 20, 3])
    n = 6
    q, k, v = (randn(n, h, hd, g=g) for h in (4, kv, kv))
    before = kc.clone(), vc.clone()
    cos, sin = tables(hd, 24)
    out = P.kv_append(q, k, v, kc, vc, table, seq, pos, cos, sin)
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])
    inside = (pos >= 0) & (pos < 24)
    assert torch.equal(out[~inside], q[~inside])
    assert torch.equal(out[inside].double(), R.rotate(q, cos[pos.long().clamp(0, 23)],
                                                      sin[pos.long().clamp(0, 23)])[inside])
    rk, rv = P.kv_read(kc, vc, table, seq, pos, hd)
    assert not rk.any() and not rv.any()


def test_q8_blocks_of_zeros_large_values_and_nan():
    kv, hd = 1, 64
    kc, vc = P.kv_cache("q8_0", 1, kv, 16, hd, DEV)
    k = torch.zeros((3, 1, hd), device=DEV)
    k[1, 0, :32] = torch.linspace(-1e6, 1e6, 32, device=DEV)
    k[1, 0, 40] = math.inf
    k[2, 0, 5] = math.nan
    k[2, 0, 32:] = 1.0
    table, seq, pos = i32([[0]]), i32([0, 0, 0]), i32([0, 1, 2])
    P.kv_append(None, k, torch.zeros_like(k), kc, vc, table, seq, pos)
    rk, rv = P.kv_read(kc, vc, table, seq, pos, hd)
    assert not rk[0].any() and not rv.any()
    assert float(rk[1].abs().max()) == R.KV_LIMIT and float(rk[1, 0, 40]) == R.KV_LIMIT
    assert torch.isnan(rk[2, 0, :32]).all() and torch.equal(rk[2, 0, 32:], R.cached_values(k[2:, :, 32:], "q8_0")[0, 0].float())


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def batch(new, past, heads, kv, hd, page, cache, dtype, seed=0, spare=2):
    """A batch's q, caches, block table, q_start, kv_len; unused rows of the caches hold NaN."""
    g = gen(seed)
    kv_len = [a + b for a, b in zip(new, past)]
    width = max(1, max(-(-max(x, 1) // page) for x in kv_len))
    pages = len(new) * width + spare
    kc, vc = make_cache(cache, pages, kv, page, hd, g)
    table = torch.randperm(pages, generator=g, device=DEV)[:len(new) * width].reshape(len(new), width).to(torch.int32)
    used = torch.zeros((pages, page), dtype=torch.bool, device=DEV)
    for s, length in enumerate(kv_len):
        pos = torch.arange(max(length, 0), device=DEV)
        used[table[s].long()[pos // page], pos % page] = True
    for c in (kc, vc):
        if cache == "bf16":
            c.masked_fill_(~used[:, None, :, None], math.nan)
        else:
            R.q8_parts(c)[1].masked_fill_(~used[:, None, :, None], math.nan)
    starts = [0]
    for a in new:
        starts.append(starts[-1] + a)
    q = (randn(starts[-1], heads, hd, g=g) * 1.5).to(dtype)
    return q, kc, vc, table, i32(starts), i32(kv_len)


def check(q, kc, vc, table, q_start, kv_len, out, scale=None):
    want, bound = R.attention(q, kc, vc, table, q_start.tolist(), kv_len.tolist(), scale)
    some = ~torch.isnan(bound)
    got = out.double()
    fine = torch.isfinite(want) & some
    assert torch.equal(torch.isfinite(got)[some], torch.isfinite(want)[some])
    over = ((got - want).abs() / bound)[fine]
    assert over.numel() == 0 or float(over.max()) <= 1.0, float(over.max())


SHAPES = [  # heads, kv_heads, head_dim, page
    (8, 4, 32, 16), (4, 4, 64, 32), (6, 1, 96, 16), (32, 8, 128, 64), (7, 7, 128, 16), (8, 2, 256, 32)]
BATCHES = [  # new tokens, tokens cached before
    ([1], [0]), ([1, 1, 1, 1], [0, 15, 16, 700]), ([5, 1, 3], [40, 2, 1000]), ([33, 2], [0, 70]), ([130], [300])]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cache", ["bf16", "q8_0"])
@pytest.mark.parametrize("heads,kv,hd,page", SHAPES)
@pytest.mark.parametrize("new,past", BATCHES)
def test_attention(new, past, heads, kv, hd, page, cache, dtype):
    b = batch(new, past, heads, kv, hd, page, cache, dtype, seed=hd + sum(new))
    check(*b, P.attention_paged(*b, max_q=max(new), max_kv=int(b[5].max())))
    if sum(new) < 10:  # loose bounds choose other launches
        check(*b, P.attention_paged(*b))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cache", ["bf16", "q8_0"])
def test_attention_of_long_sequences_is_split_and_merged(cache, dtype):
    b = batch([1, 4], [9001, 5000], 8, 2, 128, 64, cache, dtype, seed=5)
    first = P.attention_paged(*b, max_q=4, max_kv=9002)
    check(*b, first)
    for _ in range(5):  # the merge's order and its counters do not depend on the run
        assert torch.equal(P.attention_paged(*b, max_q=4, max_kv=9002), first)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cache", ["bf16", "q8_0"])
def test_attention_of_empty_sequences_and_tokens_that_see_nothing(cache, dtype):
    # no tokens; no keys; fewer keys than tokens: the first tokens see none
    new, past = [0, 2, 4, 0, 1], [30, -2, -3, 0, 5]
    b = batch(new, past, 4, 2, 64, 16, cache, dtype, seed=9)
    out = torch.full((sum(new) + 3, 4, 64), 7.0, device=DEV, dtype=dtype)
    q = torch.cat([b[0], torch.full((3, 4, 64), math.nan, device=DEV, dtype=dtype)])
    got = P.attention_paged(q, *b[1:], max_q=4, max_kv=40, out=out)
    assert got is out and bool((out[sum(new):] == 7.0).all())  # rows behind the last sequence
    check(*b, out[:sum(new)])
    assert not out[:2].any() and not out[2:5].any()


@pytest.mark.parametrize("cache", ["bf16", "q8_0"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(cache, bad, dtype):
    if cache == "q8_0" and bad != bad:
        bad = math.nan
    for new, past in (([40], [100]), ([200], [0]), ([3], [17])):
        b = batch(new, past, 4, 2, 64, 16, cache, dtype, seed=11)
        q, kc, vc, table = b[0], b[1], b[2], b[3]
        pos = past[0] + new[0] // 2  # a new token of the chunk
        page, off = int(table[0, pos // 16]), pos % 16
        if cache == "bf16":
            vc[page, 1, off, 3] = bad
        else:
            R.q8_parts(vc)[1][page, 1, off, 1] = bad
            R.q8_parts(vc)[0][page, 1, off, 32:].clamp_(min=1)
        out = P.attention_paged(*b, max_q=new[0], max_kv=new[0] + past[0])
        check(*b, out)
        assert bool(torch.isfinite(out[:new[0] // 2]).all()) and not bool(torch.isfinite(out[new[0] // 2:, 2:]).all())


@pytest.mark.parametrize("cache", ["bf16", "q8_0"])
def test_keys_that_are_not_finite_in_masked_places(cache):
    b = batch([20], [30], 4, 2, 64, 16, cache, BF16, seed=12)
    kc, table = b[1], b[3]
    page, off = int(table[0, 45 // 16]), 45 % 16
    if cache == "bf16":
        kc[page, 0, off] = math.inf
    else:
        R.q8_parts(kc)[1][page, 0, off] = math.nan
    out = P.attention_paged(*b, max_q=20, max_kv=50)
    clean = b[1].clone()
    if cache == "bf16":
        clean[page, 0, off] = 0
    else:
        R.q8_parts(clean)[1][page, 0, off] = 0
    ref = P.attention_paged(b[0], clean, *b[2:], max_q=20, max_kv=50)
    assert torch.equal(out[:15], ref[:15]) and torch.equal(out[:, 2:], ref[:, 2:])


def test_pages_outside_the_cache_read_as_zeros_and_pages_are_shared():
    b = batch([2, 3], [60, 90], 4, 2, 128, 16, "q8_0", F32, seed=13)
    table = b[3].clone()
    table[0, 1], table[0, 2], table[1, 0] = 10 ** 6, -5, table[0, 0]
    b = b[:3] + (table,) + b[4:]
    check(*b, P.attention_paged(*b, max_q=3, max_kv=93))


def test_kv_len_beyond_the_block_table_is_cut():
    b = batch([1, 1], [31, 15], 4, 2, 64, 16, "bf16", F32, seed=14)
    out = P.attention_paged(*b[:5], i32([10 ** 9, 16]), max_q=1, max_kv=32)
    check(*b, out)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_q_own_scale_and_in_place_output(dtype):
    b = batch([3, 1], [20, 33], 4, 2, 64, 16, "bf16", dtype, seed=15)
    wide = torch.zeros((4, 9, 64), device=DEV, dtype=dtype)
    wide[:, 2:6] = b[0]
    q = wide[:, 2:6]
    out = P.attention_paged(q, *b[1:], scale=0.37, out=q)
    assert out.data_ptr() == q.data_ptr()
    check(*b, out, scale=0.37)
    assert not wide[:, :2].any() and not wide[:, 6:].any()


@pytest.mark.parametrize("cache", ["bf16", "q8_0"])
def test_large_queries_and_scores(cache):
    """Scores of some hundreds: all weight on one key, and fp32 queries outside fp16's range."""
    b = batch([2], [200], 4, 2, 64, 16, cache, F32, seed=16)
    q = b[0] * 1e6
    out = P.attention_paged(q, *b[1:], max_q=2, max_kv=202)
    want, _ = R.attention(q, *b[1:4], b[4].tolist(), b[5].tolist())
    assert torch.isfinite(out).all() and float((out.double() - want).abs().max()) < 1e-5
    out = P.attention_paged(q * 0, *b[1:], max_q=2, max_kv=202)
    want, bound = R.attention(q * 0, *b[1:4], b[4].tolist(), b[5].tolist())
    assert bool(((out.double() - want).abs() <= bound).all())


def test_many_sequences():
    """More sequences than a warp's lanes: the tile search takes a second round."""
    new = [(s * 7) % 4 for s in range(75)]
    past = [(s * 37) % 90 for s in range(75)]
    b = batch(new, past, 4, 2, 64, 16, "bf16", F32, seed=17)
    check(*b, P.attention_paged(*b, max_q=3, max_kv=93))


def test_more_sequences_than_a_grid_s_second_dimension():
    """70000 sequences of a token or two over one shared table row, with the default bounds."""
    g = gen(33)
    kc, vc = make_cache("bf16", 4, 1, 16, 32, g)
    table = i32([[2, 0, 3]]).expand(70000, -1)
    n = 70000 + 65
    starts = torch.arange(70001, dtype=torch.int32, device=DEV)
    starts[40000:] += 65  # one of them has 66
    kv_len = torch.randint(1, 49, (70000,), generator=g, device=DEV).to(torch.int32)
    kv_len[39999] = 40
    q = randn(n, 1, 32, g=g, dtype=BF16)
    out = P.attention_paged(q, kc, vc, table, starts, kv_len)
    pick = [0, 1, 39998, 39999, 40000, 65535, 65536, 69999]
    rows = torch.cat([torch.arange(int(starts[s]), int(starts[s + 1]), device=DEV) for s in pick])
    sub = [0]
    for s in pick:
        sub.append(sub[-1] + int(starts[s + 1] - starts[s]))
    check(q[rows], kc, vc, table[:8], i32(sub), kv_len[torch.tensor(pick, device=DEV)], out[rows])


def test_bounds_above_any_length_are_taken_as_none():
    b = batch([2, 1], [100, 3], 4, 2, 64, 16, "bf16", F32, seed=34)
    want = P.attention_paged(*b)
    assert torch.equal(P.attention_paged(*b, max_q=2 ** 32, max_kv=2 ** 40), want)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes: its last pages."""
    pages, kv, page, hd = 17000, 8, 128, 128
    kc, vc = (torch.empty((pages, kv, page, hd), dtype=BF16, device=DEV) for _ in range(2))
    assert kc.numel() * 2 > 2 ** 32
    g = gen(18)
    table = i32([[pages - 1, pages - 2], [3, pages - 3]])
    for c in (kc, vc):
        for p in set(table.flatten().tolist()):
            c[p] = randn(kv, page, hd, g=g).to(BF16)
    new, kv_len = [2, 200], [150, 250]
    q = randn(202, 16, hd, g=g, dtype=BF16)
    out = P.attention_paged(q, kc, vc, table, i32([0, 2, 202]), i32(kv_len), max_q=200, max_kv=250)
    small_t = torch.tensor([[0, 1], [2, 3]], device=DEV, dtype=torch.int32)
    idx = table.flatten().long()
    check(q, kc[idx].contiguous(), vc[idx].contiguous(), small_t, i32([0, 2, 202]), i32(kv_len), out)


def test_two_streams_and_captured_calls_that_replay_together():
    b = batch([1, 1], [4000, 3000], 8, 2, 128, 64, "q8_0", BF16, seed=19)
    want = P.attention_paged(*b, max_q=1, max_kv=4001)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(8):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(P.attention_paged(*b, max_q=1, max_kv=4001))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs, gouts = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            gouts.append(P.attention_paged(*b, max_q=1, max_kv=4001))
        graphs.append(g)
    for _ in range(5):
        for o in gouts:
            o.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in gouts)


def test_own_workspace():
    b = batch([1], [3000], 8, 2, 128, 64, "bf16", F32, seed=20)
    need = P.attention_paged_workspace_nbytes(*b[1:4], 1, 8, 128, 1, 3001, F32)
    ws = torch.zeros(need, dtype=torch.uint8, device=DEV)
    out = P.attention_paged(*b, max_q=1, max_kv=3001, workspace=ws)
    check(*b, out)
    assert torch.equal(P.attention_paged(*b, max_q=1, max_kv=3001, workspace=ws), out)
    with pytest.raises(ValueError, match="workspace"):
        P.attention_paged(*b, max_q=1, max_kv=3001, workspace=ws[:need - 16])


@pytest.mark.parametrize("heads,kv,hd,page", [(32, 8, 128, 64), (6, 1, 96, 16), (40, 2, 64, 32)])
@pytest.mark.parametrize("cache", ["bf16", "q8_0"])
def test_long_and_short_sequences_in_one_batch(heads, kv, hd, page, cache):
    """Chunks, drafts, single tokens and sequences of none side by side: every
    sequence is taken by one of the kernels."""
    new = [200, 1, 0, 3, 64, 33, 17, 129, 1]
    b = batch(new, [100, 700, 30, 0, 50, 0, 15, 1000, 0], heads, kv, hd, page, cache, BF16, seed=21)
    out = torch.full_like(b[0], math.nan)
    P.attention_paged(*b, max_q=200, max_kv=1129, out=out)
    check(*b, out)
    check(*b, P.attention_paged(*b))  # loose bounds


@pytest.mark.parametrize("cache", ["bf16", "q8_0"])
def test_long_chunk_of_one_head_is_split_and_merged(cache):
    b = batch([150], [9000], 4, 1, 128, 64, cache, BF16, seed=22)
    out = P.attention_paged(*b, max_q=150, max_kv=9150)
    check(*b, out)
    for _ in range(3):
        assert torch.equal(P.attention_paged(*b, max_q=150, max_kv=9150), out)  # merged in a fixed order


def test_one_table_row_for_all_sequences():
    q, kc, vc, table, q_start, _ = batch([3, 3, 3], [40, 40, 40], 4, 2, 64, 16, "q8_0", F32, seed=23)
    rows, lens = table[1:2].expand(3, -1), i32([43, 43, 43])
    out = P.attention_paged(q, kc, vc, rows, q_start, lens, max_q=3, max_kv=43)
    check(q, kc, vc, rows, q_start, lens, out)
    k, v = P.kv_read(kc, vc, rows, i32([0, 1, 2]), i32([5, 5, 5]), 64)
    assert torch.equal(k[0], k[1]) and torch.equal(k[0], k[2])
    assert torch.equal(k[0].double(), R.values(kc)[int(table[1, 0]), :, 5])


def test_arguments_that_are_refused():
    q, kc, vc, table, q_start, kv_len = batch([2], [10], 4, 2, 64, 16, "bf16", F32, seed=24)
    seq, pos = i32([0, 0]), i32([10, 11])
    k, v = q[:, :2], q[:, 2:]
    cos, sin = tables(64, 32)
    ok = P.kv_append(q, k, v, kc, vc, table, seq, pos, cos, sin)
    assert ok.shape == q.shape
    half = torch.float16
    from dracort_b200.exceptions import DracoFormatError
    for err, call in [
            (ValueError, lambda: P.kv_append(q.to(half), k.to(half), v.to(half), kc, vc, table, seq, pos)),
            (ValueError, lambda: P.kv_append(q, k.bfloat16(), v, kc, vc, table, seq, pos)),
            (ValueError, lambda: P.kv_append(q, k, v, kc, vc, table, seq.long(), pos)),
            (ValueError, lambda: P.kv_append(q, k, v, kc, vc, table.long(), seq, pos)),
            (ValueError, lambda: P.kv_append(q, k, v, kc, vc, table.cpu(), seq, pos)),
            (ValueError, lambda: P.kv_append(q, k, v, kc, vc, table, seq, pos, cos)),
            (ValueError, lambda: P.kv_append(None, k, v, kc, vc, table, seq, pos, q_out=q)),
            (ValueError, lambda: P.kv_append(q.transpose(1, 2).contiguous().transpose(1, 2), k, v, kc, vc, table, seq,
                                             pos)),
            (DracoFormatError, lambda: P.kv_append(q, k, v[:1], kc, vc, table, seq, pos)),
            (DracoFormatError, lambda: P.kv_append(q, k[:, :1], v[:, :1], kc, vc, table, seq, pos)),
            (DracoFormatError, lambda: P.kv_append(q, k, v, kc, vc, table, seq[:1], pos)),
            (DracoFormatError, lambda: P.kv_append(q, k, v, kc, vc, table, seq, pos, cos[:, :16], sin[:, :16])),
            (DracoFormatError, lambda: P.kv_append(q, k, v, kc, vc[:-1], table, seq, pos)),
            (DracoFormatError, lambda: P.kv_append(q, k, v, kc, vc, table[0], seq, pos)),
            (DracoFormatError, lambda: P.kv_append(q[..., :32], k[..., :32], v[..., :32], kc, vc, table, seq, pos)),
            (ValueError, lambda: P.kv_append(q, k, v, kc.half(), vc.half(), table, seq, pos)),
            (ValueError, lambda: P.kv_read(kc, vc, table, seq, pos, 64, half)),
            (DracoFormatError, lambda: P.kv_read(kc, vc, table, seq, pos[:1], 64)),
            (DracoFormatError, lambda: P.kv_read(kc, vc, table, seq, pos, 32)),
            (ValueError, lambda: P.attention_paged(q.to(half), kc, vc, table, q_start, kv_len)),
            (DracoFormatError, lambda: P.attention_paged(q[:, :3], kc, vc, table, q_start, kv_len)),
            (DracoFormatError, lambda: P.attention_paged(q, kc, vc, table, q_start[:1], kv_len)),
            (DracoFormatError, lambda: P.attention_paged(q, kc, vc, table, q_start, i32([12, 12]))),
            (ValueError, lambda: P.attention_paged(q, kc, vc, table, q_start, kv_len, scale=0.0)),
            (ValueError, lambda: P.attention_paged(q, kc, vc, table, q_start, kv_len, scale=math.nan)),
            (ValueError, lambda: P.attention_paged(q, kc, vc, table, q_start, kv_len, out=q.bfloat16())),
            (DracoFormatError, lambda: P.attention_paged(q, kc, vc, table, q_start, kv_len, max_q=-1)),
            (DracoFormatError, lambda: P.attention_paged(q[:1].expand(2, -1, -1), kc, vc, table, q_start, kv_len,
                                                         out=q[:1].expand(2, -1, -1))),
            (ValueError, lambda: P.attention_paged(q, kc, vc, table, q_start, kv_len,
                                                   workspace=torch.zeros(64, dtype=torch.uint8)))]:
        with pytest.raises(err):
            call()
    a = verify_inputs([2, 1], 50, 1)
    for err, call in [
            (ValueError, lambda: P.verify_drafts(a[0].to(half), *a[1:5])),
            (ValueError, lambda: P.verify_drafts(a[0], a[1], a[2].long(), *a[3:5])),
            (ValueError, lambda: P.verify_drafts(*a[:5], temperature=-1.0)),
            (ValueError, lambda: P.verify_drafts(*a[:5], max_rows=0)),
            (ValueError, lambda: P.verify_drafts(*a[:5], draft_probs=a[5].double())),
            (DracoFormatError, lambda: P.verify_drafts(*a[:5], draft_probs=a[5][:, 1:])),
            (DracoFormatError, lambda: P.verify_drafts(a[0].t(), *a[1:5])),
            (DracoFormatError, lambda: P.verify_drafts(*a[:4], a[4][:1])),
            (DracoFormatError, lambda: P.verify_drafts(a[0], a[1][0], *a[2:5]))]:
        with pytest.raises(err):
            call()


def test_status_of_the_workspaces():
    b = batch([1], [300], 8, 2, 128, 64, "bf16", F32, seed=25)
    P.attention_paged(*b)
    assert P.attention_paged_status() == 0
    ws = torch.zeros(P.attention_paged_workspace_nbytes(*b[1:4], 1, 8, 128, 1, 301, F32), dtype=torch.uint8, device=DEV)
    ws[8192] = 5  # as a kernel records it
    assert P.attention_paged_status(ws) == 5
    assert P.attention_paged_status(ws) == 0 and int(ws.sum()) == 0
    check(*b, P.attention_paged(*b, max_q=1, max_kv=301, workspace=ws))


# ---------------------------------------------------------------------------
# a serving step: append, attend, verify
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cache", ["bf16", "q8_0"])
def test_a_step_of_prompts_drafts_and_single_tokens(cache, dtype):
    """The operators as a step runs them, eager and replayed from a graph whose
    inputs change: each is compared with its statement on what it was given."""
    heads, kv, hd, page, vocab = 8, 2, 64, 16, 500
    new, past = [5, 1, 80, 3], [60, 33, 0, 15]
    g = gen(31)
    n, seqs = sum(new), len(new)
    kc, vc = make_cache(cache, 40, kv, page, hd, g)
    table = torch.randperm(40, generator=g, device=DEV)[:24].reshape(4, 6).to(torch.int32)
    cos, sin = tables(hd, 128)
    head = randn(heads * hd, vocab, g=g) * 0.2
    starts = [0]
    for a in new:
        starts.append(starts[-1] + a)
    q_start = i32(starts)
    seq = i32([s for s in range(seqs) for _ in range(new[s])])
    pos, kv_len = i32([0] * n), i32([0] * seqs)
    qkv = torch.zeros(n, heads + 2 * kv, hd, dtype=dtype, device=DEV)
    drafts, au, su = i32([0] * n), torch.zeros(n, device=DEV), torch.zeros(seqs, device=DEV)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]

    def step():
        rq = P.kv_append(q, k, v, kc, vc, table, seq, pos, cos, sin)
        o = P.attention_paged(rq, kc, vc, table, q_start, kv_len, max_q=80, max_kv=96)
        logits = torch.matmul(o.reshape(n, -1).float(), head)
        return rq, o, logits, P.verify_drafts(logits, q_start, drafts, au, su, temperature=0.9, max_rows=80)

    def fill(seed):
        gg = gen(seed)
        at = [p + seed % 3 for p in past]
        qkv.copy_(randn(n, heads + 2 * kv, hd, g=gg, dtype=dtype))
        pos.copy_(i32([at[s] + j for s in range(seqs) for j in range(new[s])]))
        kv_len.copy_(i32([at[s] + new[s] for s in range(seqs)]))
        drafts.copy_(torch.randint(0, 8, (n,), generator=gg, device=DEV).to(torch.int32))
        au.copy_(torch.rand(n, generator=gg, device=DEV) * 0.02)
        su.copy_(torch.rand(seqs, generator=gg, device=DEV))

    def verify_step(got):
        rq, o, logits, (count, tokens) = got
        # the largest count of accepted drafts and the tokens
        want_c, want_t, margin = R.verify(logits.cpu(), q_start.cpu(), drafts.cpu(), au.cpu(), su.cpu(), None, 0.9, 80)
        assert margin > 1e-6
        assert count.tolist() == want_c and tokens.tolist() == want_t
        check(rq, kc, vc, table, q_start, kv_len, o)
        ck, cv = P.kv_read(kc, vc, table, seq, pos, hd)
        at = pos.long()
        assert torch.equal(ck.double(), R.cached_values(R.rotate(k, cos[at], sin[at]), cache))
        assert torch.equal(cv.double(), R.cached_values(v, cache))
        turned = R.rotate(q, cos[at], sin[at])
        assert torch.equal(rq.double(), turned.to(dtype).double())

    fill(0)
    step()  # (the matrix product's own workspace is made outside the capture)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(1, 4):
        fill(seed)
        graph.replay()
        verify_step(captured)
        eager = step()
        verify_step(eager)
        assert torch.equal(eager[1], captured[1]) and torch.equal(eager[3][1], captured[3][1])


# ---------------------------------------------------------------------------
# verification of drafts
# ---------------------------------------------------------------------------
def verify_inputs(rows, vocab, seed, dtype=F32, probs=True, near=0.5):
    g = gen(seed)
    n = sum(rows)
    logits = randn(n, vocab, g=g) * 2
    logits.scatter_add_(1, torch.randint(0, vocab, (n, 3), generator=g, device=DEV),
                        torch.tensor([8.0, 7.0, 6.0], device=DEV).expand(n, 3).contiguous())
    logits = logits.to(dtype)
    q = torch.softmax(logits.float() + near * randn(n, vocab, g=g), -1)
    drafts = torch.multinomial(q, 1, generator=g)[:, 0].to(torch.int32)
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    return (logits, i32(starts), drafts, torch.rand(n, generator=g, device=DEV),
            torch.rand(len(rows), generator=g, device=DEV), q if probs else None)


@pytest.mark.parametrize("vocab", [1, 7, 509, 32000, 128001])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0])
def test_verify(vocab, dtype, probs, temperature):
    rows = [5, 1, 3, 0, 8, 2]
    for seed in range(3):
        a = verify_inputs(rows, vocab, 100 * seed + vocab, dtype, probs)
        count, tokens = P.verify_drafts(*a[:5], draft_probs=a[5], temperature=temperature, max_rows=8)
        want_c, want_t, margin = R.verify(*[x.cpu() if x is not None else None for x in a], temperature, 8)
        assert margin > 1e-6 or temperature == 0.0
        assert count.tolist() == want_c and tokens.tolist() == want_t


def test_verify_takes_drafts_with_the_target_s_probability():
    """With q = p every draft is taken; frequencies of plain sampling follow p."""
    a = verify_inputs([4] * 8, 1000, 3, near=0.0)
    count, tokens = P.verify_drafts(*a[:5], draft_probs=a[5] * (1 - 1e-5), max_rows=4)
    assert count.tolist() == [3] * 8
    n, vocab = 20000, 5
    p = torch.tensor([0.5, 0.25, 0.0, 0.2, 0.05], device=DEV)
    logits = p.log()[None].expand(n, vocab)
    u = (torch.arange(n, device=DEV) + 0.5) / n
    _, t = P.verify_drafts(logits, torch.arange(n + 1, dtype=torch.int32, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV),
                           torch.zeros(n, device=DEV), u, max_rows=1)
    got = torch.bincount(t[:, 0].long(), minlength=vocab).double() / n
    assert float((got - p.double()).abs().max()) <= 1.5 / n  # evenly spaced u: at most one off at a border


def test_verify_at_the_edges():
    inf = math.inf
    logits = torch.tensor([[0.0, 5.0, 5.0, -inf], [inf, 0.0, inf, 1.0], [-inf] * 4, [math.nan, 1.0, math.nan, 0.0],
                           [1.0, 1.0, 1.0, 1.0], [0.0, 0.0, 9.0, 0.0]], device=DEV)
    one = torch.ones(6, dtype=torch.float32, device=DEV)
    starts = i32([0, 1, 2, 3, 4, 6])
    u = torch.tensor([0.99999, 0.6, 0.5, 0.999999, 0.0], device=DEV)
    for t in (1.0, 0.0):
        args = (logits, starts, i32([0, 0, 0, 0, 7, 0]), one * 0, u)
        count, tokens = P.verify_drafts(*args, temperature=t, max_rows=3)
        want = R.verify(*[x.cpu() for x in args], None, t, 3)
        assert count.tolist() == want[0] and tokens.tolist() == want[1]
        assert tokens[2].tolist() == [-1, -1, -1]  # no token in a row of -infinity
        assert count[4] == 0  # a draft outside the vocabulary
    # a rejected certain draft is not drawn again; u at its ends
    two = torch.tensor([[2.0, 2.0], [0.0, 0.0]], device=DEV)
    for us in (0.0, 0.5, 0.99999994):
        c, t = P.verify_drafts(two, i32([0, 2]), i32([1, 0]), torch.tensor([0.75, 0.0], device=DEV),
                               torch.tensor([us], device=DEV), max_rows=2)
        assert c.tolist() == [0] and t.tolist() == [[0, -1]]
    # p <= q everywhere: drawn from p
    q = torch.tensor([[1.0, 1.0], [0.0, 0.0]], device=DEV)
    c, t = P.verify_drafts(two, i32([0, 2]), i32([0, 0]), torch.tensor([0.75, 0.0], device=DEV),
                           torch.tensor([0.75], device=DEV), draft_probs=q, max_rows=2)
    assert c.tolist() == [0] and t.tolist() == [[1, -1]]


def test_verify_of_more_rows_than_are_held_at_a_time_and_strided_logits():
    a = verify_inputs([150], 300, 4, near=0.0, probs=True)
    wide = torch.full((150, 331), math.nan, device=DEV)
    wide[:, 5:305] = a[0]
    probs = a[5] * (1 - 1e-5)
    args = (wide[:, 5:305], *a[1:5])
    count, tokens = P.verify_drafts(*args, draft_probs=probs, max_rows=150)
    want = R.verify(*[x.cpu() for x in (a[0], *a[1:5], probs)], 1.0, 150)
    assert count.tolist() == want[0] == [149] and tokens.tolist() == want[1]
    count, short = P.verify_drafts(*args, draft_probs=probs, max_rows=10)
    assert count.tolist() == [149] and short.tolist() == [want[1][0][:10]]


@pytest.mark.parametrize("temperature", [1e-29, 1e-18, 1e-9, 1e-3, 1e29])
@pytest.mark.parametrize("offset", [0.0, 37.0, -3e4, 1e30])
def test_verify_at_extreme_temperatures_and_logits(temperature, offset):
    """Nearly greedy and nearly uniform, with logits far from zero: the two
    largest are equal, and share the weight when the others have none."""
    n, vocab = 64, 1000
    g = gen(35)
    logits = randn(n, vocab, g=g) + offset
    top = logits.amax(-1, keepdim=True) + 1.0
    logits.scatter_(1, torch.tensor([[300, 700]], device=DEV).expand(n, 2), top.expand(n, 2))
    u = (torch.arange(n, device=DEV) + 0.5) / n
    starts = torch.arange(n + 1, dtype=torch.int32, device=DEV)
    _, t = P.verify_drafts(logits, starts, i32([0] * n), torch.zeros(n, device=DEV), u, temperature=temperature,
                           max_rows=1)
    _, want, margin = R.verify(logits.cpu(), starts.cpu(), torch.zeros(n, dtype=torch.int32), torch.zeros(n), u.cpu(),
                               None, float(torch.tensor(temperature, dtype=torch.float32)), 1)
    assert margin > 1e-9 and t.tolist() == want


def test_verify_of_no_rows_at_all():
    for t in (0.0, 1.0):
        count, tokens = P.verify_drafts(torch.zeros((0, 50), device=DEV), i32([0, 0, 0]), i32([]),
                                        torch.zeros(0, device=DEV), torch.zeros(2, device=DEV), temperature=t,
                                        max_rows=3)
        assert count.tolist() == [0, 0] and tokens.tolist() == [[-1] * 3] * 2
    count, tokens = P.verify_drafts(torch.zeros((0, 50), device=DEV), i32([0]), i32([]), torch.zeros(0, device=DEV),
                                    torch.zeros(0, device=DEV))
    assert count.shape == (0,) and tokens.shape == (0, 1)


def test_verify_in_a_graph():
    a = verify_inputs([5, 3], 4000, 6)
    want = P.verify_drafts(*a[:5], draft_probs=a[5], max_rows=5)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = P.verify_drafts(*a[:5], draft_probs=a[5], max_rows=5)
    for _ in range(3):
        got[0].zero_(), got[1].zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
