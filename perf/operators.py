"""Serving operators over a paged key/value cache: workloads, plain forms and work counts.

Four kinds of case:

* ``write``  - new keys and values of some sequences are rotated (rotate-half
  RoPE), rounded to the cache's type (bf16, or Q8_0 blocks of 32) and written
  to the sequences' pages; then the same rows are read back as values.
* ``read``   - rows of a filled cache are read back as dense values (moving a
  sequence elsewhere, sharing a prefix).
* ``attend`` - causal attention of each sequence's newest tokens over all of
  its cached keys: one token (a decode step), a few (drafted tokens), a chunk
  of a prompt, or a whole prompt; grouped-query heads, ragged lengths.
* ``verify`` - drafted tokens are accepted or rejected against the target's
  probabilities from given random numbers, and the token after the last
  accepted one is drawn.

The cache of one layer is two buffers (keys, values) of pages
``[pages][kv_heads][page][head_dim]``: bf16 values, or for Q8_0, per page and
head, ``page * head_dim`` int8 quants followed by ``page * head_dim / 32``
fp16 scales (``value = scale * quant``).  A block table gives each sequence's
pages.
"""

import math
import random

import torch

own = False

KV_LIMIT = 65024.0  # Q8_0 cache values are clamped to +-65024 = 127 * 512
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _write(name, seqs, lo, hi, heads, kv_heads, head_dim, page, cache, dtype, mix):
    return {"name": name, "kind": "write", "seqs": seqs, "new_lo": lo, "new_hi": hi, "past_lo": 0, "past_hi": 2000,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "cache": cache, "dtype": dtype,
            "mix": mix}


def _read(name, rows, kv_heads, head_dim, page, cache, dtype, mix):
    return {"name": name, "kind": "read", "seqs": 1, "new_lo": rows, "new_hi": rows, "past_lo": 0, "past_hi": 0,
            "heads": kv_heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "cache": cache,
            "dtype": dtype, "mix": mix}


def _attend(name, seqs, new, past, heads, kv_heads, head_dim, page, cache, dtype, mix):
    return {"name": name, "kind": "attend", "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "past_lo": past[0],
            "past_hi": past[1], "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "cache": cache, "dtype": dtype, "mix": mix}


def _verify(name, seqs, lo, hi, vocab, probs, temperature, dtype, mix):
    return {"name": name, "kind": "verify", "seqs": seqs, "rows_lo": lo, "rows_hi": hi, "vocab": vocab,
            "draft_probs": probs, "temperature": temperature, "dtype": dtype, "mix": mix}


def listed():
    return [
        # one decode step's append for one sequence of a 32-head model: latency
        _write("write_step", 1, 1, 1, 32, 32, 128, 64, "bf16", "float32", 1),
        # a whole batch's prompts enter a quantised cache
        _write("write_prompts_q8", 7, 300, 2100, 32, 8, 128, 64, "q8_0", "bfloat16", 2),
        # a ragged chunk of a small model, small pages
        _write("write_ragged_q8", 5, 3, 40, 8, 4, 32, 16, "q8_0", "float32", 3),
        # a long sequence leaves the quantised cache as bf16
        _read("read_long_q8", 20011, 8, 128, 64, "q8_0", "bfloat16", 4),
        # a short prefix is read as fp32
        _read("read_prefix", 333, 32, 128, 32, "bf16", "float32", 5),
        # a decode step of one sequence with 1024 cached positions, fp32 activations
        _attend("decode_one", 1, (1, 1), (1024, 1024), 32, 32, 128, 64, "bf16", "float32", 6),
        # a decode step of a serving batch over long quantised caches
        _attend("decode_batch_q8", 48, (1, 1), (900, 8000), 32, 8, 128, 64, "q8_0", "bfloat16", 7),
        # drafted tokens of several sequences at once
        _attend("drafts_q8", 9, (4, 7), (100, 6000), 32, 8, 128, 32, "q8_0", "float32", 8),
        # whole prompts of different lengths
        _attend("prompts", 4, (700, 4000), (0, 0), 32, 8, 128, 64, "bf16", "bfloat16", 9),
        # the next chunk of a long prompt over a quantised cache
        _attend("chunk_q8", 1, (512, 512), (16384, 16384), 32, 8, 128, 64, "q8_0", "bfloat16", 10),
        # a few drafts looked up in the text (no draft probabilities)
        _verify("verify_lookup", 1, 5, 5, 32000, False, 1.0, "float32", 11),
        # a batch of draft-model proposals over a large vocabulary
        _verify("verify_batch", 48, 2, 8, 128000, True, 0.8, "float32", 12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def _draw(rng):
    kind = rng.choice(["write", "write", "read", "attend", "attend", "attend", "attend", "verify", "verify"])
    mix = rng.randrange(1 << 20)
    dtype = rng.choice(["float32", "bfloat16"])
    if kind == "verify":
        lo = rng.randint(1, 3)
        return _verify("", _log_int(rng, 1, 48), lo, lo + rng.randint(0, 6), _log_int(rng, 500, 128000),
                       rng.random() < 0.5, rng.choice([0.0, 0.6, 1.0, 1.3]), dtype, mix)
    head_dim = rng.choice([32, 64, 96, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16, 32])
    heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 6, 7, 8) if g * kv_heads <= 64])
    page, cache = rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "q8_0"])
    if kind == "read":
        return _read("", _log_int(rng, 1, 20011), kv_heads, head_dim, page, cache, dtype, mix)
    if kind == "write":
        lo = _log_int(rng, 1, 1000)
        return _write("", _log_int(rng, 1, 48), lo, lo + rng.randint(0, lo), heads, kv_heads, head_dim, page, cache,
                      dtype, mix)
    form = rng.choice(["step", "drafts", "chunk", "prompt"])
    if form == "step":
        new, seqs, past = (1, 1), _log_int(rng, 1, 64), _log_int(rng, 1, 16384)
    elif form == "drafts":
        new, seqs, past = (rng.randint(1, 4), rng.randint(4, 9)), _log_int(rng, 1, 32), _log_int(rng, 1, 8192)
    elif form == "chunk":
        n = _log_int(rng, 10, 600)
        new, seqs, past = (rng.randint(1, n), n), _log_int(rng, 1, 6), _log_int(rng, 1, 16384)
    else:
        n = _log_int(rng, 10, 4000)
        new, seqs, past = (rng.randint(1, n), n), _log_int(rng, 1, 6), 0
    return _attend("", seqs, new, (past // rng.randint(1, 8), past), heads, kv_heads, head_dim, page, cache, dtype,
                   mix)


def _largest(kind):
    """(weight, padded scores) of the largest listed case of a kind."""
    ws = [(_weight(c), _padded(c)) for c in listed() if c["kind"] == kind]
    return max(w for w, _ in ws), max(p for _, p in ws)


def _weight(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 200.0)


def _padded(case):
    if case["kind"] != "attend":
        return 0
    new, past = lengths(case)
    return case["seqs"] * case["heads"] * max(new) * max(n + p for n, p in zip(new, past))


def draw(rng):
    while True:
        case = _draw(rng)
        weight, padded = _largest(case["kind"])
        if _weight(case) <= weight and _padded(case) <= padded:
            case.pop("name")
            return case


def lengths(case):
    """(new, past): tokens of this pass and tokens already cached, per sequence (verify: rows, None)."""
    rng = random.Random(case["mix"])
    if case["kind"] == "verify":
        return [rng.randint(case["rows_lo"], case["rows_hi"]) for _ in range(case["seqs"])], None
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    past = [rng.randint(case["past_lo"], case["past_hi"]) for _ in range(case["seqs"])]
    return new, past


def _row_bytes(case):
    """Cache bytes of one key (or value) row of one head."""
    return case["head_dim"] * 2 if case["cache"] == "bf16" else case["head_dim"] // 32 * 34


def work(case):
    new, past = lengths(case)
    n = sum(new)
    es = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "verify":
        rows = n * case["vocab"] * es
        return {"bytes": rows + (case["seqs"] * case["vocab"] * 4 if case["draft_probs"] else 0) + 12 * n,
                "flops": 3 * n * case["vocab"]}
    h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    cached = 2 * kv * _row_bytes(case)  # a position's key and value rows
    if case["kind"] == "read":
        return {"bytes": n * (cached + 2 * kv * hd * es), "flops": n * 2 * kv * hd}
    if case["kind"] == "write":
        activations = n * (2 * h + 2 * kv) * hd * es  # q in and out, k, v
        return {"bytes": activations + n * hd * 4 + 2 * n * cached + n * 2 * kv * hd * 4,
                "flops": n * (h + kv) * hd * 3 + n * 2 * kv * hd * 3}
    total = sum(a + p for a, p in zip(new, past))
    pairs = sum(a * p + a * (a + 1) // 2 for a, p in zip(new, past))
    return {"bytes": total * cached + 2 * n * h * hd * es, "flops": 4 * hd * h * pairs}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def quantise(x):
    """Q8_0 blocks of 32 along the last dimension: (int8 quants, fp16 scales).  scale = max|x| / 127."""
    b = x.float().clamp(-KV_LIMIT, KV_LIMIT).unflatten(-1, (-1, 32))
    d = b.abs().amax(-1, keepdim=True).clamp_min(1e-12) / torch.full((), 127.0, device=x.device)
    q = torch.round(b / d).nan_to_num(0.0).clamp(-127, 127)
    return q.flatten(-2).to(torch.int8), d.squeeze(-1).to(torch.float16)


def pack_q8(x):
    """[pages, kv_heads, page, head_dim] values -> the Q8_0 cache buffer (uint8, page rows of head_dim / 32 * 34 bytes)."""
    pages, kv, page, hd = x.shape
    q, d = quantise(x)
    flat = torch.cat([q.reshape(pages, kv, -1).view(torch.uint8), d.reshape(pages, kv, -1).view(torch.uint8)], -1)
    return flat.reshape(pages, kv, page, hd // 32 * 34)


def unpack_q8(buf):
    """The values of a Q8_0 cache buffer, fp32 [pages, kv_heads, page, head_dim]."""
    pages, kv, page, rb = buf.shape
    hd = rb // 34 * 32
    flat = buf.reshape(pages, kv, -1)
    q = flat[..., :page * hd].view(torch.int8).reshape(pages, kv, page, hd // 32, 32)
    d = flat[..., page * hd:].view(torch.float16).reshape(pages, kv, page, hd // 32, 1)
    return (d.float() * q.float()).reshape(pages, kv, page, hd)


def _cache(case, pages, gen, dev):
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
    x = torch.randn(shape, generator=gen, device=dev)
    return x.to(torch.bfloat16) if case["cache"] == "bf16" else pack_q8(x)


def _int32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _starts(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed * 1000003 + case["mix"])
    dtype = DTYPES[case["dtype"]]
    new, past = lengths(case)
    starts, n = _starts(new), sum(new)
    if case["kind"] == "verify":
        return _prepare_verify(case, new, starts, gen, dev, dtype)
    h, kv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    kv_len = [a + p for a, p in zip(new, past)]
    width = max(-(-k // page) for k in kv_len)
    pages = case["seqs"] * width + 3
    table = torch.randperm(pages, generator=gen, device=dev)[:case["seqs"] * width].reshape(case["seqs"], width)
    state = {"kind": case["kind"], "head_dim": hd, "dtype": dtype, "table": table.to(torch.int32).contiguous(),
             "k_cache": _cache(case, pages, gen, dev), "v_cache": _cache(case, pages, gen, dev),
             "start": _int32(starts, dev), "kv_len": _int32(kv_len, dev), "max_q": max(new), "max_kv": max(kv_len)}
    if case["kind"] != "attend":
        state["seq"] = _int32([s for s, c in enumerate(new) for _ in range(c)], dev)
        state["pos"] = _int32([p + i for c, p in zip(new, past) for i in range(c)], dev)
    if case["kind"] != "read":
        state["q"] = (torch.randn((n, h, hd), generator=gen, device=dev) * 1.5).to(dtype)
    if case["kind"] == "write":
        state["k"] = torch.randn((n, kv, hd), generator=gen, device=dev).to(dtype)
        state["v"] = torch.randn((n, kv, hd), generator=gen, device=dev).to(dtype)
        # a channel or two of a key is far larger than the rest
        state["k"][..., hd // 2 - 1] *= 12
        angle = (torch.arange(max(kv_len), device=dev, dtype=torch.float64)[:, None]
                 * 10000.0 ** (-torch.arange(0, hd, 2, device=dev, dtype=torch.float64) / hd))
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    return state


def _prepare_verify(case, rows, starts, gen, dev, dtype):
    n, vocab = sum(rows), case["vocab"]
    logits = torch.randn((n, vocab), generator=gen, device=dev) * 2.0
    top = torch.randint(0, vocab, (n, 4), generator=gen, device=dev)
    logits.scatter_add_(1, top, torch.tensor([9.0, 8.0, 7.0, 6.0], device=dev).expand(n, 4).contiguous())
    logits = logits.to(dtype)
    state = {"kind": "verify", "logits": logits, "start": _int32(starts, dev), "max_rows": max(rows),
             "temperature": case["temperature"], "draft_probs": None,
             "accept_u": torch.rand(n, generator=gen, device=dev),
             "sample_u": torch.rand(case["seqs"], generator=gen, device=dev)}
    # proposals of a model whose logits are near the target's
    near = logits.float() + torch.randn((n, vocab), generator=gen, device=dev) * 0.5
    probs = torch.softmax(near, -1)
    state["drafts"] = torch.multinomial(probs, 1, generator=gen)[:, 0].to(torch.int32)
    if case["draft_probs"]:
        state["draft_probs"] = probs
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else PLAIN[state["kind"]](state)


def _run_own(s):
    from dracort_b200 import paged_ops as P

    if s["kind"] == "write":
        q = P.kv_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["seq"], s["pos"], s["cos"],
                        s["sin"])
        return (q,) + P.kv_read(s["k_cache"], s["v_cache"], s["table"], s["seq"], s["pos"], s["head_dim"],
                                torch.float32)
    if s["kind"] == "read":
        return P.kv_read(s["k_cache"], s["v_cache"], s["table"], s["seq"], s["pos"], s["head_dim"], s["dtype"])
    if s["kind"] == "attend":
        return P.attention_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["start"], s["kv_len"],
                                 max_q=s["max_q"], max_kv=s["max_kv"])
    return P.verify_drafts(s["logits"], s["start"], s["drafts"], s["accept_u"], s["sample_u"],
                           draft_probs=s["draft_probs"], temperature=s["temperature"], max_rows=s["max_rows"])


def _rotate(x, cos, sin):
    """Rotate-half RoPE in fp32: products and sums each rounded once."""
    a, b = x.float().chunk(2, -1)
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _plain_write(s):
    cos, sin = s["cos"][s["pos"].long()], s["sin"][s["pos"].long()]
    q = _rotate(s["q"], cos, sin).to(s["q"].dtype)
    page, offset = _places(s, s["seq"].long(), s["pos"].long())
    _store(s["k_cache"], _rotate(s["k"], cos, sin), page, offset)
    _store(s["v_cache"], s["v"].float(), page, offset)
    return q, _rows(s["k_cache"], page, offset, torch.float32), _rows(s["v_cache"], page, offset, torch.float32)


def _places(s, seq, pos):
    size = s["k_cache"].shape[2]
    return s["table"].long()[seq, pos // size], pos % size


def _store(cache, x, page, offset):
    """Write x [n, kv_heads, head_dim] to the rows (page, offset) of every head."""
    if cache.dtype == torch.bfloat16:
        cache[page, :, offset] = x.to(torch.bfloat16)
        return
    quants, scales = _q8_views(cache, x.shape[-1])
    q, d = quantise(x)
    quants[page, :, offset] = q
    scales[page, :, offset] = d


def _q8_views(cache, hd):
    pages, kv, page, _ = cache.shape
    flat = cache.view(pages, kv, -1)
    return (flat[..., :page * hd].view(torch.int8).unflatten(-1, (page, hd)),
            flat[..., page * hd:].view(torch.float16).unflatten(-1, (page, hd // 32)))


def _rows(cache, page, offset, dtype):
    if cache.dtype == torch.bfloat16:
        return cache[page, :, offset].to(dtype)
    quants, scales = _q8_views(cache, cache.shape[-1] // 34 * 32)
    q, d = quants[page, :, offset], scales[page, :, offset]
    return (q.float().unflatten(-1, (-1, 32)) * d.float()[..., None]).flatten(-2).to(dtype)


def _plain_read(s):
    page, offset = _places(s, s["seq"].long(), s["pos"].long())
    return _rows(s["k_cache"], page, offset, s["dtype"]), _rows(s["v_cache"], page, offset, s["dtype"])


def _plain_attend(s):
    """softmax(q K^T / sqrt(head_dim)) V over sequences padded to the longest, in fp32."""
    dev, dtype = s["q"].device, s["q"].dtype
    start, kv_len = s["start"].long(), s["kv_len"].long()
    new = start[1:] - start[:-1]
    n, heads, hd = s["q"].shape
    kv, seqs, max_q, max_kv = s["k_cache"].shape[1], len(kv_len), s["max_q"], s["max_kv"]
    rows, keys = torch.arange(max_q, device=dev), torch.arange(max_kv, device=dev)
    q = s["q"][(start[:-1, None] + rows).clamp_max(n - 1)].float()  # [seqs, max_q, heads, hd]
    q = q.unflatten(2, (kv, -1)).permute(0, 2, 3, 1, 4).reshape(seqs, kv, -1, hd)
    at = torch.minimum(keys, kv_len[:, None] - 1)
    page, offset = _places(s, torch.arange(seqs, device=dev)[:, None], at)
    k = _rows(s["k_cache"], page, offset, torch.float32).transpose(1, 2)  # [seqs, kv, max_kv, hd]
    scores = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(hd))
    last = (kv_len - new)[:, None] + rows  # the last key that each row sees
    seen = (keys <= last[..., None]) & (keys < kv_len[:, None, None])
    scores = scores.view(seqs, kv, -1, max_q, max_kv).masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    p = scores.exp_()
    total = p.sum(-1, keepdim=True)
    v = _rows(s["v_cache"], page, offset, torch.float32).transpose(1, 2)
    o = (p.view(seqs, kv, -1, max_kv) @ v).view(seqs, kv, -1, max_q, hd) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs, max_q, heads, hd)
    token = torch.arange(n, device=dev)
    seq = torch.searchsorted(start, token, right=True) - 1
    return o[seq, token - start[seq]].to(dtype)


def _plain_verify(s):
    """Accept draft i while u_i * q_i < p_i; then draw from max(p - q, 0) of the first rejected row, or from p of the last row."""
    dev, start = s["logits"].device, s["start"].long()
    n, vocab = s["logits"].shape
    row = torch.arange(n, device=dev)
    seqs = len(start) - 1
    seq = torch.searchsorted(start, row, right=True) - 1
    drafts, is_draft = s["drafts"].long(), row + 1 < start[seq + 1]
    logits = s["logits"].double()
    if s["temperature"] == 0.0:
        best = logits.argmax(-1)
        taken = is_draft & (best == drafts)
    else:
        p = torch.softmax(logits / s["temperature"], -1)
        px = p.gather(1, drafts[:, None])[:, 0]
        qx = 1.0 if s["draft_probs"] is None else s["draft_probs"].gather(1, drafts[:, None])[:, 0].double()
        taken = is_draft & (s["accept_u"].double() * qx < px)
    # accepted drafts of a sequence: its rows before the first one that is not taken
    count = torch.full((seqs,), vocab + n, device=dev, dtype=torch.long)
    place = torch.where(taken, vocab + n, row - start[seq])
    count = count.scatter_reduce(0, seq, place, "amin")
    at = start[:-1] + count
    if s["temperature"] == 0.0:
        last = best[at]
    else:
        w = p[at]
        rejected = is_draft[at]
        if s["draft_probs"] is None:
            gone = torch.zeros_like(w).scatter_(1, drafts[at][:, None], w.gather(1, drafts[at][:, None]))
        else:
            gone = s["draft_probs"][at].double()
        left = (w - torch.where(rejected[:, None], gone, 0.0)).clamp_min(0.0)
        left = torch.where(left.sum(-1, keepdim=True) > 0, left, w)
        upto = left.cumsum(-1)
        over = upto > s["sample_u"].double()[:, None] * upto[:, -1:]
        last = over.int().argmax(-1)
    j = torch.arange(s["max_rows"], device=dev)
    given = drafts[(start[:-1, None] + j).clamp_max(n - 1)]
    tokens = torch.where(j < count[:, None], given, torch.where(j == count[:, None], last[:, None], -1))
    return count.to(torch.int32), tokens.to(torch.int32)


PLAIN = {"write": _plain_write, "read": _plain_read, "attend": _plain_attend, "verify": _plain_verify}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"write": _exact_write, "read": _exact_read, "attend": _exact_attend, "verify": _exact_verify}[
        case["kind"]](s)


def _values64(cache):
    return cache.double() if cache.dtype == torch.bfloat16 else unpack_q8(cache).double()


def _turned64(x, cos, sin):
    half = x.shape[-1] // 2
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for j in range(half):
        c, n = cos[:, j, None].double(), sin[:, j, None].double()
        a, b = x[..., j].double(), x[..., j + half].double()
        out[..., j], out[..., j + half] = a * c - b * n, b * c + a * n
    return out


def _to32(x):
    """64-bit numbers rounded once to 32 bits."""
    return x.to(torch.float32).double()


def _key64(k, cos, sin):
    """The rotated key that the cache's rounding starts from: by definition its products and its sum are 32-bit numbers."""
    half = k.shape[-1] // 2
    a, b, c, n = k[..., :half].double(), k[..., half:].double(), cos[:, None].double(), sin[:, None].double()
    return torch.cat([_to32(_to32(a * c) - _to32(b * n)), _to32(_to32(b * c) + _to32(a * n))], -1)


def _rounded64(x, kind):
    """The values that a cache of this kind holds for 32-bit numbers x.  A block's scale and its
    quotients are 32-bit numbers by the block format's definition."""
    if kind == torch.bfloat16:
        return x.to(torch.bfloat16).double()
    out = torch.empty_like(x)
    for b in range(0, x.shape[-1], 32):
        part = x[..., b:b + 32].clamp(-KV_LIMIT, KV_LIMIT)
        d = _to32(part.abs().max(-1, keepdim=True).values.clamp_min(1e-12) / 127.0)
        out[..., b:b + 32] = torch.round(_to32(part / d)) * d.to(torch.float16).double()
    return out


def _exact_write(s):
    cos, sin = s["cos"][s["pos"].long()], s["sin"][s["pos"].long()]
    kind = s["k_cache"].dtype
    return (_turned64(s["q"], cos, sin), _rounded64(_key64(s["k"], cos, sin), kind),
            _rounded64(s["v"].double(), kind))


def _gathered64(s, values, b, length):
    size = values.shape[2]
    ids = s["table"][b, :-(-length // size)].long()
    return values[ids].transpose(0, 1).reshape(values.shape[1], -1, values.shape[3])[:, :length]


def _exact_read(s):
    n = len(s["pos"])
    return tuple(_gathered64(s, _values64(s[c]), 0, n).transpose(0, 1).contiguous() for c in ("k_cache", "v_cache"))


def _exact_attend(s):
    keys, values = _values64(s["k_cache"]), _values64(s["v_cache"])
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    n, heads, hd = s["q"].shape
    group = heads // keys.shape[1]
    start, kv_len = s["start"].tolist(), s["kv_len"].tolist()
    for b, length in enumerate(kv_len):
        k, v = _gathered64(s, keys, b, length), _gathered64(s, values, b, length)
        new = start[b + 1] - start[b]
        hidden = torch.ones((new, length), dtype=torch.bool, device=k.device).triu(length - new + 1)
        for h in range(heads):
            q = s["q"][start[b]:start[b + 1], h].double()
            w = (q @ k[h // group].T) / hd ** 0.5
            w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
            out[start[b]:start[b + 1], h] = w @ v[h // group]
    return out


def _exact_verify(s):
    start, counts, tokens = s["start"].tolist(), [], []
    drafts, u, last_u = s["drafts"].tolist(), s["accept_u"].tolist(), s["sample_u"].tolist()
    for b in range(len(start) - 1):
        said, r = [], start[b]
        while True:
            x = s["logits"][r].double()
            drafted = r + 1 < start[b + 1]
            if s["temperature"] == 0.0:
                t = int((x == x.max()).nonzero()[0])
                if drafted and t == drafts[r]:
                    said.append(t)
                    r += 1
                    continue
                break
            e = torch.exp((x - x.max()) / s["temperature"])
            p = e / e.sum()
            q = None
            if drafted:
                q = torch.zeros_like(p)
                if s["draft_probs"] is None:
                    q[drafts[r]] = 1.0
                else:
                    q = s["draft_probs"][r].double()
                if u[r] * float(q[drafts[r]]) < float(p[drafts[r]]):
                    said.append(drafts[r])
                    r += 1
                    continue
            rest = p if q is None else (p - q).clamp_min(0.0)
            if float(rest.sum()) <= 0.0:
                rest = p
            upto = torch.cumsum(rest, 0)
            t = int((upto > last_u[b] * upto[-1]).nonzero()[0])
            break
        counts.append(len(said))
        tokens.append(said + [t] + [-1] * (s["max_rows"] - len(said) - 1))
    dev = s["logits"].device
    return _int32(counts, dev), _int32(tokens, dev)
