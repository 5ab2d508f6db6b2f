"""Plain 64-bit statements of the paged cache's operators, with the bounds that
their tests hold the kernels to.  The bounds count roundings: a rounding to t
is off by at most half a step, relative u(t) = torch.finfo(t).eps / 2 (bf16
2^-8, fp16 2^-11, fp32 2^-24).  Runs on any device."""

import math

import torch

U16, UB, U32 = 2.0 ** -11, 2.0 ** -8, 2.0 ** -24
KV_LIMIT = 65024.0


def to32(x):
    return x.to(torch.float32).double()


def rotate(x, cos, sin):
    """Rotate-half RoPE of [n, heads, hd] with every product and sum rounded to fp32; cos, sin [n, hd / 2]."""
    h = x.shape[-1] // 2
    a, b = x[..., :h].double(), x[..., h:].double()
    c, s = cos.double()[:, None], sin.double()[:, None]
    return torch.cat([to32(to32(a * c) - to32(b * s)), to32(to32(b * c) + to32(a * s))], -1)


def cached_values(x, cache_type):
    """The values that the cache holds for fp32 numbers x (as float64)."""
    if cache_type == "bf16":
        return x.to(torch.float32).to(torch.bfloat16).double()
    b = x.double().unflatten(-1, (-1, 32)).clamp(-KV_LIMIT, KV_LIMIT)
    d = to32(b.abs().amax(-1, keepdim=True).clamp_min(1e-12) / 127.0)
    return (torch.round(to32(b / d)) * d.to(torch.float16).double()).flatten(-2)


def q8_parts(cache):
    """(quants [pages, kv, page, hd] int8, scales [pages, kv, page, hd / 32] fp16) views of a Q8_0 cache tensor."""
    pages, kv, page, row = cache.shape
    hd = row // 34 * 32
    flat = cache.view(pages, kv, -1)
    return (flat[..., :page * hd].view(torch.int8).unflatten(-1, (page, hd)),
            flat[..., page * hd:].view(torch.float16).unflatten(-1, (page, hd // 32)))


def values(cache):
    """All values of a cache tensor, float64 [pages, kv, page, hd]."""
    if cache.dtype == torch.bfloat16:
        return cache.double()
    q, d = q8_parts(cache)
    return (q.double().unflatten(-1, (-1, 32)) * d.double()[..., None]).flatten(-2)


def fill(cache, x):
    """Store x [pages, kv, page, hd] as the cache holds it."""
    if cache.dtype == torch.bfloat16:
        cache.copy_(x.to(torch.bfloat16))
        return
    q, d = q8_parts(cache)
    b = x.float().unflatten(-1, (-1, 32))
    scale = (b.abs().amax(-1) / 127).clamp_min(1e-12)
    q.copy_(torch.round(b / scale[..., None]).clamp(-127, 127).flatten(-2).to(torch.int8))
    d.copy_(scale.to(torch.float16))


def sequence(vals, table_row, length, n_pages):
    """Rows 0..length-1 of a sequence [kv, length, hd]; rows of pages outside the cache are zeros."""
    page = vals.shape[2]
    pos = torch.arange(length, device=vals.device)
    ids = table_row.long()[pos // page]
    ok = (ids >= 0) & (ids < n_pages)
    rows = vals[ids.clamp(0, n_pages - 1), :, pos % page]  # [length, kv, hd]
    return torch.where(ok[:, None, None], rows, torch.zeros((), dtype=rows.dtype, device=rows.device)).transpose(0, 1)


def attention(q, k_cache, v_cache, table, q_start, kv_len, scale=None):
    """(out, bound) float64 [n, heads, hd]: the attention of every sequence's tokens and how far a kernel may be
    off.  Rows of no sequence stay NaN.

    Bound of a row, with A = sum_j P_j |v_j| (each value counted by its weight) and e the largest error of its
    scores: 2 e A (a score's error moves numerator and denominator) + the roundings of P and V relative to A +
    the output's rounding.
      fp32 activations: q and P keep 22 bits or more, products are summed in fp32 by the tensor core (a sum of
        some 16 products may lose 2 steps of its largest): e = scale |q|.|k| (2^-22 + (4 + hd / 4) 2^-23), and
        2^-20 + (64 + keys / 8) 2^-24 of A for exp2, P and the sums over the keys;
      bf16 activations: P is rounded to bf16 (2^-8) or, with Q8_0, q stays exact, K, V and P are fp16 (2^-11 each)
        or, in the chunk kernel, bf16/fp16 likewise."""
    n, heads, hd = q.shape
    kv = k_cache.shape[1]
    group, n_pages = heads // kv, k_cache.shape[0]
    scale = 1 / math.sqrt(hd) if scale is None else scale
    keys, vals = values(k_cache), values(v_cache)
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    bound = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    q8, f32 = k_cache.dtype == torch.uint8, q.dtype == torch.float32
    for s in range(len(kv_len)):
        a, b, length = int(q_start[s]), int(q_start[s + 1]), int(kv_len[s])
        m = b - a
        if m <= 0:
            continue
        k, v = (sequence(x, table[s], length, n_pages).repeat_interleave(group, 0) for x in (keys, vals))
        x = q[a:b].double().transpose(0, 1)  # [heads, m, hd]
        hidden = torch.ones((m, length), dtype=torch.bool, device=q.device).triu(length - m + 1)
        w = (x @ k.transpose(1, 2) * scale).masked_fill(hidden, -math.inf)
        p = torch.softmax(w, -1)
        p = torch.where(hidden.all(-1)[:, None], torch.zeros_like(p), p)  # a token that sees nothing
        # a value that is not finite reaches only the rows that see it
        bad = ~torch.isfinite(v)
        o = p @ v.masked_fill(bad, 0)
        for h, j, d in bad.nonzero().tolist():
            o[h, :, d] += torch.where(hidden[:, j], torch.zeros_like(p[h, :, j]), p[h, :, j] * v[h, j, d])
        A = p @ v.masked_fill(bad, 0).abs()
        e = (x.abs() @ k.nan_to_num(0, 0, 0).abs().transpose(1, 2) * scale).masked_fill(hidden, 0)
        e = e.amax(-1, keepdim=True) if length else torch.zeros((heads, m, 1), device=q.device)
        if f32:
            lim = 2 * e * (2.0 ** -22 + (4 + hd / 4) * 2.0 ** -23) * A + (2.0 ** -20 + (64 + length / 8) * U32) * A
            lim = lim + U32 * o.abs()
        elif q8:
            lim = 2 * e * (U16 + 2.0 ** -18) * A + (2 * U16 + 2.0 ** -18) * A + UB * o.abs()
        else:
            lim = 2 * e * 2.0 ** -18 * A + (UB + 2.0 ** -16) * A + UB * o.abs()
        out[a:b], bound[a:b] = o.transpose(0, 1), (lim + 1e-30).transpose(0, 1)
    return out, bound


def verify(logits, row_start, drafts, accept_u, sample_u, draft_probs, temperature, max_rows):
    """(accepted, tokens) as lists, sequence by sequence in float64, and the
    smallest distance of a decision from its border (a test's inputs keep away
    from borders by more than the sums' errors)."""
    counts, tokens, margin = [], [], math.inf
    for s in range(len(row_start) - 1):
        said, r, end, last = [], int(row_start[s]), int(row_start[s + 1]), -1
        while r < end:
            x = logits[r].double()
            x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
            top, drafted = float(x.max()), r + 1 < end
            if top == -math.inf:
                break
            if temperature == 0.0:
                last = int((x == top).nonzero()[0])
                if drafted and int(drafts[r]) == last:
                    said.append(last)
                    last, r = -1, r + 1
                    continue
                break
            w = torch.where(x == top, torch.ones_like(x), torch.exp((x - top) / temperature))
            p = w / w.sum()
            d = int(drafts[r])
            q = torch.zeros_like(p)
            if drafted and draft_probs is not None:
                q = draft_probs[r].double()
            elif drafted and 0 <= d < len(p):
                q[d] = 1.0
            if drafted and 0 <= d < len(p):
                left, right = float(accept_u[r]) * float(q[d]), float(p[d])
                margin = min(margin, abs(left - right) / max(right, 1e-30))
                if left < right:
                    said.append(d)
                    r += 1
                    continue
            rest = (p - q).clamp_min(0.0) if drafted else p
            if not float(rest.sum()) > 0.0:
                rest = p
            upto = torch.cumsum(rest, 0) / rest.sum()
            over = (upto > float(sample_u[s])) & (rest > 0)
            last = int(over.nonzero()[0]) if bool(over.any()) else int((rest > 0).nonzero()[-1])
            margin = min(margin, float((upto - float(sample_u[s])).abs().min()) * 1e6)
            break
        counts.append(len(said))
        row = (said + [last] if end > int(row_start[s]) else []) + [-1] * max_rows
        tokens.append(row[:max_rows])
    return counts, tokens, margin
