"""Serving operators over a paged key/value cache (C ABI: draco_kv_append,
draco_kv_read, draco_attention_paged, draco_verify_drafts).

One layer's cache is two tensors, keys and values, from ``kv_cache``:

* ``"bf16"``  [pages, kv_heads, page_size, head_dim] bfloat16;
* ``"q8_0"``  [pages, kv_heads, page_size, head_dim // 32 * 34] uint8: GGUF
  Q8_0 blocks (int8 quants and an fp16 scale per 32 values), per page and head
  all quants first, then the scales.

``block_table`` [sequences, pages per sequence] (int32) names each sequence's
pages; position ``p`` is row ``p % page_size`` of entry ``p // page_size``.
Sequences may share pages.

A step of a batch (one token each, drafted tokens, a prompt's chunk, whole
prompts, or all of these together) is, per layer,

    q = kv_append(q, k, v, k_cache, v_cache, table, seq, pos, cos, sin)
    o = attention_paged(q, k_cache, v_cache, table, q_start, kv_len, max_q=..., max_kv=...)

and, with drafted tokens, ``verify_drafts`` on the step's logits decides which
of them stay.  The calls enqueue on the current stream, never wait for the GPU,
and can be captured in a CUDA graph.  Reference code in the neighbourhood:
draco/attention/paged.py:26-269, draco/kv_cache/block.py:119-441,
draco/runtime/cpu/speculative.py.
"""

from __future__ import annotations

import ctypes
import threading
from typing import Dict, Optional, Tuple

import torch

from dracort_b200 import _native as N
from dracort_b200.exceptions import DracoFormatError

CACHE_TYPES = {"bf16": N.KV_BF16, "q8_0": N.KV_Q8_0}
_DTYPES = {torch.float32: N.DTYPE_F32, torch.bfloat16: N.DTYPE_BF16}


def kv_cache_nbytes(cache_type: str, pages: int, kv_heads: int, page_size: int, head_dim: int) -> int:
    """Bytes of a layer's key (or value) tensor."""
    n = N.load().draco_kv_cache_bytes(_cache_type(cache_type), pages, kv_heads, page_size, head_dim)
    if n < 0:
        raise DracoFormatError(f"no {cache_type} cache of {pages} pages of {page_size} positions, {kv_heads} heads of "
                               f"{head_dim} (pages: a power of two from 16 to 1024; head_dim 32, 64, 96, 128 or 256)")
    return int(n)


def kv_cache(cache_type: str, pages: int, kv_heads: int, page_size: int, head_dim: int,
             device) -> Tuple[torch.Tensor, torch.Tensor]:
    """A layer's key and value tensors, zero-filled."""
    kv_cache_nbytes(cache_type, pages, kv_heads, page_size, head_dim)
    if cache_type == "bf16":
        shape, dtype = (pages, kv_heads, page_size, head_dim), torch.bfloat16
    else:
        shape, dtype = (pages, kv_heads, page_size, head_dim // 32 * 34), torch.uint8
    return torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)


def _cache_type(name: str) -> int:
    try:
        return CACHE_TYPES[name]
    except KeyError:
        raise ValueError(f"unknown cache type {name!r}; expected one of {sorted(CACHE_TYPES)}") from None


def _on(t: torch.Tensor, name: str, device: torch.device, dtype: torch.dtype) -> None:
    if t.device != device or t.dtype != dtype:
        raise ValueError(f"{name} must be a {dtype} tensor on {device}, not {t.dtype} on {t.device}")


def _vector(t: torch.Tensor, name: str, device: torch.device, n: int, dtype: torch.dtype = torch.int32) -> int:
    _on(t, name, device, dtype)
    if t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise DracoFormatError(f"{name} must be a contiguous tensor of {n} values, not {tuple(t.shape)}")
    return t.data_ptr()


def _rows(t: torch.Tensor, name: str, device: torch.device, n: Optional[int], dtype: Optional[torch.dtype],
          head_dim: int) -> int:
    """Token stride of [n, heads, head_dim] with contiguous heads."""
    if t.device != device or t.dtype not in _DTYPES or (dtype is not None and t.dtype != dtype):
        raise ValueError(f"{name} must be a float32 or bfloat16 tensor on {device} (all activations of a call one "
                         f"type), not {t.dtype} on {t.device}")
    if t.dim() != 3 or (n is not None and t.shape[0] != n) or t.shape[2] != head_dim:
        raise DracoFormatError(f"{name} must be [tokens, heads, {head_dim}], not {tuple(t.shape)}")
    if t.shape[0] == 0:
        return t.shape[1] * head_dim
    if (t.stride(2) != 1 and head_dim > 1) or (t.shape[1] > 1 and t.stride(1) != head_dim):
        raise ValueError(f"{name} must have contiguous heads (a token stride is free)")
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1] * head_dim)


def _cache_struct(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                  head_dim: int) -> N.KvCache:
    if not k_cache.is_cuda:
        raise ValueError("k_cache must be a CUDA tensor (this library has no CPU path)")
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype:
        raise DracoFormatError(f"k_cache {tuple(k_cache.shape)} and v_cache {tuple(v_cache.shape)} must be alike, "
                               f"[pages, kv_heads, page_size, row]")
    if v_cache.device != k_cache.device or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache and v_cache must be contiguous tensors on one device")
    pages, kv_heads, page, row = k_cache.shape
    if k_cache.dtype == torch.bfloat16:
        kind, want = N.KV_BF16, head_dim
    elif k_cache.dtype == torch.uint8:
        kind, want = N.KV_Q8_0, head_dim // 32 * 34
    else:
        raise ValueError(f"a cache is bfloat16 or uint8 (Q8_0 blocks), not {k_cache.dtype}")
    if row != want:
        raise DracoFormatError(f"cache rows of {row} do not hold head_dim {head_dim}")
    _on(block_table, "block_table", k_cache.device, torch.int32)
    if block_table.dim() != 2 or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise DracoFormatError("block_table must be [sequences, pages] with contiguous rows")
    c = N.KvCache()
    c.type, c.kv_heads, c.head_dim, c.page_size, c.n_pages = kind, kv_heads, head_dim, page, pages
    c.n_seqs, c.max_pages = block_table.shape
    c.table_stride = block_table.stride(0)  # 0: all sequences share one row
    c.k, c.v, c.block_table = k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr()
    return c


class _Device:
    """The tensors' device made current for a call (the library launches on the current one)."""

    def __init__(self, device: torch.device) -> None:
        self.index = device.index
        self.back = torch.cuda.current_device()

    def __enter__(self) -> int:
        if self.back != self.index:
            torch.cuda.set_device(self.index)
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc) -> None:
        if self.back != self.index:
            torch.cuda.set_device(self.back)


def kv_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
              v_cache: torch.Tensor, block_table: torch.Tensor, seq: torch.Tensor, pos: torch.Tensor,
              cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
              q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Rotate q and k (rotate-half RoPE with the fp32 tables cos / sin
    [positions, head_dim / 2]; none: no rotation), write the keys and values
    of token i to position pos[i] of sequence seq[i] in the cache's type, and
    return the rotated q (in q_out, which may be q).

    q [n, heads, head_dim], k and v [n, kv_heads, head_dim], all float32 or all
    bfloat16, any token stride that keeps rows on 16 bytes (slices of a fused
    projection); seq, pos int32 [n].  Tokens of a call go to distinct
    positions.  A token outside the block table or the tables writes nothing."""
    if k.dim() != 3:
        raise DracoFormatError(f"k must be [tokens, kv_heads, head_dim], not {tuple(k.shape)}")
    n, kv_heads, hd = k.shape
    c = _cache_struct(k_cache, v_cache, block_table, hd)
    dev = k_cache.device
    if kv_heads != c.kv_heads or v.shape != k.shape:
        raise DracoFormatError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not match the cache's {c.kv_heads} heads")
    a = N.KvAppendArgs()
    a.ldk, a.ldv = _rows(k, "k", dev, n, None, hd), _rows(v, "v", dev, n, k.dtype, hd)
    a.k, a.v, a.n = k.data_ptr(), v.data_ptr(), n
    if q is not None:
        a.ldq = _rows(q, "q", dev, n, k.dtype, hd)
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        elif q_out.shape != q.shape:
            raise DracoFormatError(f"q_out {tuple(q_out.shape)} is not shaped like q {tuple(q.shape)}")
        a.ldqo = _rows(q_out, "q_out", dev, n, k.dtype, hd)
        a.q, a.q_out, a.heads = q.data_ptr(), q_out.data_ptr(), q.shape[1]
    elif q_out is not None:
        raise ValueError("q_out needs q")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        for t, name in ((cos, "cos"), (sin, "sin")):
            _on(t, name, dev, torch.float32)
            if t.dim() != 2 or t.shape != cos.shape or t.shape[1] != hd // 2 or not t.is_contiguous():
                raise DracoFormatError(f"{name} must be a contiguous [positions, {hd // 2}] table")
        a.cos_table, a.sin_table, a.max_positions = cos.data_ptr(), sin.data_ptr(), cos.shape[0]
    a.seq, a.pos = _vector(seq, "seq", dev, n), _vector(pos, "pos", dev, n)
    with _Device(dev) as stream:
        N.check(N.load().draco_kv_append(ctypes.byref(c), ctypes.byref(a), _DTYPES[k.dtype], stream), "kv_append")
    return q_out


def kv_read(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, seq: torch.Tensor,
            pos: torch.Tensor, head_dim: int, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values at position pos[i] of sequence seq[i] (int32 [n]), as
    [n, kv_heads, head_dim] float32 (exact) or bfloat16 (rounded once); rows
    outside the cache are zeros."""
    c = _cache_struct(k_cache, v_cache, block_table, head_dim)
    dev, n = k_cache.device, seq.shape[0]
    if dtype not in _DTYPES:
        raise ValueError(f"kv_read gives float32 or bfloat16, not {dtype}")
    s, p = _vector(seq, "seq", dev, n), _vector(pos, "pos", dev, n)
    out = torch.empty((2, n, c.kv_heads, head_dim), dtype=dtype, device=dev)
    ld = c.kv_heads * head_dim
    with _Device(dev) as stream:
        N.check(N.load().draco_kv_read(ctypes.byref(c), s, p, n, out.data_ptr(),
                                       out.data_ptr() + n * ld * out.element_size(), ld, ld, _DTYPES[dtype], stream),
                "kv_read")
    return out[0], out[1]


# Workspace of attention_paged per (device, stream), zeroed once; the kernels
# leave its counters at zero.  A call that is being captured gets one of its
# own, zeroed in the graph: two graphs may replay at the same time.
_ws_lock = threading.Lock()
_workspaces: Dict[Tuple[int, int], torch.Tensor] = {}


def _workspace(device: torch.device, stream: int, nbytes: int) -> torch.Tensor:
    if torch.cuda.is_current_stream_capturing():
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        ws[:N.PAGED_WORKSPACE_HEAD].zero_()  # counters and status; the rest is written before it is read
        return ws
    key = (device.index, stream)
    with _ws_lock:
        ws = _workspaces.get(key)
        if ws is None or ws.numel() < nbytes:
            ws = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
            _workspaces[key] = ws
        return ws


def attention_paged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    q_start: torch.Tensor, kv_len: torch.Tensor, max_q: Optional[int] = None,
                    max_kv: Optional[int] = None, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of each sequence's newest tokens over its cached keys.

    q [n, heads, head_dim] float32 or bfloat16 (rotated); sequence s has the
    tokens q_start[s] .. q_start[s + 1] - 1 (int32 [sequences + 1], ascending)
    and kv_len[s] cached positions, these tokens' included.  Token i of m sees
    positions 0 .. kv_len - m + i; query head h reads key/value head
    h // (heads // kv_heads).  Returns out, shaped like q; tokens that see
    nothing get zeros, rows behind the last sequence are left as they are.

    max_q, max_kv are upper bounds of a sequence's tokens and positions (default:
    all tokens; the whole block table); they choose the kernels and size the
    launch, so tight bounds are faster (tokens past max_q may be left out).  scale defaults to 1 / sqrt(head_dim).
    workspace: a zeroed uint8 tensor of attention_paged_workspace_nbytes that
    the caller keeps (one per call that may overlap another); by default one
    per stream is kept here, and a captured call gets its own."""
    if q.dim() != 3:
        raise DracoFormatError(f"q must be [tokens, heads, head_dim], not {tuple(q.shape)}")
    n, heads, hd = q.shape
    c = _cache_struct(k_cache, v_cache, block_table, hd)
    dev = k_cache.device
    a = N.AttentionPagedArgs()
    a.ldq = _rows(q, "q", dev, n, None, hd)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    elif out.shape != q.shape:
        raise DracoFormatError(f"out {tuple(out.shape)} is not shaped like q {tuple(q.shape)}")
    a.ldo = _rows(out, "out", dev, n, q.dtype, hd)
    a.q, a.out, a.n, a.heads = q.data_ptr(), out.data_ptr(), n, heads
    a.q_start, a.kv_len = _vector(q_start, "q_start", dev, c.n_seqs + 1), _vector(kv_len, "kv_len", dev, c.n_seqs)
    a.max_q = n if max_q is None else int(max_q)
    a.max_kv = c.max_pages * c.page_size if max_kv is None else int(max_kv)
    if scale is not None and not 0.0 < scale < 1e30:
        raise ValueError(f"scale {scale} must be positive")
    a.scale = 0.0 if scale is None else float(scale)
    dt = _DTYPES[q.dtype]
    with _Device(dev) as stream:
        lib = N.load()
        if workspace is None:
            need = lib.draco_attention_paged_workspace_bytes(ctypes.byref(c), n, heads, a.max_q, a.max_kv, dt)
            if need:  # otherwise the call below says what is wrong
                workspace = _workspace(dev, stream, need)
        if workspace is not None:
            a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        N.check(lib.draco_attention_paged(ctypes.byref(c), ctypes.byref(a), dt, stream), "attention_paged")
    return out


def attention_paged_workspace_nbytes(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                                     n: int, heads: int, head_dim: int, max_q: int, max_kv: int,
                                     dtype: torch.dtype) -> int:
    """Bytes of the workspace of an attention_paged call of n tokens."""
    c = _cache_struct(k_cache, v_cache, block_table, head_dim)
    need = N.load().draco_attention_paged_workspace_bytes(ctypes.byref(c), n, heads, max_q, max_kv, _DTYPES[dtype])
    if need == 0:
        raise DracoFormatError(N.last_error() or "attention_paged: unsupported arguments")
    return int(need)


def verify_drafts(logits: torch.Tensor, row_start: torch.Tensor, drafts: torch.Tensor, accept_u: torch.Tensor,
                  sample_u: torch.Tensor, draft_probs: Optional[torch.Tensor] = None, temperature: float = 1.0,
                  max_rows: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Which drafted tokens stay, and the token after them.

    Sequence s owns rows row_start[s] .. row_start[s + 1] - 1 (int32) of logits
    [n, vocab] (float32 or bfloat16): one per draft and one more.  drafts[r]
    (int32 [n]) is the token proposed after row r (unused for a sequence's last
    row).  With p = softmax(logits / temperature) and q = draft_probs ([n, vocab]
    float32; none: each draft was certain), draft x of row r is taken while
    accept_u[r] * q(x) < p(x); at the first that is not, the next token is drawn
    from max(p - q, 0), after the last from p: the first index whose cumulative
    weight exceeds sample_u[s] times the total.  temperature 0 is greedy.
    accept_u [n] and sample_u [sequences] are float32 in [0, 1).

    Returns accepted (int32 [sequences]) and tokens (int32 [sequences, max_rows]:
    the drafts taken, the next token, then -1); max_rows (default n) is the
    largest number of rows of a sequence.  One row per sequence is plain
    sampling."""
    if not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor (this library has no CPU path)")
    dev = logits.device
    if logits.dtype not in _DTYPES:
        raise ValueError(f"logits must be float32 or bfloat16, not {logits.dtype}")
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise DracoFormatError("logits must be [rows, vocab] with contiguous rows")
    n, vocab = logits.shape
    seqs = row_start.shape[0] - 1
    if row_start.dim() != 1 or seqs < 0:
        raise DracoFormatError("row_start must be [sequences + 1]")
    v = N.VerifyArgs()
    v.logits, v.ld_logits, v.dtype = logits.data_ptr(), logits.stride(0), _DTYPES[logits.dtype]
    if draft_probs is not None:
        _on(draft_probs, "draft_probs", dev, torch.float32)
        if draft_probs.shape != logits.shape or (vocab > 1 and draft_probs.stride(1) != 1):
            raise DracoFormatError("draft_probs must be shaped like logits with contiguous rows")
        v.draft_probs, v.ld_probs = draft_probs.data_ptr(), draft_probs.stride(0)
    v.row_start, v.drafts = _vector(row_start, "row_start", dev, seqs + 1), _vector(drafts, "drafts", dev, n)
    v.accept_u = _vector(accept_u, "accept_u", dev, n, torch.float32)
    v.sample_u = _vector(sample_u, "sample_u", dev, seqs, torch.float32)
    rows = max(n, 1) if max_rows is None else int(max_rows)
    if rows < 1:
        raise ValueError(f"max_rows {rows} must be at least 1")
    accepted = torch.empty(seqs, dtype=torch.int32, device=dev)
    tokens = torch.empty((seqs, rows), dtype=torch.int32, device=dev)
    v.accepted, v.tokens, v.ld_tokens = accepted.data_ptr(), tokens.data_ptr(), rows
    v.temperature, v.n, v.n_seqs, v.vocab, v.max_rows = float(temperature), n, seqs, vocab, rows
    with _Device(dev) as stream:
        N.check(N.load().draco_verify_drafts(ctypes.byref(v), stream), "verify_drafts")
    return accepted, tokens
