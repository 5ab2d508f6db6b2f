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
import struct
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


# The checks run on every call of a decode loop: the fast path touches each
# tensor's properties once, the messages are put together only on failure, and
# the argument structures are packed as bytes (the mirrors of _native take three
# times as long to fill).
_KV_CACHE = struct.Struct("@7iq3P")           # draco_kv_cache
_KV_APPEND = struct.Struct("@4P4q2Pq2P2i")    # draco_kv_append_args
_ATTENTION = struct.Struct("@2P2q2P4if2P")    # draco_attention_paged_args
_VERIFY = struct.Struct("@8P3qf5i")           # draco_verify_args


class _Functions:
    """The library's functions, with structures taken as packed bytes."""

    def __init__(self) -> None:
        lib, vp, ci = N.load(), ctypes.c_void_p, ctypes.c_int

        def fn(name, *args, restype=ci):
            f = lib[name]  # (an object of its own: _native's prototypes stay)
            f.argtypes, f.restype = list(args), restype
            return f

        i64 = ctypes.c_int64
        self.kv_append = fn("draco_kv_append", vp, vp, ci, vp)
        self.kv_read = fn("draco_kv_read", vp, vp, vp, ci, vp, vp, i64, i64, ci, vp)
        self.attention_paged = fn("draco_attention_paged", vp, vp, ci, vp)
        self.workspace_bytes = fn("draco_attention_paged_workspace_bytes", vp, ci, ci, ci, ci, ci,
                                  restype=ctypes.c_size_t)
        self.verify_drafts = fn("draco_verify_drafts_at", vp, ctypes.c_double, vp)


_functions: Optional[_Functions] = None


def _lib() -> _Functions:
    global _functions
    if _functions is None:
        _functions = _Functions()
    return _functions


_I32, _F32 = torch.int32, torch.float32
_current_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _vector(t: torch.Tensor, name: str, dev: int, n: int, dtype: torch.dtype = _I32) -> int:
    if t.dtype is dtype and t.get_device() == dev and t.shape == (n,) and t.is_contiguous():
        return t.data_ptr()
    if t.dtype is not dtype or t.get_device() != dev:
        raise ValueError(f"{name} must be a {dtype} tensor on cuda:{dev}, not {t.dtype} on {t.device}")
    raise DracoFormatError(f"{name} must be a contiguous tensor of {n} values, not {tuple(t.shape)}")


def _rows(t: torch.Tensor, name: str, dev: int, n: int, dtype: torch.dtype, head_dim: int) -> int:
    """Token stride of [n, heads, head_dim] with contiguous heads."""
    shape, stride = t.shape, t.stride()
    if (t.dtype is dtype and t.get_device() == dev and len(shape) == 3 and shape[0] == n and shape[2] == head_dim
            and stride[2] == 1 and (stride[1] == head_dim or shape[1] == 1)):
        return stride[0] if n > 1 else shape[1] * head_dim
    if t.dtype is not dtype or t.get_device() != dev:
        raise ValueError(f"{name} must be a float32 or bfloat16 tensor on cuda:{dev} (all activations of a call one "
                         f"type), not {t.dtype} on {t.device}")
    if len(shape) != 3 or shape[0] != n or shape[2] != head_dim:
        raise DracoFormatError(f"{name} must be [{n}, heads, {head_dim}], not {tuple(shape)}")
    if n == 0 or shape[1] == 0:
        return shape[1] * head_dim
    raise ValueError(f"{name} must have contiguous heads (a token stride is free)")


def _cache_struct(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                  head_dim: int) -> Tuple[bytes, int, int, int]:
    """(packed draco_kv_cache, kv_heads, sequences, positions of a sequence at most)"""
    shape, dtype, dev = k_cache.shape, k_cache.dtype, k_cache.get_device()
    if dev < 0:
        raise ValueError("k_cache must be a CUDA tensor (this library has no CPU path)")
    if len(shape) != 4 or v_cache.shape != shape or v_cache.dtype is not dtype:
        raise DracoFormatError(f"k_cache {tuple(shape)} and v_cache {tuple(v_cache.shape)} must be alike, "
                               f"[pages, kv_heads, page_size, row]")
    if v_cache.get_device() != dev or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache and v_cache must be contiguous tensors on one device")
    pages, kv_heads, page, row = shape
    if dtype is torch.bfloat16:
        kind, want = N.KV_BF16, head_dim
    elif dtype is torch.uint8:
        kind, want = N.KV_Q8_0, head_dim // 32 * 34
    else:
        raise ValueError(f"a cache is bfloat16 or uint8 (Q8_0 blocks), not {dtype}")
    if row != want:
        raise DracoFormatError(f"cache rows of {row} do not hold head_dim {head_dim}")
    if block_table.dtype is not _I32 or block_table.get_device() != dev:
        raise ValueError(f"block_table must be an int32 tensor on cuda:{dev}, not {block_table.dtype} on "
                         f"{block_table.device}")
    tshape = block_table.shape
    tstride = block_table.stride()
    if len(tshape) != 2 or (tshape[1] > 1 and tstride[1] != 1):
        raise DracoFormatError("block_table must be [sequences, pages] with contiguous rows")
    # (a table stride of 0: all sequences share one row)
    seqs, width = tshape
    return _KV_CACHE.pack(kind, kv_heads, head_dim, page, pages, seqs, width, tstride[0], k_cache.data_ptr(),
                          v_cache.data_ptr(), block_table.data_ptr()), kv_heads, seqs, width * page


def _dtype(t: torch.Tensor, name: str) -> int:
    dt = _DTYPES.get(t.dtype)
    if dt is None:
        raise ValueError(f"{name} must be float32 or bfloat16, not {t.dtype}")
    return dt


def _table(t: torch.Tensor, name: str, dev: int, positions: int, half: int) -> int:
    if t.dtype is _F32 and t.get_device() == dev and t.shape == (positions, half) and t.is_contiguous():
        return t.data_ptr()
    if t.dtype is not _F32 or t.get_device() != dev:
        raise ValueError(f"{name} must be a float32 tensor on cuda:{dev}, not {t.dtype} on {t.device}")
    raise DracoFormatError(f"{name} must be a contiguous [positions, {half}] table, not {tuple(t.shape)}")


def _like(t: torch.Tensor, shape) -> torch.Tensor:
    """A new contiguous tensor of t's type and device."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(shape)


def _call(dev: int, fn, *args) -> int:
    """fn(*args, stream) on device `dev` and its current stream."""
    if _current_device() == dev:
        return fn(*args, _current_stream(dev))
    with torch.cuda.device(dev):
        return fn(*args, _current_stream(dev))


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
    shape = k.shape
    if len(shape) != 3:
        raise DracoFormatError(f"k must be [tokens, kv_heads, head_dim], not {tuple(shape)}")
    n, kv_heads, hd = shape
    c, cache_heads, _, _ = _cache_struct(k_cache, v_cache, block_table, hd)
    dev, dtype, dt = k_cache.get_device(), k.dtype, _dtype(k, "k")
    ldk, ldv = _rows(k, "k", dev, n, dtype, hd), _rows(v, "v", dev, n, dtype, hd)
    if kv_heads != cache_heads or v.shape != shape:
        raise DracoFormatError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not match the cache's {cache_heads} heads")
    ldq = ldqo = heads = 0
    q_ptr = qo_ptr = 0
    if q is not None:
        ldq = _rows(q, "q", dev, n, dtype, hd)
        heads = q.shape[1]
        if q_out is None:
            q_out, ldqo = _like(q, (n, heads, hd)), heads * hd
        elif q_out.shape != q.shape:
            raise DracoFormatError(f"q_out {tuple(q_out.shape)} is not shaped like q {tuple(q.shape)}")
        else:
            ldqo = _rows(q_out, "q_out", dev, n, dtype, hd)
        q_ptr, qo_ptr = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out needs q")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    cos_ptr = sin_ptr = 0
    positions = 0
    if cos is not None:
        positions = cos.shape[0] if cos.dim() else 0
        cos_ptr, sin_ptr = _table(cos, "cos", dev, positions, hd // 2), _table(sin, "sin", dev, positions, hd // 2)
    a = _KV_APPEND.pack(q_ptr, k.data_ptr(), v.data_ptr(), qo_ptr, ldq, ldk, ldv, ldqo, cos_ptr, sin_ptr, positions,
                        _vector(seq, "seq", dev, n), _vector(pos, "pos", dev, n), n, heads)
    rc = _call(dev, _lib().kv_append, c, a, dt)
    if rc:
        N.check(rc, "kv_append")
    return q_out


def kv_read(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, seq: torch.Tensor,
            pos: torch.Tensor, head_dim: int, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values at position pos[i] of sequence seq[i] (int32 [n]), as
    [n, kv_heads, head_dim] float32 (exact) or bfloat16 (rounded once); rows
    outside the cache are zeros.  For a host that moves a sequence to another
    cache type, device or process, or keeps a prefix outside the pages; attention
    reads the pages themselves."""
    c, kv_heads, _, _ = _cache_struct(k_cache, v_cache, block_table, head_dim)
    dev, n = k_cache.get_device(), seq.shape[0] if seq.dim() else 0
    if dtype not in _DTYPES:
        raise ValueError(f"kv_read gives float32 or bfloat16, not {dtype}")
    s, p = _vector(seq, "seq", dev, n), _vector(pos, "pos", dev, n)
    k = k_cache.new_empty((n, kv_heads, head_dim), dtype=dtype)
    v = torch.empty_like(k)
    ld = kv_heads * head_dim
    rc = _call(dev, _lib().kv_read, c, s, p, n, k.data_ptr(), v.data_ptr(), ld, ld, _DTYPES[dtype])
    if rc:
        N.check(rc, "kv_read")
    return k, v


# Workspace of attention_paged per (device, stream), its head zeroed once; the
# kernels leave its counters at zero.  A call that is being captured gets one of
# its own, zeroed in the graph: two graphs may replay at the same time.
_ws_lock = threading.Lock()
_workspaces: Dict[Tuple[int, int], torch.Tensor] = {}


def _new_workspace(like: torch.Tensor, nbytes: int) -> torch.Tensor:
    ws = like.new_empty(nbytes, dtype=torch.uint8)
    ws[:N.PAGED_WORKSPACE_HEAD].zero_()  # counters and status; the rest is written before it is read
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
    launch, so tight bounds are faster (tokens past max_q may be left out).
    scale defaults to 1 / sqrt(head_dim).
    workspace: a uint8 tensor of attention_paged_workspace_nbytes, zeroed once,
    that the caller keeps (one per call that may overlap another); by default one
    per stream is kept here, and a captured call gets its own."""
    shape = q.shape
    if len(shape) != 3:
        raise DracoFormatError(f"q must be [tokens, heads, head_dim], not {tuple(shape)}")
    n, heads, hd = shape
    c, _, seqs, held = _cache_struct(k_cache, v_cache, block_table, hd)
    dev = k_cache.get_device()
    if _current_device() != dev:  # the plan, the capture and the workspace are those of the tensors' device
        with torch.cuda.device(dev):
            return attention_paged(q, k_cache, v_cache, block_table, q_start, kv_len, max_q, max_kv, scale, out,
                                   workspace)
    dtype, dt = q.dtype, _dtype(q, "q")
    ldq = _rows(q, "q", dev, n, dtype, hd)
    if out is None:
        out, ldo = _like(q, shape), heads * hd
    elif out.shape != shape:
        raise DracoFormatError(f"out {tuple(out.shape)} is not shaped like q {tuple(shape)}")
    else:
        ldo = _rows(out, "out", dev, n, dtype, hd)
    if scale is not None and not 1e-30 < scale <= 65536.0:
        raise ValueError(f"scale {scale} must be positive and at most 65536")
    max_q = n if max_q is None or max_q > n else max(int(max_q), -1)
    max_kv = held if max_kv is None or max_kv > held else max(int(max_kv), -1)
    lib = _lib()
    start_ptr, len_ptr = _vector(q_start, "q_start", dev, seqs + 1), _vector(kv_len, "kv_len", dev, seqs)

    def run(ws: Optional[torch.Tensor]) -> int:
        ptr, nbytes = (0, 0) if ws is None else (ws.data_ptr(), ws.numel() * ws.element_size())
        a = _ATTENTION.pack(q.data_ptr(), out.data_ptr(), ldq, ldo, start_ptr, len_ptr, n, heads, max_q, max_kv,
                            0.0 if scale is None else scale, ptr, nbytes)
        return lib.attention_paged(c, a, dt, _current_stream(dev))

    if workspace is not None:
        if workspace.get_device() != dev or not workspace.is_contiguous():
            raise ValueError(f"workspace must be a contiguous tensor on cuda:{dev}")
        rc = run(workspace)
    elif torch.cuda.is_current_stream_capturing():
        need = lib.workspace_bytes(c, n, heads, max_q, max_kv, dt)
        rc = run(_new_workspace(k_cache, max(need, N.PAGED_WORKSPACE_HEAD)))
    else:
        key = (dev, _current_stream(dev))
        rc = run(_workspaces.get(key))
        if rc == N.DRACO_ERR_WORKSPACE:  # none yet, or too small
            need = lib.workspace_bytes(c, n, heads, max_q, max_kv, dt)
            with _ws_lock:
                ws = _workspaces[key] = _new_workspace(k_cache, max(need, 1 << 20))
            rc = run(ws)
    if rc:
        N.check(rc, "attention_paged")
    return out


def attention_paged_status(workspace: Optional[torch.Tensor] = None) -> int:
    """Device status of attention_paged: 0, or DRACO_ERR_TIMEOUT after a bounded
    wait inside a kernel ran out (the outputs of that call are then invalid).
    Waits for the GPU.  Without a workspace: of all calls on the current device
    since the last one that asked, those replayed from graphs and those with
    workspaces of their callers included.  With one: of the calls that used it.
    A workspace that reports an error, the given one or any that this module
    keeps, is made ready for use again (a caller's own only when it is given)."""
    rc = 0
    if workspace is None:
        dev = _current_device()
        with _ws_lock:
            kept = [ws for (d, _), ws in _workspaces.items() if d == dev]
        torch.cuda.synchronize(dev)
        word = ctypes.c_int()
        N.check(N.load().draco_attention_paged_status(0, ctypes.byref(word)), "attention_paged_status")
        rc = word.value
    else:
        dev = workspace.device
        kept = [workspace]
        torch.cuda.synchronize(dev)
    for ws in kept:
        found = int(ws[N.PAGED_WORKSPACE_STATUS:N.PAGED_WORKSPACE_STATUS + 4].view(torch.int32).item())
        if found:
            ws[:N.PAGED_WORKSPACE_HEAD].zero_()
            rc = rc or found
    torch.cuda.synchronize(dev)
    return rc


def attention_paged_workspace_nbytes(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                                     n: int, heads: int, head_dim: int, max_q: int, max_kv: int,
                                     dtype: torch.dtype) -> int:
    """Bytes of the workspace of an attention_paged call of n tokens."""
    c, _, _, held = _cache_struct(k_cache, v_cache, block_table, head_dim)
    if dtype not in _DTYPES:
        raise ValueError(f"dtype must be float32 or bfloat16, not {dtype}")
    with torch.cuda.device(k_cache.get_device()):
        need = _lib().workspace_bytes(c, n, heads, max(min(max_q, n), -1), max(min(max_kv, held), -1), _DTYPES[dtype])
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
    weight exceeds sample_u[s] times the total.  temperature (1e-30 .. 1e30, taken
    as the 64-bit number it is) 0 is greedy.
    accept_u [n] and sample_u [sequences] are float32 in [0, 1).

    Returns accepted (int32 [sequences]) and tokens (int32 [sequences, max_rows]:
    the drafts taken, the next token, then -1); max_rows (default n) is the
    largest number of rows of a sequence.  One row per sequence is plain
    sampling."""
    dev = logits.get_device()
    if dev < 0:
        raise ValueError("logits must be a CUDA tensor (this library has no CPU path)")
    dt = _dtype(logits, "logits")
    shape, stride = logits.shape, logits.stride()
    if len(shape) != 2 or (shape[1] > 1 and stride[1] != 1) or shape[0] > 0x7FFFFFFF:
        raise DracoFormatError("logits must be [rows, vocab] with contiguous rows")
    n, vocab = shape
    seqs = row_start.shape[0] - 1 if row_start.dim() == 1 else -1
    if seqs < 0:
        raise DracoFormatError("row_start must be [sequences + 1]")
    probs_ptr, ld_probs = 0, 0
    if draft_probs is not None:
        if draft_probs.dtype is not _F32 or draft_probs.get_device() != dev:
            raise ValueError(f"draft_probs must be a float32 tensor on cuda:{dev}, not {draft_probs.dtype} on "
                             f"{draft_probs.device}")
        if draft_probs.shape != shape or (vocab > 1 and draft_probs.stride(1) != 1):
            raise DracoFormatError("draft_probs must be shaped like logits with contiguous rows")
        probs_ptr, ld_probs = draft_probs.data_ptr(), draft_probs.stride(0)
    rows = max(n, 1) if max_rows is None else int(max_rows)
    if rows < 1:
        raise ValueError(f"max_rows {rows} must be at least 1")
    temperature = float(temperature)
    if not (temperature == 0.0 or 1e-30 <= temperature <= 1e30):
        raise ValueError(f"temperature {temperature} must be 0 (greedy) or lie in 1e-30 .. 1e30")
    accepted = row_start.new_empty(seqs)
    tokens = row_start.new_empty((seqs, rows))
    v = _VERIFY.pack(logits.data_ptr(), probs_ptr, _vector(row_start, "row_start", dev, seqs + 1),
                     _vector(drafts, "drafts", dev, n), _vector(accept_u, "accept_u", dev, n, _F32),
                     _vector(sample_u, "sample_u", dev, seqs, _F32), accepted.data_ptr(), tokens.data_ptr(),
                     stride[0], ld_probs, rows, 0.0, dt, n, seqs, vocab, rows)
    rc = _call(dev, _lib().verify_drafts, v, temperature)
    if rc:
        N.check(rc, "verify_drafts")
    return accepted, tokens
