"""The paged cache's operators without a GPU: what the C interface refuses (by
status and message, before any launch), what the Python functions refuse, the
sizes of caches, and the host logic of GPUExecutionBackend's paged cache and of
its n-gram drafts."""

import ctypes
import re
from pathlib import Path

import pytest
import torch

from dracort_b200 import _native as N
from dracort_b200 import paged_ops as P
from dracort_b200.exceptions import DracoFormatError
from dracort_b200.format.gguf_file import GGUFFile
from dracort_b200.gguf_executor import GPUExecutionBackend, LlamaConfig, ngram_drafts, page_pool

FIXTURE = Path(__file__).resolve().parent / "golden" / "tiny_llama_decode.gguf"
PTR = 1 << 20  # an aligned address; every call below returns before it would be read

lib = N.load()


def cache(**kw):
    f = dict(type=N.KV_BF16, kv_heads=2, head_dim=64, page_size=16, n_pages=8, n_seqs=2, max_pages=4, table_stride=4,
             k=PTR, v=PTR, block_table=PTR)
    f.update(kw)
    return N.KvCache(**f)


def append(c=None, dtype=N.DTYPE_F32, **kw):
    f = dict(q=PTR, k=PTR, v=PTR, q_out=PTR, ldq=256, ldk=128, ldv=128, ldqo=256, cos_table=PTR, sin_table=PTR,
             max_positions=64, seq=PTR, pos=PTR, n=3, heads=4)
    f.update(kw)
    return lib.draco_kv_append(c or cache(), N.KvAppendArgs(**f), dtype, None)


def read(c=None, dtype=N.DTYPE_F32, seq=PTR, pos=PTR, n=3, k=PTR, v=PTR, ldk=128, ldv=128):
    return lib.draco_kv_read(c or cache(), seq, pos, n, k, v, ldk, ldv, dtype, None)


def attend(c=None, dtype=N.DTYPE_F32, **kw):
    f = dict(q=PTR, out=PTR, ldq=256, ldo=256, q_start=PTR, kv_len=PTR, n=3, heads=4, max_q=3, max_kv=64, scale=0.0,
             workspace=PTR, workspace_bytes=1 << 30)
    f.update(kw)
    return lib.draco_attention_paged(c or cache(), N.AttentionPagedArgs(**f), dtype, None)


def verify(**kw):
    f = dict(logits=PTR, draft_probs=None, row_start=PTR, drafts=PTR, accept_u=PTR, sample_u=PTR, accepted=PTR,
             tokens=PTR, ld_logits=100, ld_probs=0, ld_tokens=4, temperature=1.0, dtype=N.DTYPE_F32, n=5, n_seqs=2,
             vocab=100, max_rows=4)
    f.update(kw)
    return lib.draco_verify_drafts(N.VerifyArgs(**f), None)


TYPE, SHAPE, ALIGN, ARG = N.DRACO_ERR_TYPE, N.DRACO_ERR_SHAPE, N.DRACO_ERR_ALIGN, N.DRACO_ERR_ARG


@pytest.mark.parametrize("call", [append, read, attend])
@pytest.mark.parametrize("status,kw", [
    (TYPE, dict(type=0)), (TYPE, dict(type=2)), (SHAPE, dict(kv_heads=0)), (SHAPE, dict(kv_heads=1025)),
    (SHAPE, dict(head_dim=48)), (SHAPE, dict(head_dim=512)), (SHAPE, dict(page_size=8)), (SHAPE, dict(page_size=48)),
    (SHAPE, dict(page_size=2048)), (SHAPE, dict(n_pages=0)), (SHAPE, dict(n_seqs=-1)), (SHAPE, dict(max_pages=0)),
    (SHAPE, dict(max_pages=1 << 27)), (SHAPE, dict(max_pages=(1 << 27) - 1)), (SHAPE, dict(table_stride=-1)), (ARG, dict(k=None)), (ARG, dict(v=None)),
    (ARG, dict(block_table=None)), (ALIGN, dict(k=PTR + 8)), (ALIGN, dict(v=PTR + 2)),
    (ALIGN, dict(block_table=PTR + 2))])
def test_caches_that_are_refused(call, status, kw):
    assert call(cache(**kw)) == status
    assert N.last_error()


@pytest.mark.parametrize("status,kw", [
    (TYPE, dict(dtype=2)), (SHAPE, dict(n=-1)), (SHAPE, dict(heads=-1)), (ARG, dict(q_out=None)), (ARG, dict(q=None)),
    (ARG, dict(cos_table=None)), (ARG, dict(sin_table=None)), (ARG, dict(k=None)), (ARG, dict(v=None)),
    (ARG, dict(seq=None)), (ARG, dict(pos=None)), (SHAPE, dict(ldq=255)), (SHAPE, dict(ldk=124)), (SHAPE, dict(ldv=0)),
    (SHAPE, dict(ldqo=128)), (ALIGN, dict(ldq=258)), (ALIGN, dict(k=PTR + 4)), (ALIGN, dict(q_out=PTR + 8)),
    (ALIGN, dict(dtype=N.DTYPE_BF16, ldv=132)), (SHAPE, dict(max_positions=0)), (ALIGN, dict(cos_table=PTR + 4)),
    (ALIGN, dict(seq=PTR + 1)), (SHAPE, dict(n=0x7FFFFFFF))])
def test_appends_that_are_refused(status, kw):
    assert append(**kw) == status


@pytest.mark.parametrize("status,kw", [
    (TYPE, dict(dtype=-1)), (SHAPE, dict(n=-2)), (ARG, dict(seq=None)), (ARG, dict(pos=None)), (ARG, dict(k=None)),
    (ARG, dict(v=None)), (SHAPE, dict(ldk=127)), (ALIGN, dict(ldk=130)), (ALIGN, dict(v=PTR + 4)),
    (ALIGN, dict(pos=PTR + 2)), (SHAPE, dict(n=0x60000000))])
def test_reads_that_are_refused(status, kw):
    assert read(**kw) == status


@pytest.mark.parametrize("status,kw", [
    (TYPE, dict(dtype=7)), (SHAPE, dict(n=-1)), (SHAPE, dict(heads=0)), (SHAPE, dict(heads=5)),
    (SHAPE, dict(max_q=-1)), (SHAPE, dict(max_kv=-1)), (ARG, dict(scale=-1.0)), (ARG, dict(scale=float("nan"))),
    (ARG, dict(scale=float("inf"))), (ARG, dict(scale=65537.0)), (ARG, dict(q=None)), (ARG, dict(out=None)), (ARG, dict(q_start=None)),
    (ARG, dict(kv_len=None)), (SHAPE, dict(ldq=252)), (SHAPE, dict(ldo=0)), (ALIGN, dict(q=PTR + 4)),
    (ALIGN, dict(ldo=257)), (ALIGN, dict(kv_len=PTR + 1)), (SHAPE, dict(n=0x7FFFFFF0))])
def test_attention_calls_that_are_refused(status, kw):
    assert attend(**kw) == status


@pytest.mark.parametrize("status,kw", [
    (TYPE, dict(dtype=9)), (SHAPE, dict(n=-1)), (SHAPE, dict(n_seqs=-1)), (SHAPE, dict(vocab=0)),
    (SHAPE, dict(max_rows=0)), (SHAPE, dict(vocab=(1 << 30) + 1)), (ARG, dict(temperature=-0.5)), (ARG, dict(temperature=1e-38)),
    (ARG, dict(temperature=float("nan"))), (ARG, dict(row_start=None)), (ARG, dict(accepted=None)),
    (ARG, dict(tokens=None)), (ARG, dict(logits=None)), (ARG, dict(drafts=None)), (ARG, dict(accept_u=None)),
    (ARG, dict(sample_u=None)), (SHAPE, dict(ld_logits=-1)), (SHAPE, dict(ld_tokens=3)),
    (SHAPE, dict(draft_probs=PTR, ld_probs=-4)), (ALIGN, dict(logits=PTR + 2)),
    (ALIGN, dict(dtype=N.DTYPE_BF16, logits=PTR + 1)), (ALIGN, dict(draft_probs=PTR + 2)),
    (ALIGN, dict(tokens=PTR + 3))])
def test_verifications_that_are_refused(status, kw):
    assert verify(**kw) == status


def test_calls_of_nothing_succeed():
    assert append(n=0) == N.DRACO_OK and read(n=0) == N.DRACO_OK and attend(n=0) == N.DRACO_OK
    assert attend(cache(n_seqs=0, block_table=None)) == N.DRACO_OK
    assert verify(n_seqs=0) == N.DRACO_OK
    assert lib.draco_kv_append(None, N.KvAppendArgs(), 0, None) == ARG
    assert lib.draco_verify_drafts(None, None) == ARG


def test_packed_structures_are_laid_out_as_the_c_ones():
    def ctype(code):
        return {"i": ctypes.c_int, "q": ctypes.c_int64, "P": ctypes.c_void_p, "f": ctypes.c_float}[code]

    for packed, mirror in ((P._KV_CACHE, N.KvCache), (P._KV_APPEND, N.KvAppendArgs), (P._ATTENTION, N.AttentionPagedArgs),
                           (P._VERIFY, N.VerifyArgs)):
        codes = re.sub(r"(\d+)(\w)", lambda m: m[2] * int(m[1]), packed.format.lstrip("@"))
        types = [t for _, t in mirror._fields_]
        assert [ctype(c) if t is not ctypes.c_size_t else t for c, t in zip(codes, types, strict=True)] == types
        assert packed.size == ctypes.sizeof(mirror)  # (with the same order and sizes: the same native alignment)
        values = [0.5 if t is ctypes.c_float else 16 * i + 16 for i, t in enumerate(types)]
        assert packed.pack(*values) == bytes(mirror(*values))


def test_cache_sizes():
    # bf16: 2 bytes a value; Q8_0: 34 bytes for 32 values
    assert P.kv_cache_nbytes("bf16", 7, 3, 16, 96) == 7 * 3 * 16 * 96 * 2
    assert P.kv_cache_nbytes("q8_0", 7, 3, 16, 96) == 7 * 3 * 16 * 96 // 32 * 34
    assert P.kv_cache_nbytes("q8_0", 1 << 20, 8, 64, 128) == (1 << 20) * 8 * 64 * 136  # past 32 bits
    for kind, want in (("bf16", (5, 2, 32, 64)), ("q8_0", (5, 2, 32, 68))):
        k, v = P.kv_cache(kind, 5, 2, 32, 64, "cpu")
        assert tuple(k.shape) == tuple(v.shape) == want
        assert k.numel() * k.element_size() == P.kv_cache_nbytes(kind, 5, 2, 32, 64)
    for bad in ((0, 2, 32, 64), (5, 0, 32, 64), (5, 2, 33, 64), (5, 2, 32, 80)):
        with pytest.raises(DracoFormatError):
            P.kv_cache("bf16", *bad, "cpu")
    with pytest.raises(ValueError, match="cache type"):
        P.kv_cache("f16", 5, 2, 32, 64, "cpu")


def test_tensors_of_the_host_are_refused():
    k, v = P.kv_cache("bf16", 4, 2, 16, 64, "cpu")
    i = torch.zeros(3, dtype=torch.int32)
    q = torch.zeros(3, 4, 64)
    table = torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        P.kv_append(q, q[:, :2], q[:, :2], k, v, table, i, i)
    with pytest.raises(ValueError, match="CUDA"):
        P.kv_read(k, v, table, i, i, 64)
    with pytest.raises(ValueError, match="CUDA"):
        P.attention_paged(q, k, v, table, i, i[:2])
    with pytest.raises(ValueError, match="CUDA"):
        P.verify_drafts(torch.zeros(3, 10), i[:2], i, torch.zeros(3), torch.zeros(1))


def test_workspace_size_covers_smaller_bounds_and_refuses_what_the_call_refuses():
    def need(**kw):
        f = dict(n=4, heads=4, max_q=1, max_kv=64, dtype=N.DTYPE_F32)
        f.update(kw)
        return lib.draco_attention_paged_workspace_bytes(cache(), f["n"], f["heads"], f["max_q"], f["max_kv"],
                                                         f["dtype"])

    assert need() >= N.PAGED_WORKSPACE_HEAD
    for bad in (dict(n=-1), dict(heads=0), dict(heads=3), dict(max_q=-1), dict(max_kv=-1), dict(dtype=5)):
        assert need(**bad) == 0
    assert lib.draco_attention_paged_workspace_bytes(cache(head_dim=40), 4, 4, 1, 64, 0) == 0


# ---------------------------------------------------------------------------
# the GPU executor's paged cache, host side
# ---------------------------------------------------------------------------
@pytest.fixture(scope="module")
def cfg():
    gf = GGUFFile(str(FIXTURE))
    try:
        return LlamaConfig.from_gguf(gf)
    finally:
        gf.close()


def test_page_pool(cfg):
    # 2 layers of keys and values, 4 heads of 32, a context of 64
    page = 2 * 2 * 4 * 16 * 32 * 2  # bf16 pages of 16 positions
    assert page_pool(cfg, "bf16", 3, page_size=16) == (12, 64)
    assert page_pool(cfg, "bf16", 3, max_seq_len=20, page_size=16) == (6, 20)
    assert page_pool(cfg, "bf16", 3, max_seq_len=1000, page_size=16) == (12, 64)
    assert page_pool(cfg, "bf16", 3, kv_budget_bytes=5 * page + 1, page_size=16) == (5, 64)
    assert page_pool(cfg, "bf16", 3, kv_budget_bytes=2 * page, page_size=16) == (2, 32)
    assert page_pool(cfg, "q8_0", 3, kv_budget_bytes=5 * page, page_size=16) == (9, 64)  # 34 bytes for 32 values
    assert page_pool(cfg, "q8_0", 1) == (1, 64)
    with pytest.raises(ValueError, match="no page"):
        page_pool(cfg, "bf16", 3, kv_budget_bytes=page - 1, page_size=16)
    with pytest.raises(ValueError, match="no page"):
        page_pool(cfg, "bf16", 3, max_seq_len=0)
    with pytest.raises(DracoFormatError):
        page_pool(cfg, "bf16", 3, page_size=24)


def test_backend_refuses_cache_types():
    for name in ("f16", "q4_0", ""):
        with pytest.raises(ValueError, match="bf16"):
            GPUExecutionBackend(str(FIXTURE), 1, name)


def test_ngram_drafts():
    ids = [1, 2, 3, 4, 1, 2, 3, 9, 8, 1, 2, 3]
    assert ngram_drafts(ids, 4) == [9, 8, 1, 2]  # the latest occurrence of 1 2 3
    assert ngram_drafts(ids, 2) == [9, 8]
    assert ngram_drafts(ids, 0) == []
    assert ngram_drafts([5, 6, 7], 3) == []
    assert ngram_drafts([7, 5, 7], 3) == [5, 7]  # one token of context, cut at the end
    assert ngram_drafts([5, 5], 3) == [5]
    assert ngram_drafts([5], 3) == ngram_drafts([], 3) == []
    assert ngram_drafts([1, 2, 8, 3, 2, 9, 1, 2], 1, ngram=2) == [8]
    assert ngram_drafts([1, 2, 8, 3, 2, 9, 1, 2], 1, ngram=1) == [9]
